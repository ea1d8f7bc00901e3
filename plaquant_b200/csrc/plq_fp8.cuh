// Shared pieces of the E4M3 kernels: conversions, the unscaled 8-bit tcgen05.mma and its descriptors.
//
// E4M3 here: 1 sign, 4 exponent, 3 mantissa bits, largest value 448, smallest step 2^-9, codes 0x7F / 0xFF are NaN.
#pragma once

#include "plq_tc.cuh"

namespace plq {

constexpr float kE4m3Max = 448.0f;
constexpr int kFp8Block = 128;               // columns (and weight rows) that share a scale of a quantised matrix
constexpr int kCacheBlock = 64;              // tokens of a cache that share a scale
constexpr float kFp8Floor = 7.888609052210118e-31f;     // 2^-100: smallest block maximum of a matrix, smallest scale of a cache

#ifdef __CUDACC__

// two float32 -> two E4M3 codes (nearest even, saturating), the first in the low byte
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(b), "f"(a));
  return d;
}
// two E4M3 codes (low byte first) -> two float32
__device__ __forceinline__ float2 e4m3x2_to_f32x2(uint32_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(c)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
// Two float32 in [0, 448] -> their nearest E4M3 codes (low half) and those of what is left (high half), by way of f16, whose
// rounding (2^-11) is far below that of the second code.
__device__ __forceinline__ uint32_t e4m3_split(float a, float b) {
  uint32_t x, back;
  uint16_t hi, lo;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(hi) : "r"(x));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(hi));
  const __half2 rest = __hsub2(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&back));
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(lo) : "r"(*reinterpret_cast<const uint32_t*>(&rest)));
  return hi | static_cast<uint32_t>(lo) << 16;
}
// Instruction descriptor of kind::f8f6f4 with E4M3 operands and a float32 accumulator:
//   [4,6) accumulator 1 = float32  [7,10), [10,13) operand formats 0 = E4M3  [15], [16] A, B with M / N contiguous instead of K
//   [17,23) N / 8  [24,29) M / 16
__host__ __device__ constexpr uint32_t make_idesc_e4m3(uint32_t m, uint32_t n, bool a_mn_major = false, bool b_mn_major = false) {
  return (1u << 4) | (a_mn_major ? 1u << 15 : 0u) | (b_mn_major ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// D[tmem] (+)= A B^T, 32 elements of K per instruction
template <int CG>
__device__ __forceinline__ void tc_mma_e4m3(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                            uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo),
                 "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
                 "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %5, p;\n\t}" ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo),
                 "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}

// The same with A in tensor memory (row = lane, four consecutive elements of K per 32-bit column), block-scaled (descriptor:
// make_idesc): every row of A and of B has an E8M0 scale for the 32 elements of K, a byte of the word that 512 bytes copied
// to these columns put there (row r: lane r % 32, column r / 32); which one, the descriptor and bits 30 and 31 of the address say.
__device__ __forceinline__ void tc_mma_mxf8_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t sfa_tmem,
                                               uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %7, 0;\n\tmov.b64 db, {%2, %3};\n\t"
               "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], [%1], db, %4, [%5], [%6], p;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo),
               "r"(b_hi), "r"(idesc), "r"(sfa_tmem), "r"(sfb_tmem), "r"(accumulate) : "memory");
}
constexpr uint32_t kIdescBMnMajor = 1u << 16;          // N contiguous instead of K

// 16 consecutive 32-bit columns of a warp's 32 lanes
__device__ __forceinline__ void tc_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
      "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 lanes x 16 consecutive 32-bit columns
__device__ __forceinline__ void tc_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// four bytes global -> shared, and an arrival on the mbarrier when all earlier ones of this thread have landed
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// An arrival that orders nothing but the tensor-memory reads that a tcgen05 fence in front of it covers: the release of
// mbar_arrive_cluster costs a memory barrier.
__device__ __forceinline__ void mbar_arrive_relaxed_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The warps of a warpgroup hand registers back, or take more.
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const void* tmap, int32_t x, int32_t y, int32_t z, uint32_t bar) {
  tma_load_3d_cg<1>(dst, tmap, x, y, z, bar);
}

#endif  // __CUDACC__

// Host side.  Raises the kernel's shared-memory limit, once per thread and device.
template <typename K>
int allow_smem(K kernel, size_t bytes, int* done_dev) {
  int dev = 0;
  PLQ_CUDA_TRY(cudaGetDevice(&dev));
  if (*done_dev != dev) {
    PLQ_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    *done_dev = dev;
  }
  return PLQ_OK;
}

}  // namespace plq
