// E4M3 quantisers with one float32 scale per block of 128 columns:
//
//   rows    [h = bf16(residual + x)] -> [RMSNorm] -> codes [rows, k], scales [rows, ceil(k / 128)]
//             r = rsqrt(mean(h^2) + eps),  y = gamma * (h * r)       (float32: y is not rounded to 16 bits in between)
//             a = max(max |y|, 2^-100) over the row's 128 columns,  code = e4m3(y * (448 / a)),  scale = a / 448
//   weights codes [n, k], scales [ceil(n / 128), ceil(k / 128)], a over 128 x 128 elements
//
// The last block of a row may be shorter (k is a multiple of 16).  A block with a value that is not finite has the scale
// NaN and codes of zero: its values are NaN, and no code ever is.  The floor keeps 448 / a finite; a block below it has
// the scale 2^-109 and steps of 2^-118, far below anything a bf16 product can show.
//
// Bound by memory: 7 bytes per element with a residual (two bf16 in, one bf16 and one code out), 3 without.  8192 x 8192 with
// residual and norm: 71.5 us replayed from a graph (6.6 TB/s), 333 x 4112 2.5 us, one row of 4096 2.1 us (a launch and the
// chain load, sum, maximum, store).  The row stays in registers between its sum and its codes, so it is read once.
#include "plq_fp8.cuh"
#include "plq_quant.cuh"

namespace plq {

struct Fp8PackArgs {
  const uint4* x;
  const uint4* residual;
  uint4* h_out;
  const uint4* gamma;
  uint2* codes;
  float* scales;
  long long ldx8, ldr8;        // row strides of x and residual in 16-byte units
  int vecs;                    // k / 8
  int blocks;                  // ceil(k / 128)
  float inv_k, eps;
};

// eight bf16 -> four pairs of float32
__device__ __forceinline__ void widen8(const uint4& q, float2 (&f)[4]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(bf16lo_to_f32(w[i]), bf16hi_to_f32(w[i]));
}
__device__ __forceinline__ uint2 codes8(const float2 (&y)[4]) {
  return make_uint2(e4m3x2(y[0].x, y[0].y) | e4m3x2(y[1].x, y[1].y) << 16, e4m3x2(y[2].x, y[2].y) | e4m3x2(y[3].x, y[3].y) << 16);
}
// the larger of a and |y|; NaN if one of them is
__device__ __forceinline__ float max_abs(float a, float y) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(a), "f"(y));
  return r;
}
__device__ __forceinline__ float max_abs8(const float2 (&y)[4]) {
  float a = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) a = max_abs(max_abs(a, y[j].x), y[j].y);
  return a;
}
// What a block's codes are multiplied with, and its scale, from its largest magnitude.
struct BlockScale {
  float inv, scale;
  bool finite;
  __device__ __forceinline__ explicit BlockScale(float top) {
    finite = top < __uint_as_float(0x7F800000u);
    const float amax = fmaxf(top, kFp8Floor);              // a number for a top of NaN as well
    inv = __fdiv_rn(kE4m3Max, amax);
    scale = finite ? __fdiv_rn(amax, kE4m3Max) : __uint_as_float(0x7FFFFFFFu);
  }
};

// One CTA per row; a thread holds VPT vectors of eight elements, 16 neighbouring lanes hold a block of 128 columns.
template <int VPT, bool NORM, bool ADD>
__global__ void __launch_bounds__(512) fp8_pack_kernel(const Fp8PackArgs a) {
  __shared__ float warp_sum[16];
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, step = blockDim.x;
  const uint4* x = a.x + row * a.ldx8;
  uint4 v[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int at = tid + i * step;
    v[i] = at < a.vecs ? x[at] : make_uint4(0, 0, 0, 0);
  }
  if constexpr (ADD) {
    const uint4* res = a.residual + row * a.ldr8;
    uint4 w[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int at = tid + i * step;
      w[i] = at < a.vecs ? res[at] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float2 f[4], g[4];
      widen8(v[i], f);
      widen8(w[i], g);
      uint32_t* o = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = f32x2_to_bf16x2(g[j].x + f[j].x, g[j].y + f[j].y);
      const int at = tid + i * step;
      if (at < a.vecs) a.h_out[row * a.vecs + at] = v[i];
    }
  }
  float r = 1.0f;
  if constexpr (NORM) {
    float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float2 f[4];
      widen8(v[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) sums = __ffma2_rn(f[j], f[j], sums);
    }
    float sum = sums.x + sums.y;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    if ((tid & 31) == 0) warp_sum[tid >> 5] = sum;
    __syncthreads();
    const int warps = step >> 5;
    sum = (tid & 31) < warps ? warp_sum[tid & 31] : 0.0f;
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    sum = __shfl_sync(0xFFFFFFFFu, sum, 0);
    r = rsqrtf(fmaf(sum, a.inv_k, a.eps));
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int at = tid + i * step;
    if (VPT > 1 && i * step >= a.vecs) break;              // the same for the whole CTA
    float2 y[4];
    widen8(v[i], y);
    if constexpr (NORM) {
      const uint4 gv = at < a.vecs ? a.gamma[at] : make_uint4(0, 0, 0, 0);
      float2 g[4];
      widen8(gv, g);
      const float2 r2 = make_float2(r, r);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = __fmul2_rn(g[j], __fmul2_rn(y[j], r2));
    }
    float top = max_abs8(y);
    if (at >= a.vecs) top = 0.0f;                          // 0 * r is NaN where the row is not finite
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) top = max_abs(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    const BlockScale s(top);
    const float2 inv = make_float2(s.inv, s.inv);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = s.finite ? __fmul2_rn(y[j], inv) : make_float2(0.0f, 0.0f);
    if (at < a.vecs) {
      a.codes[row * a.vecs + at] = codes8(y);
      if ((tid & 15) == 0) a.scales[row * a.blocks + (at >> 4)] = s.scale;
    }
  }
}

// One CTA of 256 threads per 128 x 128 block: thread t has the 8-element vectors (row t / 16 + 16 i, column t % 16).
__global__ void __launch_bounds__(256) fp8_pack_weight_kernel(const uint4* w, uint2* codes, float* scales, long long n, int vecs, int blocks) {
  __shared__ float warp_top[8];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const long long row0 = static_cast<long long>(blockIdx.y) * kFp8Block + (tid >> 4);
  const int at = blockIdx.x * 16 + (tid & 15);
  uint4 v[8];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = row0 + 16 * i < n && at < vecs;
    v[i] = in ? w[(row0 + 16 * i) * vecs + at] : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 f[4];
    widen8(v[i], f);
    top = max_abs(top, max_abs8(f));
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) top = max_abs(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  if ((tid & 31) == 0) warp_top[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max_abs(top, warp_top[i]);
  const BlockScale s(top);
  const float2 inv = make_float2(s.inv, s.inv);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float2 f[4];
    widen8(v[i], f);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = s.finite ? __fmul2_rn(f[j], inv) : make_float2(0.0f, 0.0f);
    if (row0 + 16 * i < n && at < vecs) codes[(row0 + 16 * i) * vecs + at] = codes8(f);
  }
  if (tid == 0) scales[static_cast<long long>(blockIdx.y) * blocks + blockIdx.x] = s.scale;
}

// code * scale, rounded to bf16
__global__ void __launch_bounds__(256) fp8_unpack_kernel(const uint2* codes, const float* scales, uint4* y, long long total, int vecs, int blocks,
                                                         int block_rows) {
  pdl_launch_dependents();
  pdl_wait();
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const long long row = i / vecs;
  const int at = static_cast<int>(i - row * vecs);
  const float s = scales[row / block_rows * blocks + (at >> 4)];
  const uint2 c = codes[i];
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = e4m3x2_to_f32x2((j < 2 ? c.x : c.y) >> (16 * (j & 1)));
    o[j] = f32x2_to_bf16x2(f.x * s, f.y * s);
  }
  y[i] = make_uint4(o[0], o[1], o[2], o[3]);
}

template <typename... P, typename... A>
static int launch_pdl(void (*kernel)(P...), dim3 grid, unsigned threads, void* stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
  return PLQ_OK;
}

static int check_fp8_matrix(int64_t rows, int64_t k) {
  if (rows < 0 || k < 16 || k % 16 != 0) return PLQ_ERR_SHAPE;
  if (k > 32768 || rows > 0x7FFFFFFF) return PLQ_ERR_LIMIT;
  return PLQ_OK;
}

template <bool NORM, bool ADD>
static int launch_fp8_pack(const Fp8PackArgs& a, int64_t rows, void* stream) {
  const dim3 grid(static_cast<unsigned>(rows));
  // Vectors per thread: enough threads for a row's loads to be issued at once, and at most eight vectors each.
  const int want = (a.vecs + 31) / 32 * 32;
  if (want <= 128) return launch_pdl(fp8_pack_kernel<1, NORM, ADD>, grid, static_cast<unsigned>(want), stream, a);
  if (want <= 512) return launch_pdl(fp8_pack_kernel<2, NORM, ADD>, grid, static_cast<unsigned>((a.vecs + 63) / 64 * 32), stream, a);
  if (want <= 2048) return launch_pdl(fp8_pack_kernel<4, NORM, ADD>, grid, static_cast<unsigned>((a.vecs + 127) / 128 * 32), stream, a);
  return launch_pdl(fp8_pack_kernel<8, NORM, ADD>, grid, static_cast<unsigned>((a.vecs + 255) / 256 * 32), stream, a);
}

}  // namespace plq

extern "C" int plq_fp8_pack(const void* x_bf16, int64_t ldx, const void* residual_bf16, int64_t ldr, void* h_out_bf16,
                            const void* gamma_bf16, float eps, int64_t rows, int64_t k, void* codes, void* scales_f32, void* stream) {
  using namespace plq;
  int st = check_fp8_matrix(rows, k);
  if (st != PLQ_OK) return st;
  if (ldx < k || ldx % 8 != 0 || (residual_bf16 && (ldr < k || ldr % 8 != 0))) return PLQ_ERR_SHAPE;
  if (rows == 0) return PLQ_OK;
  if (!x_bf16 || !codes || !scales_f32 || (residual_bf16 && (!h_out_bf16 || !gamma_bf16))) return PLQ_ERR_NULL;
  if (!aligned16(x_bf16) || !aligned16(residual_bf16) || !aligned16(h_out_bf16) || !aligned16(gamma_bf16) || !aligned16(codes) ||
      (reinterpret_cast<uintptr_t>(scales_f32) & 3u))
    return PLQ_ERR_ALIGN;
  if ((st = device_check()) != PLQ_OK) return st;
  Fp8PackArgs a;
  a.x = static_cast<const uint4*>(x_bf16);
  a.residual = static_cast<const uint4*>(residual_bf16);
  a.h_out = static_cast<uint4*>(h_out_bf16);
  a.gamma = static_cast<const uint4*>(gamma_bf16);
  a.codes = static_cast<uint2*>(codes);
  a.scales = static_cast<float*>(scales_f32);
  a.ldx8 = ldx / 8;
  a.ldr8 = ldr / 8;
  a.vecs = static_cast<int>(k / 8);
  a.blocks = static_cast<int>((k + kFp8Block - 1) / kFp8Block);
  a.inv_k = 1.0f / static_cast<float>(k);
  a.eps = eps;
  if (residual_bf16) return launch_fp8_pack<true, true>(a, rows, stream);
  if (gamma_bf16) return launch_fp8_pack<true, false>(a, rows, stream);
  return launch_fp8_pack<false, false>(a, rows, stream);
}

extern "C" int plq_fp8_pack_weight(const void* w_bf16, int64_t n, int64_t k, void* codes, void* scales_f32, void* stream) {
  using namespace plq;
  int st = check_fp8_matrix(n, k);
  if (st != PLQ_OK) return st;
  if ((n + kFp8Block - 1) / kFp8Block > 65535) return PLQ_ERR_LIMIT;
  if (n == 0) return PLQ_OK;
  if (!w_bf16 || !codes || !scales_f32) return PLQ_ERR_NULL;
  if (!aligned16(w_bf16) || !aligned16(codes) || (reinterpret_cast<uintptr_t>(scales_f32) & 3u)) return PLQ_ERR_ALIGN;
  if ((st = device_check()) != PLQ_OK) return st;
  const int blocks = static_cast<int>((k + kFp8Block - 1) / kFp8Block);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((n + kFp8Block - 1) / kFp8Block));
  return launch_pdl(fp8_pack_weight_kernel, grid, 256, stream, static_cast<const uint4*>(w_bf16), static_cast<uint2*>(codes),
                    static_cast<float*>(scales_f32), static_cast<long long>(n), static_cast<int>(k / 8), blocks);
}

extern "C" int plq_fp8_unpack(const void* codes, const void* scales_f32, int64_t rows, int64_t k, int64_t block_rows, void* y_bf16, void* stream) {
  using namespace plq;
  int st = check_fp8_matrix(rows, k);
  if (st != PLQ_OK) return st;
  if (block_rows != 1 && block_rows != kFp8Block) return PLQ_ERR_SHAPE;
  if (rows == 0) return PLQ_OK;
  if (!codes || !scales_f32 || !y_bf16) return PLQ_ERR_NULL;
  if (!aligned16(codes) || !aligned16(y_bf16) || (reinterpret_cast<uintptr_t>(scales_f32) & 3u)) return PLQ_ERR_ALIGN;
  const long long total = rows * (k / 8), grid = (total + 255) / 256;
  if (grid > 0x7FFFFFFF) return PLQ_ERR_LIMIT;
  if ((st = device_check()) != PLQ_OK) return st;
  return launch_pdl(fp8_unpack_kernel, dim3(static_cast<unsigned>(grid)), 256, stream, static_cast<const uint2*>(codes),
                    static_cast<const float*>(scales_f32), static_cast<uint4*>(y_bf16), total, static_cast<int>(k / 8),
                    static_cast<int>((k + kFp8Block - 1) / kFp8Block), static_cast<int>(block_rows));
}
