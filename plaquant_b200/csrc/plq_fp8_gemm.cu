// E4M3 product with a float32 scale per block of 128:
//
//   Y[m, n] = sum over K blocks b of  sa[m, b] * sw[n / 128, b] * sum_{k in b} A[m, k] W[n, k]
//
// A: codes [m, k], scales [m, ceil(k / 128)] (plq_fp8_pack);  W: codes [n, k], scales [ceil(n / 128), ceil(k / 128)].
// The scales are arbitrary float32 numbers, so the tensor core cannot apply them: each K block of 128 is a product of its
// own into a fresh tensor-memory accumulator (four tcgen05.mma kind::f8f6f4), and the epilogue warps add it, times its
// scale, to float32 sums in registers while the next block's MMAs run into another accumulator.
//
// Two kernels:
//   fp8_gemv_kernel         up to 16 rows (64 on request): the weights are the 128-row side of the MMA and the activations the narrow one, so
//                           that a few rows stream the weights once; bound by HBM (n k bytes).
//   fp8_gemm_kernel<BN, CG> more rows: 128 x 128 tiles of one CTA, 256 x 128 or 256 x 256 of a CTA pair; bound by the
//                           tensor pipe (2 m n k) and the epilogue next to it or, for few tiles, by the chain of one tile.
//
// Every wait is bounded; on expiry PLQ_DEV_TIMEOUT goes to the caller's status word and all roles leave their loops.
#include <cstring>

#include "plq_fp8.cuh"
#include "plq_quant.cuh"

namespace plq {

struct Fp8GemmArgs {
  const float* sa;             // [m, kb]
  const float* sw;             // [ceil(n / 128), kb]
  void* y;
  long long ldy;
  int32_t* status;
  int m, n, kb;                // kb: K blocks of 128
  int tiles_m, tiles_n;
  int vec;                     // rows of y allow stores of 32 (2), 16 (1) bytes or neither (0)
  int pairs;                   // bf16: rows begin at multiples of four bytes and n is even
  int static_w;                // weights may be read before the programmatic dependency wait
  int band;                    // row tiles per band of the tile order
};
struct Fp8GemmMaps { CUtensorMap a, w; };
constexpr int kMaxSlices = 8;                          // CTAs that may share a tile along K

template <typename T> __device__ __forceinline__ T round_out(float v);
template <> __device__ __forceinline__ float round_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 round_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- a few rows ------------------------------------------------------------------------------------------------------
// A tile is 128 weight rows x a group of 16 activation rows (accumulator columns); groups of the same weight rows are
// neighbours.  Where there are fewer tiles than CTA slots a cluster of S CTAs shares a tile along K; each leaves its
// sums in the shared memory of the CTA that owns the activation row (row j: CTA j mod S), which adds them in the order of the
// slices: results do not depend on timing and no scratch in HBM is needed.  They are stored there as whole 128-byte lines, one
// activation row of 32 neighbouring weight rows (scattered 16-byte stores cost 2 us more).
//   warp 0 producer, warp 1 MMA issuer, warps 2 - 5 epilogue (one weight row per thread)
// Bound by the weights' bytes: 1 x 4096 -> 128256 in 85.8 us (6.1 TB/s, 0.95 of the measured copy rate), 16 x 8192 -> 8192 in
// 14.1 us (4.8 TB/s); the rest is the launch, the first load and the reduction, 3 - 4 us.
struct GvCfg {
  static constexpr int kRows = 16;
  static constexpr int kStages = 5;
  static constexpr int kXBytes = kRows * kStageKBytes;
  static constexpr int kStageBytes = kABytes + kXBytes;
  static constexpr int kAcc = 8;                                      // accumulators in flight
  static constexpr int kTmemCols = kAcc * kRows;                      // two CTAs share an SM
  static constexpr int kSlotRows = kRows + kMaxSlices;                // S slices x ceil(kRows / S) rows
  static constexpr int kSlotBytes = kSlotRows * 128 * 4;
  static constexpr size_t kSmemBytes = 1024 + static_cast<size_t>(kStages) * kStageBytes + kSlotBytes + 4 * kRows * 4 + 512;
  static constexpr int kThreads = 192;
  static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
};

template <typename OUT>
__global__ void __launch_bounds__(192, 2) fp8_gemv_kernel(const __grid_constant__ Fp8GemmMaps maps, const Fp8GemmArgs g) {
  using C = GvCfg;
  constexpr int kRows = C::kRows;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* slots = reinterpret_cast<float*>(smem + static_cast<size_t>(C::kStages) * C::kStageBytes);       // [slice][owned row][128]
  float* factors = slots + C::kSlotBytes / 4;                         // [4 warps][kRows] scales of the K block at hand
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(factors + 4 * kRows);
  uint64_t* empty_bar = full_bar + C::kStages;
  uint64_t* acc_full = empty_bar + C::kStages;
  uint64_t* acc_empty = acc_full + C::kAcc;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + C::kAcc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  uint32_t nslice_u;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nslice_u));
  const int nslice = static_cast<int>(nslice_u), slice = static_cast<int>(cluster_ctarank());

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int s = 0; s < C::kAcc; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], 4); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && elect_one()) { prefetch_tmap(&maps.a); prefetch_tmap(&maps.w); }
  if (warp == 1) {
    tmem_alloc<1>(tmem_holder, C::kTmemCols);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  if (nslice > 1) cluster_arrive_release();            // waited for in front of the first store to another CTA
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_launch_dependents();

  const int kb0 = g.kb * slice / nslice, kb1 = g.kb * (slice + 1) / nslice;
  const int first_tile = static_cast<int>(cluster_id_x()), tile_step = static_cast<int>(nclusters_x());
  const int num_tiles = g.tiles_n * g.tiles_m;         // tiles_m: groups of activation rows, neighbours share a weight tile
  const uint32_t smem_base = smem_u32(smem);

  float acc[kRows];                                       // epilogue: this weight row's sums

  if (warp == 0) {
    if (elect_one()) {
      auto load_w = [&](uint32_t slot, int tile, int kb) {
        mbar_arrive_expect_tx(&full_bar[slot], C::kStageBytes);
        tma_load_2d_cg<1>(smem_base + slot * C::kStageBytes, &maps.w, kb * kStageKBytes, tile / g.tiles_m * kBM, smem_u32(&full_bar[slot]));
      };
      auto load_x = [&](uint32_t slot, int tile, int kb) {
        tma_load_2d_cg<1>(smem_base + slot * C::kStageBytes + kABytes, &maps.a, kb * kStageKBytes, tile % g.tiles_m * kRows, smem_u32(&full_bar[slot]));
      };
      // Static weights: the first ring fill of weight bytes is requested while the previous kernel drains.
      uint32_t early = 0;
      if (g.static_w)
        for (int tile = first_tile; tile < num_tiles && early < C::kStages; tile += tile_step)
          for (int kb = kb0; kb < kb1 && early < C::kStages; ++kb, ++early) load_w(early, tile, kb);
      pdl_wait();
      uint32_t gs = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step)
        for (int kb = kb0; kb < kb1; ++kb, ++gs) {
          const uint32_t slot = gs % C::kStages;
          if (gs >= early) {
            ok = mbar_wait_bounded(&empty_bar[slot], ((gs / C::kStages) & 1u) ^ 1u, abort_flag);
            if (!ok) break;
            load_w(slot, tile, kb);
          }
          load_x(slot, tile, kb);
        }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc = make_idesc_e4m3(128, kRows);
      uint32_t gs = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step)
        for (int kb = kb0; kb < kb1; ++kb, ++gs) {
          const uint32_t slot = gs % C::kStages, as = gs % C::kAcc;
          ok = mbar_wait_bounded(&acc_empty[as], ((gs / C::kAcc) & 1u) ^ 1u, abort_flag) &&
               mbar_wait_bounded(&full_bar[slot], (gs / C::kStages) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t w_lo = desc_lo_sw128(smem_base + slot * C::kStageBytes), x_lo = desc_lo_sw128(smem_base + slot * C::kStageBytes + kABytes);
#pragma unroll
          for (int h = 0; h < 4; ++h)
            tc_mma_e4m3<1>(tmem_base + as * kRows, w_lo + 2 * h, kDescHiSw128, x_lo + 2 * h, kDescHiSw128, idesc, h != 0);
          tc_commit<1>(smem_u32(&empty_bar[slot]));
          tc_commit<1>(smem_u32(&acc_full[as]));
        }
    }
  } else {
    // ---- epilogue: thread = weight row; lane l of a warp fetches the scales of activation row l ----
    const int trow = (warp & 3) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    float* my_factors = factors + (warp - 2) * kRows;
    pdl_wait();
    uint32_t gs = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) acc[j] = 0.0f;
      const int row0 = tile % g.tiles_m * kRows;
      const float* sw = g.sw + static_cast<long long>(tile / g.tiles_m) * g.kb;
      auto scale = [&](int kb) {
        return kb < kb1 && row0 + lane < g.m && lane < kRows ? g.sa[static_cast<long long>(row0 + lane) * g.kb + kb] * sw[kb] : 0.0f;
      };
      float next[4];                                   // scales of the next four K blocks, on their way
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = scale(kb0 + i);
      for (int kb = kb0; ok && kb < kb1; kb += 4) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[i] = next[i]; next[i] = scale(kb + 4 + i); }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!ok || kb + i >= kb1) break;
          __syncwarp();
          if (lane < kRows) my_factors[lane] = f[i];
          const uint32_t as = gs % C::kAcc;
          ok = mbar_wait_bounded_lanes(&acc_full[as], (gs / C::kAcc) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          uint32_t r[kRows];
          tc_ld_32x32b_x16(tmem_base + lane_base + as * kRows, r);
          tc_wait_ld();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty[as]);
#pragma unroll
          for (int j = 0; j < kRows; ++j) acc[j] = fmaf(__uint_as_float(r[j]), my_factors[j], acc[j]);
          ++gs;
        }
      }
      if (nslice == 1 && ok) {
        const long long row = static_cast<long long>(tile / g.tiles_m) * kBM + trow;
        OUT* y = static_cast<OUT*>(g.y) + row0 * g.ldy + row;
        if (row < g.n) {
#pragma unroll
          for (int j = 0; j < kRows; ++j)
            if (row0 + j < g.m) y[j * g.ldy] = round_out<OUT>(acc[j]);
        }
      }
    }
  }
  if (nslice > 1) {                                    // one tile per cluster
    const int trow = (warp & 3) * 32 + lane, row0 = first_tile % g.tiles_m * kRows, rows = min(kRows, g.m - row0), per = (kRows + nslice - 1) / nslice;
    __syncwarp();
    cluster_wait_acquire();                            // every CTA of the cluster is there
    if (warp >= 2) {
      const uint32_t own = smem_u32(slots) + static_cast<uint32_t>((slice * per * 128 + trow) * 4);
      int cta = 0, at = 0;                             // row j: CTA j % S, its row j / S
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (j < rows) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(own + at * 512u, static_cast<uint32_t>(cta))), "f"(acc[j]) : "memory");
        if (++cta == nslice) { cta = 0; ++at; }
      }
    }
    __syncwarp();
    cluster_arrive_release();
    cluster_wait_acquire();
    const long long row = static_cast<long long>(first_tile / g.tiles_m) * kBM + trow;
    if (warp >= 2 && !*abort_flag && row < g.n) {
      OUT* y = static_cast<OUT*>(g.y) + row0 * g.ldy + row;
      for (int j = slice, at = 0; j < rows; j += nslice, ++at) {
        float sum = 0.0f;
#pragma unroll
        for (int s = 0; s < kMaxSlices; ++s)
          if (s < nslice) sum += slots[(s * per + at) * 128 + trow];
        y[j * g.ldy] = round_out<OUT>(sum);
      }
    }
  }
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(g.status, PLQ_DEV_TIMEOUT);
    const long long t0 = clock64();                    // copies still in flight get time to land
    while (clock64() - t0 < 400000ll) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, C::kTmemCols);
  }
}

// ---- many rows -------------------------------------------------------------------------------------------------------
// Persistent; warps 0 and 3 producers (alternate K blocks), warp 1 MMA issuer (leader CTA of a pair), warp 2 fetches scales, warps 4 and up epilogue: four
// warps (the quadrants of tensor memory) for every 64 columns of the tile, each thread one row x 64 float32 sums.
// Per K block an epilogue warp reads its columns from tensor memory and does one packed multiply-add per two of them,
// beside the 256 (128 x 128) or 512 cycles of the block's MMAs.  The scales travel ahead of the epilogue through a ring of
// their own (cp.async, 16 K blocks deep): loaded by the epilogue itself their latency was longer than a K block.
// 8192 x 14336 -> 4096 in 476 us as a burst (2.0 PFLOP/s; 570 - 590 under the power cap).  The sums bound it: a 256 x 256 tile has
// two accumulators, so the epilogue of a K block has to be done within the MMAs of the next one (512 cycles), and the chain commit,
// wait, load, add, release is longer: 0.60 us a K block, without the additions 0.43 us (334 us in all).  Eight warps of 128 columns took
// 575 us, accumulators of 128 columns 533 (A read twice), 256 x 128 tiles 507, 128 x 128 tiles 524 (feed from L2: 14 TB/s).
template <int BN, int CG>
struct GmCfg {
  static constexpr int kBRows = BN / CG;
  static constexpr int kStageBytes = kABytes + kBRows * kStageKBytes;
  static constexpr int kStages = 196608 / kStageBytes;                      // 6 x 32 KiB or 8 x 24 KiB
  static constexpr int kAcc = 512 / BN;
  static constexpr int kCols = 64;                                          // per epilogue warp
  static constexpr int kEpiWarps = 4 * BN / kCols;
  static constexpr int kSfSlots = 16;
  static constexpr int kSfBytes = 512 + 16;                                 // 128 row scales, the scales of the tile's weight blocks
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr size_t kSmemBytes = 1024 + static_cast<size_t>(kStages) * kStageBytes + kSfSlots * kSfBytes + 640 + kEpiWarps * 32 * 36;
  static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// Tile order: bands of `band` row tiles, M fastest inside a band, so that the CTAs running together share operands in L2.
__device__ __forceinline__ void fp8_tile(int tile, const Fp8GemmArgs& g, int& tm, int& tn) {
  const int per = g.band * g.tiles_n, b = tile / per, r = tile - b * per, rows = min(g.band, g.tiles_m - b * g.band);
  tn = r / rows;
  tm = b * g.band + (r - tn * rows);
}

// 16 neighbouring columns of 32 rows, a row per lane.  Where rows or the edge do not allow wide stores the columns go through
// 1152 bytes of the warp's own (rows 36 bytes apart: no bank twice), so that neighbouring lanes still store neighbouring columns:
// 2549 x 336 -> 5057 takes 25 us, with each lane storing its row by elements 135; 1079 x 816 -> 12188 30 and 150.
constexpr int kStoreBytes = 32 * 36;
template <typename OUT>
__device__ __forceinline__ void store16(const Fp8GemmArgs& g, int row0, int lane, int col, const float2* s, uint8_t* scratch) {
  if (g.vec && col + 16 <= g.n) {
    OUT* y = static_cast<OUT*>(g.y) + (row0 + lane) * g.ldy;
    if (row0 + lane >= g.m) return;
    if constexpr (sizeof(OUT) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) __stcs(reinterpret_cast<float4*>(y + col) + i, make_float4(s[2 * i].x, s[2 * i].y, s[2 * i + 1].x, s[2 * i + 1].y));
    } else {
      uint32_t d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = f32x2_to_bf16x2(s[i].x, s[i].y);
      if (g.vec == 2) {
        asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(y + col), "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]),
                     "r"(d[4]), "r"(d[5]), "r"(d[6]), "r"(d[7]) : "memory");
      } else {
        __stcs(reinterpret_cast<uint4*>(y + col), make_uint4(d[0], d[1], d[2], d[3]));
        __stcs(reinterpret_cast<uint4*>(y + col + 8), make_uint4(d[4], d[5], d[6], d[7]));
      }
    }
    return;
  }
  constexpr int kPart = 32 / static_cast<int>(sizeof(OUT));          // columns that go through at a time
  const uint32_t base = smem_u32(scratch);
#pragma unroll
  for (int part = 0; part < 16; part += kPart) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t d;
      if constexpr (sizeof(OUT) == 4) d = __float_as_uint(i & 1 ? s[(part + i) / 2].y : s[(part + i) / 2].x);
      else d = f32x2_to_bf16x2(s[i].x, s[i].y);
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + lane * 36 + i * 4), "r"(d) : "memory");
    }
    __syncwarp();
    if (sizeof(OUT) == 4 || g.pairs) {                  // eight words a row, four rows at a time
      const int c = col + part + (lane & 7) * (4 / static_cast<int>(sizeof(OUT)));
#pragma unroll 1
      for (int i = lane >> 3; i < 32; i += 4) {
        uint32_t d;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(d) : "r"(base + i * 36 + (lane & 7) * 4) : "memory");
        if (row0 + i < g.m && c < g.n) *reinterpret_cast<uint32_t*>(static_cast<OUT*>(g.y) + (row0 + i) * g.ldy + c) = d;
      }
    } else {                                            // sixteen elements a row, two rows at a time
      const int c = col + (lane & 15);
#pragma unroll 1
      for (int i = lane >> 4; i < 32; i += 2) {
        uint16_t d;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(d) : "r"(base + i * 36 + (lane & 15) * 2) : "memory");
        if (row0 + i < g.m && c < g.n) *reinterpret_cast<uint16_t*>(static_cast<OUT*>(g.y) + (row0 + i) * g.ldy + c) = d;
      }
    }
  }
}

template <int BN, int CG, typename OUT>
__global__ void __launch_bounds__(GmCfg<BN, CG>::kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Fp8GemmMaps maps, const Fp8GemmArgs g) {
  using C = GmCfg<BN, CG>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_ring = smem + static_cast<size_t>(C::kStages) * C::kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sf_ring + C::kSfSlots * C::kSfBytes);
  uint64_t* empty_bar = full_bar + C::kStages;
  uint64_t* acc_full = empty_bar + C::kStages;
  uint64_t* acc_empty = acc_full + C::kAcc;
  uint64_t* sf_full = acc_empty + C::kAcc;
  uint64_t* sf_empty = sf_full + C::kSfSlots;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(sf_empty + C::kSfSlots);
  uint8_t* store_s = smem + C::kSmemBytes - 1024 - C::kEpiWarps * kStoreBytes;        // the epilogue warps' way out
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int s = 0; s < C::kAcc; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], C::kEpiWarps * CG); }
    for (int s = 0; s < C::kSfSlots; ++s) { mbar_init(&sf_full[s], 32); mbar_init(&sf_empty[s], C::kEpiWarps); }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && elect_one()) { prefetch_tmap(&maps.a); prefetch_tmap(&maps.w); }
  if (warp == 1) {
    tmem_alloc<CG>(tmem_holder, 512);
    tmem_relinquish<CG>();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) {
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_launch_dependents();

  const int num_tiles = g.tiles_m * g.tiles_n;
  const int first = static_cast<int>(cluster_id_x()), step = static_cast<int>(nclusters_x());
  // without a pair the CTAs of a cluster share a tile along K
  uint32_t cluster_size;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(cluster_size));
  const int slices = CG == 2 ? 1 : static_cast<int>(cluster_size), slice = CG == 2 ? 0 : static_cast<int>(cluster_ctarank());
  const int kb0 = g.kb * slice / slices, kb1 = g.kb * (slice + 1) / slices, kbs = kb1 - kb0;
  const uint32_t smem_base = smem_u32(smem);

  float2 acc[C::kCols / 2];                            // epilogue: 64 columns of this thread's row
  if (warp == 0 || warp == 3) {
    if (elect_one()) {
      pdl_wait();
      const uint32_t mine = warp == 0 ? 0u : 1u;       // K blocks of this producer: every other one, over all tiles
      uint32_t gs = 0;
      bool ok = true;
      for (int tile = first; ok && tile < num_tiles; tile += step) {
        int tm, tn;
        fp8_tile(tile, g, tm, tn);
        const int row_a = (tm * CG + static_cast<int>(rank)) * kBM, row_b = tn * BN + static_cast<int>(rank) * C::kBRows;
        for (int i = static_cast<int>((gs ^ mine) & 1u); i < kbs; i += 2) {
          const uint32_t x = gs + i, slot = x % C::kStages;
          const int kb = kb0 + i;
          ok = mbar_wait_bounded(&empty_bar[slot], ((x / C::kStages) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          const uint32_t st = smem_base + slot * C::kStageBytes;
          // in a pair every load of both CTAs is counted on the leader's barrier
          const uint32_t bar = smem_u32(&full_bar[slot]) & (CG == 2 ? 0xFEFFFFFFu : 0xFFFFFFFFu);
          if (leader) mbar_arrive_expect_tx(&full_bar[slot], CG * C::kStageBytes);
          tma_load_2d_cg<CG>(st, &maps.a, kb * kStageKBytes, row_a, bar);
          tma_load_2d_cg<CG>(st + kABytes, &maps.w, kb * kStageKBytes, row_b, bar);
        }
        gs += kbs;
      }
    }
  } else if (warp == 1) {
    if (elect_one() && leader) {
      constexpr uint32_t idesc = make_idesc_e4m3(128 * CG, BN);
      const uint32_t peer_off = CG == 2 ? map_to_cta(smem_u32(full_bar), 1u) - smem_u32(full_bar) : 0u;
      auto commit_all = [&](uint64_t* bar) {
        tc_commit<CG>(smem_u32(bar));
        if constexpr (CG == 2) tc_commit<CG>(smem_u32(bar) + peer_off);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return CG == 2 ? mbar_wait_bounded_cluster(bar, parity, abort_flag) : mbar_wait_bounded(bar, parity, abort_flag);
      };
      const uint32_t a_lo0 = desc_lo_sw128(smem_base), b_lo0 = desc_lo_sw128(smem_base + kABytes);
      uint32_t gs = 0;
      bool ok = true;
      for (int tile = first; ok && tile < num_tiles; tile += step)
        for (int kb = kb0; kb < kb1; ++kb, ++gs) {
          const uint32_t slot = gs % C::kStages, as = gs % C::kAcc;
          ok = wait(&acc_empty[as], ((gs / C::kAcc) & 1u) ^ 1u) && wait(&full_bar[slot], (gs / C::kStages) & 1u);
          if (!ok) break;
          tc_fence_after();
          const uint32_t off = slot * (C::kStageBytes >> 4);
#pragma unroll
          for (int h = 0; h < 4; ++h)
            tc_mma_e4m3<CG>(tmem_base + as * BN, a_lo0 + off + 2 * h, kDescHiSw128, b_lo0 + off + 2 * h, kDescHiSw128, idesc, h != 0);
          commit_all(&empty_bar[slot]);
          commit_all(&acc_full[as]);
        }
    }
  } else if (warp == 2) {
    pdl_wait();
    uint32_t gs = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles; tile += step) {
      int tm, tn;
      fp8_tile(tile, g, tm, tn);
      // rows and columns behind the end: their operands are zeros, any scale will do that can be read
      const float* src[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        src[i] = g.sa + static_cast<long long>(min((tm * CG + static_cast<int>(rank)) * kBM + lane + 32 * i, g.m - 1)) * g.kb;
      const float* sw = g.sw + static_cast<long long>(min(tn * BN + (lane & 1) * 128, g.n - 1) / kFp8Block) * g.kb;
      for (int kb = kb0; kb < kb1; ++kb, ++gs) {
        const uint32_t slot = gs % C::kSfSlots;
        ok = mbar_wait_bounded_lanes(&sf_empty[slot], ((gs / C::kSfSlots) & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        const uint32_t dst = smem_u32(sf_ring) + slot * C::kSfBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) cp_async4(dst + (lane + 32 * i) * 4, src[i] + kb);
        if (lane < BN / 128) cp_async4(dst + 512 + lane * 4, sw + kb);
        cp_async_arrive(&sf_full[slot]);
      }
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, cgp = (warp - 4) >> 2;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t empty_addr = CG == 2 ? map_to_cta(smem_u32(acc_empty), 0u) : smem_u32(acc_empty);
    pdl_wait();
    uint32_t gs = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles; tile += step) {
      int tm, tn;
      fp8_tile(tile, g, tm, tn);
      const int row0 = (tm * CG + static_cast<int>(rank)) * kBM + quad * 32;
      const int col0 = tn * BN + cgp * C::kCols;
#pragma unroll
      for (int j = 0; j < C::kCols / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
      for (int kb = kb0; kb < kb1; ++kb, ++gs) {
        const uint32_t as = gs % C::kAcc, slot = gs % C::kSfSlots;
        ok = mbar_wait_bounded_lanes(&sf_full[slot], (gs / C::kSfSlots) & 1u, abort_flag);
        if (!ok) break;
        const float* sf = reinterpret_cast<const float*>(sf_ring + slot * C::kSfBytes);
        const float f = sf[quad * 32 + lane] * sf[128 + cgp / 2];
        const float2 f2 = make_float2(f, f);
        ok = mbar_wait_bounded_lanes(&acc_full[as], (gs / C::kAcc) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + lane_base + as * BN + cgp * C::kCols;
#pragma unroll
        for (int c = 0; c < C::kCols / 16; ++c) {
          uint32_t r[16];
          tc_ld_32x32b_x16(taddr + c * 16, r);
          tc_wait_ld();
          if (c == C::kCols / 16 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 2) mbar_arrive_relaxed_cluster(empty_addr + 8u * as);
              else mbar_arrive(&acc_empty[as]);
              mbar_arrive(&sf_empty[slot]);
            }
          }
#pragma unroll
          for (int j = 0; j < 8; ++j)
            acc[c * 8 + j] = __ffma2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), f2, acc[c * 8 + j]);
        }
      }
      if (!ok) break;
      if (slices == 1) {
#pragma unroll
        for (int v = 0; v < C::kCols / 16; ++v) store16<OUT>(g, row0, lane, col0 + v * 16, acc + v * 8, store_s + (warp - 4) * kStoreBytes);
      }
    }
  }
  if constexpr (CG == 1) {
    if (slices > 1) {
      // One tile per cluster.  Each CTA adds, in the order of the slices, the 16-column groups g with g mod S = its rank; the
      // others' sums come to it through its ring, which is idle in every CTA behind the first barrier.
      const int quad = warp & 3, cgp = (warp - 4) >> 2, trow = quad * 32 + lane, per = (8 + slices - 1) / slices;
      float* slots = reinterpret_cast<float*>(smem);             // [slice][owned group][16 columns][128 rows]: whole lines per store
      __syncwarp();
      cluster_arrive_release();
      cluster_wait_acquire();
      if (warp >= 4) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int group = cgp * 4 + v, owner = group % slices;
          const uint32_t dst = map_to_cta(smem_u32(slots + (slice * per + group / slices) * 2048 + trow), static_cast<uint32_t>(owner));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 x = acc[v * 8 + i];
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 1024 * i), "f"(x.x) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 1024 * i + 512), "f"(x.y) : "memory");
          }
        }
      }
      __syncwarp();
      cluster_arrive_release();
      cluster_wait_acquire();
      if (warp >= 4 && !*abort_flag) {
        int tm, tn;
        fp8_tile(first, g, tm, tn);
        for (int at = cgp; at < per; at += 2) {
          const int group = at * slices + slice;
          if (group >= 8) break;
          float2 sum[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) sum[i] = make_float2(0.0f, 0.0f);
          for (int sl = 0; sl < slices; ++sl) {
            const float* src = slots + (sl * per + at) * 2048 + trow;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = make_float2(sum[i].x + src[256 * i], sum[i].y + src[256 * i + 128]);
          }
          store16<OUT>(g, tm * kBM + quad * 32, lane, tn * BN + group * 16, sum, store_s + (warp - 4) * kStoreBytes);
        }
      }
    }
  }

  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(g.status, PLQ_DEV_TIMEOUT);
    const long long t0 = clock64();                    // copies still in flight get time to land
    while (clock64() - t0 < 400000ll) __nanosleep(1000);
    __syncthreads();
  }
  if constexpr (CG == 2) {          // the leader's MMAs read the peer's shared memory: leave together
    tc_fence_before();
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, 512);
  }
}

// ---- host side -------------------------------------------------------------------------------------------------------
template <typename K>
static int launch_clusters(K kernel, unsigned grid, unsigned cluster, unsigned threads, size_t smem, void* stream, const Fp8GemmMaps& tm,
                           const Fp8GemmArgs& g) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tm, g));
  return PLQ_OK;
}

struct Fp8Ptrs { const void *a, *w; int64_t k; };

// How many clusters of 1 .. kMaxSlices CTAs of a kernel the device holds at once; looked up once per thread and device.
struct ClusterTable { int dev = -1, n[kMaxSlices + 1]; };
template <typename K>
static int clusters_at_once(K kernel, unsigned threads, size_t smem, int slices, ClusterTable* t) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (t->dev != dev) {
    for (int s = 1; s <= kMaxSlices; ++s) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(static_cast<unsigned>(s * 64), 1, 1);
      cfg.blockDim = dim3(threads, 1, 1);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = static_cast<unsigned>(s);
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
      t->n[s] = n;
    }
    (void)cudaGetLastError();
    t->dev = dev;
  }
  return t->n[slices];
}

// CTAs per tile: as many as keep all clusters on the device at once, none with fewer than `least` K blocks.  The occupancy
// query counts one CTA per SM for these kernels where `per_sm` run (16 x 8192 -> 8192 with 256 CTAs 13.8 us, with 128 16.1).
template <typename K>
static int k_slices(K kernel, unsigned threads, size_t smem, int64_t tiles, int per_sm, int kb, int least, ClusterTable* t) {
  int64_t s = static_cast<int64_t>(per_sm) * sm_count() / tiles;
  if (s > kMaxSlices) s = kMaxSlices;
  if (s > kb / least) s = kb / least;
  while (s > 1 && per_sm * clusters_at_once(kernel, threads, smem, static_cast<int>(s), t) < tiles) --s;
  return s > 1 ? static_cast<int>(s) : 1;
}

template <typename OUT>
static int launch_gemv(const Fp8Ptrs& p, Fp8GemmArgs& g, void* stream) {
  using C = GvCfg;
  auto kernel = fp8_gemv_kernel<OUT>;
  static thread_local int done_dev = -1;
  int st = allow_smem(kernel, C::kSmemBytes, &done_dev);
  if (st != PLQ_OK) return st;
  Fp8GemmMaps tm;
  memset(&tm, 0, sizeof(tm));
  if ((st = make_tmap(&tm.w, p.w, g.n, p.k, kBM)) != PLQ_OK) return st;
  if ((st = make_tmap(&tm.a, p.a, g.m, p.k, C::kRows)) != PLQ_OK) return st;
  g.tiles_n = (g.n + kBM - 1) / kBM;
  g.tiles_m = (g.m + C::kRows - 1) / C::kRows;
  const int slots = 2 * sm_count(), tiles = g.tiles_n * g.tiles_m;
  static thread_local ClusterTable table;
  const int slices = k_slices(kernel, C::kThreads, C::kSmemBytes, tiles, 2, g.kb, 1, &table);
  const int grid = slices > 1 ? tiles * slices : (tiles < slots ? tiles : slots);
  return launch_clusters(kernel, static_cast<unsigned>(grid), static_cast<unsigned>(slices), C::kThreads, C::kSmemBytes, stream, tm, g);
}

template <int BN, int CG, typename OUT>
static int launch_gemm_fp8(const Fp8Ptrs& p, Fp8GemmArgs& g, void* stream) {
  using C = GmCfg<BN, CG>;
  auto kernel = fp8_gemm_kernel<BN, CG, OUT>;
  static thread_local int done_dev = -1;
  int st = allow_smem(kernel, C::kSmemBytes, &done_dev);
  if (st != PLQ_OK) return st;
  Fp8GemmMaps tm;
  memset(&tm, 0, sizeof(tm));
  if ((st = make_tmap(&tm.a, p.a, g.m, p.k, kBM)) != PLQ_OK) return st;
  if ((st = make_tmap(&tm.w, p.w, g.n, p.k, C::kBRows)) != PLQ_OK) return st;
  g.tiles_m = (g.m + kBM * CG - 1) / (kBM * CG);
  g.tiles_n = (g.n + BN - 1) / BN;
  // The operand walked in the inner direction should stay in L2: narrow bands when A is the larger one and too big for that.
  const int64_t a_bytes = static_cast<int64_t>(g.m) * p.k, w_bytes = static_cast<int64_t>(g.n) * p.k;
  g.band = a_bytes > w_bytes && a_bytes > (32ll << 20) ? 4 : g.tiles_m;
  if (g.band > g.tiles_m) g.band = g.tiles_m;
  const int slots = sm_count() / CG, tiles = g.tiles_m * g.tiles_n;
  if constexpr (CG == 1) {
    static thread_local ClusterTable table;
    const int slices = k_slices(kernel, C::kThreads, C::kSmemBytes, tiles, 1, g.kb, 4, &table);
    if (slices > 1) return launch_clusters(kernel, static_cast<unsigned>(tiles * slices), static_cast<unsigned>(slices), C::kThreads, C::kSmemBytes, stream, tm, g);
  }
  return launch_clusters(kernel, static_cast<unsigned>((tiles < slots ? tiles : slots) * CG), CG, C::kThreads, C::kSmemBytes, stream, tm, g);
}

template <typename OUT>
static int launch_fp8(const Fp8Ptrs& p, Fp8GemmArgs& g, int variant, void* stream) {
  if (variant == PLQ_FP8_AUTO) {
    // Up to 16 rows the weights' bytes count.  Above, the shape with the smallest waves x time of a wave; per K block of a wave,
    // measured at 1024 x 8192 x 8192 and 8192 x 4096 x 14336: 128 x 128 0.34 us (the feed from L2: 14 TB/s), 256 x 128 of a pair
    // 0.32, 256 x 256 0.60.  Tiles that leave half of the SMs idle are split along K instead (128 x 128): 128 x 4096 x 8192
    // 22.2 -> 11.9 us, 77 x 6144 x 4096 12.8 -> 10.6.
    const int64_t sms = sm_count(), pairs = sms / 2 > 0 ? sms / 2 : 1, mt = (g.m + 127ll) / 128, nt = (g.n + 127ll) / 128;
    const auto waves = [](int64_t tiles, int64_t slots) { return (tiles + slots - 1) / slots; };
    const int64_t small = waves(mt * nt, sms) * 34, wide = waves((mt + 1) / 2 * nt, pairs) * 32, square = waves((mt + 1) / 2 * ((nt + 1) / 2), pairs) * 60;
    if (g.m <= 16) variant = PLQ_FP8_ROWS;
    else if (2 * mt * nt <= sms) variant = PLQ_FP8_128x128;
    else variant = square <= wide && square <= small ? PLQ_FP8_PAIR_256x256 : wide <= small && mt > 1 ? PLQ_FP8_PAIR_256x128 : PLQ_FP8_128x128;
  }
  if (variant == PLQ_FP8_ROWS) {
    if (g.m > 64) return PLQ_ERR_SHAPE;
    return launch_gemv<OUT>(p, g, stream);
  }
  if (variant == PLQ_FP8_128x128) return launch_gemm_fp8<128, 1, OUT>(p, g, stream);
  if (variant == PLQ_FP8_PAIR_256x256) return launch_gemm_fp8<256, 2, OUT>(p, g, stream);
  if (variant == PLQ_FP8_PAIR_256x128) return launch_gemm_fp8<128, 2, OUT>(p, g, stream);
  return PLQ_ERR_SHAPE;
}

}  // namespace plq

extern "C" int plq_fp8_gemm(const void* a_codes, const void* a_scales_f32, const void* w_codes, const void* w_scales_f32, int64_t m, int64_t n,
                            int64_t k, void* y, int64_t ldy, int y_is_f32, int32_t* dev_status, int flags, void* stream) {
  using namespace plq;
  const int variant = flags >> 4;
  if (m < 1 || n < 1 || k < 16 || k % 16 != 0 || ldy < n || variant < 0 || variant > PLQ_FP8_PAIR_256x128) return PLQ_ERR_SHAPE;
  if (m > (1 << 30) || n > (1 << 30) || k > (1 << 24) || (m + 127) / 128 * ((n + 127) / 128) > 0x7FFFFFFF) return PLQ_ERR_LIMIT;
  if (!a_codes || !a_scales_f32 || !w_codes || !w_scales_f32 || !y || !dev_status) return PLQ_ERR_NULL;
  const uintptr_t es = y_is_f32 ? 4 : 2;
  if (!aligned16(a_codes) || !aligned16(w_codes) || (reinterpret_cast<uintptr_t>(a_scales_f32) & 3u) || (reinterpret_cast<uintptr_t>(w_scales_f32) & 3u) ||
      reinterpret_cast<uintptr_t>(y) % es != 0)
    return PLQ_ERR_ALIGN;
  const int st = device_check();
  if (st != PLQ_OK) return st;
  Fp8GemmArgs g;
  memset(&g, 0, sizeof(g));
  g.sa = static_cast<const float*>(a_scales_f32);
  g.sw = static_cast<const float*>(w_scales_f32);
  g.y = y;
  g.ldy = ldy;
  g.status = dev_status;
  g.m = static_cast<int>(m);
  g.n = static_cast<int>(n);
  g.kb = static_cast<int>((k + kFp8Block - 1) / kFp8Block);
  g.static_w = flags & PLQ_FP8_STATIC_W;
  const auto fits = [&](uintptr_t bytes) { return reinterpret_cast<uintptr_t>(y) % bytes == 0 && static_cast<uintptr_t>(ldy) * es % bytes == 0; };
  g.vec = fits(32) ? 2 : fits(16) ? 1 : 0;
  g.pairs = reinterpret_cast<uintptr_t>(y) % 4 == 0 && ldy % 2 == 0 && n % 2 == 0;
  const Fp8Ptrs p = {a_codes, w_codes, k};
  return y_is_f32 ? launch_fp8<float>(p, g, variant, stream) : launch_fp8<__nv_bfloat16>(p, g, variant, stream);
}
