// A key / value cache in E4M3 with one scale per block of 64 tokens and head, and attention that reads it.
//
// Cache: codes u8 [batch, t_max, kv_heads, 128], scales float32 [batch, kv_heads, ceil(t_max / 64)], keys and values each.
// Scales are powers of two: a block is filled token by token, and when a new token does not fit the block's scale the rows
// that are already there move to the larger one.  By a power of two that is a change of exponent, exact but for the
// smallest codes; with arbitrary scales every growth would round all of the block again.
#include <cstring>

#include "plq_fp8.cuh"
#include "plq_quant.cuh"

namespace plq {

constexpr int kHeadDim = 128;

// ---- append ----------------------------------------------------------------------------------------------------------
struct Fp8AppendArgs {
  const uint4* qkv;            // bf16 [batch * t, ld]: [q heads | k heads | v heads]
  const float* cos;            // float32 [t, 128], or [batch, t, 128] (cs_batch != 0)
  const float* sin;
  uint4* q_out;                // bf16 [batch * t, heads, 128]
  uint8_t* codes[2];           // keys, values
  float* scales[2];
  const long long* pos_dev;    // first new position, one for all sequences (pos_batch = 0) or one each; or nullptr
  long long pos, t_max, ld8, cs_batch;
  long long q_threads;         // batch * t * heads * 8
  int* status;
  int t, heads, kv_heads, pos_batch, units_per_head;
  int scale_blocks;            // ceil(t_max / 64)
  unsigned q_blocks;
};

// The smallest 2^e with amax <= 448 * 2^e, e >= -100; `bits`: amax as an integer.
__device__ __forceinline__ float cache_scale(uint32_t bits) {
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
  return __uint_as_float(static_cast<uint32_t>(max(e, 127 - 100)) << 23);
}

// RoPE of four elements of a head: (2 l, 2 l + 1) and (64 + 2 l, 65 + 2 l) of lane l; every operation rounded on its own, then to
// bf16, as rope_kv_append_kernel does it.
__device__ __forceinline__ uint2 rope4(uint2 w, const float* cos, const float* sin, int lane) {
  const float2 c1 = *reinterpret_cast<const float2*>(cos + 2 * lane), c2 = *reinterpret_cast<const float2*>(cos + 64 + 2 * lane);
  const float2 s1 = *reinterpret_cast<const float2*>(sin + 2 * lane), s2 = *reinterpret_cast<const float2*>(sin + 64 + 2 * lane);
  const float ax = bf16lo_to_f32(w.x), ay = bf16hi_to_f32(w.x), bx = bf16lo_to_f32(w.y), by = bf16hi_to_f32(w.y);
  return make_uint2(f32x2_to_bf16x2(__fadd_rn(__fmul_rn(ax, c1.x), __fmul_rn(-bx, s1.x)), __fadd_rn(__fmul_rn(ay, c1.y), __fmul_rn(-by, s1.y))),
                    f32x2_to_bf16x2(__fadd_rn(__fmul_rn(bx, c2.x), __fmul_rn(ax, s2.x)), __fadd_rn(__fmul_rn(by, c2.y), __fmul_rn(ay, s2.y))));
}

// One launch: the first q_blocks blocks rotate the queries (eight threads per head, 16 elements each), every other block
// quantises one (sequence, head, keys or values, 64-token block) of the new rows, a warp per row and up to eight rows per
// warp.  Bound by the bytes of the projection (read once) and of the outputs; a decode step by its launch and the chain
// load -> maximum -> scale -> store.
__global__ void __launch_bounds__(256) rope_kv_append_fp8_kernel(const Fp8AppendArgs a) {
  __shared__ uint32_t warp_top[8];
  pdl_launch_dependents();
  pdl_wait();
  if (blockIdx.x < a.q_blocks) {
    const long long idx = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (idx >= a.q_threads) return;
    const int j = static_cast<int>(idx & 7);
    const long long hr = idx >> 3, row = hr / a.heads, b = row / a.t;
    const int head = static_cast<int>(hr - row * a.heads), tt = static_cast<int>(row - b * a.t);
    const uint4* src = a.qkv + row * a.ld8 + head * 16 + j;
    const uint4 lo = src[0], hi = src[8];
    const float* cos = a.cos + b * a.cs_batch + static_cast<long long>(tt) * kHeadDim + 8 * j;
    const float* sin = a.sin + b * a.cs_batch + static_cast<long long>(tt) * kHeadDim + 8 * j;
    const uint32_t lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
    uint32_t ol[4], oh[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 o = rope4(make_uint2(lw[i], hw[i]), cos, sin, i);
      ol[i] = o.x;
      oh[i] = o.y;
    }
    uint4* dst = a.q_out + hr * 16 + j;
    dst[0] = make_uint4(ol[0], ol[1], ol[2], ol[3]);
    dst[8] = make_uint4(oh[0], oh[1], oh[2], oh[3]);
    return;
  }
  const unsigned unit = blockIdx.x - a.q_blocks;
  const int u = static_cast<int>(unit % a.units_per_head);
  const unsigned rest = unit / a.units_per_head;
  const int side = static_cast<int>(rest & 1u), kh = static_cast<int>((rest >> 1) % a.kv_heads);
  const long long b = (rest >> 1) / a.kv_heads;
  const long long pos = a.pos_dev != nullptr ? a.pos_dev[b * a.pos_batch] : a.pos;
  if (pos < 0) return;                                // the sequence sits out
  if (pos > a.t_max - a.t) {                          // does not fit: nothing is stored, the caller is told
    if (threadIdx.x == 0 && a.status != nullptr) atomicExch(a.status, PLQ_DEV_RANGE);
    return;
  }
  const long long block = pos / kCacheBlock + u, lo = block * kCacheBlock;
  if (lo >= pos + a.t) return;
  const long long start = max(lo, pos);               // first new row of the block; [lo, start) hold earlier ones
  const int fresh = static_cast<int>(min(lo + kCacheBlock, pos + a.t) - start), before = static_cast<int>(start - lo);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = a.heads + (side ? a.kv_heads : 0) + kh;
  float* scale_at = a.scales[side] + (b * a.kv_heads + kh) * a.scale_blocks + block;
  const float old = before > 0 ? *scale_at : 0.0f;

  uint2 w[8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = warp + 8 * i;
    w[i] = make_uint2(0, 0);
    if (r < fresh) {
      const long long tt = start - pos + r;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(a.qkv + (b * a.t + tt) * a.ld8 + head * 16) + lane;
      w[i] = make_uint2(src[0], src[32]);
      if (!side) w[i] = rope4(w[i], a.cos + b * a.cs_batch + tt * kHeadDim, a.sin + b * a.cs_batch + tt * kHeadDim, lane);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    top = max(max(top, max((w[i].x << 16) & 0x7FFF0000u, w[i].x & 0x7FFF0000u)), max((w[i].y << 16) & 0x7FFF0000u, w[i].y & 0x7FFF0000u));
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
  if (lane == 0) warp_top[warp] = top;
  __syncthreads();                                    // also: every thread has read the old scale
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, warp_top[i]);
  // A value that is not finite, or an earlier one of the block that was not: the scale is NaN and the new codes are zeros.
  const bool finite = top < 0x7F800000u && old == old;
  const float s = finite ? fmaxf(cache_scale(top), old) : __uint_as_float(0x7FFFFFFFu);
  uint8_t* rows = a.codes[side] + ((b * a.t_max + lo) * a.kv_heads + kh) * kHeadDim;
  const long long row_bytes = static_cast<long long>(a.kv_heads) * kHeadDim;
  if (before > 0 && finite && s != old) {             // move the earlier rows to the new scale
    const float f = old / s;                          // a power of two (or whatever scale the caller put there)
    for (int r = warp; r < before; r += 8) {
      uint32_t* p = reinterpret_cast<uint32_t*>(rows + r * row_bytes) + lane;
      const uint32_t c = *p;
      const float2 x = e4m3x2_to_f32x2(c & 0xFFFFu), y = e4m3x2_to_f32x2(c >> 16);
      *p = e4m3x2(x.x * f, x.y * f) | e4m3x2(y.x * f, y.y * f) << 16;
    }
  }
  const float inv = finite ? 1.0f / s : 0.0f;         // exact for a power of two
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = warp + 8 * i;
    if (r >= fresh) break;
    uint16_t* p = reinterpret_cast<uint16_t*>(rows + (before + r) * row_bytes) + lane;
    p[0] = static_cast<uint16_t>(finite ? e4m3x2(bf16lo_to_f32(w[i].x) * inv, bf16hi_to_f32(w[i].x) * inv) : 0u);
    p[32] = static_cast<uint16_t>(finite ? e4m3x2(bf16lo_to_f32(w[i].y) * inv, bf16hi_to_f32(w[i].y) * inv) : 0u);
  }
  if (threadIdx.x == 0) *scale_at = s;
}

// ---- attention -------------------------------------------------------------------------------------------------------
// out[row] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * q_row . k_t),  over the positions t <= pos + i of a query i.
//
// One pass over the cache with the 8-bit codes fed to the tensor core as they are (tcgen05 kind::f8f6f4): no thread
// converts or scales a key or a value.  For that the other operand has to be 8-bit too, without losing its precision, and
// is the sum of two E4M3 numbers, which are two sets of columns of one product:
//   q      hi + lo / 16 (4 + 4 significant bits: exact for bf16 within 2^-22 of the largest query of the tile; one
//          power-of-two scale per tile of queries)
//   256 p  hi + lo, 256 p <= 256 within a tile of 128 tokens: off by at most 2^-9 of itself (a bf16 would be by 2^-8) or by
//          half a step of 2^-9, which is 2^-18 of the tile's largest weight
// With S^T = K Q^T the 128 tokens of a tile are the lanes of tensor memory and the query rows its columns (R = 8, 16 or 32 of
// them: heads of a group x queries), so a thread owns one token, and the scale of its key is a factor of the whole warp;
// O^T = V^T P^T has the 128 elements of the head as its lanes.  Each 64-token block of V gets an accumulator of its own, to
// which the block's scale is applied in float32 on the way into the running sums in registers.
//   warp 0 producer (TMA: 128 tokens x 128 bytes of keys, of values), warp 1 MMA issuer, warps 2 - 5 softmax and sums
// The cache's tiles can be split over several CTAs whose partial sums fp8_attention_join_kernel adds in a fixed order.
struct Fp8AttnArgs {
  const __nv_bfloat16* q;      // [batch, t, heads, 128]
  const float* k_scale;        // [batch, kv_heads, scale_blocks]
  const float* v_scale;
  __nv_bfloat16* out;          // [batch, t, heads, 128]
  float* part;                 // [splits][batch * t * heads][128] sums, then [splits][batch * t * heads][2] (maximum, weight)
  const long long* pos_dev;
  long long pos, t_max, rows_all;      // rows_all = batch * t * heads
  int* status;
  float scale_log2;            // scale * log2(e)
  int batch, t, heads, kv_heads, group, pos_batch, scale_blocks, splits, row_tiles;
};

template <int R>
struct AtCfg {
  static constexpr int kN = 2 * R;                     // columns of either product: hi | lo
  static constexpr int kPBytes = kN * 128;
  static constexpr int kQBytes = kN * 128;
  static constexpr int kKStages = 3, kVStages = R == 32 ? 2 : 3;
  static constexpr int kTile = 128 * kHeadDim;         // 16 KiB
  static constexpr int kDCol0 = 2 * kN;                // two S accumulators, then one D per 64-token block
  static constexpr int kTmemCols = 8 * R;
  static constexpr int kStatFloats = 2 * 4 * R /* warp maxima */ + 4 * 2 * 2 * R /* per warp: factors */ + 4 * R /* per warp: maxima */ + 4 * R;
  static constexpr size_t kSmemBytes = 1024 + kQBytes + kPBytes + static_cast<size_t>(kKStages + kVStages) * kTile + kStatFloats * 4 + R * 4 + 256;
  static_assert(2 * (kSmemBytes + 1024) <= 233472, "two CTAs per SM");
};

// 128-byte swizzled tile with the M side contiguous (V: 128 bytes of a token are the 128 rows of the MMA): groups of eight
// tokens 1024 bytes apart, as for the K-major tiles.  P: 16 rows x 8 tokens without swizzle, 128 bytes; eight-token groups
// 128 bytes apart (leading offset), 16-row groups 2048 bytes apart (stride offset).
constexpr uint32_t kDescHiP = (2048u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t desc_lo_p(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | ((128u >> 4) << 16); }

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(r) : "f"(v));
  return r;
}
// barrier of the 128 softmax threads; true where `ok` is in all of them, so that they leave a loop together
__device__ __forceinline__ bool softmax_barrier(bool ok = true) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %1, 0;\n\tbar.red.and.pred p, 1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(r) : "r"(static_cast<uint32_t>(ok)) : "memory");
  return r != 0;
}

constexpr float kNegInf = -__builtin_huge_valf();

template <int R>
__global__ void __launch_bounds__(192, 2) fp8_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                               const Fp8AttnArgs a) {
  using C = AtCfg<R>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                                            // [2 R rows x 128 bytes], 128-byte swizzle
  uint8_t* p_s = q_s + C::kQBytes;                                // [piece][16-row group][token][16]
  uint8_t* k_s = p_s + C::kPBytes;
  uint8_t* v_s = k_s + C::kKStages * C::kTile;
  float* wmax = reinterpret_cast<float*>(v_s + C::kVStages * C::kTile);      // [2][4 warps][R]
  float* fac = wmax + 2 * 4 * R;                                  // [4 warps][2][2: alpha, beta][R]
  float* mloc = fac + 4 * 2 * 2 * R;                              // [4 warps][R]: the tile's maxima
  float* red = mloc + 4 * R;                                      // [4 warps][R]
  int* lim_s = reinterpret_cast<int*>(red + 4 * R);               // [R] last position a row sees, relative to the tile loop's base
  uint64_t* bars = reinterpret_cast<uint64_t*>(lim_s + R);
  uint64_t* k_full = bars, *k_empty = k_full + C::kKStages, *v_full = k_empty + C::kKStages, *v_empty = v_full + C::kVStages;
  uint64_t* s_full = v_empty + C::kVStages, *s_empty = s_full + 2, *p_full = s_empty + 2, *d_full = p_full + 1, *q_full = d_full + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(q_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kKStages; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
    for (int s = 0; s < C::kVStages; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(&s_full[s], 1); mbar_init(&s_empty[s], 4); }
    mbar_init(p_full, 4);
    mbar_init(d_full, 1);
    mbar_init(q_full, 4);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && elect_one()) { prefetch_tmap(&map_k); prefetch_tmap(&map_v); }
  if (warp == 1) {
    tmem_alloc<1>(tmem_holder, C::kTmemCols);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's work: rows [row0, row0 + nrows) of (sequence b, key head kh), tiles [tile0, tile1) of the cache ----
  const int split = static_cast<int>(blockIdx.x);
  const int rt = a.row_tiles - 1 - static_cast<int>(blockIdx.y);       // the rows that see most first
  const int kh = static_cast<int>(blockIdx.z) % a.kv_heads;
  const long long b = blockIdx.z / static_cast<unsigned>(a.kv_heads);
  const int row0 = rt * R, nrows = min(R, a.t * a.group - row0);
  const long long pos = a.pos_dev != nullptr ? a.pos_dev[b * a.pos_batch] : a.pos;
  const bool fits = pos <= a.t_max - a.t;
  if (!fits && threadIdx.x == 0 && a.status != nullptr) atomicExch(a.status, PLQ_DEV_RANGE);
  int tiles = 0;
  const int i_min = row0 / a.group, i_max = (row0 + nrows - 1) / a.group;
  if (pos >= 0 && fits) tiles = static_cast<int>((pos + i_max) / 128) + 1;
  const int tile0 = static_cast<int>(static_cast<long long>(tiles) * split / a.splits);
  const int tile1 = static_cast<int>(static_cast<long long>(tiles) * (split + 1) / a.splits);
  const int n = tile1 - tile0;
  const uint32_t k_base = smem_u32(k_s), v_base = smem_u32(v_s);

  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      for (int j = 0; ok && j < n; ++j) {
        const int ks = j % C::kKStages, vs = j % C::kVStages;
        ok = mbar_wait_bounded(&k_empty[ks], ((j / C::kKStages) & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(&k_full[ks], C::kTile);
        tma_load_3d(k_base + ks * C::kTile, &map_k, kh * kHeadDim, (tile0 + j) * 128, static_cast<int>(b), smem_u32(&k_full[ks]));
        ok = mbar_wait_bounded(&v_empty[vs], ((j / C::kVStages) & 1u) ^ 1u, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(&v_full[vs], C::kTile);
        tma_load_3d(v_base + vs * C::kTile, &map_v, kh * kHeadDim, (tile0 + j) * 128, static_cast<int>(b), smem_u32(&v_full[vs]));
      }
    }
  } else if (warp == 1) {
    if (elect_one() && n > 0) {
      constexpr uint32_t idesc_s = make_idesc_e4m3(128, C::kN), idesc_d = make_idesc_e4m3(128, C::kN, true, true);
      const uint32_t q_lo = desc_lo_sw128(smem_u32(q_s)), p_lo = desc_lo_p(smem_u32(p_s));
      bool ok = mbar_wait_bounded(q_full, 0, abort_flag);
      for (int j = 0; ok && j <= n; ++j) {
        if (j < n) {                                  // S of tile j
          const int ks = j % C::kKStages;
          ok = mbar_wait_bounded(&s_empty[j & 1], ((j >> 1) & 1u) ^ 1u, abort_flag) &&
               mbar_wait_bounded(&k_full[ks], (j / C::kKStages) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t k_lo = desc_lo_sw128(k_base + ks * C::kTile);
#pragma unroll
          for (int h = 0; h < 4; ++h)
            tc_mma_e4m3<1>(tmem_base + (j & 1) * C::kN, k_lo + 2 * h, kDescHiSw128, q_lo + 2 * h, kDescHiSw128, idesc_s, h != 0);
          tc_commit<1>(smem_u32(&s_full[j & 1]));
          tc_commit<1>(smem_u32(&k_empty[ks]));
        }
        if (j > 0) {                                  // P V of tile j - 1
          const int vs = (j - 1) % C::kVStages;
          ok = mbar_wait_bounded(&v_full[vs], ((j - 1) / C::kVStages) & 1u, abort_flag) &&
               mbar_wait_bounded(p_full, (j - 1) & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t v_lo = desc_lo_sw128(v_base + vs * C::kTile);
#pragma unroll
          for (int h = 0; h < 4; ++h)                 // 32 tokens each; two 64-token blocks, two accumulators
            tc_mma_e4m3<1>(tmem_base + C::kDCol0 + (h >> 1) * C::kN, v_lo + h * (4096 >> 4), kDescHiSw128, p_lo + h * (512 >> 4), kDescHiP,
                           idesc_d, h & 1);
          tc_commit<1>(smem_u32(d_full));
          tc_commit<1>(smem_u32(&v_empty[vs]));
        }
      }
    }
  } else {
    const int sw = warp - 2, quad = warp & 3, tok = quad * 32 + lane, tid = static_cast<int>(threadIdx.x) - 64;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    float* my_fac = fac + sw * 4 * R;
    float* my_max = mloc + sw * R;

    // ---- the queries: tile-wide power-of-two scale, hi and lo codes ----
    constexpr int kPer = R > 16 ? R / 16 : 1;         // 16-element chunks per thread
    const bool has_q = R >= 16 || tid < 8 * R;
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u, keep = a.scale_log2 == 0.0f ? 0u : 0xFFFFFFFFu;      // a negative or no scale
    const __nv_bfloat16* q_base = a.q + ((b * a.t) * a.heads + static_cast<long long>(kh) * a.group) * kHeadDim;
    uint4 qv[kPer][2];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const int r = (tid >> 3) + 16 * c, row = row0 + r;
      qv[c][0] = qv[c][1] = make_uint4(0, 0, 0, 0);
      if (r < nrows) {
        const int i = row / a.group, h = row - i * a.group;
        const uint4* src = reinterpret_cast<const uint4*>(q_base + (static_cast<long long>(i) * a.heads + h) * kHeadDim) + 2 * (tid & 7);
        qv[c][0] = src[0];
        qv[c][1] = src[1];
      }
      uint32_t* w = reinterpret_cast<uint32_t*>(qv[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = (w[e] & keep) ^ flip;
        const uint32_t lo = (w[e] << 16) & 0x7FFF0000u, hi = w[e] & 0x7FFF0000u;
        if (lo < 0x7F800000u) top = max(top, lo);
        if (hi < 0x7F800000u) top = max(top, hi);
      }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    if (lane == 0) reinterpret_cast<uint32_t*>(red)[sw] = top;
    if (tid < R) {
      const int i = (row0 + tid) / a.group;
      lim_s[tid] = tid < nrows ? static_cast<int>(min(pos + i, 0x7FFFFFFFll)) : 0x7FFFFFFF;
    }
    softmax_barrier();
    top = max(max(reinterpret_cast<uint32_t*>(red)[0], reinterpret_cast<uint32_t*>(red)[1]),
              max(reinterpret_cast<uint32_t*>(red)[2], reinterpret_cast<uint32_t*>(red)[3]));
    softmax_barrier();
    // largest query in [128, 256): multiply by 2^e
    const int e = top == 0 ? 0 : min(max(134 - static_cast<int>(top >> 23), -120), 120);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
      const int r = (tid >> 3) + 16 * c, chunk = (tid & 7);
      uint32_t hi[4], lo[4];
      const uint32_t* w = reinterpret_cast<const uint32_t*>(qv[c]);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        uint32_t h2[2], l2[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float f0 = bf16lo_to_f32(w[2 * d + x]) * up, f1 = bf16hi_to_f32(w[2 * d + x]) * up;
          if (isinf(f0)) f0 = __uint_as_float(0x7FFFFFFFu);      // an infinite query is NaN, not the largest number
          if (isinf(f1)) f1 = __uint_as_float(0x7FFFFFFFu);
          h2[x] = e4m3x2(f0, f1);
          const float2 back = e4m3x2_to_f32x2(h2[x]);
          l2[x] = e4m3x2((f0 - back.x) * 16.0f, (f1 - back.y) * 16.0f);
        }
        hi[d] = h2[0] | h2[1] << 16;
        lo[d] = l2[0] | l2[1] << 16;
      }
      auto at = [&](int rr) { return reinterpret_cast<uint4*>(q_s + (rr >> 3) * 1024 + (rr & 7) * 128 + ((chunk ^ (rr & 7)) << 4)); };
      if (has_q) {
        *at(r) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *at(R + r) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);

    // ---- the tiles ----
    float o[R], l[R], m_run = kNegInf;                // o: element `tok` of the head; m_run: row `lane`
#pragma unroll
    for (int r = 0; r < R; ++r) o[r] = l[r] = 0.0f;
    const long long head_scales = (b * a.kv_heads + kh) * a.scale_blocks;
    const int lim_min = static_cast<int>(min(pos + i_min, 0x7FFFFFFFll));
    const long long written = pos + a.t;              // rows behind the last sequence position may hold anything
    bool ok = true;

    // adds the product of the tile before: o = o * alpha + (D0 * vs0 + D1 * vs1) * beta / 256
    auto promote = [&](int j, float vs0, float vs1) {
      ok = mbar_wait_bounded_lanes(d_full, j & 1u, abort_flag);
      if (!ok) return;
      tc_fence_after();
      const float* f = my_fac + (j & 1) * 2 * R;
      const bool finite = fabsf(vs0) < 3e38f && fabsf(vs1) < 3e38f;
      auto add = [&](int r, float d0, float d1, float al, float be) {
        if (!finite) {                                // a block of NaN: not for the rows that end before it
          d0 = lim_s[r] >= (tile0 + j) * 128 ? d0 * vs0 : 0.0f;
          d1 = lim_s[r] >= (tile0 + j) * 128 + kCacheBlock ? d1 * vs1 : 0.0f;
          o[r] = fmaf(o[r], al, (d0 + d1) * be);
        } else {
          o[r] = fmaf(o[r], al, fmaf(d0, vs0, d1 * vs1) * be);
        }
      };
      if constexpr (R == 8) {
        uint32_t d0[16], d1[16];
        tc_ld_32x32b_x16(tmem_base + lane_base + C::kDCol0, d0);
        tc_ld_32x32b_x16(tmem_base + lane_base + C::kDCol0 + C::kN, d1);
        tc_wait_ld();
#pragma unroll
        for (int r = 0; r < 8; ++r)
          add(r, __uint_as_float(d0[r]) + __uint_as_float(d0[8 + r]), __uint_as_float(d1[r]) + __uint_as_float(d1[8 + r]), f[r], f[R + r]);
      } else {
#pragma unroll
        for (int c = 0; c < R / 8; ++c) {
          uint32_t h0[8], l0[8], h1[8], l1[8];
          const uint32_t at = tmem_base + lane_base + C::kDCol0 + c * 8;
          tc_ld_32x32b_x8(at, h0);
          tc_ld_32x32b_x8(at + R, l0);
          tc_ld_32x32b_x8(at + C::kN, h1);
          tc_ld_32x32b_x8(at + C::kN + R, l1);
          tc_wait_ld();
#pragma unroll
          for (int x = 0; x < 8; ++x)
            add(c * 8 + x, __uint_as_float(h0[x]) + __uint_as_float(l0[x]), __uint_as_float(h1[x]) + __uint_as_float(l1[x]), f[c * 8 + x], f[R + c * 8 + x]);
        }
      }
      tc_fence_before();
    };
    float vs0 = 0.0f, vs1 = 0.0f;                     // scales of the tile whose product is on its way
    const float* k_scale = a.k_scale + head_scales;
    const float* v_scale = a.v_scale + head_scales;
    const int last_block = static_cast<int>((written - 1) / kCacheBlock);       // the last one that holds a position
    auto scale_of = [&](const float* side, int block) { return block <= last_block ? side[block] : 1.0f; };
    float next_k = 1.0f, next_v0 = 1.0f, next_v1 = 1.0f;
    const float per_k = down * (a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2));
    if (n > 0) {
      next_k = scale_of(k_scale, tile0 * 2 + (quad >> 1));
      next_v0 = scale_of(v_scale, tile0 * 2);
      next_v1 = scale_of(v_scale, tile0 * 2 + 1);
    }
    for (int j = 0; j < n; ++j) {                     // `ok` is looked at by all warps together, at the barrier
      const int tile = tile0 + j;
      const float nv0 = next_v0, nv1 = next_v1;
      float ksc = next_k * per_k;                     // of the warp's tokens
      if (ksc < 1.2e-38f) ksc = 1.2e-38f;             // a score of zero, and minus infinity stays what it is
      if (j + 1 < n) {                                // a tile ahead: they come from L2
        next_k = scale_of(k_scale, tile * 2 + 2 + (quad >> 1));
        next_v0 = scale_of(v_scale, tile * 2 + 2);
        next_v1 = scale_of(v_scale, tile * 2 + 3);
      }
      if (ok) ok = mbar_wait_bounded_lanes(&s_full[j & 1], (j >> 1) & 1u, abort_flag);
      tc_fence_after();
      float s[R];                                      // scores without the scale of the keys
      {
        const uint32_t at = tmem_base + lane_base + (j & 1) * C::kN;
        if constexpr (R == 8) {
          uint32_t x[16];
          tc_ld_32x32b_x16(at, x);
          tc_wait_ld();
#pragma unroll
          for (int r = 0; r < 8; ++r) s[r] = fmaf(__uint_as_float(x[8 + r]), 0.0625f, __uint_as_float(x[r]));
        } else {
#pragma unroll
          for (int c = 0; c < R / 16; ++c) {
            uint32_t x[16], y[16];
            tc_ld_32x32b_x16(at + c * 16, x);
            tc_ld_32x32b_x16(at + R + c * 16, y);
            tc_wait_ld();
#pragma unroll
            for (int r = 0; r < 16; ++r) s[c * 16 + r] = fmaf(__uint_as_float(y[r]), 0.0625f, __uint_as_float(x[r]));
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[j & 1]);
      }
      const int token = tile * 128 + tok;
      const bool masked = tile * 128 + 127 > lim_min;            // the same for the whole CTA
      if (masked) {
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (token > lim_s[r]) s[r] = kNegInf;
      }
      float mine = kNegInf;                            // lane r: the warp's maximum of row r
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float m = warp_max(s[r]);
        if (lane == r) mine = m;
      }
      float* wm = wmax + (j & 1) * 4 * R;
      if (lane < R) wm[sw * R + lane] = mine * ksc;
      ok = softmax_barrier(ok);
      if (!ok) break;
      if (lane < R) {
        const float m = fmaxf(fmaxf(wm[lane], wm[R + lane]), fmaxf(wm[2 * R + lane], wm[3 * R + lane]));
        const float m_new = fmaxf(m_run, m);
        my_fac[(j & 1) * 2 * R + lane] = m_run > kNegInf ? ex2_approx(m_run - m_new) : 0.0f;
        my_fac[(j & 1) * 2 * R + R + lane] = m > kNegInf ? ex2_approx(m - m_new - 8.0f) : 0.0f;
        my_max[lane] = m > kNegInf ? 8.0f - m : 0.0f;
        m_run = m_new;
      }
      __syncwarp();
      const float* f = my_fac + (j & 1) * 2 * R;
      uint32_t hi[R / 4], lo[R / 4];
#pragma unroll
      for (int r = 0; r < R; r += 4) {
        const float4 mx = *reinterpret_cast<const float4*>(my_max + r), al = *reinterpret_cast<const float4*>(f + r), be = *reinterpret_cast<const float4*>(f + R + r);
        float p[4] = {ex2_approx(fmaf(s[r], ksc, mx.x)), ex2_approx(fmaf(s[r + 1], ksc, mx.y)), ex2_approx(fmaf(s[r + 2], ksc, mx.z)),
                      ex2_approx(fmaf(s[r + 3], ksc, mx.w))};      // 256 p
        if (masked) {                                  // whatever the scale of their block is
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (token > lim_s[r + x]) p[x] = 0.0f;
        }
        l[r] = fmaf(l[r], al.x, p[0] * be.x);
        l[r + 1] = fmaf(l[r + 1], al.y, p[1] * be.y);
        l[r + 2] = fmaf(l[r + 2], al.z, p[2] * be.z);
        l[r + 3] = fmaf(l[r + 3], al.w, p[3] * be.w);
        const uint32_t c0 = e4m3_split(p[0], p[1]), c1 = e4m3_split(p[2], p[3]);
        hi[r / 4] = __byte_perm(c0, c1, 0x5410);
        lo[r / 4] = __byte_perm(c0, c1, 0x7632);
      }
      if (j > 0) {                                     // the product of tile j - 1 is done: its P may be overwritten
        promote(j - 1, vs0, vs1);
        if (!ok) continue;
      }
      vs0 = nv0;
      vs1 = nv1;
      if constexpr (R == 8) {
        *reinterpret_cast<uint4*>(p_s + tok * 16) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
      } else {
#pragma unroll
        for (int c = 0; c < R / 16; ++c) {
          *reinterpret_cast<uint4*>(p_s + c * 2048 + tok * 16) = make_uint4(hi[4 * c], hi[4 * c + 1], hi[4 * c + 2], hi[4 * c + 3]);
          *reinterpret_cast<uint4*>(p_s + (R / 16 + c) * 2048 + tok * 16) = make_uint4(lo[4 * c], lo[4 * c + 1], lo[4 * c + 2], lo[4 * c + 3]);
        }
      }
      if (static_cast<long long>(tile) * 128 + 128 > written) {  // rows that nobody has written: 0 x NaN would be NaN
        const int vs = j % C::kVStages;
        ok = mbar_wait_bounded_lanes(&v_full[vs], (j / C::kVStages) & 1u, abort_flag);
        if (!ok) continue;
        if (static_cast<long long>(tile) * 128 + tok >= written) {
          uint4* row = reinterpret_cast<uint4*>(v_s + vs * C::kTile + tok * 128);
#pragma unroll
          for (int x = 0; x < 8; ++x) row[x] = make_uint4(0, 0, 0, 0);
        }
      }
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (ok && n > 0) promote(n - 1, vs0, vs1);

    // ---- weights of the rows: over the lanes, then over the warps ----
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], d);
    }
    float mine = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (lane == r) mine = l[r];
    if (lane < R) red[sw * R + lane] = mine;
    softmax_barrier();
    float total = 0.0f;
    if (lane < R) total = (red[lane] + red[R + lane]) + (red[2 * R + lane] + red[3 * R + lane]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float sum = __shfl_sync(0xFFFFFFFFu, total, r), m = __shfl_sync(0xFFFFFFFFu, m_run, r);
      if (r >= nrows) continue;
      const int row = row0 + r, i = row / a.group, h = row - i * a.group;
      const long long at = (b * a.t + i) * a.heads + static_cast<long long>(kh) * a.group + h;
      if (a.splits == 1) {
        a.out[at * kHeadDim + tok] = __float2bfloat16_rn(sum == 0.0f ? 0.0f : o[r] / sum);
      } else {
        if (n > 0) a.part[(split * a.rows_all + at) * kHeadDim + tok] = o[r];
        if (tok == 0) *reinterpret_cast<float2*>(a.part + a.splits * a.rows_all * kHeadDim + (split * a.rows_all + at) * 2) = make_float2(m, sum);
      }
    }
  }

  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && a.status != nullptr) atomicExch(a.status, PLQ_DEV_TIMEOUT);
    const long long t0 = clock64();                    // copies still in flight get time to land
    while (clock64() - t0 < 400000ll) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, C::kTmemCols);
  }
}

// Adds the splits' partial sums, in order: one CTA of 128 threads per row.
__global__ void __launch_bounds__(128) fp8_attention_join_kernel(const float* part, __nv_bfloat16* out, long long rows, int splits) {
  extern __shared__ float weight[];                    // [splits]
  pdl_launch_dependents();
  pdl_wait();
  const long long row = blockIdx.x;
  const float2* stat = reinterpret_cast<const float2*>(part + splits * rows * kHeadDim);
  float top = kNegInf;
  for (int s = 0; s < splits; ++s) {
    const float2 st = stat[s * rows + row];
    if (st.y != 0.0f) top = fmaxf(top, st.x);
  }
  float total = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const float2 st = stat[s * rows + row];
    const float w = st.y == 0.0f ? 0.0f : ex2_approx(st.x - top);
    if (threadIdx.x == 0) weight[s] = st.y == 0.0f ? -1.0f : w;
    total = fmaf(st.y, w, total);
  }
  __syncthreads();
  float sum = 0.0f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float w = weight[s];
    if (w != -1.0f) sum = fmaf(part[(s * rows + row) * kHeadDim + threadIdx.x], w, sum);
  }
  out[row * kHeadDim + threadIdx.x] = __float2bfloat16_rn(total == 0.0f ? 0.0f : sum / total);
}

// ---- host side -------------------------------------------------------------------------------------------------------
// u8 cache [batch, t_max, kv_heads * 128]: boxes of 128 tokens x 128 bytes, 128-byte swizzle, zeros behind t_max.
static int make_cache_tmap(CUtensorMap* tm, const void* base, int64_t batch, int64_t t_max, int64_t kv_heads) {
  return make_tmap_3d(tm, base, kv_heads * kHeadDim, t_max, batch, kHeadDim, 128);
}

template <int R>
static int launch_attention(const CUtensorMap& mk, const CUtensorMap& mv, const Fp8AttnArgs& a, void* stream) {
  using C = AtCfg<R>;
  static thread_local int done_dev = -1;
  int dev = 0;
  PLQ_CUDA_TRY(cudaGetDevice(&dev));
  if (done_dev != dev) {
    PLQ_CUDA_TRY(cudaFuncSetAttribute(fp8_attention_kernel<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmemBytes)));
    done_dev = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.splits), static_cast<unsigned>(a.row_tiles), static_cast<unsigned>(a.batch * a.kv_heads));
  cfg.blockDim = dim3(192, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_attention_kernel<R>, mk, mv, a));
  if (a.splits > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows_all));
    cfg.blockDim = dim3(128, 1, 1);
    cfg.dynamicSmemBytes = a.splits * sizeof(float);
    PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_attention_join_kernel, const_cast<const float*>(a.part), a.out, static_cast<long long>(a.rows_all), a.splits));
  }
  return PLQ_OK;
}

// Rows of a CTA and splits of the cache for a call that sees up to `ctx` positions.
struct AttnPlan { int rows, row_tiles, splits; };
static AttnPlan attn_plan(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t ctx) {
  AttnPlan p;
  const int64_t rows = t * (heads / kv_heads);
  p.rows = rows <= 8 ? 8 : rows <= 16 ? 16 : 32;
  p.row_tiles = static_cast<int>((rows + p.rows - 1) / p.rows);
  // Two CTAs fit an SM.  As many splits as fill the device once, none shorter than four tiles of 128 tokens: a CTA's
  // set-up and its share of the join cost about what two tiles do.
  const int64_t ctas = batch * kv_heads * p.row_tiles, slots = 2 * static_cast<int64_t>(sm_count());
  int64_t splits = slots / ctas;
  const int64_t most = ((ctx + 127) / 128 + 3) / 4;
  if (splits > most) splits = most;
  if (splits < 1) splits = 1;
  p.splits = static_cast<int>(splits);
  return p;
}

}  // namespace plq

extern "C" int plq_rope_kv_append_fp8(const void* qkv_bf16, int64_t ld, const void* cos_f32, const void* sin_f32, int64_t cs_batch_stride,
                                      int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, void* q_out_bf16, void* k_codes,
                                      void* k_scales_f32, void* v_codes, void* v_scales_f32, int64_t t_max, const int64_t* pos_dev,
                                      int pos_per_sequence, int64_t pos, int32_t* dev_status, void* stream) {
  using namespace plq;
  if (batch < 0 || t < 0 || heads < 1 || kv_heads < 1 || t_max < 1) return PLQ_ERR_SHAPE;
  if (ld < (heads + 2 * kv_heads) * kHeadDim || ld % 8 != 0 || cs_batch_stride < 0 || cs_batch_stride % 4 != 0) return PLQ_ERR_SHAPE;
  if (pos_dev == nullptr && pos >= 0 && (t > t_max || pos > t_max - t)) return PLQ_ERR_SHAPE;
  if (heads + 2 * kv_heads > 4096 || batch > 0x7FFFFFFF || t > 0x7FFFFFFF || t_max > 0x7FFFFFFF - 128) return PLQ_ERR_LIMIT;
  if (batch == 0 || t == 0) return PLQ_OK;
  if (!qkv_bf16 || !cos_f32 || !sin_f32 || !q_out_bf16 || !k_codes || !k_scales_f32 || !v_codes || !v_scales_f32) return PLQ_ERR_NULL;
  if (!aligned16(qkv_bf16) || !aligned16(cos_f32) || !aligned16(sin_f32) || !aligned16(q_out_bf16) || !aligned16(k_codes) || !aligned16(v_codes) ||
      ((reinterpret_cast<uintptr_t>(k_scales_f32) | reinterpret_cast<uintptr_t>(v_scales_f32)) & 3u) || (reinterpret_cast<uintptr_t>(pos_dev) & 7u))
    return PLQ_ERR_ALIGN;
  int st = device_check();
  if (st != PLQ_OK) return st;
  Fp8AppendArgs a;
  a.qkv = static_cast<const uint4*>(qkv_bf16);
  a.cos = static_cast<const float*>(cos_f32);
  a.sin = static_cast<const float*>(sin_f32);
  a.q_out = static_cast<uint4*>(q_out_bf16);
  a.codes[0] = static_cast<uint8_t*>(k_codes);
  a.codes[1] = static_cast<uint8_t*>(v_codes);
  a.scales[0] = static_cast<float*>(k_scales_f32);
  a.scales[1] = static_cast<float*>(v_scales_f32);
  a.pos_dev = reinterpret_cast<const long long*>(pos_dev);
  a.pos = pos;
  a.t_max = t_max;
  a.ld8 = ld / 8;
  a.cs_batch = cs_batch_stride;
  a.q_threads = batch * t * heads * 8;
  a.status = dev_status;
  a.t = static_cast<int>(t);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.pos_batch = pos_per_sequence ? 1 : 0;
  a.scale_blocks = static_cast<int>((t_max + kCacheBlock - 1) / kCacheBlock);
  a.units_per_head = static_cast<int>((t + kCacheBlock - 2) / kCacheBlock + 1);      // blocks that t rows can touch
  const int64_t q_blocks = (a.q_threads + 255) / 256, blocks = q_blocks + batch * kv_heads * 2 * a.units_per_head;
  if (blocks > 0x7FFFFFFF) return PLQ_ERR_LIMIT;
  a.q_blocks = static_cast<unsigned>(q_blocks);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, rope_kv_append_fp8_kernel, a));
  return PLQ_OK;
}

extern "C" int64_t plq_fp8_attention_workspace_bytes(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t ctx) {
  using namespace plq;
  if (batch < 1 || t < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || ctx < 1) return 0;
  const AttnPlan p = attn_plan(batch, t, heads, kv_heads, ctx);
  return p.splits == 1 ? 0 : p.splits * batch * t * heads * static_cast<int64_t>((kHeadDim + 2) * sizeof(float));
}

extern "C" int plq_fp8_attention(const void* q_bf16, const void* k_codes, const void* k_scales_f32, const void* v_codes, const void* v_scales_f32,
                                 int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t t_max, const int64_t* pos_dev,
                                 int pos_per_sequence, int64_t pos, int64_t ctx, float scale, void* out_bf16, void* workspace,
                                 int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  using namespace plq;
  if (batch < 0 || t < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || t_max < 1 || ctx < 1 || ctx > t_max) return PLQ_ERR_SHAPE;
  if (pos_dev == nullptr && pos >= 0 && (t > t_max || pos > t_max - t)) return PLQ_ERR_SHAPE;
  if (pos_dev == nullptr && pos >= 0 && pos + t > ctx) return PLQ_ERR_SHAPE;
  if (heads > 4096 || batch * kv_heads > 65535 || t > (1 << 24) || t_max > 0x7FFFFFFF - 128) return PLQ_ERR_LIMIT;
  if (batch == 0 || t == 0) return PLQ_OK;
  if (!q_bf16 || !k_codes || !k_scales_f32 || !v_codes || !v_scales_f32 || !out_bf16) return PLQ_ERR_NULL;
  if (!aligned16(q_bf16) || !aligned16(k_codes) || !aligned16(v_codes) || !aligned16(out_bf16) || !aligned16(workspace) ||
      ((reinterpret_cast<uintptr_t>(k_scales_f32) | reinterpret_cast<uintptr_t>(v_scales_f32)) & 3u) || (reinterpret_cast<uintptr_t>(pos_dev) & 7u))
    return PLQ_ERR_ALIGN;
  int st = device_check();
  if (st != PLQ_OK) return st;
  const AttnPlan p = attn_plan(batch, t, heads, kv_heads, ctx);
  if (p.row_tiles > 65535) return PLQ_ERR_LIMIT;
  if (p.splits > 1 && !workspace) return PLQ_ERR_NULL;
  if (workspace_bytes < plq_fp8_attention_workspace_bytes(batch, t, heads, kv_heads, ctx)) return PLQ_ERR_LIMIT;
  Fp8AttnArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q_bf16);
  a.k_scale = static_cast<const float*>(k_scales_f32);
  a.v_scale = static_cast<const float*>(v_scales_f32);
  a.out = static_cast<__nv_bfloat16*>(out_bf16);
  a.part = static_cast<float*>(workspace);
  a.pos_dev = reinterpret_cast<const long long*>(pos_dev);
  a.pos = pos;
  a.t_max = t_max;
  a.rows_all = batch * t * heads;
  a.status = dev_status;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.batch = static_cast<int>(batch);
  a.t = static_cast<int>(t);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(heads / kv_heads);
  a.pos_batch = pos_per_sequence ? 1 : 0;
  a.scale_blocks = static_cast<int>((t_max + kCacheBlock - 1) / kCacheBlock);
  a.splits = p.splits;
  a.row_tiles = p.row_tiles;
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  if ((st = make_cache_tmap(&mk, k_codes, batch, t_max, kv_heads)) != PLQ_OK) return st;
  if ((st = make_cache_tmap(&mv, v_codes, batch, t_max, kv_heads)) != PLQ_OK) return st;
  if (p.rows == 8) return launch_attention<8>(mk, mv, a, stream);
  return p.rows == 16 ? launch_attention<16>(mk, mv, a, stream) : launch_attention<32>(mk, mv, a, stream);
}
