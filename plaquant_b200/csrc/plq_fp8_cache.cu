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
  long long q_threads;         // batch * t * heads * 8 / HT
  int* status;
  int t, heads, kv_heads, pos_batch, units_per_head;
  int scale_blocks;            // ceil(t_max / 64)
  unsigned long long unit_rate;  // 2^32 * units / blocks, rounded up: block i has floor(i * rate / 2^32) units before it
};

// The smallest 2^e with amax <= 448 * 2^e, e >= -100; `bits`: amax as an integer.
__device__ __forceinline__ float cache_scale(uint32_t bits) {
  const int e = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);      // 448 = 1.75 * 2^8
  return __uint_as_float(static_cast<uint32_t>(max(e, 127 - 100)) << 23);
}

// 16 bytes that are read once: not kept in L1, where the angles are
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// RoPE of two elements of a head's first half (x) and the two 64 behind them (y); every operation rounded on its own, then to
// bf16, as rope_kv_append_kernel does it.
__device__ __forceinline__ uint2 rope4(uint2 w, float2 c1, float2 c2, float2 s1, float2 s2) {
  const float ax = bf16lo_to_f32(w.x), ay = bf16hi_to_f32(w.x), bx = bf16lo_to_f32(w.y), by = bf16hi_to_f32(w.y);
  return make_uint2(f32x2_to_bf16x2(__fadd_rn(__fmul_rn(ax, c1.x), __fmul_rn(-bx, s1.x)), __fadd_rn(__fmul_rn(ay, c1.y), __fmul_rn(-by, s1.y))),
                    f32x2_to_bf16x2(__fadd_rn(__fmul_rn(bx, c2.x), __fmul_rn(ax, s2.x)), __fadd_rn(__fmul_rn(by, c2.y), __fmul_rn(ay, s2.y))));
}

// One launch.  Most blocks rotate queries (eight threads per head, 16 elements each of HT neighbouring heads: the angles are
// four times the bytes of a head's elements and come from L1 once per thread); a unit quantises one (sequence, head, keys or
// values, 64-token block) of the new rows, a warp per row and up to eight rows per warp.  Units lie evenly between the others:
// their chain load -> maximum -> scale -> store leaves time that the queries' streams fill.  Bound by the bytes of the
// projection (read once) and of the outputs; a decode step by its launch and that chain.  4 x 2048 tokens of 64 + 2 x 8 heads:
// 56 us (0.88 of the measured copy rate; 68 with the units last and the rows of a unit loaded one after the other); 16 tokens of 16
// sequences 2.6 us.
template <int HT>
__global__ void __launch_bounds__(256, 4) rope_kv_append_fp8_kernel(const Fp8AppendArgs a) {
  __shared__ uint32_t warp_top[8];
  pdl_launch_dependents();
  pdl_wait();
  // blocks of either kind alternate, so that the ones' waits are filled by the others' streams
  const unsigned units_before = static_cast<unsigned>(blockIdx.x * a.unit_rate >> 32);
  if (static_cast<unsigned>((blockIdx.x + 1) * a.unit_rate >> 32) == units_before) {
    const long long idx = static_cast<long long>(blockIdx.x - units_before) * blockDim.x + threadIdx.x;
    if (idx >= a.q_threads) return;
    const int j = static_cast<int>(idx & 7), groups = a.heads / HT;
    const long long hr = idx >> 3, row = hr / groups, b = row / a.t;
    const int head = static_cast<int>(hr - row * groups) * HT, tt = static_cast<int>(row - b * a.t);
    const uint4* src = a.qkv + row * a.ld8 + head * 16 + j;
    uint4 lo[HT], hi[HT];
#pragma unroll
    for (int x = 0; x < HT; ++x) { lo[x] = load_once(src + 16 * x); hi[x] = load_once(src + 16 * x + 8); }
    const float* cos = a.cos + b * a.cs_batch + static_cast<long long>(tt) * kHeadDim + 8 * j;
    const float* sin = a.sin + b * a.cs_batch + static_cast<long long>(tt) * kHeadDim + 8 * j;
    uint4* dst = a.q_out + (row * a.heads + head) * 16 + j;
    float c1[8], c2[8], s1[8], s2[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<float4*>(c1 + 4 * i) = *reinterpret_cast<const float4*>(cos + 4 * i);
      *reinterpret_cast<float4*>(c2 + 4 * i) = *reinterpret_cast<const float4*>(cos + 64 + 4 * i);
      *reinterpret_cast<float4*>(s1 + 4 * i) = *reinterpret_cast<const float4*>(sin + 4 * i);
      *reinterpret_cast<float4*>(s2 + 4 * i) = *reinterpret_cast<const float4*>(sin + 64 + 4 * i);
    }
#pragma unroll
    for (int x = 0; x < HT; ++x) {
      uint32_t* lw = reinterpret_cast<uint32_t*>(&lo[x]);
      uint32_t* hw = reinterpret_cast<uint32_t*>(&hi[x]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 o = rope4(make_uint2(lw[i], hw[i]), make_float2(c1[2 * i], c1[2 * i + 1]), make_float2(c2[2 * i], c2[2 * i + 1]),
                              make_float2(s1[2 * i], s1[2 * i + 1]), make_float2(s2[2 * i], s2[2 * i + 1]));
        lw[i] = o.x;
        hw[i] = o.y;
      }
      dst[16 * x] = lo[x];
      dst[16 * x + 8] = hi[x];
    }
    return;
  }
  const unsigned unit = units_before;
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
  if (fresh == kCacheBlock) {                          // a whole block: all loads are on their way before the first is used
    const uint32_t* src = reinterpret_cast<const uint32_t*>(a.qkv + (b * a.t + (start - pos) + warp) * a.ld8 + head * 16) + lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = make_uint2(src[32 * i * a.ld8], src[32 * i * a.ld8 + 32]);
    if (!side) {
      const long long at = b * a.cs_batch + (start - pos + warp) * kHeadDim;
      const float2* cos = reinterpret_cast<const float2*>(a.cos + at) + lane;
      const float2* sin = reinterpret_cast<const float2*>(a.sin + at) + lane;
#pragma unroll
      for (int g = 0; g < 8; g += 4) {
        float2 c[4][2], n[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            c[i][x] = cos[8 * (g + i) * (kHeadDim / 2) + 32 * x];
            n[i][x] = sin[8 * (g + i) * (kHeadDim / 2) + 32 * x];
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[g + i] = rope4(w[g + i], c[i][0], c[i][1], n[i][0], n[i][1]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = warp + 8 * i;
      w[i] = make_uint2(0, 0);
      if (r < fresh) {
        const long long tt = start - pos + r;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(a.qkv + (b * a.t + tt) * a.ld8 + head * 16) + lane;
        w[i] = make_uint2(src[0], src[32]);
        if (!side) {
          const float2* cos = reinterpret_cast<const float2*>(a.cos + b * a.cs_batch + tt * kHeadDim) + lane;
          const float2* sin = reinterpret_cast<const float2*>(a.sin + b * a.cs_batch + tt * kHeadDim) + lane;
          w[i] = rope4(w[i], cos[0], cos[32], sin[0], sin[32]);
        }
      }
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
//   q      hi + lo / 16 at a power of two of the row's own that brings its largest element to [128, 256): exact for what is at
//          least 2^-13 of that, off by 2^-21 of it below
//   256 p  hi + lo, 256 p <= 256 within a block of 64 tokens: off by at most 2^-9 + 2^-11 (f16 on the way) of itself or by half
//          a step of 2^-9, which is 2^-18 of the block's largest weight, whatever the other block's weights and values are
// With S^T = K Q^T the 128 tokens of a tile are the lanes of tensor memory and the query rows its columns (R = 8 or 16 of
// them: heads of a group x queries), so a thread owns one token, and the scale of its key is a factor of the whole warp;
// O^T = V^T P^T has the 128 elements of the head as its lanes.  Each 64-token block of V gets an accumulator of its own, to
// which the block's scale is applied in float32 on the way into the running sums in registers.
//   warp 0 producer (TMA: 128 tokens x 128 bytes of keys, of values), warp 1 MMA issuer, warps 2 - 5 softmax and sums
// Work: the tiles of all sequences in one row, cut into as many equal runs as CTAs fit the device, so that sequences of
// different lengths load it evenly and no length has to be known on the host.  A run is one or several segments (tiles of one
// sequence); a sequence that lies in several runs leaves partial sums, at most two per run (its first and its last segment),
// which fp8_attention_join_kernel adds in a fixed order.
// Bound by the cache's bytes for long ones: one sequence of 131072 positions (64 heads on 8) 51 us, 5.2 TB/s; 16 of 4096 (32 on 8)
// 31 us, 4.3 TB/s, and 25 us of different lengths.  A tile is a chain of some 2000 cycles for a CTA (scores, maxima over the
// lanes, weights, product), which two CTAs per SM turn into the memory's rate; about 2.5 us before the first tile and 4 us for
// the join come on top, which is what a short cache consists of (1 x 4096: 9.3 us).  A join in the kernel itself by the
// last CTA of a sequence took 64 and 36 us: its counters are six round trips to L2.
constexpr int kMaxFlat = 256;                          // sequences whose tiles are cut as one row

struct Fp8AttnArgs {
  const __nv_bfloat16* q;      // [batch, t, heads, 128]
  const float* k_scale;        // [batch, kv_heads, scale_blocks]
  const float* v_scale;
  __nv_bfloat16* out;          // [batch, t, heads, 128]
  float* part;                 // [units][runs][2][R][128] sums, then [units][runs][2][R][2] (maximum, weight); fp8_prefill_kernel:
                               // [batch][units][runs][128][128], [batch][units][runs][128][2].  A unit is a row tile of a key head
  const long long* pos_dev;
  long long pos, t_max;
  int* status;
  float scale_log2;            // scale * log2(e)
  int batch, t, heads, kv_heads, group, pos_batch, scale_blocks, row_tiles;
  int runs;                    // runs of the row of tiles (fp8_prefill_kernel: of each sequence), or 0: one CTA per sequence
};

// Tiles of 128 positions that sequence b has (0: it sits out, or does not fit).
__device__ __forceinline__ int sequence_tiles(const Fp8AttnArgs& a, long long b, long long* pos_out = nullptr) {
  const long long pos = a.pos_dev != nullptr ? a.pos_dev[b * a.pos_batch] : a.pos;
  if (pos_out != nullptr) *pos_out = pos;
  return pos < 0 || pos > a.t_max - a.t ? 0 : static_cast<int>((pos + a.t - 1) / 128) + 1;
}
// Run r holds the tiles [r * run_length, (r + 1) * run_length) of the row of tiles; the last runs may be empty.
__device__ __forceinline__ int run_length(int total, int runs) { return max(1, (total + runs - 1) / runs); }

template <int R>
struct AtCfg {
  static_assert(R == 8 || R == 16, "rows of a key head: queries x heads of a group");
  static constexpr int kN = 2 * R;                     // columns of either product: hi | lo
  static constexpr int kPBytes = kN * 128;
  static constexpr int kQBytes = kN * 128;
  static constexpr int kKStages = 3, kVStages = 3;
  static constexpr int kTile = 128 * kHeadDim;         // 16 KiB
  static constexpr int kDCol0 = 2 * kN;                // two S accumulators, then one D per 64-token block
  static constexpr int kTmemCols = 8 * R;
  static constexpr int kStatFloats = 2 * 4 * R /* warp maxima */ + 4 * 2 * 3 * R /* per warp: factors */ + 4 * 3 * R /* per warp: of its tokens */ + 4 * R + R;
  static constexpr size_t kSmemBytes = 1024 + kQBytes + kPBytes + static_cast<size_t>(kKStages + kVStages) * kTile + kStatFloats * 4 + R * 4 + (2 * kMaxFlat + 6) * 4 + 256;
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
// Behind scores (base 2) far beyond 2^21 the 8 of 8 - m has no bits left and the weights would be anything.  Inside a block such
// scores are scaled down to 2^21, so that differences of 2^-21 of their size are one; between blocks they count as they are.
constexpr float kVast = 2097152.0f;
__device__ __forceinline__ float vast_factor(float m) { return fminf(1.0f, kVast * rcp_approx(fabsf(m))); }

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
  float* fac = wmax + 2 * 4 * R;                                  // [4 warps][2][3: alpha, factor of either block's product][R]
  float* mloc = fac + 4 * 2 * 3 * R;                              // [4 warps][3: maxima of the block, factor of its weights, scale of its scores][R]
  float* red = mloc + 4 * 3 * R;                                  // [4 warps][R]
  float* down_s = red + 4 * R;                                    // [R] scale of a row's scores without that of the keys
  int* lim_s = reinterpret_cast<int*>(down_s + R);               // [R] last position a row sees, relative to the tile loop's base
  int* first_s = lim_s + R;                                       // [batch + 1] first tile of each sequence in the row of tiles
  int* pos_s = first_s + kMaxFlat + 1;                            // their positions
  int* start_s = pos_s + kMaxFlat;                                // the run: first and last tile, sequence of the first
  uint64_t* bars = reinterpret_cast<uint64_t*>(start_s + 5);
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

  // ---- this CTA's work: all rows of key head kh, tiles [run0, run1) of the row of tiles ----
  const int kh = static_cast<int>(blockIdx.x), run = static_cast<int>(blockIdx.y), nrows = a.t * a.group;
  int run0 = 0, run1 = 0;
  pdl_wait();
  pdl_launch_dependents();                             // behind the wait: what joins the sums reads the positions before its own
  if (a.runs) {
    if (warp == 0) {                                   // prefix sums of the sequences' tiles
      int sum = 0;
      for (int b0 = 0; b0 < a.batch; b0 += 32) {
        long long pos = -1;
        const int own = b0 + lane < a.batch ? sequence_tiles(a, b0 + lane, &pos) : 0;
        int x = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int y = __shfl_up_sync(0xFFFFFFFFu, x, d);
          if (lane >= d) x += y;
        }
        if (b0 + lane < a.batch) {
          first_s[b0 + lane] = sum + x - own;
          pos_s[b0 + lane] = own ? static_cast<int>(pos) : -1;
        }
        sum += __shfl_sync(0xFFFFFFFFu, x, 31);
      }
      const int length = run_length(sum, a.runs), from = min(run * length, sum);
      __syncwarp();
      int begun = 0;                                   // sequences that start at or before the run's first tile
      for (int b0 = 0; b0 < a.batch; b0 += 32)
        begun += __popc(__ballot_sync(0xFFFFFFFFu, b0 + lane < a.batch && first_s[b0 + lane] <= from));
      if (lane == 0) {
        first_s[a.batch] = sum;
        start_s[0] = from;
        start_s[1] = min(from + length, sum);
        start_s[2] = begun - 1;
      }
    }
    __syncthreads();
    run0 = start_s[0];
    run1 = start_s[1];
  }
  // the segments of the run, in order; false behind the last one
  struct Segment { int b, tile0, n; long long pos; bool whole; };
  int next_b = a.runs ? start_s[2] : run;
  auto next_segment = [&](Segment& g) {
    if (!a.runs) {
      if (next_b != run) return false;
      ++next_b;
      g.b = run;
      g.tile0 = 0;
      g.n = sequence_tiles(a, run, &g.pos);
      g.whole = true;
    } else {
      while (next_b < a.batch && first_s[next_b] < run1 && first_s[next_b + 1] <= max(run0, first_s[next_b])) ++next_b;     // empty ones
      if (next_b >= a.batch || first_s[next_b] >= run1) return false;
      g.b = next_b++;
      const int f = first_s[g.b], all = first_s[g.b + 1] - f;
      g.pos = pos_s[g.b];
      g.tile0 = max(run0 - f, 0);
      const int end = min(run1 - f, all);
      g.whole = g.tile0 == 0 && end == all;
      g.n = end - g.tile0;
    }
    return true;
  };
  if (kh == 0 && (run == 0 || !a.runs) && a.status != nullptr) {
    const int first = a.runs ? static_cast<int>(threadIdx.x) : run;
    for (int b = first; b < (a.runs ? a.batch : run + 1); b += 192) {
      const long long pos = a.pos_dev != nullptr ? a.pos_dev[b * a.pos_batch] : a.pos;
      if (pos > a.t_max - a.t && (a.runs || threadIdx.x == 0)) atomicExch(a.status, PLQ_DEV_RANGE);
    }
  }
  const uint32_t k_base = smem_u32(k_s), v_base = smem_u32(v_s);

  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      uint32_t gs = 0;
      Segment g;
      while (ok && next_segment(g))
        for (int j = 0; j < g.n; ++j, ++gs) {
          const uint32_t ks = gs % C::kKStages, vs = gs % C::kVStages;
          ok = mbar_wait_bounded(&k_empty[ks], ((gs / C::kKStages) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&k_full[ks], C::kTile);
          tma_load_3d(k_base + ks * C::kTile, &map_k, kh * kHeadDim, (g.tile0 + j) * 128, g.b, smem_u32(&k_full[ks]));
          ok = mbar_wait_bounded(&v_empty[vs], ((gs / C::kVStages) & 1u) ^ 1u, abort_flag);
          if (!ok) break;
          mbar_arrive_expect_tx(&v_full[vs], C::kTile);
          tma_load_3d(v_base + vs * C::kTile, &map_v, kh * kHeadDim, (g.tile0 + j) * 128, g.b, smem_u32(&v_full[vs]));
        }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_e4m3(128, C::kN), idesc_d = make_idesc_e4m3(128, C::kN, true, true);
      const uint32_t q_lo = desc_lo_sw128(smem_u32(q_s)), p_lo = desc_lo_p(smem_u32(p_s));
      bool ok = true;
      uint32_t gs = 0, seg = 0;
      Segment g;
      while (ok && next_segment(g)) {
        if (g.n == 0) continue;
        ok = mbar_wait_bounded(q_full, seg++ & 1u, abort_flag);
        for (int j = 0; ok && j <= g.n; ++j) {
          if (j < g.n) {                              // S of tile j
            const uint32_t x = gs + j, ks = x % C::kKStages;
            ok = mbar_wait_bounded(&s_empty[x & 1], ((x >> 1) & 1u) ^ 1u, abort_flag) &&
                 mbar_wait_bounded(&k_full[ks], (x / C::kKStages) & 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t k_lo = desc_lo_sw128(k_base + ks * C::kTile);
#pragma unroll
            for (int h = 0; h < 4; ++h)
              tc_mma_e4m3<1>(tmem_base + (x & 1) * C::kN, k_lo + 2 * h, kDescHiSw128, q_lo + 2 * h, kDescHiSw128, idesc_s, h != 0);
            tc_commit<1>(smem_u32(&s_full[x & 1]));
            tc_commit<1>(smem_u32(&k_empty[ks]));
          }
          if (j > 0) {                                // P V of tile j - 1
            const uint32_t x = gs + j - 1, vs = x % C::kVStages;
            ok = mbar_wait_bounded(&v_full[vs], (x / C::kVStages) & 1u, abort_flag) && mbar_wait_bounded(p_full, x & 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t v_lo = desc_lo_sw128(v_base + vs * C::kTile);
#pragma unroll
            for (int h = 0; h < 4; ++h)               // 32 tokens each; two 64-token blocks, two accumulators
              tc_mma_e4m3<1>(tmem_base + C::kDCol0 + (h >> 1) * C::kN, v_lo + h * (4096 >> 4), kDescHiSw128, p_lo + h * (512 >> 4), kDescHiP,
                             idesc_d, h & 1);
            tc_commit<1>(smem_u32(d_full));
            tc_commit<1>(smem_u32(&v_empty[vs]));
          }
        }
        gs += g.n;
      }
    }
  } else {
    const int sw = warp - 2, quad = warp & 3, tok = quad * 32 + lane, tid = static_cast<int>(threadIdx.x) - 64;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    float* my_fac = fac + sw * 6 * R;
    float* my_max = mloc + sw * 3 * R;
    const bool second = quad >= 2;                    // the tile's second block of 64

    bool ok = true;
    uint32_t gs = 0;
    Segment g;
    while (ok && next_segment(g)) {
    const long long b = g.b, pos = g.pos;
    const int n = g.n, tile0 = g.tile0;
    // ---- the queries: a row's scale, hi and lo codes ----
    const bool has_q = tid < 8 * R;                   // 16 elements each
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u, keep = a.scale_log2 == 0.0f ? 0u : 0xFFFFFFFFu;      // a negative or no scale
    const __nv_bfloat16* q_base = a.q + ((b * a.t) * a.heads + static_cast<long long>(kh) * a.group) * kHeadDim;
    uint4 qv[2];
    uint32_t top = 0;
    const int r = tid >> 3;
    qv[0] = qv[1] = make_uint4(0, 0, 0, 0);
    if (r < nrows) {
      const int i = r / a.group, h = r - i * a.group;
      const uint4* src = reinterpret_cast<const uint4*>(q_base + (static_cast<long long>(i) * a.heads + h) * kHeadDim) + 2 * (tid & 7);
      qv[0] = src[0];
      qv[1] = src[1];
    }
    uint32_t* w = reinterpret_cast<uint32_t*>(qv);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      w[e] = (w[e] & keep) ^ flip;
      const uint32_t lo = (w[e] << 16) & 0x7FFF0000u, hi = w[e] & 0x7FFF0000u;
      if (lo < 0x7F800000u) top = max(top, lo);
      if (hi < 0x7F800000u) top = max(top, hi);
    }
#pragma unroll
    for (int d = 4; d >= 1; d >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
    softmax_barrier();                                // the segment before has been read out
    if (tid < R) {
      const int i = tid / a.group;
      lim_s[tid] = tid < nrows ? static_cast<int>(min(pos + i, 0x7FFFFFFFll)) : 0x7FFFFFFF;
    }
    // largest element in [128, 256): multiply by 2^e
    const int e = top == 0 ? 0 : min(max(134 - static_cast<int>(top >> 23), -120), 120);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23), down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
    if (has_q && (tid & 7) == 0) down_s[r] = down * (a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2));
    {
      const int chunk = tid & 7;
      uint32_t hi[4], lo[4];
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
    softmax_barrier();
    if (lane == 0 && n > 0) mbar_arrive(q_full);
    const float down_lane = lane < R ? down_s[lane] : 1.0f;

    // ---- the tiles ----
    float o[R], l[R], m_run = kNegInf;                // o: element `tok` of the head; m_run: row `lane`
#pragma unroll
    for (int r = 0; r < R; ++r) o[r] = l[r] = 0.0f;
    const long long head_scales = (b * a.kv_heads + kh) * a.scale_blocks;
    const int lim_min = static_cast<int>(min(pos, 0x7FFFFFFFll));
    const long long written = pos + a.t;              // rows behind the last sequence position may hold anything

    // adds the product of the tile before: o = o * alpha + D0 * (vs0 * beta0 / 256) + D1 * (vs1 * beta1 / 256)
    auto promote = [&](int j, float vs0, float vs1) {
      ok = mbar_wait_bounded_lanes(d_full, (gs + j) & 1u, abort_flag);
      if (!ok) return;
      tc_fence_after();
      const float* f = my_fac + (j & 1) * 3 * R;
      const bool finite = fabsf(vs0) < 3e38f && fabsf(vs1) < 3e38f;
      auto add = [&](int r, float d0, float d1, float al, float f0, float f1) {
        if (!finite) {                                // a block of NaN: not for the rows that end before it
          d0 = lim_s[r] >= (tile0 + j) * 128 ? d0 * f0 : 0.0f;
          d1 = lim_s[r] >= (tile0 + j) * 128 + kCacheBlock ? d1 * f1 : 0.0f;
          o[r] = fmaf(o[r], al, d0 + d1);
        } else {
          o[r] = fmaf(o[r], al, fmaf(d0, f0, d1 * f1));
        }
      };
      if constexpr (R == 8) {
        uint32_t d0[16], d1[16];
        tc_ld_32x32b_x16(tmem_base + lane_base + C::kDCol0, d0);
        tc_ld_32x32b_x16(tmem_base + lane_base + C::kDCol0 + C::kN, d1);
        tc_wait_ld();
#pragma unroll
        for (int r = 0; r < 8; ++r)
          add(r, __uint_as_float(d0[r]) + __uint_as_float(d0[8 + r]), __uint_as_float(d1[r]) + __uint_as_float(d1[8 + r]), f[r], f[R + r], f[2 * R + r]);
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
          for (int x = 0; x < 8; x += 4) {
            const float4 al = *reinterpret_cast<const float4*>(f + c * 8 + x), f0 = *reinterpret_cast<const float4*>(f + R + c * 8 + x),
                         f1 = *reinterpret_cast<const float4*>(f + 2 * R + c * 8 + x);
            const auto d = [&](const uint32_t (&h)[8], const uint32_t (&l)[8], int y) { return __uint_as_float(h[y]) + __uint_as_float(l[y]); };
            add(c * 8 + x, d(h0, l0, x), d(h1, l1, x), al.x, f0.x, f1.x);
            add(c * 8 + x + 1, d(h0, l0, x + 1), d(h1, l1, x + 1), al.y, f0.y, f1.y);
            add(c * 8 + x + 2, d(h0, l0, x + 2), d(h1, l1, x + 2), al.z, f0.z, f1.z);
            add(c * 8 + x + 3, d(h0, l0, x + 3), d(h1, l1, x + 3), al.w, f0.w, f1.w);
          }
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
    if (n > 0) {
      next_k = scale_of(k_scale, tile0 * 2 + (quad >> 1));
      next_v0 = scale_of(v_scale, tile0 * 2);
      next_v1 = scale_of(v_scale, tile0 * 2 + 1);
    }
    for (int j = 0; j < n; ++j) {                     // `ok` is looked at by all warps together, at the barrier
      const int tile = tile0 + j;
      const float nv0 = next_v0, nv1 = next_v1;
      float ksc = next_k * down_lane;                 // of the warp's tokens and row `lane`
      if (ksc < 1.2e-38f) ksc = 1.2e-38f;             // a score of zero, and minus infinity stays what it is
      if (j + 1 < n) {                                // a tile ahead: they come from L2
        next_k = scale_of(k_scale, tile * 2 + 2 + (quad >> 1));
        next_v0 = scale_of(v_scale, tile * 2 + 2);
        next_v1 = scale_of(v_scale, tile * 2 + 3);
      }
      const uint32_t x = gs + j;                      // running index over the segments
      if (ok) ok = mbar_wait_bounded_lanes(&s_full[x & 1], (x >> 1) & 1u, abort_flag);
      tc_fence_after();
      float s[R];                                      // scores without the scale of the keys
      {
        const uint32_t at = tmem_base + lane_base + (x & 1) * C::kN;
        if constexpr (R == 8) {
          uint32_t v[16];
          tc_ld_32x32b_x16(at, v);
          tc_wait_ld();
#pragma unroll
          for (int r = 0; r < 8; ++r) s[r] = fmaf(__uint_as_float(v[8 + r]), 0.0625f, __uint_as_float(v[r]));
        } else {
          uint32_t v[16], y[16];
          tc_ld_32x32b_x16(at, v);
          tc_ld_32x32b_x16(at + 16, y);
          tc_wait_ld();
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = fmaf(__uint_as_float(y[r]), 0.0625f, __uint_as_float(v[r]));
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_empty[x & 1]);
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
        // warps 2 and 3 of the four have the first 64 tokens
        const float m0 = fmaxf(wm[2 * R + lane], wm[3 * R + lane]), m1 = fmaxf(wm[lane], wm[R + lane]), m = second ? m1 : m0;
        const float m_new = fmaxf(m_run, fmaxf(m0, m1));
        const float b0 = m0 > kNegInf ? ex2_approx(m0 - m_new - 8.0f) : 0.0f, b1 = m1 > kNegInf ? ex2_approx(m1 - m_new - 8.0f) : 0.0f;
        float* f = my_fac + (j & 1) * 3 * R;
        f[lane] = m_run > kNegInf ? ex2_approx(m_run - m_new) : 0.0f;
        f[R + lane] = b0 * nv0;
        f[2 * R + lane] = b1 * nv1;
        const float v = vast_factor(m);
        my_max[lane] = m > kNegInf ? fmaf(-m, v, 8.0f) : 0.0f;
        my_max[R + lane] = second ? b1 : b0;
        my_max[2 * R + lane] = ksc * v;
        m_run = m_new;
      }
      __syncwarp();
      const float* f = my_fac + (j & 1) * 3 * R;
      uint32_t hi[R / 4], lo[R / 4];
#pragma unroll
      for (int r = 0; r < R; r += 4) {
        const float4 mx = *reinterpret_cast<const float4*>(my_max + r), al = *reinterpret_cast<const float4*>(f + r), be = *reinterpret_cast<const float4*>(my_max + R + r),
                     ks = *reinterpret_cast<const float4*>(my_max + 2 * R + r);
        float p[4] = {ex2_approx(fmaf(s[r], ks.x, mx.x)), ex2_approx(fmaf(s[r + 1], ks.y, mx.y)), ex2_approx(fmaf(s[r + 2], ks.z, mx.z)),
                      ex2_approx(fmaf(s[r + 3], ks.w, mx.w))};      // 256 p
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
        *reinterpret_cast<uint4*>(p_s + tok * 16) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(p_s + 2048 + tok * 16) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      if (static_cast<long long>(tile) * 128 + 128 > written) {  // rows that nobody has written: 0 x NaN would be NaN
        const uint32_t vs = x % C::kVStages;
        ok = mbar_wait_bounded_lanes(&v_full[vs], (x / C::kVStages) & 1u, abort_flag);
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

    // ---- weights of the rows: over the lanes (each exchange halves the rows a lane still carries), then over the warps ----
#pragma unroll
    for (int d = 16, cnt = R / 2; cnt >= 1; d >>= 1, cnt >>= 1) {
      const bool up = (lane & d) != 0;
#pragma unroll
      for (int r = 0; r < cnt; ++r) {
        const float give = up ? l[r] : l[r + cnt], keep_l = up ? l[r + cnt] : l[r];
        l[r] = keep_l + __shfl_xor_sync(0xFFFFFFFFu, give, d);
      }
    }
#pragma unroll
    for (int d = 16 / R; d >= 1; d >>= 1) l[0] += __shfl_xor_sync(0xFFFFFFFFu, l[0], d);
    red[sw * R + lane / (32 / R)] = l[0];             // lane 32 / R * r and its neighbours have row r
    ok = softmax_barrier(ok);
    float total = 0.0f;
    if (lane < R) {
      total = (red[lane] + red[R + lane]) + (red[2 * R + lane] + red[3 * R + lane]);
      my_max[lane] = total == 0.0f ? 0.0f : 1.0f / total;
    }
    __syncwarp();
    const long long out_row = b * a.t * a.heads + static_cast<long long>(kh) * a.group;
    if (g.whole) {
      int h = 0;
      __nv_bfloat16* dst = a.out + out_row * kHeadDim + tok;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r < nrows) *dst = __float2bfloat16_rn(o[r] * my_max[r]);
        if (++h == a.group) { h = 0; dst += static_cast<long long>(a.heads - a.group) * kHeadDim; }
        dst += kHeadDim;
      }
    } else {
      const long long slot = (static_cast<long long>(kh) * a.runs + run) * 2 + (first_s[b] + tile0 == run0 ? 0 : 1);
      float* dst = a.part + slot * R * kHeadDim + tok;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < nrows) dst[r * kHeadDim] = o[r];
      if (sw == 0 && lane < nrows)
        *reinterpret_cast<float2*>(a.part + static_cast<long long>(gridDim.x) * a.runs * 2 * R * kHeadDim + (slot * R + lane) * 2) = make_float2(m_run, total);
    }
    gs += n;
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

// fp8_prefill_kernel, below
struct PfCfg {
  static constexpr int kRows = 128;
  static constexpr int kTile = 128 * kHeadDim;          // 16 KiB
  static constexpr int kBlock = kCacheBlock * kHeadDim; // 8 KiB: 64 positions of K or V
  static constexpr int kStages = 4;
  static constexpr int kScaleBytes = 512;               // 128 rows, a word each
  static constexpr size_t kSmemBytes = 1024 + 2 * kTile + 2 * kStages * kBlock + 2 * kScaleBytes + 256;
  // 128 registers a thread at launch (256 x 128); the warps with a row of scores per thread take what the others leave.
  static constexpr int kRegsMain = 56, kRegsRows = 200;
  static_assert(128 * kRegsMain + 128 * kRegsRows <= 256 * 128, "register split");
  static constexpr size_t kAlone = 116 * 1024;          // more than half of an SM's
  static_assert(kAlone >= kSmemBytes && 2 * (kSmemBytes + 1024) <= 233472, "shared memory budget");
};

// Adds the partial sums of the sequences that lie in several runs, in a fixed order, and clears the output of those that have
// no tiles: one CTA of four warps per row, a warp taking every fourth run and a lane four elements.
__global__ void __launch_bounds__(128) fp8_attention_join_kernel(const Fp8AttnArgs a, int rows_per_tile) {
  __shared__ int sum_s[4][2];
  __shared__ float4 acc_s[4][32];
  pdl_launch_dependents();
  // Up to the wait only the positions are read, which are older than the kernel before: that one lets this one begin when all
  // of its CTAs have waited for them.
  const int at = static_cast<int>(blockIdx.x), bi = at / a.heads, b = bi / a.t;
  const int head = at - bi * a.heads, i = bi - b * a.t, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = sequence_tiles(a, b);
  __nv_bfloat16* dst = a.out + static_cast<long long>(at) * kHeadDim;
  if (tiles == 0) {
    pdl_wait();
    dst[threadIdx.x] = __float2bfloat16_rn(0.0f);
    return;
  }
  int before = 0, all = 0;                             // tiles of the sequences in front, of all
  const bool own_runs = rows_per_tile == PfCfg::kRows;  // every sequence is cut into runs of its own
  if (own_runs) {
    all = tiles;
  } else if (a.pos_dev != nullptr && a.pos_batch) {
    for (int x = threadIdx.x; x < a.batch; x += 128) {
      const int n = sequence_tiles(a, x);
      all += n;
      if (x < b) before += n;
    }
    before = __reduce_add_sync(0xFFFFFFFFu, before);
    all = __reduce_add_sync(0xFFFFFFFFu, all);
    if (lane == 0) { sum_s[warp][0] = before; sum_s[warp][1] = all; }
    __syncthreads();
    before = sum_s[0][0] + sum_s[1][0] + sum_s[2][0] + sum_s[3][0];
    all = sum_s[0][1] + sum_s[1][1] + sum_s[2][1] + sum_s[3][1];
  } else {
    before = tiles * b;
    all = tiles * a.batch;
  }
  const int length = run_length(all, a.runs), r0 = before / length, n = (before + tiles - 1) / length - r0 + 1;
  const int kh = head / a.group, row = i * a.group + (head - kh * a.group), rt = row / rows_per_tile;
  const long long unit = static_cast<long long>(a.row_tiles - 1 - rt) * a.kv_heads + kh;
  const long long units = static_cast<long long>(a.row_tiles) * a.kv_heads;
  const int each = own_runs ? rows_per_tile : 2 * rows_per_tile;                 // partial sums of a run
  const float2* stat = reinterpret_cast<const float2*>(a.part + (own_runs ? a.batch : 1) * units * a.runs * each * kHeadDim);
  // the sequence is the first segment of every run but perhaps of the one it starts in
  const long long base = ((own_runs ? b * units + unit : unit) * a.runs + r0) * each + (row - rt * rows_per_tile);
  const int late = r0 * length < before ? rows_per_tile : 0;
  auto slot = [&](int x) { return base + (x == 0 ? late : static_cast<long long>(x) * each); };
  pdl_wait();
  if (n == 1) return;                                  // written whole
  // One round of loads: a warp's sums, and the maxima and weights of all runs in its lanes.
  float4 ahead[4];
#pragma unroll
  for (int y = 0; y < 4; ++y)
    ahead[y] = warp + 4 * y < n ? *reinterpret_cast<const float4*>(a.part + slot(warp + 4 * y) * kHeadDim + 4 * lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float2 own[2];
#pragma unroll
  for (int y = 0; y < 2; ++y) own[y] = lane + 32 * y < n ? stat[slot(lane + 32 * y)] : make_float2(kNegInf, 0.0f);
  float top = kNegInf;
#pragma unroll
  for (int y = 0; y < 2; ++y)
    if (own[y].y != 0.0f) top = fmaxf(top, own[y].x);
  for (int x = lane + 64; x < n; x += 32) {
    const float2 s = stat[slot(x)];
    if (s.y != 0.0f) top = fmaxf(top, s.x);
  }
  top = warp_max(top);
  auto factor = [&](const float2 s) { return s.y == 0.0f ? 0.0f : ex2_approx(s.x - top); };      // a run of which the row sees nothing left zeros
  const float w0 = factor(own[0]), w1 = factor(own[1]);
  float weight = fmaf(own[0].y, w0, own[1].y * w1);     // of the lane's runs
  for (int x = lane + 64; x < n; x += 32) {
    const float2 s = stat[slot(x)];
    weight = fmaf(s.y, factor(s), weight);
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) weight += __shfl_xor_sync(0xFFFFFFFFu, weight, d);
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float w, const float4 v) { acc = make_float4(fmaf(v.x, w, acc.x), fmaf(v.y, w, acc.y), fmaf(v.z, w, acc.z), fmaf(v.w, w, acc.w)); };
#pragma unroll
  for (int y = 0; y < 4; ++y) add(__shfl_sync(0xFFFFFFFFu, w0, warp + 4 * y), ahead[y]);
#pragma unroll 4
  for (int x = warp + 16; x < n; x += 4) {
    const float4 v = *reinterpret_cast<const float4*>(a.part + slot(x) * kHeadDim + 4 * lane);
    add(x < 64 ? __shfl_sync(0xFFFFFFFFu, x < 32 ? w0 : w1, x & 31) : factor(stat[slot(x)]), v);
  }
  acc_s[warp][lane] = acc;
  __syncthreads();
  const float* part = reinterpret_cast<const float*>(acc_s) + threadIdx.x;
  const float sum = (part[0] + part[128]) + (part[256] + part[384]);
  dst[threadIdx.x] = __float2bfloat16_rn(weight == 0.0f ? 0.0f : sum / weight);
}

// ---- attention of many queries -----------------------------------------------------------------------------------------
// The same sums with the queries as the 128 lanes: S = Q K^T, O = P V, a thread owning a row (a query and a head of the group),
// so that a row's maximum and weight need no exchange.  A CTA has 128 rows and two CTAs share an SM: while one of them begins
// or ends, or turns scores into weights, the tensor core works for the other.
//   q      hi + lo, both E4M3 at the scale of the row (a power of two that brings its largest element to [128, 256)): exact
//          for what is at least 2^-9 of that, off by 2^-17 of 128 below
//   S      of 64 positions, twice in tensor memory: the product of block j + 2 is issued behind the one that reads the weights
//          of block j, so the scores of j + 1 lie ready when the weights of j are done
//   p      w = exp2(score + log2 vs - e + 8) with e the row's largest score + log2 vs in the block of 64, rounded up: the scale of
//          V is part of the weight, and the block's largest is 128 to 256.  hi + lo, both E4M3, in tensor memory (A operand), in
//          the place of the scores they come from: off by at most 2^-9 + 2^-11 (f16 on the way) of itself or by half a step of
//          2^-9, which is 2^-17 of the block's largest weight
//   O      stays in tensor memory, in units of 2^R, R = e - 8 of the first block.  The tensor core applies 2^(e - 8 - R), an E8M0
//          scale per row and 32 positions (kind::mxf8f6f4), so no block's weights share an exponent with another's: a long tail of
//          small weights keeps its bits behind a position that outweighs each of them, and ordinary values behind a block of
//          large ones.  R moves only when a block is 2^60 above it.  The sum of the weights takes w / vs.  (With one running
//          exponent for the row two prompts of 2048 take 82 us instead of 84, 104 instead of 87 where scores spread four times
//          as wide and O is scaled often, but weights 12 nats below the row's largest are off by 24 % and those beyond 13 gone.)
//   warp 0 producer, warp 1 MMA issuer, warps 4 - 7 the rows
// 128 positions of two row tiles are 2048 cycles of the tensor core (four products of 128 x 128 x 128 each) and as many of
// exponentials (16 a cycle).  They take 2.2 us (about 4000 cycles): without the weights' arithmetic 1.2 us, with exponentials
// alone 1.9 us.  Bound by the instructions that turn scores into weights (some 11 an element, of which 3 the two codes), not by
// their latency: twice the warps with half of the blocks each took 5 % longer, codes by integer arithmetic 3 to 5 % longer.
// 8192 tokens of 32 heads on 8: 490 us (1.12 PFLOP/s); two prompts of 2048: 84 us.  Of these a CTA's beginning and end take
// 6 us each; they were 12 with the loops over queries and output unrolled, since code that runs once costs its fetch, and with
// both row tiles in one CTA nothing hid them: 102 us.  A CTA that took further work over from CTAs that had not started yet
// (the next queries prepared meanwhile by two warps) was slower, 110 us: two warps take longer for that than the tiles before.
// Few CTAs and a long past: each sequence is cut into runs, whose sums O and weight in units of their 2^R go to the join (64
// tokens of 32 heads on 8 behind 8000 positions 88 -> 26 us).
constexpr int kScaleBias = 127 - 8;                     // e - R = 8 is the scale one
constexpr int kScaleTop = 127 + 60;                     // beyond it R moves: O stays below 2^60 * 2^8 * 448 * positions
constexpr float kFarBelow = 92.0f;                      // blocks further below R than this share its scale, 2^-100

// RUNS: every sequence in a.runs runs of its own, for the join; as a branch it would cost the other calls 4 %
template <bool RUNS>
__global__ void __launch_bounds__(256, 2) fp8_prefill_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                             const Fp8AttnArgs a) {
  using C = PfCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* q_s = smem;                                  // [hi | lo][128 x 128 bytes]
  uint8_t* k_s = q_s + 2 * C::kTile;
  uint8_t* v_s = k_s + C::kStages * C::kBlock;
  uint8_t* w_scale_s = v_s + C::kStages * C::kBlock;    // two blocks' words: byte 0 scale of the row's weights, byte 1 that of V (one)
  uint64_t* k_full = reinterpret_cast<uint64_t*>(w_scale_s + 2 * C::kScaleBytes);
  uint64_t* k_empty = k_full + C::kStages, *v_full = k_empty + C::kStages, *v_empty = v_full + C::kStages;
  uint64_t* q_full = v_empty + C::kStages, *s_full = q_full + 1, *p_full = s_full + 2, *o_done = p_full + 2, *o_full = o_done + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(o_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);

  const int warp = warp_index(), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
    for (int x = 0; x < 2; ++x) { mbar_init(&s_full[x], 1); mbar_init(&p_full[x], 4); }
    mbar_init(q_full, 4);
    mbar_init(o_done, 1);
    mbar_init(o_full, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && elect_one()) { prefetch_tmap(&map_k); prefetch_tmap(&map_v); }
  if (warp == 1) {
    tmem_alloc<1>(tmem_holder, 256);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;              // two blocks of 64 columns of S (and P), 128 of O
  if constexpr (!RUNS) pdl_launch_dependents();
  pdl_wait();
  if constexpr (RUNS) pdl_launch_dependents();          // behind the wait where the join follows, as in fp8_attention_kernel

  // the rows that see most first, of all sequences and key heads
  const int pairs = a.batch * a.kv_heads, pair = static_cast<int>(blockIdx.x) % pairs, b = pair / a.kv_heads, kh = pair - b * a.kv_heads;
  const int rt = a.row_tiles - 1 - static_cast<int>(blockIdx.x) / pairs;
  const int rows = a.t * a.group, row0 = rt * 128;
  const long long pos = a.pos_dev != nullptr ? a.pos_dev[static_cast<long long>(b) * a.pos_batch] : a.pos;
  const bool fits = pos <= a.t_max - a.t;
  if (!fits && threadIdx.x == 0 && a.status != nullptr) atomicExch(a.status, PLQ_DEV_RANGE);
  // blocks of 64 positions that the rows see
  const int seen = pos < 0 || !fits ? 0 : static_cast<int>((pos + (min(row0 + 128, rows) - 1) / a.group) / kCacheBlock) + 1;
  // of these the CTA's run: blocks [j0, j0 + n)
  int j0 = 0, n = seen;
  bool whole = true, idle = false;
  if constexpr (RUNS) {
    const int tiles = sequence_tiles(a, b), length = run_length(tiles, a.runs), run = static_cast<int>(blockIdx.y);
    j0 = 2 * run * length;
    idle = run * length >= tiles;
    whole = tiles <= length;
    n = idle ? 0 : max(0, min(seen, j0 + 2 * length) - j0);
  }
  const uint32_t q_base = smem_u32(q_s), k_base = smem_u32(k_s), v_base = smem_u32(v_s);

  if (warp < 4) registers_down<C::kRegsMain>();
  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      for (int j = 0; ok && j < n; ++j) {
        const int st = j % C::kStages;
        const uint32_t parity = ((j / C::kStages) & 1u) ^ 1u;
        ok = mbar_wait_bounded(&k_empty[st], parity, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(&k_full[st], C::kBlock);
        tma_load_3d(k_base + st * C::kBlock, &map_k, kh * kHeadDim, (j0 + j) * kCacheBlock, b, smem_u32(&k_full[st]));
        ok = j == 0 ? mbar_wait_bounded(q_full, 0, abort_flag) : mbar_wait_bounded(&v_empty[st], parity, abort_flag);     // the queries lay there
        if (!ok) break;
        mbar_arrive_expect_tx(&v_full[st], C::kBlock);
        tma_load_3d(v_base + st * C::kBlock, &map_v, kh * kHeadDim, (j0 + j) * kCacheBlock, b, smem_u32(&v_full[st]));
      }
    }
  } else if (warp == 1) {
    if (elect_one() && n > 0) {
      constexpr uint32_t idesc_s = make_idesc_e4m3(128, 64), idesc_o = make_idesc(0u /*E4M3*/, 128, 128, 1u /*E8M0*/) | kIdescBMnMajor | (1u << 4 /*B: byte 1*/);
      bool ok = true;
      auto scores = [&](int j) {
        const int st = j % C::kStages;
        ok = ok && mbar_wait_bounded(&k_full[st], (j / C::kStages) & 1u, abort_flag);
        if (!ok) return;
        tc_fence_after();
        const uint32_t q_lo = desc_lo_sw128(q_base), k_lo = desc_lo_sw128(k_base + st * C::kBlock);
#pragma unroll
        for (int h = 0; h < 8; ++h)
          tc_mma_e4m3<1>(tmem_base + 64 * (j & 1), q_lo + (h >> 2) * (C::kTile >> 4) + 2 * (h & 3), kDescHiSw128, k_lo + 2 * (h & 3), kDescHiSw128, idesc_s, h != 0);
        tc_commit<1>(smem_u32(&s_full[j & 1]));
        tc_commit<1>(smem_u32(&k_empty[st]));
      };
      ok = mbar_wait_bounded(q_full, 0, abort_flag);
      scores(0);
      if (n > 1) scores(1);
      for (int j = 0; ok && j < n; ++j) {
        const int st = j % C::kStages;
        ok = mbar_wait_bounded(&v_full[st], (j / C::kStages) & 1u, abort_flag) && mbar_wait_bounded(&p_full[j & 1], (j >> 1) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t v_lo = desc_lo_sw128(v_base + st * C::kBlock), p = tmem_base + 64 * (j & 1), o = tmem_base + 128;
        tc_cp_32x128b_warpx4<1>(p + 32, desc_lo_sf(smem_u32(w_scale_s + (j & 1) * C::kScaleBytes)), kDescHiSf);
        const uint32_t sfa = p + 32, sfb = sfa + (1u << 30);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                   // 32 positions each: codes of hi, then of lo
          tc_mma_mxf8_ts(o, p + 16 * h, v_lo + h * (4096 >> 4), kDescHiSw128, idesc_o, sfa, sfb, j > 0 || h > 0);
          tc_mma_mxf8_ts(o, p + 16 * h + 8, v_lo + h * (4096 >> 4), kDescHiSw128, idesc_o, sfa, sfb, 1u);
        }
        tc_commit<1>(smem_u32(&v_empty[st]));
        tc_commit<1>(smem_u32(j + 1 == n ? o_full : o_done));
        if (j + 2 < n) scores(j + 2);                   // behind the product that still reads P: same pipe, in order
      }
    }
  } else if (warp >= 4) {
    registers_up<C::kRegsRows>();
    const int quad = warp & 3, r = quad * 32 + lane, row = row0 + r;
    const int i = row / a.group;
    const bool real = row < rows;
    const uint32_t s_at = tmem_base + (static_cast<uint32_t>(quad * 32) << 16), o_at = s_at + 128;

    // ---- the queries: whole lines to where V will be, then a row per thread: scale, hi and lo codes ----
    // Rolled loops: a CTA passes here once, and straight-line code costs more to fetch than to run.
    const uint32_t raw = v_base + quad * 8192;          // the warp's 32 rows of 256 bytes, 16-byte pieces exchanged by row
    // copies: two rows at a time, 16 bytes a lane
    const int first = row0 + quad * 32 + (lane >> 4), first_i = first / a.group, first_h = first - first_i * a.group;
    const int step_h = a.group == 1 ? 0 : a.group == 2 ? 0 : 2, step = (a.group == 1 ? 2 * a.heads : a.group == 2 ? a.heads : 2) * kHeadDim;
    const int wrap = (a.heads - a.group) * kHeadDim;
    const long long copy_at = ((static_cast<long long>(b) * a.t + first_i) * a.heads + static_cast<long long>(kh) * a.group + first_h) * kHeadDim + 8 * (lane & 15);
    {
      const __nv_bfloat16* src = a.q + copy_at;
      int at_row = first, at_h = first_h;
      uint32_t dst = raw + (lane >> 4) * 256;
      const uint32_t piece = lane & 15;
#pragma unroll 4
      for (int y = 0; y < 16; ++y) {
        const bool in = at_row < rows;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + ((piece ^ ((2 * y + (lane >> 4)) & 7)) << 4)), "l"(in ? src : a.q), "r"(in ? 16 : 0) : "memory");
        dst += 512;
        at_row += 2;
        src += step;
        at_h += step_h;
        if (at_h >= a.group) { at_h -= a.group; src += wrap; }
      }
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
      __syncwarp();
    }
    float down;
    {
      auto piece = [&](int c) {
        uint4 w;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(raw + lane * 256 + ((c ^ (lane & 7)) << 4)));
        return w;
      };
      uint32_t most = 0;                                // two magnitudes
#pragma unroll 4
      for (int c = 0; c < 16; ++c) {
        const uint4 w = piece(c);
        most = __vmaxu2(most, __vmaxu2(__vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu), __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu)));
      }
      uint32_t top = max(most & 0xFFFFu, most >> 16);
      const bool finite = top < 0x7F80u;
      if (!finite) {                                    // infinities and NaN do not set the scale
        top = 0;
#pragma unroll 1
        for (int c = 0; c < 64; ++c) {
          uint32_t w;
          asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(raw + lane * 256 + (((c >> 2) ^ (lane & 7)) << 4) + 4 * (c & 3)));
          if ((w & 0x7FFFu) < 0x7F80u) top = max(top, w & 0x7FFFu);
          if ((w >> 16 & 0x7FFFu) < 0x7F80u) top = max(top, w >> 16 & 0x7FFFu);
        }
      }
      const int e = top == 0 ? 0 : min(max(134 - static_cast<int>(top >> 7), -120), 120);
      const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * (a.scale_log2 < 0.0f ? -1.0f : 1.0f);
      const uint32_t keep = a.scale_log2 == 0.0f ? 0u : 0xFFFFFFFFu;
      down = finite || a.scale_log2 == 0.0f ? __uint_as_float(static_cast<uint32_t>(127 - e) << 23) : __uint_as_float(0x7FFFFFFFu);      // such a row is NaN
      const uint32_t dst = q_base + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        const uint4 w0 = piece(2 * c), w1 = piece(2 * c + 1);
        const uint32_t w[8] = {w0.x & keep, w0.y & keep, w0.z & keep, w0.w & keep, w1.x & keep, w1.y & keep, w1.z & keep, w1.w & keep};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t h2[2], l2[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float f0 = bf16lo_to_f32(w[2 * d + y]) * up, f1 = bf16hi_to_f32(w[2 * d + y]) * up;
            h2[y] = e4m3x2(f0, f1);
            const float2 back = e4m3x2_to_f32x2(h2[y]);
            l2[y] = e4m3x2(f0 - back.x, f1 - back.y);
          }
          hi[d] = h2[0] | h2[1] << 16;
          lo[d] = l2[0] | l2[1] << 16;
        }
        const uint32_t at = dst + ((c ^ (r & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + C::kTile), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }

    // ---- the tiles ----
    const long long scales = (static_cast<long long>(b) * a.kv_heads + kh) * a.scale_blocks;
    const float* k_scale = a.k_scale + scales;
    const float* v_scale = a.v_scale + scales;
    // a sequence with positions ends below 2^31
    const int written = static_cast<int>(n > 0 ? pos + a.t : 0);                      // positions behind may hold anything
    const int last_block = (written - 1) / kCacheBlock;
    const float per_k = down * (a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2));
    const int lim = real ? written - a.t + i : written - 1;                             // last position the row sees
    const int lim_min = written - a.t + row0 / a.group;                       // ... of any row of the tile
    float R = 0.0f, weight = 0.0f;
    const uint32_t scale_at = smem_u32(w_scale_s) + lane * 16 + quad * 4;
    bool ok = true;
    float next_k = 1.0f, next_v = 1.0f;
    auto fetch = [&](int j) {
      if (j0 + j <= last_block) { next_k = k_scale[j0 + j]; next_v = v_scale[j0 + j]; }
    };
    if (n > 0) fetch(0);
    for (int j = 0; ok && j < n; ++j) {
      const int t0 = (j0 + j) * kCacheBlock;
      const bool sees = lim >= t0;
      float ck = sees ? next_k * per_k : 0.0f;
      if (ck < 1.2e-38f) ck = 1.2e-38f;                 // a score of zero, and minus infinity stays what it is
      float vs = sees ? next_v : 1.0f;
      if (vs < 1e-36f) vs = 1e-36f;
      const float lv = __log2f(vs), inv_v = rcp_approx(vs);
      if (j + 1 < n) fetch(j + 1);
      ok = mbar_wait_bounded_lanes(&s_full[j & 1], (j >> 1) & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const bool masked = t0 + 63 > lim_min;            // the same for the whole row tile
      const uint32_t sp_at = s_at + 64 * (j & 1);
      uint32_t v[2][32];
#pragma unroll
      for (int c = 0; c < 2; ++c) tc_ld_32x32b_x32(sp_at + 32 * c, v[c]);
      tc_wait_ld();
      if (masked) {
        const int cut = max(-1, min(lim - t0, 63));         // last visible position of the block
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int d = 0; d < 32; ++d)
            if (32 * c + d > cut) v[c][d] = 0xFF800000u;
      }
      float m[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) m[d] = fmaxf(__uint_as_float(v[0][d]), __uint_as_float(v[1][d]));
#pragma unroll
      for (int d = 4; d < 32; ++d) m[d & 3] = fmaxf(m[d & 3], fmaxf(__uint_as_float(v[0][d]), __uint_as_float(v[1][d])));
      const float s_max = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), t_max = fmaf(s_max, ck, lv);
      ck *= vast_factor(t_max);
      if (ck < 1.2e-38f) ck = 1.2e-38f;
      float e = ceilf(t_max);
      if (j == 0) {
        R = e > kNegInf ? e - 8.0f : 0.0f;
      } else {
        const bool far = e - R > static_cast<float>(kScaleTop - kScaleBias);
        if (__any_sync(0xFFFFFFFFu, far)) {
          ok = mbar_wait_bounded_lanes(o_done, (j - 1) & 1u, abort_flag);        // the product of the block before is in O
          if (!ok) break;
          tc_fence_after();
          const float alpha = far ? ex2_approx(R + 8.0f - e) : 1.0f;
          if (far) R = e - 8.0f;
          weight *= alpha;
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t w[16];
            tc_ld_32x32b_x16(o_at + 16 * c, w);
            tc_wait_ld();
#pragma unroll
            for (int d = 0; d < 16; ++d) w[d] = __float_as_uint(__uint_as_float(w[d]) * alpha);
            tc_st_32x32b_x16(o_at + 16 * c, w);
          }
        }
      }
      if (t0 + kCacheBlock > written) {                 // positions that nobody has written: 0 x NaN would be NaN
        const int st = j % C::kStages;
        ok = mbar_wait_bounded_lanes(&v_full[st], (j / C::kStages) & 1u, abort_flag);
        if (!ok) break;
        if (t0 + (r >> 1) >= written) {
          uint4* dst = reinterpret_cast<uint4*>(v_s + st * C::kBlock + (r >> 1) * 128) + 4 * (r & 1);
#pragma unroll
          for (int c = 0; c < 4; ++c) dst[c] = make_uint4(0, 0, 0, 0);
        }
      }
      e = fmaxf(e, R - kFarBelow);                      // a number whatever the scores are
      // e - R is a whole number from -92 to 68: the low byte of the sum's bits is the scale, without a conversion
      const uint32_t ws = __float_as_uint((e - R) + (12582912.0f + kScaleBias)) & 0xFFu;
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(scale_at + (j & 1) * C::kScaleBytes), "r"(ws | 0x7F00u) : "memory");
      fence_proxy_async_smem();
      // A block that the row sees and whose scale is NaN makes the row NaN, its masked positions included.
      const float shift = fmaf(-fmaxf(s_max, -3e38f), ck, (t_max - e) + 8.0f);
      const float2 ck2 = make_float2(ck, ck), shift2 = make_float2(shift, shift);
      float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int d = 0; d < 32; d += 4) {
          float w[4];
#pragma unroll
          for (int y = 0; y < 4; y += 2) {
            const float2 z = __ffma2_rn(make_float2(__uint_as_float(v[c][d + y]), __uint_as_float(v[c][d + y + 1])), ck2, shift2);
            w[y] = ex2_approx(z.x);
            w[y + 1] = ex2_approx(z.y);
            sum = __fadd2_rn(sum, make_float2(w[y], w[y + 1]));
          }
          const uint32_t c0 = e4m3_split(w[0], w[1]), c1 = e4m3_split(w[2], w[3]);
          p[d / 4] = __byte_perm(c0, c1, 0x5410);
          p[8 + d / 4] = __byte_perm(c0, c1, 0x7632);
        }
        tc_st_32x32b_x16(sp_at + 16 * c, p);            // columns of S that have been read
      }
      weight = fmaf(sum.x + sum.y, inv_v * __uint_as_float(ws << 23), weight);
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[j & 1]);
    }

    // ---- out: a run's sums as they are, for the join ----
    if (RUNS && !whole) {
      if (ok && n > 0) ok = mbar_wait_bounded_lanes(o_full, 0, abort_flag);
      tc_fence_after();
      const long long units = static_cast<long long>(a.row_tiles) * a.kv_heads;
      const long long slot = ((b * units + static_cast<long long>(a.row_tiles - 1 - rt) * a.kv_heads + kh) * a.runs + blockIdx.y) * C::kRows + r;
      float* dst = a.part + slot * kHeadDim;
      const bool wide = reinterpret_cast<uintptr_t>(a.part) % 32 == 0;
#pragma unroll 1
      for (int c = 0; c < 8; ++c) {
        uint32_t v[16];
        if (n > 0) {
          tc_ld_32x32b_x16(o_at + 16 * c, v);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int d = 0; d < 16; ++d) v[d] = 0;
        }
        if (real && !idle) {
#pragma unroll
          for (int d = 0; d < 16; d += 8) {              // the workspace is 16-byte aligned; by 32 bytes 64 tokens behind 8000 take 27.6 us, by 16 28.8
            if (wide)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + 16 * c + d), "r"(v[d]), "r"(v[d + 1]), "r"(v[d + 2]),
                           "r"(v[d + 3]), "r"(v[d + 4]), "r"(v[d + 5]), "r"(v[d + 6]), "r"(v[d + 7]) : "memory");
            else
#pragma unroll
              for (int y = d; y < d + 8; y += 4) *reinterpret_cast<uint4*>(dst + 16 * c + y) = make_uint4(v[y], v[y + 1], v[y + 2], v[y + 3]);
          }
        }
      }
      if (real && !idle)                                // both in units of 2^R
        *reinterpret_cast<float2*>(a.part + a.batch * units * a.runs * C::kRows * kHeadDim + 2 * slot) = make_float2(R, weight);
      tc_fence_before();
    }
    // ---- or the result: by way of the queries' memory, so that the stores are whole lines ----
    const uint32_t o_base = q_base + quad * 8192;       // 32 rows of 256 bytes; nothing reads the queries any more
    if (whole && n > 0) {
      if (ok) ok = mbar_wait_bounded_lanes(o_full, 0, abort_flag);
      tc_fence_after();
      const float inv = weight == 0.0f ? 0.0f : 1.0f / weight;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tc_ld_32x32b_x32(o_at + 32 * c, v);
        tc_wait_ld();
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          uint32_t o[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) o[y] = f32x2_to_bf16x2(__uint_as_float(v[8 * d + 2 * y]) * inv, __uint_as_float(v[8 * d + 2 * y + 1]) * inv);
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(o_base + lane * 256 + (((4 * c + d) ^ (lane & 7)) << 4)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
        }
      }
      tc_fence_before();
      __syncwarp();
    }
    __nv_bfloat16* dst = a.out + copy_at;
    int at_row = first, at_h = first_h;
#pragma unroll 1
    for (int y0 = 0; y0 < 32; y0 += 8) {
      uint4 o[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int y = y0 + 2 * d + (lane >> 4);
        o[d] = make_uint4(0, 0, 0, 0);
        if (n > 0)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(o[d].x), "=r"(o[d].y), "=r"(o[d].z), "=r"(o[d].w) : "r"(o_base + y * 256 + (((lane & 15) ^ (y & 7)) << 4)) : "memory");
      }
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if (at_row < rows && whole && !idle) *reinterpret_cast<uint4*>(dst) = o[d];
        at_row += 2;
        dst += step;
        at_h += step_h;
        if (at_h >= a.group) { at_h -= a.group; dst += wrap; }
      }
    }
  }

  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && a.status != nullptr) atomicExch(a.status, PLQ_DEV_TIMEOUT);
    const long long t0 = clock64();                     // copies still in flight get time to land
    while (clock64() - t0 < 400000ll) __nanosleep(1000);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, 256);
  }
}

// ---- host side -------------------------------------------------------------------------------------------------------
// u8 cache [batch, t_max, kv_heads * 128]: boxes of `box` tokens x 128 bytes, 128-byte swizzle, zeros behind t_max.
static int make_cache_tmap(CUtensorMap* tm, const void* base, int64_t batch, int64_t t_max, int64_t kv_heads, int box) {
  return make_tmap_3d(tm, base, kv_heads * kHeadDim, t_max, batch, kHeadDim, box);
}

template <bool RUNS>
static int launch_prefill(const CUtensorMap& mk, const CUtensorMap& mv, const Fp8AttnArgs& a, void* stream) {
  static thread_local int done_dev = -1;
  const int st = allow_smem(fp8_prefill_kernel<RUNS>, PfCfg::kAlone, &done_dev);
  if (st != PLQ_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.batch) * a.kv_heads * a.row_tiles, static_cast<unsigned>(a.runs ? a.runs : 1));
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = cfg.gridDim.x * cfg.gridDim.y <= static_cast<unsigned>(sm_count()) ? PfCfg::kAlone : PfCfg::kSmemBytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_prefill_kernel<RUNS>, mk, mv, a));
  if (a.runs) {
    cfg.gridDim = dim3(static_cast<unsigned>(a.batch * a.t * a.heads));
    cfg.blockDim = dim3(128, 1, 1);
    cfg.dynamicSmemBytes = 0;
    PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_attention_join_kernel, a, PfCfg::kRows));
  }
  return PLQ_OK;
}

// Rows of a CTA, their tiles, and runs of the row of tiles (0: one CTA per sequence) for a call that sees up to `ctx` positions.
// rows = 128: fp8_prefill_kernel.
struct AttnPlan { int rows, row_tiles, runs; };
static AttnPlan attn_plan(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t ctx) {
  AttnPlan p;
  const int64_t rows = t * (heads / kv_heads), slots = 2 * static_cast<int64_t>(sm_count()), tiles = (ctx + 127) / 128;
  if (rows <= 16) {
    p.rows = rows <= 8 ? 8 : 16;
    p.row_tiles = 1;
    // Two CTAs fit an SM: as many runs as fill the device once, none shorter than four tiles of 128 positions (a CTA's set-up
    // and its share of the join cost about what two tiles do).
    int64_t runs = slots / kv_heads;
    if (runs > batch * tiles / 4) runs = batch * tiles / 4;
    p.runs = batch > kMaxFlat || batch * tiles > (1 << 30) || tiles <= 4 || runs < 2 ? 0 : static_cast<int>(runs);
    return p;
  }
  // More rows: the kernel with 128 of them per CTA, every sequence whole or in runs of its own.  A tile takes a CTA 1.4 us, with a
  // second one on the SM 2.2; runs cost 5 us and 0.3 for every 128 rows.  8 key heads with 4 heads each behind 8000 positions,
  // whole / in runs: 9 tokens 88 / 16 us, 64 tokens 88 / 26, 256 tokens 90 / 66; four sequences of 128 tokens 93 / 116.
  // (The other kernel with 32 rows takes 2.6 us a tile: 8 tokens of 16 sequences behind 4000 positions 60 us, here 50.)
  const int64_t many = batch * kv_heads * ((rows + 127) / 128);
  int64_t split = slots / many;
  if (split > tiles / 4) split = tiles / 4;
  const int64_t whole = 50 + tiles * (2 * many <= slots ? 14 : 22 * ((many + slots - 1) / slots));
  p.rows = PfCfg::kRows;
  p.row_tiles = static_cast<int>((rows + 127) / 128);
  p.runs = split >= 2 && 100 + 3 * many + (tiles + split - 1) / split * (2 * many * split <= slots ? 14 : 22) < whole ? static_cast<int>(split) : 0;
  return p;
}

template <int R>
static int launch_attention(const CUtensorMap& mk, const CUtensorMap& mv, const Fp8AttnArgs& a, void* stream) {
  using C = AtCfg<R>;
  static thread_local int done_dev = -1;
  const int st = allow_smem(fp8_attention_kernel<R>, C::kSmemBytes, &done_dev);
  if (st != PLQ_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(a.runs ? a.runs : a.batch));
  cfg.blockDim = dim3(192, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_attention_kernel<R>, mk, mv, a));
  if (a.runs) {
    cfg.gridDim = dim3(static_cast<unsigned>(a.batch * a.t * a.heads));
    cfg.blockDim = dim3(128, 1, 1);
    cfg.dynamicSmemBytes = 0;
    PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, fp8_attention_join_kernel, a, R));
  }
  return PLQ_OK;
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
  // two heads per thread where there are enough of them for every SM (four need 80 registers: three CTAs per SM, 60 us for 56)
  const int64_t head_rows = batch * t * heads;
  const int ht = head_rows * 8 < 2 * 2048 * static_cast<int64_t>(sm_count()) ? 1 : heads % 2 == 0 ? 2 : 1;
  a.q_threads = head_rows / ht * 8;
  a.status = dev_status;
  a.t = static_cast<int>(t);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.pos_batch = pos_per_sequence ? 1 : 0;
  a.scale_blocks = static_cast<int>((t_max + kCacheBlock - 1) / kCacheBlock);
  a.units_per_head = static_cast<int>((t + kCacheBlock - 2) / kCacheBlock + 1);      // blocks that t rows can touch
  const int64_t q_blocks = (a.q_threads + 255) / 256, blocks = q_blocks + batch * kv_heads * 2 * a.units_per_head;
  if (blocks > 0x7FFFFFFF) return PLQ_ERR_LIMIT;
  a.unit_rate = ((static_cast<unsigned long long>(blocks - q_blocks) << 32) + blocks - 1) / blocks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PLQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, ht == 2 ? rope_kv_append_fp8_kernel<2> : rope_kv_append_fp8_kernel<1>, a));
  return PLQ_OK;
}

extern "C" int64_t plq_fp8_attention_workspace_bytes(int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t ctx) {
  using namespace plq;
  if (batch < 1 || t < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || ctx < 1) return 0;
  const AttnPlan p = attn_plan(batch, t, heads, kv_heads, ctx);
  const int64_t each = p.rows == PfCfg::kRows ? batch : 2;             // partial sums of a run and row: of every sequence, or of two
  return kv_heads * p.row_tiles * static_cast<int64_t>(p.runs) * each * p.rows * static_cast<int64_t>((kHeadDim + 2) * sizeof(float));
}

extern "C" int plq_fp8_attention(const void* q_bf16, const void* k_codes, const void* k_scales_f32, const void* v_codes, const void* v_scales_f32,
                                 int64_t batch, int64_t t, int64_t heads, int64_t kv_heads, int64_t t_max, const int64_t* pos_dev,
                                 int pos_per_sequence, int64_t pos, int64_t ctx, float scale, void* out_bf16, void* workspace,
                                 int64_t workspace_bytes, int32_t* dev_status, void* stream) {
  using namespace plq;
  if (batch < 0 || t < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || t_max < 1 || ctx < 1 || ctx > t_max) return PLQ_ERR_SHAPE;
  if (pos_dev == nullptr && pos >= 0 && (t > t_max || pos > t_max - t)) return PLQ_ERR_SHAPE;
  if (pos_dev == nullptr && pos >= 0 && pos + t > ctx) return PLQ_ERR_SHAPE;
  if (heads > 4096 || batch > 65535 || t > (1 << 24) || batch * t * heads > 0x7FFFFFFF || t_max > 0x7FFFFFFF - 128) return PLQ_ERR_LIMIT;
  if (batch == 0 || t == 0) return PLQ_OK;
  if (!q_bf16 || !k_codes || !k_scales_f32 || !v_codes || !v_scales_f32 || !out_bf16) return PLQ_ERR_NULL;
  if (!aligned16(q_bf16) || !aligned16(k_codes) || !aligned16(v_codes) || !aligned16(out_bf16) || !aligned16(workspace) ||
      ((reinterpret_cast<uintptr_t>(k_scales_f32) | reinterpret_cast<uintptr_t>(v_scales_f32)) & 3u) || (reinterpret_cast<uintptr_t>(pos_dev) & 7u))
    return PLQ_ERR_ALIGN;
  int st = device_check();
  if (st != PLQ_OK) return st;
  const AttnPlan p = attn_plan(batch, t, heads, kv_heads, ctx);
  if (kv_heads * static_cast<int64_t>(p.row_tiles) > 0x7FFFFFFF) return PLQ_ERR_LIMIT;
  if (p.runs && !workspace) return PLQ_ERR_NULL;
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
  a.status = dev_status;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.batch = static_cast<int>(batch);
  a.t = static_cast<int>(t);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(heads / kv_heads);
  a.pos_batch = pos_per_sequence ? 1 : 0;
  a.scale_blocks = static_cast<int>((t_max + kCacheBlock - 1) / kCacheBlock);
  a.runs = p.runs;
  a.row_tiles = p.row_tiles;
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  const int box = p.rows >= 128 ? kCacheBlock : 128;
  if ((st = make_cache_tmap(&mk, k_codes, batch, t_max, kv_heads, box)) != PLQ_OK) return st;
  if ((st = make_cache_tmap(&mv, v_codes, batch, t_max, kv_heads, box)) != PLQ_OK) return st;
  if (p.rows >= 128) return p.runs ? launch_prefill<true>(mk, mv, a, stream) : launch_prefill<false>(mk, mv, a, stream);
  return p.rows == 8 ? launch_attention<8>(mk, mv, a, stream) : launch_attention<16>(mk, mv, a, stream);
}
