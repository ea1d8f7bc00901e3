// PyTorch front end of the calls that a forward pass makes most often: the pack, a whole quantised linear, a whole decoder
// layer, the E4M3 operators.
// The kernels are those of libplq_b200.so, launched one after the other on the current stream; this file only allocates
// and forwards.  Called operator by operator from Python a linear is two foreign calls and nine allocations (~40 us of
// host time against 8 - 15 us on the device for up to a few hundred rows), a layer nine foreign calls and ~30.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <dlfcn.h>

#include <array>
#include <optional>
#include <tuple>

#include "../../include/plq.h"

namespace {

using at::Tensor;

// The C entry points, out of the library that _lib has loaded (init).
struct Api {
  decltype(&::plq_pack) pack;
  decltype(&::plq_rmsnorm_pack) rmsnorm_pack;
  decltype(&::plq_add_rmsnorm_pack) add_rmsnorm_pack;
  decltype(&::plq_silu_mul_pack) silu_mul_pack;
  decltype(&::plq_gemv_tc) gemv_tc;
  decltype(&::plq_mixed_gemm) mixed_gemm;
  decltype(&::plq_mixed_gemm_silu_mul) mixed_gemm_silu_mul;
  decltype(&::plq_rope_kv_append) rope_kv_append;
  decltype(&::plq_rope_kv_append_nvfp4_values) rope_kv_append_nvfp4_values;
  decltype(&::plq_sf_tiled_bytes) sf_tiled_bytes;
  decltype(&::plq_fp8_pack) fp8_pack;
  decltype(&::plq_fp8_gemm) fp8_gemm;
  decltype(&::plq_rope_kv_append_fp8) rope_kv_append_fp8;
  decltype(&::plq_fp8_attention_workspace_bytes) fp8_attention_workspace_bytes;
  decltype(&::plq_fp8_attention) fp8_attention;
} api;

void init(const std::string& path) {
  void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  if (!lib) throw std::runtime_error(std::string("cannot load ") + path + ": " + dlerror());
  auto find = [&](auto& fn, const char* name) {
    void* at = dlsym(lib, name);
    if (!at) throw std::runtime_error(path + " has no " + name);
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(at);
  };
  find(api.pack, "plq_pack");
  find(api.rmsnorm_pack, "plq_rmsnorm_pack");
  find(api.add_rmsnorm_pack, "plq_add_rmsnorm_pack");
  find(api.silu_mul_pack, "plq_silu_mul_pack");
  find(api.gemv_tc, "plq_gemv_tc");
  find(api.mixed_gemm, "plq_mixed_gemm");
  find(api.mixed_gemm_silu_mul, "plq_mixed_gemm_silu_mul");
  find(api.rope_kv_append, "plq_rope_kv_append");
  find(api.rope_kv_append_nvfp4_values, "plq_rope_kv_append_nvfp4_values");
  find(api.sf_tiled_bytes, "plq_sf_tiled_bytes");
  find(api.fp8_pack, "plq_fp8_pack");
  find(api.fp8_gemm, "plq_fp8_gemm");
  find(api.rope_kv_append_fp8, "plq_rope_kv_append_fp8");
  find(api.fp8_attention_workspace_bytes, "plq_fp8_attention_workspace_bytes");
  find(api.fp8_attention, "plq_fp8_attention");
}

// Raises the package's PlqError for a non-zero status.
void check(int status) {
  if (status != PLQ_OK) {
    pybind11::gil_scoped_acquire gil;
    pybind11::module_::import("plaquant_b200._lib").attr("check")(status);
  }
}

int64_t up256(int64_t b) { return (b + 255) / 256 * 256; }

const void* ptr(const Tensor& t) { return t.numel() == 0 ? nullptr : t.const_data_ptr(); }

// A packed [rows, k_lo + k_hi] operand with tiled scales, laid out at `base`.
struct PackedAt {
  uint8_t *lo, *lo_sf, *hi, *hi_sf;
  int64_t bytes;
  PackedAt(void* base, int64_t rows, int64_t k_lo, int64_t k_hi) {
    uint8_t* at = static_cast<uint8_t*>(base);
    const int64_t n[4] = {up256(rows * (k_lo / 2)), up256(api.sf_tiled_bytes(rows, k_lo / 16)), up256(rows * k_hi),
                          up256(api.sf_tiled_bytes(rows, k_hi / 32))};
    lo = at; lo_sf = lo + n[0]; hi = lo_sf + n[1]; hi_sf = hi + n[2];
    bytes = n[0] + n[1] + n[2] + n[3];
  }
};

Tensor checked_gamma(const Tensor& gamma, int64_t k) {
  if (!gamma.is_cuda()) throw std::runtime_error("gamma must be a CUDA tensor: plaquant_b200 has no CPU path");
  if (gamma.scalar_type() != at::kBFloat16 || gamma.numel() != k) throw pybind11::type_error("gamma must be bfloat16 [K]");
  return gamma.contiguous();
}

// [RMSNorm] -> [Hadamard] -> pack of bf16 CUDA x[..., K] into new buffers: (lo_codes, lo_sf, hi_codes, hi_sf).
std::tuple<Tensor, Tensor, Tensor, Tensor> pack(const Tensor& x, int64_t k_hi, bool hadamard, bool tiled,
                                                const std::optional<Tensor>& gamma, double eps) {
  const int64_t k = x.size(-1), k_lo = k - k_hi;
  const Tensor g = gamma ? checked_gamma(*gamma, k) : Tensor();
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor x2 = x.reshape({-1, k}).contiguous();
  const int64_t rows = x2.size(0);
  const auto u8 = x.options().dtype(at::kByte);
  Tensor lo = at::empty({rows, k_lo / 2}, u8), hi = at::empty({rows, k_hi}, u8), lo_sf, hi_sf;
  if (tiled) {
    lo_sf = at::empty({api.sf_tiled_bytes(rows, k_lo / 16)}, u8);
    hi_sf = at::empty({api.sf_tiled_bytes(rows, k_hi / 32)}, u8);
  } else {
    lo_sf = at::empty({rows, k_lo / 16}, u8);
    hi_sf = at::empty({rows, k_hi / 32}, u8);
  }
  auto at = [](const Tensor& t) { return t.numel() == 0 ? nullptr : t.data_ptr(); };
  const int layout = tiled ? PLQ_SF_TILED : PLQ_SF_ROWMAJOR;
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  check(gamma ? api.rmsnorm_pack(ptr(x2), g.const_data_ptr(), static_cast<float>(eps), rows, k, k_hi, hadamard, at(lo), at(lo_sf),
                                 at(hi), at(hi_sf), layout, stream)
              : api.pack(ptr(x2), rows, k, k_hi, hadamard, at(lo), at(lo_sf), at(hi), at(hi_sf), layout, stream));
  return {lo, lo_sf, hi, hi_sf};
}

// A packed weight: B operand of the products, and the status word their kernels report to.
struct Linear {
  Tensor lo, lo_sf, hi, hi_sf, status;
  int64_t n, k_lo, k_hi;
  int64_t k() const { return k_lo + k_hi; }
  int64_t packed_bytes(int64_t rows) const { return PackedAt(nullptr, rows, k_lo, k_hi).bytes; }

  // `like`: the choice of kernel for another number of rows (the two sum K in different orders).
  int product(const PackedAt& a, int64_t rows, void* y, int64_t ldy, void* stream, int64_t like = 0) const {
    int32_t* st = status.data_ptr<int32_t>();
    if (std::max(rows, like) <= 16)      // decode: stream the weights once; every product here has a pack in front of it
      return api.gemv_tc(a.lo, a.lo_sf, a.hi, a.hi_sf, ptr(lo), ptr(lo_sf), ptr(hi), ptr(hi_sf), rows, n, k_lo, k_hi, y, ldy, st,
                         PLQ_GEMV_STATIC_B | PLQ_GEMV_INTERLEAVED, stream);
    return api.mixed_gemm(a.lo, a.lo_sf, a.hi, a.hi_sf, ptr(lo), ptr(lo_sf), ptr(hi), ptr(hi_sf), rows, n, k_lo, k_hi, y, ldy, st,
                          stream);
  }

  // [RMSNorm] -> [Hadamard] -> pack -> product of x[..., K]; nullopt for an input that the Python path has to look at
  // (another dtype, device or K, no rows): it raises what it always raised.
  std::optional<Tensor> forward(const Tensor& x, bool hadamard, const std::optional<Tensor>& gamma, double eps,
                                const std::optional<Tensor>& out) const {
    if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() < 1 || x.size(-1) != k() || x.device() != lo.device() ||
        x.numel() == 0)
      return std::nullopt;
    const Tensor g = gamma ? checked_gamma(*gamma, k()) : Tensor();
    pybind11::gil_scoped_release nogil;
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor x2 = x.contiguous();
    const int64_t rows = x.numel() / k();
    const Tensor ws = at::empty({packed_bytes(rows)}, x.options().dtype(at::kByte));
    Tensor y = out ? *out : at::empty({rows, n}, x.options());
    void* stream = c10::cuda::getCurrentCUDAStream().stream();
    const PackedAt p(ws.data_ptr(), rows, k_lo, k_hi);
    check(gamma ? api.rmsnorm_pack(x2.const_data_ptr(), g.const_data_ptr(), static_cast<float>(eps), rows, k(), k_hi, hadamard, p.lo,
                                   p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream)
                : api.pack(x2.const_data_ptr(), rows, k(), k_hi, hadamard, p.lo, p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream));
    check(product(p, rows, y.data_ptr(), y.stride(0), stream));
    if (x.dim() == 2 && !out) return y;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    return y.view(shape);
  }
};

Tensor heads_first(const Tensor& t) { return t.transpose(1, 2); }

// The two halves of a decoder layer around its attention.  Workspace: the packed operand of the linear that runs, `packed`
// bytes, then that linear's output.
struct LayerSizes {
  int64_t rows, hidden, ffn, packed, out0;
  bool gated;                                          // the GEMM applies SiLU(gate) * up itself: one column per pair
  LayerSizes(const Tensor& h, std::initializer_list<const Linear*> linears, int64_t ffn_)
      : rows(h.size(0) * h.size(1)), hidden(h.size(2)), ffn(ffn_), packed(0), out0(up256(2 * rows * hidden)), gated(rows > 16) {
    for (const Linear* l : linears) packed = std::max(packed, l->packed_bytes(rows));
  }
  int64_t back_bytes() const { return out0 + (gated ? 2 : 4) * rows * ffn; }
};

// h + delta -> RMSNorm(ln1) -> qkv at `out` [rows, qkv.n].  Returns the residual stream.
Tensor front_half(const LayerSizes& z, const Linear& qkv, const Tensor& ln1, float eps, const Tensor& h, const std::optional<Tensor>& delta, void* ws,
                  void* out, void* stream) {
  Tensor h1 = h;
  const PackedAt p(ws, z.rows, qkv.k_lo, qkv.k_hi);
  if (delta) {
    h1 = at::empty_like(h);
    check(api.add_rmsnorm_pack(delta->const_data_ptr(), h.const_data_ptr(), h1.data_ptr(), ln1.const_data_ptr(), eps, z.rows, z.hidden,
                               qkv.k_hi, 1, p.lo, p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream));
  } else {
    check(api.rmsnorm_pack(h.const_data_ptr(), ln1.const_data_ptr(), eps, z.rows, z.hidden, qkv.k_hi, 1, p.lo, p.lo_sf, p.hi, p.hi_sf,
                           PLQ_SF_TILED, stream));
  }
  check(qkv.product(p, z.rows, out, qkv.n, stream));
  return h1;
}

// attn -> o_proj -> residual h1, RMSNorm(ln2) -> gate_up -> SiLU * up -> down_proj, with z.back_bytes() of outputs at `act`.
// Returns (residual stream, down_proj's output not added to it yet).
std::tuple<Tensor, Tensor> back_half(const LayerSizes& z, const Linear& o, const Linear& gate_up, const Linear& down, const Tensor& ln2, float eps,
                                     Tensor h1, Tensor attn, bool last_only, void* ws, uint8_t* act, void* stream) {
  const int64_t b = h1.size(0), t = h1.size(1), hidden = z.hidden, ffn = z.ffn, like = z.rows;
  if (last_only) {
    attn = attn.slice(1, t - 1).contiguous();
    h1 = h1.slice(1, t - 1).contiguous();
  }
  const int64_t out_rows = last_only ? b : z.rows;
  Tensor h2 = at::empty_like(h1), delta2 = at::empty_like(h1);
  uint8_t* gu = act + z.out0;
  {
    const PackedAt p(ws, out_rows, o.k_lo, o.k_hi);
    check(api.pack(attn.const_data_ptr(), out_rows, o.k(), o.k_hi, 1, p.lo, p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream));
    check(o.product(p, out_rows, act, hidden, stream, like));
  }
  {
    const PackedAt p(ws, out_rows, gate_up.k_lo, gate_up.k_hi);
    check(api.add_rmsnorm_pack(act, h1.const_data_ptr(), h2.data_ptr(), ln2.const_data_ptr(), eps, out_rows, hidden, gate_up.k_hi, 1, p.lo,
                               p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream));
    if (z.gated)
      check(api.mixed_gemm_silu_mul(p.lo, p.lo_sf, p.hi, p.hi_sf, ptr(gate_up.lo), ptr(gate_up.lo_sf), ptr(gate_up.hi), ptr(gate_up.hi_sf),
                                    out_rows, ffn, gate_up.k_lo, gate_up.k_hi, gu, ffn, gate_up.status.data_ptr<int32_t>(), stream));
    else
      check(gate_up.product(p, out_rows, gu, 2 * ffn, stream, like));
  }
  {
    const PackedAt p(ws, out_rows, down.k_lo, down.k_hi);
    if (z.gated)
      check(api.pack(gu, out_rows, ffn, down.k_hi, 1, p.lo, p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream));
    else
      check(api.silu_mul_pack(gu, gu + 2 * ffn, 2 * ffn, out_rows, ffn, down.k_hi, 1, p.lo, p.lo_sf, p.hi, p.hi_sf, PLQ_SF_TILED, stream));
    check(down.product(p, out_rows, delta2.data_ptr(), hidden, stream, like));
  }
  return {h2, delta2};
}

void check_stream(const Tensor& h, const std::optional<Tensor>& delta) {
  TORCH_CHECK(h.dim() == 3 && h.is_contiguous() && h.scalar_type() == at::kBFloat16 && (!delta || (delta->is_contiguous() && delta->sizes() == h.sizes())),
              "h and delta must be contiguous bfloat16 [B, T, hidden]");
}

// The halves as calls of their own, for an attention that is not one of decoder_layer's.
// -> (residual stream, [B, T, qkv.n])
std::tuple<Tensor, Tensor> layer_front(const Linear& qkv, const Tensor& ln1, double eps, const Tensor& h, const std::optional<Tensor>& delta) {
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(h.device());
  check_stream(h, delta);
  TORCH_CHECK(qkv.k() == h.size(2), "the layer's linears do not fit together");
  const LayerSizes z(h, {&qkv}, 0);
  const Tensor ws = at::empty({z.packed}, h.options().dtype(at::kByte));
  Tensor out = at::empty({h.size(0), h.size(1), qkv.n}, h.options());
  return {front_half(z, qkv, ln1, static_cast<float>(eps), h, delta, ws.data_ptr(), out.data_ptr(), c10::cuda::getCurrentCUDAStream().stream()), out};
}

// attn: [B, T, o.k()].  -> (residual stream, down_proj's output not added to it yet)
std::tuple<Tensor, Tensor> layer_back(const Linear& o, const Linear& gate_up, const Linear& down, const Tensor& ln2, double eps, const Tensor& h,
                                      const Tensor& attn, bool last_only) {
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(h.device());
  check_stream(h, std::nullopt);
  const int64_t ffn = down.k();
  TORCH_CHECK(o.n == h.size(2) && gate_up.k() == h.size(2) && gate_up.n == 2 * ffn && down.n == h.size(2) && ffn % 128 == 0,
              "the layer's linears do not fit together");
  TORCH_CHECK(attn.is_contiguous() && attn.scalar_type() == at::kBFloat16 && attn.dim() == 3 && attn.size(0) == h.size(0) && attn.size(1) == h.size(1) &&
                  attn.size(2) == o.k() && attn.device() == h.device(),
              "the attention's output must be contiguous bfloat16 [B, T, heads * head_dim]");
  const LayerSizes z(h, {&o, &gate_up, &down}, ffn);
  const Tensor ws = at::empty({z.packed + z.back_bytes()}, h.options().dtype(at::kByte));
  uint8_t* at = static_cast<uint8_t*>(ws.data_ptr());
  return back_half(z, o, gate_up, down, ln2, static_cast<float>(eps), h, attn, last_only, at, at + z.packed, c10::cuda::getCurrentCUDAStream().stream());
}

// One decoder layer on one GPU: h + delta -> RMSNorm(ln1) -> qkv -> RoPE, cache append -> attention -> o_proj -> residual,
// RMSNorm(ln2) -> gate_up -> SiLU * up -> down_proj.  Returns (residual stream, down_proj's output not added to it yet).
// k_view / v_view: the first `ctx` positions of caches allocated for `cap`; the new rows go to `pos` (or *pos_dev).
// More than one position per sequence: all of them (a causal mask over the positions themselves) or with a mask.
// Packed caches (uint8) need `had`, the float32 Hadamard of the queries.  With `last_only` everything behind the attention
// runs for the last position of each sequence alone, results [B, 1, hidden] (the same bits: rows are independent).
std::tuple<Tensor, Tensor> decoder_layer(const Linear& qkv, const Linear& o, const Linear& gate_up, const Linear& down,
                                         const Tensor& ln1, const Tensor& ln2, int64_t heads, int64_t kv_heads, double eps_,
                                         const Tensor& h, const std::optional<Tensor>& delta, const Tensor& cos,
                                         const Tensor& sin, const Tensor& k_view, const Tensor& v_view, int64_t cap, int64_t pos,
                                         const std::optional<Tensor>& pos_dev, const std::optional<Tensor>& mask,
                                         const std::optional<Tensor>& had, bool last_only) {
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(h.device());
  check_stream(h, delta);
  const int64_t b = h.size(0), t = h.size(1), hidden = h.size(2), rows = b * t, ctx = k_view.size(1);
  const int64_t nq = (heads + 2 * kv_heads) * 128, ffn = down.k(), attn_width = heads * 128;
  TORCH_CHECK(qkv.n == nq && qkv.k() == hidden && o.k() == attn_width && o.n == hidden && gate_up.k() == hidden &&
                  gate_up.n == 2 * ffn && down.n == hidden && ffn % 128 == 0,
              "the layer's linears do not fit together");
  TORCH_CHECK(cos.numel() == t * 128 && sin.numel() == t * 128 && cos.is_contiguous() && sin.is_contiguous(), "cos / sin: one row per new position");
  const bool packed = k_view.scalar_type() == at::kByte;
  const int64_t width = packed ? 72 : 128;
  for (const Tensor* c : {&k_view, &v_view})
    TORCH_CHECK(c->size(0) == b && c->size(1) == ctx && c->size(2) == kv_heads && c->size(3) == width && ctx <= cap &&
                    c->scalar_type() == k_view.scalar_type() && (b == 1 || c->stride(0) == cap * kv_heads * width) &&
                    c->stride(1) == kv_heads * width && c->stride(2) == width && c->stride(3) == 1,
                "the caches must be the leading positions of contiguous allocations");
  TORCH_CHECK(t == 1 || mask || t == ctx, "a chunk behind a prompt needs a mask");
  const auto opts = h.options();
  // qkv's output is dead before o's is written, and the attention's operands have storage of their own.
  const LayerSizes z(h, {&qkv, &o, &gate_up, &down}, ffn);
  const Tensor ws = at::empty({z.packed + std::max(2 * rows * nq, z.back_bytes())}, opts.dtype(at::kByte));
  uint8_t* act = static_cast<uint8_t*>(ws.data_ptr()) + z.packed;
  void* stream = c10::cuda::getCurrentCUDAStream().stream();
  int32_t* status = qkv.status.data_ptr<int32_t>();
  const float eps = static_cast<float>(eps_);

  const Tensor h1 = front_half(z, qkv, ln1, eps, h, delta, ws.data_ptr(), act, stream);
  Tensor q = at::empty({b, t, heads, 128}, packed ? opts.dtype(at::kFloat) : opts), kk = k_view, vv = v_view;
  const int64_t* at_pos = pos_dev ? pos_dev->const_data_ptr<int64_t>() : nullptr;
  if (packed) {
    kk = at::empty({b, ctx, kv_heads, 128}, opts);
    vv = at::empty_like(kk);
    check(api.rope_kv_append_nvfp4_values(act, nq, cos.const_data_ptr(), sin.const_data_ptr(), b, t, heads, kv_heads, 128, q.data_ptr(),
                                          k_view.data_ptr(), v_view.data_ptr(), cap, at_pos, pos, ctx, kk.data_ptr(), vv.data_ptr(),
                                          status, stream));
    q = at::matmul(q, *had).to(at::kBFloat16);
  } else {
    check(api.rope_kv_append(act, nq, cos.const_data_ptr(), sin.const_data_ptr(), b, t, heads, kv_heads, 128, q.data_ptr(),
                             k_view.data_ptr(), v_view.data_ptr(), cap, at_pos, pos, status, stream));
  }
  Tensor attn = heads_first(at::scaled_dot_product_attention(heads_first(q), heads_first(kk), heads_first(vv), mask, 0.0,
                                                                   !mask && t > 1, std::nullopt, true))
                          .contiguous();
  return back_half(z, o, gate_up, down, ln2, eps, h1, attn, last_only, ws.data_ptr(), act, stream);
}

// Does nothing else share the memory of a or of b?  (The base that a view keeps alive does not count.)
bool alone(const Tensor& a, const Tensor& b) {
  auto one = [](const Tensor& t) { return t.storage().use_count() == (t.is_view() ? 2u : 1u); };
  return one(a) && one(b);
}

// ---- the E4M3 operators ----------------------------------------------------------------------------------------------
// From Python each was 10 - 15 us of checks, allocations and a foreign call with up to twenty arguments, as long as the
// kernels of a decode step take.  Each of these handles what needs no further look - contiguous, aligned tensors of the right
// types on one device - and returns nullopt for anything else: the Python path then copies or raises.
bool plain(const Tensor& t, at::ScalarType type, c10::Device device) {
  return t.scalar_type() == type && t.device() == device && t.is_contiguous() && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}

// at::empty on a CUDA device without the dispatcher (1.2 -> 0.6 us)
Tensor cuda_empty(c10::IntArrayRef size, at::ScalarType type, c10::Device device) {
  return at::detail::empty_cuda(size, type, device, std::nullopt);
}

// [h = residual + x] -> [RMSNorm] -> E4M3: (h or nothing, codes, scales)
std::optional<std::tuple<std::optional<Tensor>, Tensor, Tensor>> fp8_pack(const Tensor& x, const std::optional<Tensor>& residual,
                                                                          const std::optional<Tensor>& gamma, double eps) {
  if (!x.is_cuda() || x.dim() < 1 || x.numel() == 0 || !plain(x, at::kBFloat16, x.device())) return std::nullopt;
  const int64_t k = x.size(-1), rows = x.numel() / k;
  if (residual && (residual->sizes() != x.sizes() || !plain(*residual, at::kBFloat16, x.device()))) return std::nullopt;
  if (gamma && (gamma->numel() != k || !plain(*gamma, at::kBFloat16, x.device()))) return std::nullopt;
  if (residual && !gamma) return std::nullopt;
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor codes = cuda_empty({rows, k}, at::kByte, x.device()), scales = cuda_empty({rows, (k + 127) / 128}, at::kFloat, x.device());
  std::optional<Tensor> h;
  if (residual) h = cuda_empty(x.sizes(), at::kBFloat16, x.device());
  check(api.fp8_pack(x.const_data_ptr(), k, residual ? residual->const_data_ptr() : nullptr, k, h ? h->data_ptr() : nullptr,
                     gamma ? gamma->const_data_ptr() : nullptr, static_cast<float>(eps), rows, k, codes.data_ptr(), scales.data_ptr(),
                     c10::cuda::getCurrentCUDAStream().stream()));
  return std::make_tuple(h, codes, scales);
}

std::optional<Tensor> fp8_gemm(const Tensor& a, const Tensor& sa, int64_t a_rows, const Tensor& w, const Tensor& sw, int64_t w_rows,
                               const Tensor& status, bool f32, int64_t flags) {
  const auto dev = a.device();
  if (!a.is_cuda() || a.dim() != 2 || w.dim() != 2 || a_rows != 1 || w_rows != 128 || a.numel() == 0 || w.numel() == 0 ||
      !plain(a, at::kByte, dev) || !plain(w, at::kByte, dev) || !plain(sa, at::kFloat, dev) || !plain(sw, at::kFloat, dev))
    return std::nullopt;
  const int64_t m = a.size(0), n = w.size(0), k = a.size(1), kb = (k + 127) / 128;
  if (w.size(1) != k || sa.dim() != 2 || sa.size(0) != m || sa.size(1) != kb || sw.dim() != 2 || sw.size(0) != (n + 127) / 128 || sw.size(1) != kb)
    return std::nullopt;
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(dev);
  Tensor y = cuda_empty({m, n}, f32 ? at::kFloat : at::kBFloat16, dev);
  check(api.fp8_gemm(a.const_data_ptr(), sa.const_data_ptr(), w.const_data_ptr(), sw.const_data_ptr(), m, n, k, y.data_ptr(), n, f32,
                     status.data_ptr<int32_t>(), static_cast<int>(flags), c10::cuda::getCurrentCUDAStream().stream()));
  return y;
}

// A cache's sides are what kv_cache.Fp8Cache.check asks for.
bool plain_cache(const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& vs, int64_t b, int64_t kv_heads, c10::Device dev) {
  if (k.dim() != 4 || k.size(0) != b || k.size(1) < 1 || k.size(2) != kv_heads || k.size(3) != 128 || v.sizes() != k.sizes()) return false;
  const std::array<int64_t, 3> scales = {b, kv_heads, (k.size(1) + 63) / 64};
  return ks.sizes() == c10::IntArrayRef(scales) && vs.sizes() == c10::IntArrayRef(scales) && plain(k, at::kByte, dev) && plain(v, at::kByte, dev) &&
         plain(ks, at::kFloat, dev) && plain(vs, at::kFloat, dev);
}
bool plain_positions(const std::optional<Tensor>& at, int64_t b, c10::Device dev) {
  return !at || (at->scalar_type() == at::kLong && (at->numel() == 1 || at->numel() == b) && at->device() == dev && at->is_contiguous());
}

std::optional<Tensor> rope_kv_append_fp8(const Tensor& qkv, const Tensor& cos, const Tensor& sin, int64_t heads, int64_t kv_heads, const Tensor& k,
                                         const Tensor& ks, const Tensor& v, const Tensor& vs, const std::optional<Tensor>& pos_dev, int64_t pos,
                                         const Tensor& status) {
  const auto dev = qkv.device();
  if (!qkv.is_cuda() || qkv.dim() != 3 || heads < 1 || kv_heads < 1 || qkv.numel() == 0 || qkv.size(2) != (heads + 2 * kv_heads) * 128 ||
      !plain(qkv, at::kBFloat16, dev) || !plain(cos, at::kFloat, dev) || !plain(sin, at::kFloat, dev))
    return std::nullopt;
  const int64_t b = qkv.size(0), t = qkv.size(1), n = cos.numel();
  if (sin.numel() != n || (n != t * 128 && n != b * t * 128) || !plain_cache(k, ks, v, vs, b, kv_heads, dev) || !plain_positions(pos_dev, b, dev))
    return std::nullopt;
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(dev);
  Tensor q = cuda_empty({b, t, heads, 128}, at::kBFloat16, dev);
  check(api.rope_kv_append_fp8(qkv.const_data_ptr(), qkv.size(2), cos.const_data_ptr(), sin.const_data_ptr(), n == t * 128 ? 0 : t * 128, b, t, heads,
                               kv_heads, q.data_ptr(), k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), k.size(1),
                               pos_dev ? pos_dev->const_data_ptr<int64_t>() : nullptr, pos_dev && b > 1 && pos_dev->numel() == b, pos,
                               status.data_ptr<int32_t>(), c10::cuda::getCurrentCUDAStream().stream()));
  return q;
}

std::optional<Tensor> fp8_attention(const Tensor& q, const Tensor& k, const Tensor& ks, const Tensor& v, const Tensor& vs,
                                    const std::optional<Tensor>& pos_dev, int64_t pos, int64_t ctx, double scale, const Tensor& status) {
  const auto dev = q.device();
  if (!q.is_cuda() || q.dim() != 4 || q.numel() == 0 || q.size(3) != 128 || !plain(q, at::kBFloat16, dev) || k.dim() != 4 ||
      !plain_cache(k, ks, v, vs, q.size(0), k.size(2), dev) || !plain_positions(pos_dev, q.size(0), dev))
    return std::nullopt;
  const int64_t b = q.size(0), t = q.size(1), heads = q.size(2), kv_heads = k.size(2), room = k.size(1);
  if (kv_heads < 1 || heads % kv_heads != 0) return std::nullopt;
  pybind11::gil_scoped_release nogil;
  const c10::cuda::CUDAGuard guard(dev);
  if (!pos_dev && pos >= 0) ctx = std::min(pos + t, room);
  else if (ctx <= 0) ctx = room;
  Tensor out = cuda_empty(q.sizes(), at::kBFloat16, dev), ws;
  const int64_t need = api.fp8_attention_workspace_bytes(b, t, heads, kv_heads, ctx);
  if (need) ws = cuda_empty({need}, at::kByte, dev);
  check(api.fp8_attention(q.const_data_ptr(), k.const_data_ptr(), ks.const_data_ptr(), v.const_data_ptr(), vs.const_data_ptr(), b, t, heads, kv_heads,
                          room, pos_dev ? pos_dev->const_data_ptr<int64_t>() : nullptr, pos_dev && b > 1 && pos_dev->numel() == b, pos, ctx,
                          static_cast<float>(scale), out.data_ptr(), need ? ws.data_ptr() : nullptr, need, status.data_ptr<int32_t>(),
                          c10::cuda::getCurrentCUDAStream().stream()));
  return out;
}

}  // namespace

PYBIND11_MODULE(_plq_torch, m) {
  pybind11::class_<Linear>(m, "Linear")
      .def(pybind11::init([](Tensor lo, Tensor lo_sf, Tensor hi, Tensor hi_sf, Tensor status, int64_t n, int64_t k_lo, int64_t k_hi) {
        return Linear{lo, lo_sf, hi, hi_sf, status, n, k_lo, k_hi};
      }))
      .def("forward", &Linear::forward);
  m.def("init", &init);
  m.def("pack", &pack);
  m.def("alone", &alone);
  m.def("decoder_layer", &decoder_layer);
  m.def("layer_front", &layer_front);
  m.def("layer_back", &layer_back);
  m.def("fp8_pack", &fp8_pack);
  m.def("fp8_gemm", &fp8_gemm);
  m.def("rope_kv_append_fp8", &rope_kv_append_fp8);
  m.def("fp8_attention", &fp8_attention);
}
