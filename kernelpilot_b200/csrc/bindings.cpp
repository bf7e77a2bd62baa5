// torch.ops.kp.* on top of the C ABI in include/kp_b200.h.
//
// Same operator schemas and checks as kernelpilot's csrc/bindings.cpp:118-134
// (inputs on the GPU and contiguous :25-28, matching shapes/dtypes :38/:71/:88-90/:106,
// size limits :60/:73/:93/:109, variant ranges :30-33/:77/:111, launch on the current
// stream :12-17,
// fresh outputs from the caching allocator). Additions: bf16 inputs (dtype_of,
// :19-23, accepted float32/float16 only), the attention_causal operator and the decode
// step's operators (qk_norm_rope and its backward, kv_cache_write, kv_cache_read,
// paged_attention), which have no counterpart there. The latter take slices of a fused
// projection (tokens any stride apart) and run on their tensors' device whatever the
// current one is.
// Errors surface as c10::Error (Python RuntimeError) carrying kpb_last_error().
//
// Scratch (reduction partials, the aligned copy of B for odd N) comes from the
// caching allocator on the op's stream, so concurrent calls on different streams
// never share it.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "kp_b200.h"

namespace {

void* current_stream(const at::Tensor& t) {
  auto impl = c10::impl::getDeviceGuardImpl(t.device().type());
  return impl->getStream(t.device()).native_handle();
}

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KPB_F32;
    case at::kHalf: return KPB_F16;
    case at::kBFloat16: return KPB_BF16;
    default:
      TORCH_CHECK(false, "kernelpilot kernels support float32, float16 and bfloat16, got ",
                  t.scalar_type());
  }
}

void check_input(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

int64_t check_variant(const char* op, int64_t v) {
  const int64_t n = kpb_num_variants(op);
  TORCH_CHECK(v >= 0 && v < n, "variant must be in [0, ", n, ")");
  return v;
}

void check_rc(int rc, const char* op) {
  TORCH_CHECK(rc == KPB_OK, "kp.", op, " failed (status ", rc, "): ", kpb_last_error());
}

// Scratch bytes from the caching allocator, stream-ordered with the op.
at::Tensor scratch(const at::Tensor& like, size_t bytes) {
  return at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)},
                   like.options().dtype(at::kByte));
}

at::Tensor vector_add(const at::Tensor& a, const at::Tensor& b, int64_t variant) {
  check_input(a, "a");
  check_input(b, "b");
  TORCH_CHECK(a.sizes() == b.sizes() && a.scalar_type() == b.scalar_type(),
              "a and b must match in shape and dtype");
  const int v = static_cast<int>(check_variant("vector_add", variant));
  auto c = at::empty_like(a);
  check_rc(kpb_vector_add(v, dtype_of(a), a.data_ptr(), b.data_ptr(), c.data_ptr(), a.numel(),
                          current_stream(a)),
           "vector_add");
  return c;
}

at::Tensor reduce_sum(const at::Tensor& x, int64_t variant) {
  check_input(x, "x");
  const int v = static_cast<int>(check_variant("reduce_sum", variant));
  const int dt = dtype_of(x);
  // kpb writes out[0] (no zero-init needed, unlike the reference's at::zeros)
  auto out = at::empty({}, x.options().dtype(at::kFloat));
  auto ws = scratch(x, kpb_reduce_sum_workspace_bytes(v, x.numel()));
  check_rc(kpb_reduce_sum_ws(v, dt, x.data_ptr(), out.data_ptr<float>(), x.numel(),
                             ws.data_ptr(), static_cast<size_t>(ws.numel()), current_stream(x)),
           "reduce_sum");
  return out;
}

at::Tensor softmax(const at::Tensor& x, int64_t variant) {
  check_input(x, "x");
  TORCH_CHECK(x.dim() >= 1, "softmax needs at least 1 dimension");
  const int v = static_cast<int>(check_variant("softmax", variant));
  auto y = at::empty_like(x);
  const int64_t N = x.size(-1);
  const int64_t M = N == 0 ? 0 : x.numel() / N;
  TORCH_CHECK(M < (int64_t{1} << 31) && N < (int64_t{1} << 31), "softmax shape too large");
  check_rc(kpb_softmax(v, dtype_of(x), x.data_ptr(), y.data_ptr(), M, N, current_stream(x)),
           "softmax");
  return y;
}

at::Tensor matmul(const at::Tensor& a, const at::Tensor& b, int64_t variant) {
  check_input(a, "a");
  check_input(b, "b");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0),
              "matmul expects (M, K) @ (K, N), got ", a.sizes(), " and ", b.sizes());
  TORCH_CHECK(a.scalar_type() == b.scalar_type(), "a and b must have the same dtype");
  const int v = static_cast<int>(check_variant("matmul", variant));
  const int64_t M = a.size(0), K = a.size(1), N = b.size(1);
  TORCH_CHECK(M < (int64_t{1} << 31) && N < (int64_t{1} << 31) && K < (int64_t{1} << 31),
              "matmul shape too large");
  const int dt = dtype_of(a);
  auto c = at::empty({M, N}, a.options());
  if (M == 0 || N == 0) return c;
  if (K == 0) return c.zero_();
  auto ws = scratch(a, kpb_matmul_workspace_bytes(v, dt, M, N, K));
  check_rc(kpb_matmul_ws(v, dt, a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K,
                         ws.data_ptr(), static_cast<size_t>(ws.numel()), current_stream(a)),
           "matmul");
  return c;
}

at::Tensor layernorm(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, double eps,
                     int64_t variant) {
  check_input(x, "x");
  check_input(w, "weight");
  check_input(b, "bias");
  TORCH_CHECK(x.dim() >= 1, "layernorm needs at least 1 dimension");
  const int64_t N = x.size(-1);
  TORCH_CHECK(w.numel() == N && b.numel() == N, "weight and bias must have size ", N);
  TORCH_CHECK(w.scalar_type() == x.scalar_type() && b.scalar_type() == x.scalar_type(),
              "x, weight and bias must share a dtype");
  const int var = static_cast<int>(check_variant("layernorm", variant));
  auto y = at::empty_like(x);
  const int64_t M = N == 0 ? 0 : x.numel() / N;
  TORCH_CHECK(M < (int64_t{1} << 31) && N < (int64_t{1} << 31), "layernorm shape too large");
  check_rc(kpb_layernorm(var, dtype_of(x), x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(),
                         M, N, static_cast<float>(eps), current_stream(x)),
           "layernorm");
  return y;
}

at::Tensor attention_impl(const char* op, const at::Tensor& q, const at::Tensor& k,
                          const at::Tensor& v, int64_t variant) {
  check_input(q, "q");
  check_input(k, "k");
  check_input(v, "v");
  TORCH_CHECK(q.dim() == 4 && q.sizes() == k.sizes() && q.sizes() == v.sizes(),
              "q, k, v must all be (B, H, S, D)");
  TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(),
              "q, k, v must share a dtype");
  const int var = static_cast<int>(check_variant(op, variant));
  const int64_t BH = q.size(0) * q.size(1), S = q.size(2), D = q.size(3);
  TORCH_CHECK(D <= 256 && BH < 65536, "attention supports D <= 256 and B*H < 65536");
  auto o = at::empty_like(q);
  const int dt = dtype_of(q);
  const int rc = std::string(op) == "attention"
                     ? kpb_attention(var, dt, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                     o.data_ptr(), BH, S, D, current_stream(q))
                     : kpb_attention_causal(var, dt, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                            o.data_ptr(), BH, S, D, current_stream(q));
  check_rc(rc, op);
  return o;
}

at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     int64_t variant) {
  return attention_impl("attention", q, k, v, variant);
}

at::Tensor attention_causal(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            int64_t variant) {
  return attention_impl("attention_causal", q, k, v, variant);
}

// ------------------------------------------------------------------ the decode step

void check_same_device(const at::Tensor& t, const at::Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a GPU tensor");
  TORCH_CHECK(t.device() == first.device(), name, " must be on ", first.device(), ", got ",
              t.device());
}

// (T, H, D) whose tokens may be any stride apart, each token's (H, D) part contiguous.
void check_heads(const at::Tensor& t, const at::Tensor& first, const char* name) {
  check_same_device(t, first, name);
  TORCH_CHECK(t.dim() == 3, name, " must be (tokens, heads, head dim)");
  TORCH_CHECK(t.scalar_type() == first.scalar_type(), name, " must share q's or k's dtype");
  TORCH_CHECK(t.numel() == 0 || ((t.size(2) == 1 || t.stride(2) == 1) &&
                                 (t.size(1) == 1 || t.stride(1) == t.size(2))),
              name, " must hold each token's heads contiguously");
}

void check_index(const at::Tensor& t, const at::Tensor& first, const char* name,
                 at::ScalarType type, int64_t dim) {
  check_same_device(t, first, name);
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension", dim == 1 ? "" : "s");
}

struct RopeArgs {
  int dtype;
  int64_t T, Hq, Hkv, D, rot, max_pos;
};

RopeArgs check_rope(const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq,
                    const at::Tensor& wk, const at::Tensor& cos_sin,
                    const at::Tensor& positions) {
  check_heads(q, q, "q");
  check_heads(k, q, "k");
  RopeArgs a;
  a.dtype = dtype_of(q);
  a.T = q.size(0), a.Hq = q.size(1), a.Hkv = k.size(1), a.D = q.size(2);
  TORCH_CHECK(k.size(0) == a.T && k.size(2) == a.D,
              "q and k must match in tokens and head dim, got ", q.sizes(), " and ", k.sizes());
  for (const at::Tensor* w : {&wq, &wk}) {
    check_same_device(*w, q, "weight");
    TORCH_CHECK(w->is_contiguous() && w->dim() == 1 && w->size(0) == a.D,
                "weights must be contiguous and have size ", a.D);
    TORCH_CHECK(w->scalar_type() == q.scalar_type(), "q, k and weights must share a dtype");
  }
  check_same_device(cos_sin, q, "cos_sin");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2 && cos_sin.is_contiguous(),
              "cos_sin must be a contiguous float32 (positions, rotated elements) table");
  a.max_pos = cos_sin.size(0), a.rot = cos_sin.size(1);
  check_index(positions, q, "positions", at::kLong, 1);
  TORCH_CHECK(positions.is_contiguous() && positions.size(0) == a.T,
              "positions must be contiguous, one per token");
  return a;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k,
                                                const at::Tensor& wq, const at::Tensor& wk,
                                                const at::Tensor& cos_sin,
                                                const at::Tensor& positions, double eps,
                                                bool interleaved, int64_t variant) {
  const RopeArgs a = check_rope(q, k, wq, wk, cos_sin, positions);
  const int v = static_cast<int>(check_variant("qk_norm_rope", variant));
  const c10::DeviceGuard guard(q.device());
  auto q_out = at::empty({a.T, a.Hq, a.D}, q.options());
  auto k_out = at::empty({a.T, a.Hkv, a.D}, k.options());
  check_rc(kpb_qk_norm_rope(v, a.dtype, q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(),
                            cos_sin.data_ptr<float>(), positions.data_ptr<int64_t>(),
                            q_out.data_ptr(), k_out.data_ptr(), a.T, a.Hq, a.Hkv, a.D, a.rot,
                            a.max_pos, q.stride(0), k.stride(0), static_cast<float>(eps),
                            interleaved, current_stream(q)),
           "qk_norm_rope");
  return {q_out, k_out};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_backward(
    const at::Tensor& gq, const at::Tensor& gk, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& cos_sin,
    const at::Tensor& positions, double eps, bool interleaved, int64_t variant) {
  const RopeArgs a = check_rope(q, k, wq, wk, cos_sin, positions);
  check_heads(gq, q, "grad_q");
  check_heads(gk, q, "grad_k");
  TORCH_CHECK(gq.sizes() == q.sizes() && gk.sizes() == k.sizes(),
              "gradients must have the shapes of q and k");
  const int v = static_cast<int>(check_variant("qk_norm_rope_backward", variant));
  const c10::DeviceGuard guard(q.device());
  auto dq = at::empty({a.T, a.Hq, a.D}, q.options());
  auto dk = at::empty({a.T, a.Hkv, a.D}, k.options());
  auto dwq = at::empty_like(wq);
  auto dwk = at::empty_like(wk);
  auto ws = scratch(q, kpb_qk_norm_rope_backward_workspace_bytes(a.T, a.Hq, a.Hkv, a.D));
  check_rc(kpb_qk_norm_rope_backward(
               v, a.dtype, gq.data_ptr(), gk.data_ptr(), q.data_ptr(), k.data_ptr(),
               wq.data_ptr(), wk.data_ptr(), cos_sin.data_ptr<float>(),
               positions.data_ptr<int64_t>(), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(),
               dwk.data_ptr(), a.T, a.Hq, a.Hkv, a.D, a.rot, a.max_pos, gq.stride(0),
               gk.stride(0), q.stride(0), k.stride(0), static_cast<float>(eps), interleaved,
               ws.data_ptr(), static_cast<size_t>(ws.numel()), current_stream(q)),
           "qk_norm_rope_backward");
  return {dq, dk, dwq, dwk};
}

struct CacheArgs {
  int cache_dtype;
  int64_t pages, heads, page_size, dim, page_stride;
  float *k_scale, *v_scale;
};

// Both caches (pages, Hkv, page size, D): alike in shape, type and page stride, the inner
// three dimensions contiguous; scales with e4m3 caches and only with them. `like` names
// the device.
CacheArgs check_cache(const at::Tensor& kc, const at::Tensor& vc,
                      const std::optional<at::Tensor>& ks, const std::optional<at::Tensor>& vs,
                      const at::Tensor& like) {
  check_same_device(kc, like, "k_cache");
  check_same_device(vc, like, "v_cache");
  TORCH_CHECK(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.scalar_type() == vc.scalar_type(),
              "k_cache and v_cache must both be (pages, heads, page size, head dim) of one dtype");
  CacheArgs a;
  a.pages = kc.size(0), a.heads = kc.size(1), a.page_size = kc.size(2), a.dim = kc.size(3);
  for (const at::Tensor* c : {&kc, &vc})
    TORCH_CHECK(c->numel() == 0 || ((a.dim == 1 || c->stride(3) == 1) &&
                                    (a.page_size == 1 || c->stride(2) == a.dim) &&
                                    (a.heads == 1 || c->stride(1) == a.page_size * a.dim)),
                "each page of a cache must be contiguous");
  TORCH_CHECK(a.pages < 2 || kc.stride(0) == vc.stride(0),
              "k_cache and v_cache must have the same page stride");
  a.page_stride = a.pages < 2 ? a.heads * a.page_size * a.dim : kc.stride(0);
  const bool e4m3 = kc.scalar_type() == at::kFloat8_e4m3fn;
  a.cache_dtype = e4m3 ? KPB_E4M3 : dtype_of(kc);
  a.k_scale = a.v_scale = nullptr;
  TORCH_CHECK(ks.has_value() == e4m3 && vs.has_value() == e4m3,
              "k_scale and v_scale go with float8_e4m3fn caches, and only with them");
  if (e4m3) {
    for (const at::Tensor* s : {&*ks, &*vs}) {
      check_same_device(*s, like, "scale");
      TORCH_CHECK(s->scalar_type() == at::kFloat && s->is_contiguous() && s->dim() == 3 &&
                      s->size(0) == a.pages && s->size(1) == a.heads && s->size(2) == a.page_size,
                  "scales must be contiguous float32 (pages, heads, page size)");
    }
    a.k_scale = ks->data_ptr<float>();
    a.v_scale = vs->data_ptr<float>();
  }
  return a;
}

void kv_cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots,
                    at::Tensor& kc, at::Tensor& vc, const std::optional<at::Tensor>& ks,
                    const std::optional<at::Tensor>& vs, int64_t variant) {
  check_heads(k, k, "k");
  check_heads(v, k, "v");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must match in shape");
  const int dt = dtype_of(k);
  const CacheArgs a = check_cache(kc, vc, ks, vs, k);
  TORCH_CHECK(a.cache_dtype == KPB_E4M3 || a.cache_dtype == dt,
              "the caches must have k's dtype or float8_e4m3fn");
  TORCH_CHECK(k.size(1) == a.heads && k.size(2) == a.dim, "k and v must have the caches' heads (",
              a.heads, ") and head dim (", a.dim, ")");
  check_index(slots, k, "slots", at::kLong, 1);
  TORCH_CHECK(slots.is_contiguous() && slots.size(0) == k.size(0),
              "slots must be contiguous, one per token");
  const int var = static_cast<int>(check_variant("kv_cache_write", variant));
  const c10::DeviceGuard guard(k.device());
  check_rc(kpb_kv_cache_write(var, dt, a.cache_dtype, k.data_ptr(), v.data_ptr(),
                              slots.data_ptr<int64_t>(), kc.data_ptr(), vc.data_ptr(), a.k_scale,
                              a.v_scale, k.size(0), a.heads, a.dim, a.pages, a.page_size,
                              k.stride(0), v.stride(0), a.page_stride, current_stream(k)),
           "kv_cache_write");
}

std::tuple<at::Tensor, at::Tensor> kv_cache_read(const at::Tensor& kc, const at::Tensor& vc,
                                                 const at::Tensor& slots,
                                                 const std::optional<at::Tensor>& ks,
                                                 const std::optional<at::Tensor>& vs,
                                                 at::ScalarType dtype, int64_t variant) {
  const CacheArgs a = check_cache(kc, vc, ks, vs, kc);
  check_index(slots, kc, "slots", at::kLong, 1);
  TORCH_CHECK(slots.is_contiguous(), "slots must be contiguous");
  const int var = static_cast<int>(check_variant("kv_cache_read", variant));
  const c10::DeviceGuard guard(kc.device());
  auto k = at::empty({slots.size(0), a.heads, a.dim}, kc.options().dtype(dtype));
  const int dt = dtype_of(k);
  TORCH_CHECK(a.cache_dtype == KPB_E4M3 || a.cache_dtype == dt,
              "caches that are not float8_e4m3fn are read in their own dtype");
  auto v = at::empty_like(k);
  check_rc(kpb_kv_cache_read(var, dt, a.cache_dtype, kc.data_ptr(), vc.data_ptr(),
                             slots.data_ptr<int64_t>(), a.k_scale, a.v_scale, k.data_ptr(),
                             v.data_ptr(), slots.size(0), a.heads, a.dim, a.pages, a.page_size,
                             a.page_stride, current_stream(kc)),
           "kv_cache_read");
  return {k, v};
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                           const at::Tensor& table, const at::Tensor& lens,
                           const std::optional<at::Tensor>& ks,
                           const std::optional<at::Tensor>& vs, std::optional<double> scale,
                           int64_t variant) {
  check_heads(q, q, "q");
  const int dt = dtype_of(q);
  const CacheArgs a = check_cache(kc, vc, ks, vs, q);
  TORCH_CHECK(a.cache_dtype == KPB_E4M3 || a.cache_dtype == dt,
              "the caches must have q's dtype or float8_e4m3fn");
  const int64_t B = q.size(0), Hq = q.size(1);
  TORCH_CHECK(q.size(2) == a.dim, "q must have the caches' head dim (", a.dim, ")");
  TORCH_CHECK(Hq == 0 || (a.heads > 0 && Hq % a.heads == 0),
              "q's heads must be a multiple of the caches' (", a.heads, ")");
  check_index(table, q, "block_table", at::kInt, 2);
  TORCH_CHECK(table.size(0) == B && (table.size(1) < 2 || table.stride(1) == 1),
              "block_table must be (sequences, pages) with each row contiguous");
  check_index(lens, q, "seq_lens", at::kInt, 1);
  TORCH_CHECK(lens.is_contiguous() && lens.size(0) == B,
              "seq_lens must be contiguous, one per sequence");
  const int var = static_cast<int>(check_variant("paged_attention", variant));
  const c10::DeviceGuard guard(q.device());
  auto o = at::empty({B, Hq, a.dim}, q.options());
  const double sc = scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(a.dim));
  auto ws = scratch(q, kpb_paged_attention_workspace_bytes(var, B, Hq, a.heads, a.dim,
                                                           table.size(1) * a.page_size));
  check_rc(kpb_paged_attention(var, dt, a.cache_dtype, q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                               table.data_ptr<int>(), lens.data_ptr<int>(), a.k_scale, a.v_scale,
                               o.data_ptr(), B, Hq, a.heads, a.dim, a.pages, a.page_size,
                               table.size(1), q.stride(0), a.page_stride, table.stride(0),
                               static_cast<float>(sc), ws.data_ptr(),
                               static_cast<size_t>(ws.numel()), current_stream(q)),
           "paged_attention");
  return o;
}

}  // namespace

TORCH_LIBRARY(kp, m) {
  m.def("vector_add(Tensor a, Tensor b, int variant) -> Tensor");
  m.def("reduce_sum(Tensor x, int variant) -> Tensor");
  m.def("softmax(Tensor x, int variant) -> Tensor");
  m.def("matmul(Tensor a, Tensor b, int variant) -> Tensor");
  m.def("layernorm(Tensor x, Tensor weight, Tensor bias, float eps, int variant) -> Tensor");
  m.def("attention(Tensor q, Tensor k, Tensor v, int variant) -> Tensor");
  m.def("attention_causal(Tensor q, Tensor k, Tensor v, int variant) -> Tensor");
  m.def(
      "qk_norm_rope(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos_sin, "
      "Tensor positions, float eps, bool interleaved, int variant) -> (Tensor, Tensor)");
  m.def(
      "qk_norm_rope_backward(Tensor grad_q, Tensor grad_k, Tensor q, Tensor k, Tensor q_weight, "
      "Tensor k_weight, Tensor cos_sin, Tensor positions, float eps, bool interleaved, "
      "int variant) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "kv_cache_write(Tensor k, Tensor v, Tensor slots, Tensor(a!) k_cache, Tensor(b!) v_cache, "
      "Tensor(c!)? k_scale, Tensor(d!)? v_scale, int variant) -> ()");
  m.def(
      "kv_cache_read(Tensor k_cache, Tensor v_cache, Tensor slots, Tensor? k_scale, "
      "Tensor? v_scale, ScalarType dtype, int variant) -> (Tensor, Tensor)");
  m.def(
      "paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
      "Tensor seq_lens, Tensor? k_scale, Tensor? v_scale, float? scale, int variant) -> Tensor");
}

TORCH_LIBRARY_IMPL(kp, CUDA, m) {
  m.impl("vector_add", &vector_add);
  m.impl("reduce_sum", &reduce_sum);
  m.impl("softmax", &softmax);
  m.impl("matmul", &matmul);
  m.impl("layernorm", &layernorm);
  m.impl("attention", &attention);
  m.impl("attention_causal", &attention_causal);
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("qk_norm_rope_backward", &qk_norm_rope_backward);
  m.impl("kv_cache_write", &kv_cache_write);
  m.impl("kv_cache_read", &kv_cache_read);
  m.impl("paged_attention", &paged_attention);
}
