// The attention layer of a language model on the PrivateUse1 device:
//   torch_vulkan::qk_norm_rotary (+ _backward)  norm of each head and rotary positions
//   torch_vulkan::attention (+ _backward)       causal attention of packed sequences
//   torch_vulkan::kv_cache_write_, kv_cache_read, attention_paged   a paged cache and attention over it
// Queries, keys and values [tokens, heads, head_dim] are read with their strides (packed
// first where the last axis is not contiguous); outputs are contiguous, and zero in rows
// that belong to no sequence.
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <array>
#include <optional>
#include <tuple>

#include "common.h"

namespace tvk {
namespace {

using OptT = std::optional<at::Tensor>;

bool present(const OptT& t) { return t.has_value() && t->defined(); }
void launched() { counters().kernel_launches += uint64_t(mx_last_launches()); }  // by the call before

void check_dev(const char* who, const char* what, const at::Tensor& t, at::ScalarType type, const at::Tensor& like) {
  TORCH_CHECK(is_vk(t) && t.scalar_type() == type && !t.is_neg() && !t.is_conj(), who, ": ", what, " must be a ", type,
              " vulkan tensor");
  TORCH_CHECK(t.device() == like.device(), who, ": expected all tensors on one device");
}

// A packed tensor and its strides.
struct Rows {
  at::Tensor held;
  const float* at = nullptr;
  int64_t token = 0, head = 0;
  Rows() = default;
  Rows(const char* who, const char* what, const at::Tensor& t, const at::Tensor& like) {
    check_dev(who, what, t, at::kFloat, like);
    TORCH_CHECK(t.dim() == 3, who, ": ", what, " must be [tokens, heads, head_dim], got ", t.sizes());
    held = t.size(2) <= 1 || t.stride(2) == 1 || t.numel() == 0 ? t : t.contiguous();
    at = held.const_data_ptr<float>();
    token = held.stride(0), head = held.stride(1);
  }
};

at::Tensor flat(const char* who, const char* what, const at::Tensor& t, at::IntArrayRef shape, const at::Tensor& like,
                at::ScalarType type = at::kFloat) {
  check_dev(who, what, t, type, like);
  TORCH_CHECK(t.sizes().equals(shape), who, ": ", what, " has shape ", t.sizes(), ", expected ", shape);
  return t.contiguous();
}
at::Tensor flat(const char* who, const char* what, const OptT& t, at::IntArrayRef shape, const at::Tensor& like,
                at::ScalarType type = at::kFloat) {
  return present(t) ? flat(who, what, *t, shape, like, type) : at::Tensor();
}
template <class T = float>
const T* cptr(const at::Tensor& t) {
  return t.defined() ? t.const_data_ptr<T>() : nullptr;
}
float* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef shape, bool zero = false) {
  return zero ? at::zeros(shape, like.options()) : at::empty(shape, like.options());
}

// ----------------------------------------------------------- norm and rotation
struct RotaryCall {
  at::Tensor positions, qw, kw;
  mx_rotary_desc d{};
};
RotaryCall rotary_call(const char* who, const at::Tensor& like, at::IntArrayRef q, at::IntArrayRef k, const OptT& positions,
                       at::ArrayRef<double> frequencies, bool interleaved, double magnitude, const OptT& qw, const OptT& kw,
                       std::optional<double> eps) {
  TORCH_CHECK(q.size() == 3 && k.size() == 3 && q[0] == k[0] && q[2] == k[2], who, ": queries ", q, " and keys ", k, " do not fit");
  RotaryCall c;
  TORCH_CHECK(frequencies.empty() || present(positions), who, ": no positions");
  c.positions = flat(who, "positions", positions, {q[0]}, like, at::kLong);
  c.qw = flat(who, "q_weight", qw, {q[2]}, like);
  c.kw = flat(who, "k_weight", kw, {q[2]}, like);
  TORCH_CHECK(eps || (!c.qw.defined() && !c.kw.defined()), who, ": weights without a norm (eps)");
  c.d.tokens = q[0], c.d.q_heads = q[1], c.d.k_heads = k[1], c.d.head_dim = q[2];
  c.d.rotary_dim = 2 * int64_t(frequencies.size());
  c.d.positions = cptr<int64_t>(c.positions);
  c.d.frequencies = frequencies.data();
  c.d.magnitude = magnitude, c.d.eps = eps.value_or(0.0), c.d.interleaved = interleaved, c.d.norm = eps.has_value();
  return c;
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary(const at::Tensor& q, const at::Tensor& k, const OptT& positions,
                                                  at::ArrayRef<double> frequencies, bool interleaved, double magnitude,
                                                  const OptT& q_weight, const OptT& k_weight, std::optional<double> eps) {
  const char* const who = "qk_norm_rotary";
  const Rows qr(who, "q", q, q), kr(who, "k", k, q);
  RotaryCall c = rotary_call(who, q, q.sizes(), k.sizes(), positions, frequencies, interleaved, magnitude, q_weight, k_weight, eps);
  c.d.q_token = qr.token, c.d.q_head = qr.head, c.d.k_token = kr.token, c.d.k_head = kr.head;
  c10::DeviceGuard guard(q.device());
  at::Tensor qo = fresh(q, q.sizes()), ko = fresh(k, k.sizes());
  GpuTimer timer(gpu_timing_enabled() ? "qk_norm_rotary" : "");
  TVK_MX(mx_qk_norm_rotary_forward(&c.d, qr.at, kr.at, cptr(c.qw), cptr(c.kw), ptr(qo), ptr(ko), current_stream()));
  launched();
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rotary_backward(
    const at::Tensor& dq_out, const at::Tensor& dk_out, const OptT& q, const OptT& k, const OptT& positions,
    at::ArrayRef<double> frequencies, bool interleaved, double magnitude, const OptT& q_weight, const OptT& k_weight,
    std::optional<double> eps, std::array<bool, 4> mask) {
  const char* const who = "qk_norm_rotary_backward";
  const at::Tensor gq = flat(who, "dq_out", dq_out, dq_out.sizes(), dq_out), gk = flat(who, "dk_out", dk_out, dk_out.sizes(), dq_out);
  RotaryCall c =
      rotary_call(who, gq, gq.sizes(), gk.sizes(), positions, frequencies, interleaved, magnitude, q_weight, k_weight, eps);
  Rows qr, kr;
  if (eps) {
    TORCH_CHECK(present(q) && present(k) && q->sizes() == gq.sizes() && k->sizes() == gk.sizes(), who,
                ": a norm needs its inputs, of the gradients' shapes");
    qr = Rows(who, "q", *q, gq), kr = Rows(who, "k", *k, gq);
    c.d.q_token = qr.token, c.d.q_head = qr.head, c.d.k_token = kr.token, c.d.k_head = kr.head;
  }
  c10::DeviceGuard guard(gq.device());
  at::Tensor dq, dk, dqw, dkw;
  if (mask[0]) dq = fresh(gq, gq.sizes());
  if (mask[1]) dk = fresh(gk, gk.sizes());
  if (mask[2]) dqw = fresh(gq, {gq.size(2)});
  if (mask[3]) dkw = fresh(gq, {gq.size(2)});
  GpuTimer timer(gpu_timing_enabled() ? "qk_norm_rotary_backward" : "");
  TVK_MX(mx_qk_norm_rotary_backward(&c.d, cptr(gq), cptr(gk), qr.at, kr.at, cptr(c.qw), cptr(c.kw), ptr(dq), ptr(dk), ptr(dqw),
                                    ptr(dkw), nullptr, 0, current_stream()));
  launched();
  return {dq, dk, dqw, dkw};
}

// ------------------------------------------------------------------ attention
struct AttentionCall {
  Rows q, k, v;
  at::Tensor starts;
  mx_attention_desc d{};
};
AttentionCall attention_call(const char* who, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& starts,
                             int64_t sequences, int64_t window, int64_t sinks, double scale) {
  AttentionCall c;
  c.q = Rows(who, "q", q, q), c.k = Rows(who, "k", k, q), c.v = Rows(who, "v", v, q);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2), who, ": q ", q.sizes(), ", k ", k.sizes(),
              " and v ", v.sizes(), " do not fit");
  if (present(starts)) {
    TORCH_CHECK(starts->dim() == 1 && starts->numel() >= 1, who, ": starts must name every sequence's first row and the last one's end");
    c.starts = flat(who, "starts", starts, starts->sizes(), q, at::kInt);
    sequences = starts->numel() - 1;
  }
  c.d = {q.size(0), sequences, cptr<int32_t>(c.starts), q.size(1), k.size(1), q.size(2), c.q.token, c.q.head,
         c.k.token, c.k.head,  c.v.token, c.v.head,     window,    sinks,     scale};
  return c;
}

std::tuple<at::Tensor, at::Tensor> attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptT& starts,
                                             int64_t sequences, int64_t window, int64_t sinks, double scale) {
  const AttentionCall c = attention_call("attention", q, k, v, starts, sequences, window, sinks, scale);
  c10::DeviceGuard guard(q.device());
  at::Tensor out = fresh(q, q.sizes(), c.starts.defined()), lse = fresh(q, {q.size(1), q.size(0)}, c.starts.defined());
  GpuTimer timer(gpu_timing_enabled() ? "attention_forward" : "");
  TVK_MX(mx_attention_forward(&c.d, c.q.at, c.k.at, c.v.at, ptr(out), ptr(lse), nullptr, 0, current_stream()));
  launched();
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_backward(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
                                                                  const at::Tensor& v, const at::Tensor& out,
                                                                  const at::Tensor& lse, const OptT& starts, int64_t sequences,
                                                                  int64_t window, int64_t sinks, double scale,
                                                                  std::array<bool, 3> mask) {
  const char* const who = "attention_backward";
  const AttentionCall c = attention_call(who, q, k, v, starts, sequences, window, sinks, scale);
  const at::Tensor g = flat(who, "dout", dout, q.sizes(), q), o = flat(who, "out", out, q.sizes(), q),
                   l = flat(who, "lse", lse, {q.size(1), q.size(0)}, q);
  c10::DeviceGuard guard(q.device());
  const bool zero = c.starts.defined();
  at::Tensor dq, dk, dv;
  if (mask[0]) dq = fresh(q, q.sizes(), zero);
  if (mask[1]) dk = fresh(k, k.sizes(), zero);
  if (mask[2]) dv = fresh(v, v.sizes(), zero);
  GpuTimer timer(gpu_timing_enabled() ? "attention_backward" : "");
  TVK_MX(mx_attention_backward(&c.d, cptr(g), c.q.at, c.k.at, c.v.at, cptr(o), cptr(l), ptr(dq), ptr(dk), ptr(dv), nullptr, 0,
                               current_stream()));
  launched();
  return {dq, dk, dv};
}

// ------------------------------------------------------------------ the cache
struct CacheCall {
  at::Tensor table, lengths, starts;
  mx_kv_cache c{};
  mx_kv_batch b{};
};
CacheCall cache_call(const char* who, const at::Tensor& k, const at::Tensor& v, const OptT& ks, const OptT& vs,
                     const at::Tensor& table, const at::Tensor& lengths, const OptT& starts, int64_t tokens) {
  CacheCall r;
  TORCH_CHECK(is_vk(k) && k.dim() == 4 && (k.scalar_type() == at::kFloat || k.scalar_type() == at::kChar), who,
              ": the cache's k must be a float32 or int8 vulkan tensor [pages, heads, page_size, head_dim]");
  const bool i8 = k.scalar_type() == at::kChar;
  check_dev(who, "the cache's v", v, k.scalar_type(), k);
  TORCH_CHECK(v.sizes().equals({k.size(0), k.size(1), k.size(3), k.size(2)}), who, ": the cache's v has shape ", v.sizes(),
              ", expected [pages, heads, head_dim, page_size] for k ", k.sizes());
  TORCH_CHECK(present(ks) == i8 && present(vs) == i8, who, ": scales go with an int8 cache, and with no other");
  for (const OptT* s : {&ks, &vs}) {
    if (!present(*s)) continue;
    check_dev(who, "a scale", **s, at::kFloat, k);
    TORCH_CHECK((*s)->sizes().equals(k.sizes().slice(0, 3)), who, ": a scale has shape ", (*s)->sizes());
    TORCH_CHECK((*s)->is_contiguous(), who, ": the cache must be contiguous");
  }
  TORCH_CHECK(k.is_contiguous() && v.is_contiguous(), who, ": the cache must be contiguous");
  TORCH_CHECK(table.dim() == 2, who, ": table must be [sequences, pages]");
  r.table = flat(who, "table", table, table.sizes(), k, at::kInt);
  r.lengths = flat(who, "lengths", lengths, {table.size(0)}, k, at::kInt);
  r.starts = flat(who, "starts", starts, {table.size(0) + 1}, k, at::kInt);
  r.c = {k.data_ptr(), v.data_ptr(), i8 ? ks->data_ptr<float>() : nullptr, i8 ? vs->data_ptr<float>() : nullptr, k.size(0), k.size(1),
         k.size(2),    k.size(3),    i8 ? MX_KV_I8 : MX_KV_F32};
  r.b = {tokens, table.size(0), table.size(1), cptr<int32_t>(r.starts), cptr<int32_t>(r.lengths), cptr<int32_t>(r.table)};
  return r;
}

void kv_cache_write_(const at::Tensor& k_cache, const at::Tensor& v_cache, const OptT& k_scale, const OptT& v_scale,
                     const at::Tensor& table, const at::Tensor& lengths, const OptT& starts, const at::Tensor& k,
                     const at::Tensor& v) {
  const char* const who = "kv_cache_write_";
  const Rows kr(who, "k", k, k_cache), vr(who, "v", v, k_cache);
  const CacheCall r = cache_call(who, k_cache, v_cache, k_scale, v_scale, table, lengths, starts, k.size(0));
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(1) == r.c.heads && k.size(2) == r.c.head_dim, who, ": k ", k.sizes(), " and v ",
              v.sizes(), " do not fit the cache");
  c10::DeviceGuard guard(k_cache.device());
  GpuTimer timer(gpu_timing_enabled() ? "kv_cache_write" : "");
  TVK_MX(mx_kv_cache_write(&r.c, &r.b, kr.at, kr.token, kr.head, vr.at, vr.token, vr.head, current_stream()));
  launched();
}

std::tuple<at::Tensor, at::Tensor> kv_cache_read(const at::Tensor& k_cache, const at::Tensor& v_cache, const OptT& k_scale,
                                                 const OptT& v_scale, const at::Tensor& table, const at::Tensor& lengths,
                                                 const OptT& starts, int64_t tokens) {
  const char* const who = "kv_cache_read";
  const CacheCall r = cache_call(who, k_cache, v_cache, k_scale, v_scale, table, lengths, starts, tokens);
  c10::DeviceGuard guard(k_cache.device());
  const auto options = k_cache.options().dtype(at::kFloat);
  TORCH_CHECK(tokens >= 0, who, ": negative size");
  const std::array<int64_t, 3> shape{tokens, r.c.heads, r.c.head_dim};
  at::Tensor k = present(starts) ? at::zeros(shape, options) : at::empty(shape, options), v = at::empty_like(k);
  if (present(starts)) v.zero_();
  GpuTimer timer(gpu_timing_enabled() ? "kv_cache_read" : "");
  TVK_MX(mx_kv_cache_read(&r.c, &r.b, ptr(k), ptr(v), current_stream()));
  launched();
  return {k, v};
}

at::Tensor attention_paged(const at::Tensor& k_cache, const at::Tensor& v_cache, const OptT& k_scale, const OptT& v_scale,
                           const at::Tensor& table, const at::Tensor& lengths, const OptT& starts, const at::Tensor& q,
                           int64_t window, int64_t sinks, double scale) {
  const char* const who = "attention_paged";
  const Rows qr(who, "q", q, k_cache);
  const CacheCall r = cache_call(who, k_cache, v_cache, k_scale, v_scale, table, lengths, starts, q.size(0));
  TORCH_CHECK(q.size(2) == r.c.head_dim, who, ": q ", q.sizes(), " does not fit the cache");
  const mx_paged_desc d{q.size(1), qr.token, qr.head, window, sinks, scale};
  c10::DeviceGuard guard(q.device());
  at::Tensor out = fresh(q, q.sizes(), present(starts));
  GpuTimer timer(gpu_timing_enabled() ? "attention_paged" : "");
  TVK_MX(mx_attention_paged(&d, &r.c, &r.b, qr.at, ptr(out), nullptr, 0, current_stream()));
  launched();
  return out;
}

}  // namespace
}  // namespace tvk

TORCH_LIBRARY_FRAGMENT(torch_vulkan, m) {
  m.def(
      "qk_norm_rotary(Tensor q, Tensor k, Tensor? positions, float[] frequencies, bool interleaved, float magnitude, Tensor? "
      "q_weight, Tensor? k_weight, float? eps) -> (Tensor, Tensor)");
  m.def(
      "qk_norm_rotary_backward(Tensor dq_out, Tensor dk_out, Tensor? q, Tensor? k, Tensor? positions, float[] frequencies, bool "
      "interleaved, float magnitude, Tensor? q_weight, Tensor? k_weight, float? eps, bool[4] mask) -> (Tensor, Tensor, Tensor, "
      "Tensor)");
  m.def(
      "attention(Tensor q, Tensor k, Tensor v, Tensor? starts, int sequences, int window, int sinks, float scale) -> (Tensor, "
      "Tensor)");
  m.def(
      "attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor? starts, int sequences, int "
      "window, int sinks, float scale, bool[3] mask) -> (Tensor, Tensor, Tensor)");
  m.def(
      "kv_cache_write_(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, Tensor table, Tensor "
      "lengths, Tensor? starts, Tensor k, Tensor v) -> ()");
  m.def(
      "kv_cache_read(Tensor k_cache, Tensor v_cache, Tensor? k_scale, Tensor? v_scale, Tensor table, Tensor lengths, Tensor? "
      "starts, int tokens) -> (Tensor, Tensor)");
  m.def(
      "attention_paged(Tensor k_cache, Tensor v_cache, Tensor? k_scale, Tensor? v_scale, Tensor table, Tensor lengths, Tensor? "
      "starts, Tensor q, int window, int sinks, float scale) -> Tensor");
}

TORCH_LIBRARY_IMPL(torch_vulkan, PrivateUse1, m) {
  m.impl("qk_norm_rotary", TORCH_FN(tvk::qk_norm_rotary));
  m.impl("qk_norm_rotary_backward", TORCH_FN(tvk::qk_norm_rotary_backward));
  m.impl("attention", TORCH_FN(tvk::attention));
  m.impl("attention_backward", TORCH_FN(tvk::attention_backward));
  m.impl("kv_cache_write_", TORCH_FN(tvk::kv_cache_write_));
  m.impl("kv_cache_read", TORCH_FN(tvk::kv_cache_read));
  m.impl("attention_paged", TORCH_FN(tvk::attention_paged));
}
