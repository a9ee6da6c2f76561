// Layer norm, the linear layer with its epilogue, and the orthogonalised
// momentum step on the PrivateUse1 device:
//   aten::native_layer_norm (+ _backward)   nn.LayerNorm and its gradients
//   torch_vulkan::linear_act (+ _backward)  y = act(x w^T + b) + residual
//   torch_vulkan::orthogonalize             Newton-Schulz polar factors
//   torch_vulkan::muon_step_                the optimizer step around them
// FP32 operands are packed to contiguous tensors on the device and run through
// the C ABI; a layer norm of another dtype goes to the CPU and is counted, the
// custom operators refuse one.
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <array>
#include <optional>
#include <tuple>
#include <vector>

#include "common.h"

namespace tvk {
namespace {

using OptT = std::optional<at::Tensor>;

bool present(const OptT& t) { return t.has_value() && t->defined(); }
bool f32_dev(const at::Tensor& t) { return is_vk(t) && t.scalar_type() == at::kFloat && !t.is_neg() && !t.is_conj(); }
at::Tensor packed(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
at::Tensor packed(const OptT& t) { return present(t) ? packed(*t) : at::Tensor(); }
const float* cptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
float* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
OptT to_cpu(const OptT& t) { return present(t) ? OptT(t->cpu()) : OptT(); }
at::Tensor to_dev(const at::Tensor& t, const at::Device& d) { return t.defined() ? t.to(d) : t; }
void launched() { counters().kernel_launches += uint64_t(mx_last_launches()); }  // by the call before

// ---------------------------------------------------------------- LayerNorm
struct Rows {
  int64_t rows = 1, cols = 1;
  std::vector<int64_t> stat_shape;
};
Rows rows_of(const char* who, const at::Tensor& x, c10::SymIntArrayRef shape, const OptT& weight, const OptT& bias) {
  const int64_t nd = int64_t(shape.size()), lead = x.dim() - nd;
  TORCH_CHECK(nd >= 1 && lead >= 0, who, ": normalized_shape must name trailing axes of the input");
  Rows r;
  std::vector<int64_t> tail;
  for (int64_t i = 0; i < nd; ++i) {
    tail.push_back(shape[size_t(i)].expect_int());
    TORCH_CHECK(x.size(lead + i) == tail.back(), who, ": normalized_shape does not match the input's shape ", x.sizes());
    r.cols *= tail.back();
  }
  for (const OptT* t : {&weight, &bias})
    TORCH_CHECK(!present(*t) || (*t)->sizes().equals(tail), who, ": weight and bias must have the normalized shape");
  for (int64_t i = 0; i < lead; ++i) {
    r.rows *= x.size(i);
    r.stat_shape.push_back(x.size(i));
  }
  for (int64_t i = 0; i < nd; ++i) r.stat_shape.push_back(1);
  return r;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> native_layer_norm_vk(const at::Tensor& x, c10::SymIntArrayRef shape,
                                                                 const OptT& weight, const OptT& bias, double eps) {
  const Rows r = rows_of("native_layer_norm", x, shape, weight, bias);
  const bool ok = f32_dev(x) && r.cols > 0 && (!present(weight) || f32_dev(*weight)) && (!present(bias) || f32_dev(*bias));
  if (!ok) {
    note_cpu_fallback("native_layer_norm (non-FP32 / empty rows)");
    auto o = at::native_layer_norm_symint(x.cpu(), shape, to_cpu(weight), to_cpu(bias), eps);
    return {to_dev(std::get<0>(o), x.device()), to_dev(std::get<1>(o), x.device()), to_dev(std::get<2>(o), x.device())};
  }
  c10::DeviceGuard guard(x.device());
  const at::Tensor xc = packed(x), wc = packed(weight), bc = packed(bias);
  at::Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  at::Tensor mean = at::empty(r.stat_shape, x.options()), rstd = at::empty(r.stat_shape, x.options());
  GpuTimer timer(gpu_timing_enabled() ? "layer_norm_forward" : "");
  TVK_MX(mx_layer_norm_forward(cptr(xc), cptr(wc), cptr(bc), r.rows, r.cols, float(eps), ptr(y), ptr(mean), ptr(rstd),
                               current_stream()));
  launched();
  return {y, mean, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> native_layer_norm_backward_vk(
    const at::Tensor& dy, const at::Tensor& x, c10::SymIntArrayRef shape, const at::Tensor& mean, const at::Tensor& rstd,
    const OptT& weight, const OptT& bias, std::array<bool, 3> mask) {
  const Rows r = rows_of("native_layer_norm_backward", x, shape, weight, bias);
  TORCH_CHECK(dy.sizes() == x.sizes() && mean.numel() == r.rows && rstd.numel() == r.rows,
              "native_layer_norm_backward: gradient or statistics do not match the input");
  const bool ok = f32_dev(dy) && f32_dev(x) && f32_dev(mean) && f32_dev(rstd) && r.cols > 0 &&
                  (!present(weight) || f32_dev(*weight));
  if (!ok) {
    note_cpu_fallback("native_layer_norm_backward (non-FP32 / empty rows)");
    auto o = at::native_layer_norm_backward_symint(dy.cpu(), x.cpu(), shape, mean.cpu(), rstd.cpu(), to_cpu(weight),
                                                   to_cpu(bias), mask);
    return {to_dev(std::get<0>(o), x.device()), to_dev(std::get<1>(o), x.device()), to_dev(std::get<2>(o), x.device())};
  }
  c10::DeviceGuard guard(x.device());
  const auto tail = x.sizes().slice(size_t(x.dim() - int64_t(shape.size())));
  at::Tensor dx, dw, db;
  if (mask[0]) dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  if (mask[1]) dw = at::empty(tail, x.options());
  if (mask[2]) db = at::empty(tail, x.options());
  const at::Tensor dyc = packed(dy), xc = packed(x), mc = packed(mean), rc = packed(rstd), wc = packed(weight);
  GpuTimer timer(gpu_timing_enabled() ? "layer_norm_backward" : "");
  TVK_MX(mx_layer_norm_backward(cptr(dyc), cptr(xc), cptr(mc), cptr(rc), cptr(wc), r.rows, r.cols, ptr(dx), ptr(dw),
                                ptr(db), nullptr, 0, current_stream()));
  launched();
  return {dx, dw, db};
}

// ------------------------------------------------------------- linear layer
int activation_code(c10::string_view name) {
  static constexpr const char* kNames[] = {"none", "relu", "silu", "gelu", "gelu_tanh"};
  for (int i = 0; i < 5; ++i)
    if (name == kNames[i]) return i;
  TORCH_CHECK(false, "linear_act: activation must be none, relu, silu, gelu or gelu_tanh, got ", std::string(name));
}

void check_operand(const char* who, const char* what, const at::Tensor& t, const at::Tensor& like, at::IntArrayRef shape) {
  TORCH_CHECK(f32_dev(t), who, ": ", what, " must be a float32 vulkan tensor");
  TORCH_CHECK(t.device() == like.device(), who, ": expected all tensors on one device");
  TORCH_CHECK(t.sizes().equals(shape), who, ": ", what, " has shape ", t.sizes(), ", expected ", shape);
}

// (y, z): z is empty unless keep_z (the backward's argument).
std::tuple<at::Tensor, at::Tensor> linear_act(const at::Tensor& x, const at::Tensor& w, const OptT& bias, const OptT& residual,
                                             c10::string_view activation, bool keep_z) {
  const char* const who = "linear_act";
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, who, ": x and weight must be matrices");
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  const int act = activation_code(activation);
  check_operand(who, "x", x, x, {m, k});
  check_operand(who, "weight", w, x, {n, k});
  if (present(bias)) check_operand(who, "bias", *bias, x, {n});
  if (present(residual)) check_operand(who, "residual", *residual, x, {m, n});
  c10::DeviceGuard guard(x.device());
  const at::Tensor xc = packed(x), wc = packed(w), bc = packed(bias), rc = packed(residual);
  at::Tensor y = at::empty({m, n}, x.options()), z = keep_z ? at::empty({m, n}, x.options()) : at::empty({0}, x.options());
  GpuTimer timer(gpu_timing_enabled() ? "linear_forward" : "", 2.0 * double(m) * double(n) * double(k));
  TVK_MX(mx_linear_forward(cptr(xc), cptr(wc), cptr(bc), cptr(rc), m, k, n, act, ptr(y), keep_z ? ptr(z) : nullptr, nullptr,
                           0, current_stream()));
  launched();
  return {y, z};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_act_backward(const at::Tensor& dy, const at::Tensor& x,
                                                                   const at::Tensor& w, const OptT& z,
                                                                   c10::string_view activation, std::array<bool, 3> mask) {
  const char* const who = "linear_act_backward";
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2, who, ": x and weight must be matrices");
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  const int act = activation_code(activation);
  check_operand(who, "x", x, x, {m, k});
  check_operand(who, "weight", w, x, {n, k});
  check_operand(who, "dy", dy, x, {m, n});
  TORCH_CHECK(act == MX_ACT_NONE || present(z), who, ": an activation needs its input z");
  if (act != MX_ACT_NONE) check_operand(who, "z", *z, x, {m, n});
  c10::DeviceGuard guard(x.device());
  at::Tensor dx, dw, db;
  if (mask[0]) dx = at::empty({m, k}, x.options());
  if (mask[1]) dw = at::empty({n, k}, x.options());
  if (mask[2]) db = at::empty({n}, x.options());
  const at::Tensor dyc = packed(dy), xc = packed(x), wc = packed(w), zc = act != MX_ACT_NONE ? packed(z) : at::Tensor();
  GpuTimer timer(gpu_timing_enabled() ? "linear_backward" : "",
                 2.0 * double(m) * double(n) * double(k) * (int(mask[0]) + int(mask[1])));
  TVK_MX(mx_linear_backward(cptr(dyc), cptr(xc), cptr(wc), cptr(zc), m, k, n, act, ptr(dx), ptr(dw), ptr(db), nullptr, 0,
                            current_stream()));
  launched();
  return {dx, dw, db};
}

// ---------------------------------------------- orthogonalised momentum step
mx_newton_schulz newton_schulz(at::ArrayRef<double> coefficients, int64_t steps, double eps) {
  TORCH_CHECK(coefficients.size() == 3, "orthogonalize: three coefficients expected, got ", coefficients.size());
  return {steps, coefficients[0], coefficients[1], coefficients[2], eps};
}

void check_matrix(const char* who, const char* what, size_t i, const at::Tensor& t, const at::Tensor& like) {
  TORCH_CHECK(f32_dev(t) && t.dim() == 2, who, ": ", what, " ", i, " must be a float32 vulkan matrix");
  TORCH_CHECK(t.device() == like.device(), who, ": tensors on different devices");
  TORCH_CHECK(t.sizes() == like.sizes(), who, ": incompatible tensor shapes at ", i);
}

std::vector<at::Tensor> orthogonalize(at::TensorList inputs, at::ArrayRef<double> coefficients, int64_t steps, double eps) {
  const char* const who = "orthogonalize";
  const mx_newton_schulz ns = newton_schulz(coefficients, steps, eps);
  std::vector<at::Tensor> in, out;
  std::vector<mx_matrix_pair> tab;
  if (inputs.empty()) return out;
  c10::DeviceGuard guard(inputs[0].device());
  for (size_t i = 0; i < inputs.size(); ++i) {
    check_matrix(who, "input", i, inputs[i], inputs[i]);
    TORCH_CHECK(inputs[i].device() == inputs[0].device(), who, ": tensors on different devices");
    in.push_back(packed(inputs[i]));
    out.push_back(at::empty(inputs[i].sizes(), inputs[i].options().memory_format(at::MemoryFormat::Contiguous)));
    tab.push_back({cptr(in.back()), ptr(out.back()), in.back().size(0), in.back().size(1)});
  }
  GpuTimer timer(gpu_timing_enabled() ? "orthogonalize" : "");
  TVK_MX(mx_orthogonalize(tab.data(), int64_t(tab.size()), &ns, nullptr, 0, current_stream()));
  launched();
  return out;
}

void muon_step_(at::TensorList params, at::TensorList grads, at::TensorList momentum_buffers, double lr, double weight_decay,
                double momentum, bool nesterov, at::ArrayRef<double> coefficients, int64_t steps, double eps,
                c10::string_view adjust_lr) {
  const char* const who = "muon_step_";
  const size_t count = params.size();
  TORCH_CHECK(grads.size() == count && momentum_buffers.size() == count,
              "muon_step_: parameter, gradient and momentum lists must match");
  mx_muon_hparams hp{};
  hp.lr = lr;
  hp.weight_decay = weight_decay;
  hp.momentum = momentum;
  hp.nesterov = nesterov;
  hp.ns = newton_schulz(coefficients, steps, eps);
  TORCH_CHECK(adjust_lr == "original" || adjust_lr == "match_rms_adamw",
              "muon_step_: adjust_lr must be original or match_rms_adamw, got ", std::string(adjust_lr));
  hp.adjust_lr = adjust_lr == "original" ? MX_MUON_ORIGINAL : MX_MUON_MATCH_RMS_ADAMW;
  if (count == 0) return;
  c10::DeviceGuard guard(params[0].device());
  std::vector<at::Tensor> held;
  std::vector<mx_muon_tensor> tab;
  for (size_t i = 0; i < count; ++i) {
    const at::Tensor &p = params[i], &m = momentum_buffers[i];
    check_matrix(who, "param", i, p, p);
    TORCH_CHECK(p.device() == params[0].device(), who, ": tensors on different devices");
    check_matrix(who, "grad", i, grads[i], p);
    check_matrix(who, "momentum buffer", i, m, p);
    TORCH_CHECK(p.is_contiguous() && m.is_contiguous(), who, ": parameters and momentum buffers must be contiguous (", i, ")");
    held.push_back(packed(grads[i]));
    if (p.numel() == 0) continue;
    tab.push_back({ptr(p), cptr(held.back()), ptr(m), p.size(0), p.size(1)});
  }
  GpuTimer timer(gpu_timing_enabled() ? "muon_step" : "");
  TVK_MX(mx_muon_step(tab.data(), int64_t(tab.size()), &hp, nullptr, 0, current_stream()));
  launched();
}

}  // namespace
}  // namespace tvk

TORCH_LIBRARY_FRAGMENT(torch_vulkan, m) {
  m.def(
      "linear_act(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation, bool keep_z) -> (Tensor, "
      "Tensor)");
  m.def(
      "linear_act_backward(Tensor dy, Tensor x, Tensor weight, Tensor? z, str activation, bool[3] mask) -> (Tensor, "
      "Tensor, Tensor)");
  m.def("orthogonalize(Tensor[] inputs, float[] coefficients, int steps, float eps) -> Tensor[]");
  m.def(
      "muon_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momentum_buffers, float lr, float weight_decay, "
      "float momentum, bool nesterov, float[] coefficients, int steps, float eps, str adjust_lr) -> ()");
}

TORCH_LIBRARY_IMPL(torch_vulkan, PrivateUse1, m) {
  m.impl("linear_act", TORCH_FN(tvk::linear_act));
  m.impl("linear_act_backward", TORCH_FN(tvk::linear_act_backward));
  m.impl("orthogonalize", TORCH_FN(tvk::orthogonalize));
  m.impl("muon_step_", TORCH_FN(tvk::muon_step_));
}

TORCH_LIBRARY_IMPL(aten, PrivateUse1, m) {
  m.impl("native_layer_norm", TORCH_FN(tvk::native_layer_norm_vk));
  m.impl("native_layer_norm_backward", TORCH_FN(tvk::native_layer_norm_backward_vk));
}
