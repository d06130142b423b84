// torch.ops.tgcm.{gated_linear, qk_norm_rotary, window_attention}: the kernels'
// forward passes with their backward passes attached.  The graph nodes are
// native: a training step over short sequences is bound by the host, and a
// node in Python costs several times what these kernels take.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "sequence_ops.h"

namespace tgcm {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor& t) { return t.has_value() && wants(*t); }
at::Tensor undef_or(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// The upstream gradient in the result's type with a contiguous last axis.
at::Tensor rows_like(const at::Tensor& g, const at::Tensor& like) {
  if (!g.defined()) return at::zeros_like(like);
  at::Tensor r = g.scalar_type() == like.scalar_type() ? g : g.to(like.scalar_type());
  return r.size(-1) == 1 || r.stride(-1) == 1 ? r : r.contiguous();
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                            const OptTensor& bg, const OptTensor& bu, int64_t act, const OptTensor& err) {
    ctx->save_for_backward({x, wg, wu, undef_or(bg), undef_or(bu)});
    ctx->saved_data["act"] = act;
    ctx->saved_data["err"] = err;
    ctx->saved_data["x"] = wants(x);
    ctx->saved_data["w"] = wants(wg) || wants(wu);
    ctx->saved_data["b"] = wants(bg) || wants(bu);
    return gated_fwd(x, wg, wu, bg, bu, act, err);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(7);
    auto& d = ctx->saved_data;
    const at::Tensor dh = g[0].scalar_type() == at::kBFloat16 ? g[0] : g[0].to(at::kBFloat16);
    auto r = gated_bwd(dh.size(1) == 1 || dh.stride(1) == 1 ? dh : dh.contiguous(), s[0], s[1], s[2], opt(s[3]),
                       opt(s[4]), d["act"].toInt(), d["x"].toBool(), d["w"].toBool(), d["b"].toBool(),
                       d["err"].toOptional<at::Tensor>());
    return {r[0], r[1], r[2], s[3].defined() ? r[3] : at::Tensor(), s[4].defined() ? r[4] : at::Tensor(),
            at::Tensor(), at::Tensor()};
  }
};

struct QKNormRotary : torch::autograd::Function<QKNormRotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const OptTensor& table,
                               const OptTensor& positions, const OptTensor& qw, const OptTensor& kw,
                               const OptTensor& qb, const OptTensor& kb, int64_t norm, bool interleaved, double eps,
                               const OptTensor& err) {
    ctx->save_for_backward({q, k, undef_or(table), undef_or(positions), undef_or(qw), undef_or(kw)});
    auto& d = ctx->saved_data;
    d["norm"] = norm;
    d["inter"] = interleaved;
    d["eps"] = eps;
    d["err"] = err;
    d["qw"] = wants(qw);
    d["kw"] = wants(kw);
    d["qb"] = wants(qb);
    d["kb"] = wants(kb);
    return qk_norm_rotary_fwd(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    const bool qw = d["qw"].toBool(), kw = d["kw"].toBool(), qb = d["qb"].toBool(), kb = d["kb"].toBool();
    auto r = qk_norm_rotary_bwd(rows_like(g[0], s[0]), rows_like(g[1], s[1]), s[0], s[1], opt(s[2]), opt(s[3]),
                                opt(s[4]), opt(s[5]), d["norm"].toInt(), d["inter"].toBool(), d["eps"].toDouble(),
                                {qw, kw, qb, kb}, d["err"].toOptional<at::Tensor>());
    variable_list out(12);
    out[0] = r[0], out[1] = r[1];
    for (int i = 0; i < 4; ++i) out[4 + i] = r[2 + i];
    return out;
  }
};

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            int64_t window, int64_t sinks, bool causal, const OptTensor& lengths, double scale,
                            const OptTensor& err) {
    auto r = window_attention_fwd(q, k, v, window, sinks, causal, lengths, scale, err);
    ctx->save_for_backward({q, k, v, r[0], r[1], undef_or(lengths)});
    auto& d = ctx->saved_data;
    d["window"] = window;
    d["sinks"] = sinks;
    d["causal"] = causal;
    d["scale"] = scale;
    d["err"] = err;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(9);
    auto& d = ctx->saved_data;
    auto r = window_attention_bwd(rows_like(g[0], s[3]), s[0], s[1], s[2], s[3], s[4], d["window"].toInt(),
                                  d["sinks"].toInt(), d["causal"].toBool(), opt(s[5]), d["scale"].toDouble(),
                                  d["err"].toOptional<at::Tensor>());
    variable_list out(9);
    for (int i = 0; i < 3; ++i) out[i] = r[i];
    return out;
  }
};

at::Tensor gated_linear(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const OptTensor& bg,
                        const OptTensor& bu, int64_t act, const OptTensor& err) {
  return gated_fwd(x, wg, wu, bg, bu, act, err);
}
at::Tensor gated_linear_autograd(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const OptTensor& bg,
                                 const OptTensor& bu, int64_t act, const OptTensor& err) {
  if (at::GradMode::is_enabled() && (wants(x) || wants(wg) || wants(wu) || wants(bg) || wants(bu)))
    return GatedLinear::apply(x, wg, wu, bg, bu, act, err);
  at::AutoDispatchBelowADInplaceOrView below;
  return gated_fwd(x, wg, wu, bg, bu, act, err);
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rotary(const at::Tensor& q, const at::Tensor& k, const OptTensor& table,
                                                  const OptTensor& positions, const OptTensor& qw, const OptTensor& kw,
                                                  const OptTensor& qb, const OptTensor& kb, int64_t norm,
                                                  bool interleaved, double eps, const OptTensor& err) {
  auto r = qk_norm_rotary_fwd(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
  return {r[0], r[1]};
}
std::tuple<at::Tensor, at::Tensor> qk_norm_rotary_autograd(
    const at::Tensor& q, const at::Tensor& k, const OptTensor& table, const OptTensor& positions, const OptTensor& qw,
    const OptTensor& kw, const OptTensor& qb, const OptTensor& kb, int64_t norm, bool interleaved, double eps,
    const OptTensor& err) {
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(qw) || wants(kw) || wants(qb) || wants(kb))) {
    auto r = QKNormRotary::apply(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return qk_norm_rotary(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
}

at::Tensor window_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                            int64_t sinks, bool causal, const OptTensor& lengths, double scale, const OptTensor& err) {
  return window_attention_fwd(q, k, v, window, sinks, causal, lengths, scale, err)[0];
}
at::Tensor window_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                                     int64_t sinks, bool causal, const OptTensor& lengths, double scale,
                                     const OptTensor& err) {
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v)))
    return WindowAttention::apply(q, k, v, window, sinks, causal, lengths, scale, err);
  at::AutoDispatchBelowADInplaceOrView below;
  return window_attention(q, k, v, window, sinks, causal, lengths, scale, err);
}

}  // namespace
}  // namespace tgcm

TORCH_LIBRARY_FRAGMENT(tgcm, m) {
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, int act, Tensor? err) "
        "-> Tensor");
  m.def("qk_norm_rotary(Tensor q, Tensor k, Tensor? table, Tensor? positions, Tensor? q_weight, Tensor? k_weight, "
        "Tensor? q_bias, Tensor? k_bias, int norm, bool interleaved, float eps, Tensor? err) -> (Tensor, Tensor)");
  m.def("window_attention(Tensor q, Tensor k, Tensor v, int window, int sinks, bool causal, Tensor? lengths, "
        "float scale, Tensor? err) -> Tensor");
}

TORCH_LIBRARY_IMPL(tgcm, CUDA, m) {
  m.impl("gated_linear", &tgcm::gated_linear);
  m.impl("qk_norm_rotary", &tgcm::qk_norm_rotary);
  m.impl("window_attention", &tgcm::window_attention);
}

TORCH_LIBRARY_IMPL(tgcm, AutogradCUDA, m) {
  m.impl("gated_linear", &tgcm::gated_linear_autograd);
  m.impl("qk_norm_rotary", &tgcm::qk_norm_rotary_autograd);
  m.impl("window_attention", &tgcm::window_attention_autograd);
}
