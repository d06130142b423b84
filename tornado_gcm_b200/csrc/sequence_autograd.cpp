// torch.ops.tgcm.{gated_linear, qk_norm_rotary, window_attention}: the kernels'
// forward passes with their backward passes attached.  The graph nodes are
// native: a training step over short sequences is bound by the host, and a
// node in Python costs several times what these kernels take.  The one-token step
// has none and says so where one is wanted; so do all of them for forward-mode and
// second derivatives.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <cstring>

#include "sequence_ops.h"

namespace tgcm {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool wants(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor& t) { return t.has_value() && wants(*t); }
at::Tensor undef_or(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

bool dual(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool dual(const OptTensor& t) { return t.has_value() && dual(*t); }
template <class... T>
void refuse_forward_mode(const char* name, const T&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(dual(inputs) || ...), name, ": no forward-mode derivative");
}

// A graph that has saved t finds that it has changed since.
void written(const at::Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

// A node's gradients under create_graph: they have no history, so one that says so takes its place.  `of`: the
// node's inputs and the upstream gradients, on which the gradients depend.
variable_list first_only(variable_list grads, const variable_list& of, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  auto node = std::shared_ptr<torch::autograd::Error>(
      new torch::autograd::Error(std::string(name) + ": no second derivative", torch::autograd::collect_next_edges(of)),
      torch::autograd::deleteNode);
  for (auto& g : grads)
    if (g.defined()) {
      g = g.detach();
      torch::autograd::set_history(g, node);
    }
  return grads;
}

// The upstream gradient in the result's type with a contiguous last axis.
at::Tensor rows_like(const at::Tensor& g, const at::Tensor& like) {
  if (!g.defined()) return at::zeros_like(like);
  at::Tensor r = g.scalar_type() == like.scalar_type() ? g : g.to(like.scalar_type());
  return r.size(-1) == 1 || r.stride(-1) == 1 ? r : r.contiguous();
}

// What a node keeps beside its tensors: the numbers in one entry (an entry for each would cost
// more than a kernel's launch), and the error flag (not a saved variable: it is cleared between passes).
int64_t bits_of(double x) {
  int64_t b;
  std::memcpy(&b, &x, sizeof(b));
  return b;
}
double double_of(int64_t b) {
  double x;
  std::memcpy(&x, &b, sizeof(x));
  return x;
}
void keep(AutogradContext* ctx, std::vector<int64_t> v, const OptTensor& err) {
  ctx->saved_data["cfg"] = std::move(v);
  ctx->saved_data["err"] = err;
}
OptTensor flag_of(AutogradContext* ctx) { return ctx->saved_data["err"].toOptional<at::Tensor>(); }
std::vector<int64_t> kept(AutogradContext* ctx) { return ctx->saved_data["cfg"].toIntVector(); }

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu,
                            const OptTensor& bg, const OptTensor& bu, int64_t act, const OptTensor& err) {
    // rows that had to be padded are padded once for both passes
    const at::Tensor xr = gated_rows(x), wgr = gated_rows(wg), wur = gated_rows(wu);
    ctx->save_for_backward({xr, wgr, wur, undef_or(bg), undef_or(bu)});
    keep(ctx, {act, x.size(1), wants(x), wants(wg) || wants(wu), wants(bg) || wants(bu)}, err);
    return gated_fwd(xr, wgr, wur, bg, bu, act, err);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(7);
    const auto c = kept(ctx);
    const at::Tensor dh = g[0].scalar_type() == at::kBFloat16 ? g[0] : g[0].to(at::kBFloat16);
    auto r = gated_bwd(dh.size(1) == 1 || dh.stride(1) == 1 ? dh : dh.contiguous(), s[0], s[1], s[2], opt(s[3]),
                       opt(s[4]), c[0], c[1], c[2], c[3], c[4], flag_of(ctx));
    return first_only({r[0], r[1], r[2], s[3].defined() ? r[3] : at::Tensor(), s[4].defined() ? r[4] : at::Tensor(),
                       at::Tensor(), at::Tensor()},
                      {g[0], s[0], s[1], s[2], s[3], s[4]}, "gated_linear");
  }
};

struct QKNormRotary : torch::autograd::Function<QKNormRotary> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const OptTensor& table,
                               const OptTensor& positions, const OptTensor& qw, const OptTensor& kw,
                               const OptTensor& qb, const OptTensor& kb, int64_t norm, bool interleaved, double eps,
                               const OptTensor& err) {
    ctx->save_for_backward({q, k, undef_or(table), undef_or(positions), undef_or(qw), undef_or(kw)});
    keep(ctx, {norm, interleaved, bits_of(eps), wants(qw), wants(kw), wants(qb), wants(kb)}, err);
    return qk_norm_rotary_fwd(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    const auto c = kept(ctx);
    auto r = qk_norm_rotary_bwd(rows_like(g[0], s[0]), rows_like(g[1], s[1]), s[0], s[1], opt(s[2]), opt(s[3]),
                                opt(s[4]), opt(s[5]), c[0], c[1], double_of(c[2]),
                                {c[3] != 0, c[4] != 0, c[5] != 0, c[6] != 0}, flag_of(ctx));
    variable_list out(12);
    out[0] = r[0], out[1] = r[1];
    for (int i = 0; i < 4; ++i) out[4 + i] = r[2 + i];
    return first_only(std::move(out), {g[0], g[1], s[0], s[1], s[4], s[5]}, "qk_norm_rotary");
  }
};

struct WindowAttention : torch::autograd::Function<WindowAttention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            int64_t window, int64_t sinks, bool causal, const OptTensor& lengths, double scale,
                            const OptTensor& err) {
    auto r = window_attention_fwd(q, k, v, window, sinks, causal, lengths, scale, true, err);
    ctx->save_for_backward({q, k, v, r[0], r[1], undef_or(lengths), r[2]});
    keep(ctx, {window, sinks, causal, bits_of(scale)}, err);
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto s = ctx->get_saved_variables();
    if (!g[0].defined()) return variable_list(9);
    const auto c = kept(ctx);
    auto r = window_attention_bwd(rows_like(g[0], s[3]), s[0], s[1], s[2], s[3], s[6], s[4], c[0], c[1], c[2],
                                  opt(s[5]), double_of(c[3]), flag_of(ctx));
    variable_list out(9);
    for (int i = 0; i < 3; ++i) out[i] = r[i];
    return first_only(std::move(out), {g[0], s[0], s[1], s[2]}, "window_attention");
  }
};

at::Tensor gated_linear(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const OptTensor& bg,
                        const OptTensor& bu, int64_t act, const OptTensor& err) {
  return gated_fwd(x, wg, wu, bg, bu, act, err);
}
at::Tensor gated_linear_autograd(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const OptTensor& bg,
                                 const OptTensor& bu, int64_t act, const OptTensor& err) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && wg.dim() == 2 && wg.sizes() == wu.sizes() && x.size(-1) == wg.size(1),
                    "gated_linear: x (..., features) and two weights (hidden, features) expected");
  TORCH_CHECK_VALUE(bg.has_value() == bu.has_value(), "gated_linear: both biases or none");
  refuse_forward_mode("gated_linear", x, wg, wu, bg, bu);
  // Other types are rounded to bf16 here, above autograd, so that gradients come back in the caller's type.
  auto bf = [](const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? t : t.to(at::kBFloat16); };
  auto bf_opt = [&](const OptTensor& t) { return t.has_value() ? OptTensor(bf(*t)) : t; };
  const bool flat = x.dim() == 2;
  const at::Tensor x2 = flat ? bf(x) : bf(x).reshape({-1, x.size(-1)});
  const at::Tensor wg2 = bf(wg), wu2 = bf(wu);
  const OptTensor bg2 = bf_opt(bg), bu2 = bf_opt(bu);
  at::Tensor h;
  if (at::GradMode::is_enabled() && (wants(x2) || wants(wg2) || wants(wu2) || wants(bg2) || wants(bu2))) {
    h = GatedLinear::apply(x2, wg2, wu2, bg2, bu2, act, err);
  } else {
    at::AutoDispatchBelowADInplaceOrView below;
    h = gated_fwd(x2, wg2, wu2, bg2, bu2, act, err);
  }
  if (flat) return h;
  auto sizes = x.sizes().vec();
  sizes.back() = h.size(1);
  return h.reshape(sizes);
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
  refuse_forward_mode("qk_norm_rotary", q, k, table, qw, kw, qb, kb);
  TORCH_CHECK(!at::GradMode::is_enabled() || !wants(table), "qk_norm_rotary: no gradient for the table");
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(qw) || wants(kw) || wants(qb) || wants(kb))) {
    auto r = QKNormRotary::apply(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return qk_norm_rotary(q, k, table, positions, qw, kw, qb, kb, norm, interleaved, eps, err);
}

at::Tensor window_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                            int64_t sinks, bool causal, const OptTensor& lengths, double scale, const OptTensor& err) {
  return window_attention_fwd(q, k, v, window, sinks, causal, lengths, scale, false, err)[0];
}
at::Tensor window_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t window,
                                     int64_t sinks, bool causal, const OptTensor& lengths, double scale,
                                     const OptTensor& err) {
  refuse_forward_mode("window_attention", q, k, v);
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v)))
    return WindowAttention::apply(q, k, v, window, sinks, causal, lengths, scale, err);
  at::AutoDispatchBelowADInplaceOrView below;
  return window_attention(q, k, v, window, sinks, causal, lengths, scale, err);
}

at::Tensor window_attention_step_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                          at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& lengths,
                                          int64_t sinks, double scale) {
  TORCH_CHECK(!at::GradMode::is_enabled() ||
                  !(wants(q) || wants(k) || wants(v) || wants(k_cache) || wants(v_cache)),
              "window_attention_step: no gradient; call it under torch.no_grad()");
  refuse_forward_mode("window_attention_step", q, k, v, k_cache, v_cache);
  at::Tensor o;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    o = window_attention_step(q, k, v, k_cache, v_cache, lengths, sinks, scale);
  }
  written(k_cache);
  written(v_cache);
  return o;
}

at::Tensor clip_grad_norm_autograd(at::TensorList grads, at::TensorList out, double max_norm) {
  at::Tensor norm;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    norm = clip_grad_norm(grads, out, max_norm);
  }
  for (const auto& t : out.empty() ? grads : out) written(t);
  return norm;
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
  m.impl("window_attention_step", &tgcm::window_attention_step_autograd);
  m.impl("clip_grad_norm", &tgcm::clip_grad_norm_autograd);
}
