// Kernel entry points of the sequence operators.
#pragma once

#include <ATen/ATen.h>

#include <array>
#include <vector>

namespace tgcm {

using OptTensor = c10::optional<at::Tensor>;

// t itself where its rows can be read as they are, else a copy with rows padded by zeros to 16 bytes
at::Tensor gated_rows(const at::Tensor& t);
at::Tensor gated_fwd(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const OptTensor& bg,
                     const OptTensor& bu, int64_t act, const OptTensor& err);
// dx, dWg, dWu, dbg, dbu; the ones not asked for are undefined.  x and the weights as gated_rows left them
std::vector<at::Tensor> gated_bwd(const at::Tensor& dh, const at::Tensor& x, const at::Tensor& wg,
                                  const at::Tensor& wu, const OptTensor& bg, const OptTensor& bu, int64_t act,
                                  int64_t features, bool need_x, bool need_w, bool need_b, const OptTensor& err);

std::vector<at::Tensor> qk_norm_rotary_fwd(const at::Tensor& q, const at::Tensor& k, const OptTensor& table,
                                           const OptTensor& positions, const OptTensor& qw, const OptTensor& kw,
                                           const OptTensor& qb, const OptTensor& kb, int64_t norm, bool interleaved,
                                           double eps, const OptTensor& err);
// dq, dk, dq_weight, dk_weight, dq_bias, dk_bias; of the last four those that `need` names
std::vector<at::Tensor> qk_norm_rotary_bwd(const at::Tensor& dyq, const at::Tensor& dyk, const at::Tensor& q,
                                           const at::Tensor& k, const OptTensor& table, const OptTensor& positions,
                                           const OptTensor& qw, const OptTensor& kw, int64_t norm, bool interleaved,
                                           double eps, std::array<bool, 4> need, const OptTensor& err);

// o, lse and, for a backward pass, what o's rounding left over (undefined in fp32 or without `train`)
std::vector<at::Tensor> window_attention_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                             int64_t window, int64_t sinks, bool causal, const OptTensor& lengths,
                                             double scale, bool train, const OptTensor& err);
// dq, dk, dv
std::vector<at::Tensor> window_attention_bwd(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
                                             const at::Tensor& v, const at::Tensor& o, const at::Tensor& o_rest,
                                             const at::Tensor& lse, int64_t window, int64_t sinks, bool causal, const OptTensor& lengths,
                                             double scale, const OptTensor& err);

// changes the caches in place; no backward pass
at::Tensor window_attention_step(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache,
                                 at::Tensor& v_cache, const at::Tensor& lengths, int64_t sinks, double scale);

// the norm; clips into `out`, or in place where that is empty; no backward pass
at::Tensor clip_grad_norm(at::TensorList grads, at::TensorList out, double max_norm);

}  // namespace tgcm
