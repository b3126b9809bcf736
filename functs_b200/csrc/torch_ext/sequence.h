// Calls of the sequence operators on the host side (sequence.cpp): checks, allocation, launch.  Shared by the Python entry points and by
// the region operator.
#pragma once

#include <ATen/ATen.h>

#include <optional>
#include <tuple>

namespace functs_b200 {

using MaybeTensor = std::optional<at::Tensor>;

// Whether a forward derivative is asked of what is made of `t`; whether any is, or a transform (torch.func) is on its way through.
bool carriesTangent(const at::Tensor& t);
bool wantsDerivative(const at::Tensor& t);

// q [B, T, H, Dk], k [B, T, Hk, Dk], v [B, T, Hk, Dv] -> (out [B, T, H, Dv], the states)
std::tuple<at::Tensor, at::Tensor> linearAttention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                                                   double scale, const MaybeTensor& state, const MaybeTensor& slots,
                                                   const MaybeTensor& lengths, const MaybeTensor& out, const MaybeTensor& status);
// q [B, H, Dk], k [B, Hk, Dk], v [B, Hk, Dv] -> out [B, H, Dv]
at::Tensor linearAttentionStep(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& log_decay,
                               const at::Tensor& state, double scale, const MaybeTensor& slots, const MaybeTensor& out,
                               const MaybeTensor& status);
// logits [R, V], tokens [R] -> (logprobs [R], entropy [R], top_logprobs [R, top], top_ids [R, top])
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> tokenLogprobs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top,
                                                                         const MaybeTensor& status);

}  // namespace functs_b200
