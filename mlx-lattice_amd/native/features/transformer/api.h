// Operators of a transformer block over feature rows: layer norm, dropout,
// rotary positions and windowed attention, with their gradients.
#pragma once

#include <torch/extension.h>

#include <cstdint>
#include <tuple>
#include <vector>

namespace lattice_native {

// (y, statistics); statistics is undefined (None) unless kept for the gradient.
std::tuple<at::Tensor, at::Tensor> layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                                              const c10::optional<at::Tensor>& bias, double eps,
                                              const c10::optional<at::Tensor>& active_rows, bool keep_statistics);
// (grad_x, grad_weight, grad_bias); the last two are undefined (None) unless
// asked for.
std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_grad(const at::Tensor& grad_y, const at::Tensor& x,
                                                               const c10::optional<at::Tensor>& weight,
                                                               const at::Tensor& statistics,
                                                               const c10::optional<at::Tensor>& active_rows,
                                                               bool grad_weight, bool grad_bias);

at::Tensor dropout(const at::Tensor& x, const c10::optional<at::Tensor>& residual, uint64_t seed, uint64_t offset,
                   uint64_t threshold, double scale);

at::Tensor rotary_positions(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& frequencies,
                            const std::vector<int>& dims, bool interleaved, bool inverse);

// (out, lse, rest); the last two are undefined (None) unless kept for the
// gradient, rest (what rounding took from out) in float32 too.
std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
    const at::Tensor& key_offsets, const c10::optional<at::Tensor>& key_lengths, int64_t left, int64_t right,
    int64_t sinks, double scale, bool keep);
// (grad_q, grad_k, grad_v).
std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention_grad(
    const at::Tensor& grad_out, const at::Tensor& out, const at::Tensor& lse, const c10::optional<at::Tensor>& rest,
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
    const at::Tensor& key_offsets, const c10::optional<at::Tensor>& key_lengths, int64_t left, int64_t right,
    int64_t sinks, double scale);

// The same operators as differentiable nodes of torch's graph.
at::Tensor layer_norm_node(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                           const c10::optional<at::Tensor>& bias, double eps,
                           const c10::optional<at::Tensor>& active_rows);
at::Tensor dropout_node(const at::Tensor& x, const c10::optional<at::Tensor>& residual, uint64_t seed,
                        uint64_t offset, uint64_t threshold, double scale);
at::Tensor rotary_positions_node(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& frequencies,
                                 const std::vector<int>& dims, bool interleaved);
at::Tensor window_attention_node(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 const at::Tensor& offsets, const at::Tensor& key_offsets,
                                 const c10::optional<at::Tensor>& key_lengths, int64_t left, int64_t right,
                                 int64_t sinks, double scale);

}  // namespace lattice_native
