// Operators of a transformer block over feature rows: layer norm, dropout,
// rotary positions, windowed attention and the junction of two parts, with
// their gradients, and an 8-bit cache that is written, read and attended to.
#pragma once

#include <torch/extension.h>

#include <array>
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

// weight, bias, gate, post weight and post bias of a junction.
typedef std::array<c10::optional<at::Tensor>, 5> JoinVectors;
// (sum, normed, statistics); statistics is undefined (None) unless kept for the
// gradient.
std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_norm(const at::Tensor& x, const at::Tensor& residual,
                                                             const JoinVectors& vectors, double scale, bool post_norm,
                                                             bool rms, double eps,
                                                             const c10::optional<at::Tensor>& active_rows,
                                                             bool keep_statistics);
// The gradients of x, residual and the vectors; a vector's is undefined (None)
// unless wanted.  x is read with post_norm or where the gate's gradient is
// wanted, and may be undefined otherwise; so may the bias, and the post bias
// where the gate's gradient is not wanted.
std::vector<at::Tensor> residual_norm_grad(const c10::optional<at::Tensor>& grad_sum,
                                           const c10::optional<at::Tensor>& grad_normed, const at::Tensor& sum,
                                           const at::Tensor& statistics, const c10::optional<at::Tensor>& x,
                                           const JoinVectors& vectors, double scale, bool post_norm, bool rms,
                                           double eps, const c10::optional<at::Tensor>& active_rows,
                                           const std::array<bool, 5>& wanted);

// keys, values, key exponents and value exponents of a cache.
typedef std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> CacheParts;
void cache_write(const CacheParts& parts, int64_t dim, const at::Tensor& k, const at::Tensor& v,
                 const at::Tensor& offsets, const at::Tensor& lengths);
// (k, v).
std::tuple<at::Tensor, at::Tensor> cache_read(const CacheParts& parts, int64_t dim, const at::Tensor& lengths,
                                              at::ScalarType type);
at::Tensor cache_attention(const at::Tensor& q, const CacheParts& parts, int64_t dim, const at::Tensor& offsets,
                           const at::Tensor& lengths, int64_t left, int64_t right, int64_t sinks, double scale);

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
std::tuple<at::Tensor, at::Tensor> residual_norm_node(const at::Tensor& x, const at::Tensor& residual,
                                                      const JoinVectors& vectors, double scale, bool post_norm,
                                                      bool rms, double eps,
                                                      const c10::optional<at::Tensor>& active_rows);

}  // namespace lattice_native
