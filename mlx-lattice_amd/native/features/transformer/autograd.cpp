// The differentiable forms of the transformer operators: nodes of torch's
// graph that run their gradients without the interpreter.

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>
#include <utility>
#include <vector>

#include "features/transformer/api.h"

namespace lattice_native {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

typedef c10::optional<at::Tensor> MaybeTensor;

at::Tensor or_undefined(const MaybeTensor& t) { return t ? *t : at::Tensor(); }
MaybeTensor or_none(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : c10::nullopt; }
bool wants_grad(const MaybeTensor& t) { return t && t->defined() && t->requires_grad(); }

// The gradients are made outside the graph: where it is being built, they say
// so when they are differentiated, in place of passing for constants.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    std::vector<size_t> places;
    variable_list defined;
    for (size_t i = 0; i < grads.size(); ++i) {
        if (!grads[i].defined()) continue;
        places.push_back(i);
        defined.push_back(grads[i].detach().requires_grad_());
    }
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "the transformer operators can be differentiated once.", static_cast<int64_t>(defined.size()));
    defined = (*error)(std::move(defined));
    for (size_t i = 0; i < places.size(); ++i) grads[places[i]] = defined[i];
    return grads;
}

struct LayerNorm : Function<LayerNorm> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& weight,
                              const MaybeTensor& bias, double eps, const MaybeTensor& active_rows) {
        auto [y, statistics] = layer_norm(x, weight, bias, eps, active_rows, true);
        ctx->save_for_backward({x, or_undefined(weight), statistics, or_undefined(active_rows)});
        ctx->saved_data["weight"] = wants_grad(weight);
        ctx->saved_data["bias"] = wants_grad(bias);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const bool weight = ctx->saved_data["weight"].toBool(), bias = ctx->saved_data["bias"].toBool();
        auto [dx, dw, db] = layer_norm_grad(grads[0], saved[0], or_none(saved[1]), saved[2], or_none(saved[3]),
                                            weight, bias);
        return once({dx, weight ? dw : at::Tensor(), bias ? db : at::Tensor(), {}, {}});
    }
};

struct Dropout : Function<Dropout> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const MaybeTensor& residual, int64_t seed,
                              int64_t offset, int64_t threshold, double scale) {
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["threshold"] = threshold;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["x"] = wants_grad(x);
        ctx->saved_data["residual"] = wants_grad(residual);
        return dropout(x, residual, static_cast<uint64_t>(seed), static_cast<uint64_t>(offset),
                       static_cast<uint64_t>(threshold), scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        auto& data = ctx->saved_data;
        at::Tensor dx;
        if (data["x"].toBool())
            dx = once({dropout(grads[0], c10::nullopt, static_cast<uint64_t>(data["seed"].toInt()),
                               static_cast<uint64_t>(data["offset"].toInt()),
                               static_cast<uint64_t>(data["threshold"].toInt()), data["scale"].toDouble())})[0];
        return {dx, data["residual"].toBool() ? grads[0] : at::Tensor(), {}, {}, {}, {}};
    }
};

struct RotaryPositions : Function<RotaryPositions> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& positions,
                              const at::Tensor& frequencies, const std::vector<int64_t>& dims, bool interleaved) {
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["dims"] = dims;
        ctx->saved_data["interleaved"] = interleaved;
        return rotary_positions(x, positions, frequencies, {dims.begin(), dims.end()}, interleaved, false);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const std::vector<int64_t> dims = ctx->saved_data["dims"].toIntVector();
        return once({rotary_positions(grads[0], saved[0], saved[1], {dims.begin(), dims.end()},
                                      ctx->saved_data["interleaved"].toBool(), true),
                     {}, {}, {}, {}});
    }
};

struct WindowAttention : Function<WindowAttention> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const at::Tensor& offsets, const at::Tensor& key_offsets, const MaybeTensor& key_lengths,
                              int64_t left, int64_t right, int64_t sinks, double scale) {
        auto [out, lse, rest] = window_attention(q, k, v, offsets, key_offsets, key_lengths, left, right, sinks, scale,
                                           true);
        ctx->save_for_backward({q, k, v, out, lse, offsets, key_offsets, or_undefined(key_lengths), rest});
        ctx->saved_data["left"] = left;
        ctx->saved_data["right"] = right;
        ctx->saved_data["sinks"] = sinks;
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        auto& data = ctx->saved_data;
        auto [dq, dk, dv] = window_attention_grad(grads[0], saved[3], saved[4], or_none(saved[8]), saved[0], saved[1],
                                                  saved[2], saved[5], saved[6], or_none(saved[7]), data["left"].toInt(),
                                                  data["right"].toInt(), data["sinks"].toInt(),
                                                  data["scale"].toDouble());
        return once({dq, dk, dv, {}, {}, {}, {}, {}, {}, {}});
    }
};

struct ResidualNorm : Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& residual,
                                 const MaybeTensor& weight, const MaybeTensor& bias, const MaybeTensor& gate,
                                 const MaybeTensor& post_weight, const MaybeTensor& post_bias, double scale,
                                 bool post_norm, bool rms, double eps, const MaybeTensor& active_rows) {
        const JoinVectors vectors{weight, bias, gate, post_weight, post_bias};
        auto [sum, normed, statistics] = residual_norm(x, residual, vectors, scale, post_norm, rms, eps, active_rows,
                                                       true);
        std::vector<bool> wanted;
        for (const MaybeTensor& v : vectors) wanted.push_back(wants_grad(v));
        // What the gradients read: neither the residual nor the bias.
        ctx->save_for_backward({post_norm || wanted[2] ? x : at::Tensor(), sum, statistics, or_undefined(active_rows),
                                or_undefined(weight), or_undefined(gate), or_undefined(post_weight),
                                wanted[2] ? or_undefined(post_bias) : at::Tensor()});
        ctx->saved_data["wanted"] = c10::List<bool>({wanted[0], wanted[1], wanted[2], wanted[3], wanted[4]});
        ctx->saved_data["x"] = wants_grad(x);
        ctx->saved_data["residual"] = wants_grad(residual);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["post_norm"] = post_norm;
        ctx->saved_data["rms"] = rms;
        ctx->saved_data["eps"] = eps;
        ctx->set_materialize_grads(false);
        return {sum, normed};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list out(12);
        if (!grads[0].defined() && !grads[1].defined()) return out;
        const auto saved = ctx->get_saved_variables();
        auto& data = ctx->saved_data;
        const JoinVectors vectors{or_none(saved[4]), c10::nullopt, or_none(saved[5]), or_none(saved[6]),
                                  or_none(saved[7])};
        const auto list = data["wanted"].toBoolList();
        std::array<bool, 5> wanted;
        for (int i = 0; i < 5; ++i) wanted[i] = list.get(i);
        variable_list made = residual_norm_grad(
            or_none(grads[0]), or_none(grads[1]), saved[1], saved[2], or_none(saved[0]), vectors,
            data["scale"].toDouble(), data["post_norm"].toBool(), data["rms"].toBool(), data["eps"].toDouble(),
            or_none(saved[3]), wanted);
        if (!data["x"].toBool()) made[0] = at::Tensor();
        if (!data["residual"].toBool()) made[1] = at::Tensor();
        made = once(std::move(made));
        for (int i = 0; i < 7; ++i) out[i] = made[i];
        return out;
    }
};

}  // namespace

at::Tensor layer_norm_node(const at::Tensor& x, const c10::optional<at::Tensor>& weight,
                           const c10::optional<at::Tensor>& bias, double eps,
                           const c10::optional<at::Tensor>& active_rows) {
    return LayerNorm::apply(x, weight, bias, eps, active_rows);
}

at::Tensor dropout_node(const at::Tensor& x, const c10::optional<at::Tensor>& residual, uint64_t seed,
                        uint64_t offset, uint64_t threshold, double scale) {
    return Dropout::apply(x, residual, static_cast<int64_t>(seed), static_cast<int64_t>(offset),
                          static_cast<int64_t>(threshold), scale);
}

at::Tensor rotary_positions_node(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& frequencies,
                                 const std::vector<int>& dims, bool interleaved) {
    return RotaryPositions::apply(x, positions, frequencies, std::vector<int64_t>(dims.begin(), dims.end()),
                                  interleaved);
}

at::Tensor window_attention_node(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                 const at::Tensor& offsets, const at::Tensor& key_offsets,
                                 const c10::optional<at::Tensor>& key_lengths, int64_t left, int64_t right,
                                 int64_t sinks, double scale) {
    return WindowAttention::apply(q, k, v, offsets, key_offsets, key_lengths, left, right, sinks, scale);
}

std::tuple<at::Tensor, at::Tensor> residual_norm_node(const at::Tensor& x, const at::Tensor& residual,
                                                      const JoinVectors& vectors, double scale, bool post_norm,
                                                      bool rms, double eps,
                                                      const c10::optional<at::Tensor>& active_rows) {
    const variable_list out = ResidualNorm::apply(x, residual, vectors[0], vectors[1], vectors[2], vectors[3],
                                                  vectors[4], scale, post_norm, rms, eps, active_rows);
    return {out[0], out[1]};
}

}  // namespace lattice_native
