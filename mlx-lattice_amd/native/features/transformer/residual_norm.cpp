#include <ATen/DeviceGuard.h>

#include <array>
#include <stdexcept>

#include "features/transformer/api.h"
#include "features/transformer/checks.h"

namespace lattice_native {

namespace {

struct Join {
    lattice_residual_norm args;
    at::Tensor x, residual;
    std::array<at::Tensor, 5> vectors;  // weight, bias, gate, post weight, post bias
};

Join join_of(const at::Tensor& x, const at::Tensor& residual, const JoinVectors& vectors, double scale, bool post_norm,
             bool rms, double eps, const c10::optional<at::Tensor>& active_rows) {
    if (x.dim() != 2 || x.size(1) < 1) throw std::invalid_argument("residual norm rows must have shape (N, C).");
    const int dtype = dtype_code(x, "residual norm rows");
    require_row_values(1, x.size(1), "residual norm rows");
    if (!(eps >= 0.0)) throw std::invalid_argument("eps must be non-negative.");
    require_device(x, "x");
    require_same(residual, x, "residual");
    if (residual.sizes() != x.sizes()) throw std::invalid_argument("residual must match the shape of x.");
    static constexpr const char* kNames[5] = {"weight", "bias", "gate", "post_weight", "post_bias"};
    Join j;
    for (int i = 0; i < 5; ++i) j.vectors[i] = channel_vector(vectors[i], x, kNames[i]);
    if (!post_norm && (j.vectors[3].defined() || j.vectors[4].defined())) {
        throw std::invalid_argument("post_weight and post_bias need post_norm.");
    }
    j.x = unit_rows(x);
    j.residual = unit_rows(residual);
    lattice_residual_norm& a = j.args;
    a.dtype = dtype;
    a.rows = row_count(x, "x");
    a.channels = static_cast<int>(x.size(1));
    a.rms = rms;
    a.post_norm = post_norm;
    a.scale = static_cast<float>(scale);
    a.eps = static_cast<float>(eps);
    a.x = j.x.data_ptr();
    a.residual = j.residual.data_ptr();
    a.x_stride = row_stride(j.x);
    a.residual_stride = row_stride(j.residual);
    a.weight = or_null(j.vectors[0]);
    a.bias = or_null(j.vectors[1]);
    a.gate = or_null(j.vectors[2]);
    a.post_weight = or_null(j.vectors[3]);
    a.post_bias = or_null(j.vectors[4]);
    a.active_rows = active_or_null(active_rows, x);
    return j;
}

c10::OptionalDeviceGuard guard_of(const at::Tensor& t) {
    return c10::OptionalDeviceGuard(t.is_cuda() ? c10::make_optional(t.device()) : c10::nullopt);
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor> residual_norm(const at::Tensor& x, const at::Tensor& residual,
                                                             const JoinVectors& vectors, double scale, bool post_norm,
                                                             bool rms, double eps,
                                                             const c10::optional<at::Tensor>& active_rows,
                                                             bool keep_statistics) {
    refuse_tangents({x, residual});
    for (const auto& v : vectors) refuse_tangents({or_undefined(v)});
    const auto guard = guard_of(x);
    const Join j = join_of(x, residual, vectors, scale, post_norm, rms, eps, active_rows);
    at::Tensor sum = at::empty(x.sizes(), x.options()), normed = at::empty(x.sizes(), x.options());
    at::Tensor statistics;
    if (keep_statistics) statistics = at::empty({x.size(0), 4}, x.options().dtype(at::kFloat));
    check_status(lattice_hip_residual_norm(&j.args, sum.data_ptr(), normed.data_ptr(),
                                           keep_statistics ? statistics.data_ptr<float>() : nullptr,
                                           current_stream(x)));
    return {sum, normed, statistics};
}

std::vector<at::Tensor> residual_norm_grad(const c10::optional<at::Tensor>& grad_sum_in,
                                           const c10::optional<at::Tensor>& grad_normed_in, const at::Tensor& sum,
                                           const at::Tensor& statistics, const c10::optional<at::Tensor>& x_in,
                                           const JoinVectors& vectors, double scale, bool post_norm, bool rms,
                                           double eps, const c10::optional<at::Tensor>& active_rows,
                                           const std::array<bool, 5>& wanted) {
    const bool reads_x = post_norm || wanted[2];
    if (reads_x && (!x_in || !x_in->defined())) {
        throw std::invalid_argument("x is needed by post_norm and by the gate's gradient.");
    }
    // The sum stands in for rows that are not read.
    const at::Tensor& x = reads_x ? *x_in : sum;
    refuse_tangents({x, or_undefined(grad_sum_in), or_undefined(grad_normed_in)});
    const auto guard = guard_of(x);
    require_same(sum, x, "sum");
    if (sum.sizes() != x.sizes() || !sum.is_contiguous()) {
        throw std::invalid_argument("sum must be that of the forward call.");
    }
    const Join j = join_of(x, sum, vectors, scale, post_norm, rms, eps, active_rows);
    at::Tensor cotangents[2];
    const c10::optional<at::Tensor>* given[2] = {&grad_sum_in, &grad_normed_in};
    for (int i = 0; i < 2; ++i) {
        if (!*given[i] || !(*given[i])->defined()) continue;
        require_same(**given[i], x, "the cotangent");
        if ((*given[i])->sizes() != x.sizes()) {
            throw std::invalid_argument("the cotangent must match the output shape.");
        }
        cotangents[i] = (*given[i])->contiguous();
    }
    if (statistics.dim() != 2 || statistics.size(0) != x.size(0) || statistics.size(1) != 4 ||
        statistics.scalar_type() != at::kFloat || !statistics.is_contiguous() || statistics.device() != x.device()) {
        throw std::invalid_argument("statistics must be those of the forward call.");
    }
    std::vector<at::Tensor> grads(7);
    grads[0] = at::empty(x.sizes(), x.options());
    grads[1] = at::empty(x.sizes(), x.options());
    bool sums = false;
    for (int i = 0; i < 5; ++i) {
        if (!wanted[i] || (i >= 3 && !post_norm)) continue;
        grads[2 + i] = at::empty({x.size(1)}, x.options());
        sums = true;
    }
    at::Tensor ws;
    size_t bytes = 0;
    if (sums) {
        bytes = lattice_hip_residual_norm_grad_workspace_bytes(j.args.rows, j.args.channels);
        ws = workspace(bytes, x);
    }
    check_status(lattice_hip_residual_norm_grad(
        &j.args, sum.data_ptr(), statistics.data_ptr<float>(), or_null(cotangents[0]), or_null(cotangents[1]),
        grads[0].data_ptr(), grads[1].data_ptr(), or_null(grads[2]), or_null(grads[3]), or_null(grads[4]),
        or_null(grads[5]), or_null(grads[6]), or_null(ws), bytes, current_stream(x)));
    return grads;
}

}  // namespace lattice_native
