#include "features/transformer/api.h"

#include <ATen/DeviceGuard.h>

#include <algorithm>
#include <stdexcept>

#include "features/transformer/checks.h"

namespace lattice_native {

std::tuple<at::Tensor, at::Tensor> layer_norm(const at::Tensor& x_in, const c10::optional<at::Tensor>& weight_in,
                                              const c10::optional<at::Tensor>& bias_in, double eps,
                                              const c10::optional<at::Tensor>& active_rows, bool keep_statistics) {
    refuse_tangents({x_in, or_undefined(weight_in), or_undefined(bias_in)});
    if (x_in.dim() != 2 || x_in.size(1) < 1) throw std::invalid_argument("layer norm rows must have shape (N, C).");
    const int dtype = dtype_code(x_in, "layer norm rows");
    require_row_values(1, x_in.size(1), "layer norm rows");
    if (!(eps >= 0.0)) throw std::invalid_argument("eps must be non-negative.");
    require_device(x_in, "x");
    const at::DeviceGuard guard(x_in.device());
    const at::Tensor weight = channel_vector(weight_in, x_in, "weight"), bias = channel_vector(bias_in, x_in, "bias");
    const int32_t* active = active_or_null(active_rows, x_in);
    const at::Tensor x = unit_rows(x_in);
    const int rows = row_count(x, "x");
    at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor statistics;
    if (keep_statistics) statistics = at::empty({rows, 2}, x.options().dtype(at::kFloat));
    check_status(lattice_hip_layer_norm(dtype, x.data_ptr(), row_stride(x), rows, static_cast<int>(x.size(1)),
                                        or_null(weight), or_null(bias), static_cast<float>(eps), active, y.data_ptr(),
                                        keep_statistics ? statistics.data_ptr<float>() : nullptr, current_stream(x)));
    return {y, statistics};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_grad(const at::Tensor& grad_y, const at::Tensor& x_in,
                                                               const c10::optional<at::Tensor>& weight_in,
                                                               const at::Tensor& statistics,
                                                               const c10::optional<at::Tensor>& active_rows,
                                                               bool grad_weight, bool grad_bias) {
    refuse_tangents({grad_y, x_in, or_undefined(weight_in)});
    if (x_in.dim() != 2 || x_in.size(1) < 1) throw std::invalid_argument("layer norm rows must have shape (N, C).");
    const int dtype = dtype_code(x_in, "layer norm rows");
    require_row_values(1, x_in.size(1), "layer norm rows");
    require_device(x_in, "x");
    require_same(grad_y, x_in, "the cotangent");
    if (grad_y.sizes() != x_in.sizes()) throw std::invalid_argument("the cotangent must match the output shape.");
    if (statistics.dim() != 2 || statistics.size(0) != x_in.size(0) || statistics.size(1) != 2 ||
        statistics.scalar_type() != at::kFloat || !statistics.is_contiguous() ||
        statistics.device() != x_in.device()) {
        throw std::invalid_argument("statistics must be those of the forward call.");
    }
    const at::DeviceGuard guard(x_in.device());
    const at::Tensor weight = channel_vector(weight_in, x_in, "weight");
    const int32_t* active = active_or_null(active_rows, x_in);
    const at::Tensor x = unit_rows(x_in), dy = unit_rows(grad_y);
    const int rows = row_count(x, "x"), channels = static_cast<int>(x.size(1));
    at::Tensor dx = at::empty(x.sizes(), x.options());
    at::Tensor dw, db;
    if (grad_weight) dw = at::empty({channels}, x.options());
    if (grad_bias) db = at::empty({channels}, x.options());
    at::Tensor ws;
    size_t bytes = 0;
    if (grad_weight || grad_bias) {
        bytes = lattice_hip_layer_norm_grad_workspace_bytes(rows, channels);
        ws = workspace(bytes, x);
    }
    check_status(lattice_hip_layer_norm_grad(
        dtype, dy.data_ptr(), row_stride(dy), x.data_ptr(), row_stride(x), rows, channels, or_null(weight),
        statistics.data_ptr<float>(), active, dx.data_ptr(), or_null(dw), or_null(db), or_null(ws), bytes, current_stream(x)));
    return {dx, dw, db};
}

at::Tensor dropout(const at::Tensor& x_in, const c10::optional<at::Tensor>& residual_in, uint64_t seed,
                   uint64_t offset, uint64_t threshold, double scale) {
    refuse_tangents({x_in, or_undefined(residual_in)});
    const int dtype = dtype_code(x_in, "dropout values");
    require_device(x_in, "x");
    const at::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous();
    at::Tensor residual;
    if (residual_in && residual_in->defined()) {
        require_same(*residual_in, x_in, "residual");
        if (residual_in->sizes() != x_in.sizes()) throw std::invalid_argument("residual must match the shape of x.");
        residual = residual_in->contiguous();
    }
    at::Tensor y = at::empty(x.sizes(), x.options());
    check_status(lattice_hip_dropout(dtype, x.data_ptr(), or_null(residual), x.numel(), seed, offset, threshold,
                                     static_cast<float>(scale), y.data_ptr(), current_stream(x)));
    return y;
}

at::Tensor rotary_positions(const at::Tensor& x_in, const at::Tensor& positions_in, const at::Tensor& frequencies_in,
                            const std::vector<int>& dims, bool interleaved, bool inverse) {
    refuse_tangents({x_in, positions_in, frequencies_in});
    if (x_in.dim() != 3 || x_in.size(1) < 1 || x_in.size(2) < 1) {
        throw std::invalid_argument("rotary rows must have shape (N, heads, dim).");
    }
    const int dtype = dtype_code(x_in, "rotary rows");
    require_row_values(x_in.size(1), x_in.size(2), "rotary rows");
    if (x_in.size(2) > 1024) throw std::invalid_argument("rotary heads must have between 1 and 1024 channels.");
    if (dims.empty() || dims.size() > 4) throw std::invalid_argument("rotary positions need between 1 and 4 axes.");
    int64_t pairs = 0;
    for (const int d : dims) {
        if (d < 0 || d % 2 != 0) throw std::invalid_argument("rotary dims must be even and non-negative.");
        pairs += d / 2;
    }
    if (2 * pairs > x_in.size(2)) throw std::invalid_argument("rotary dims must fit the head.");
    if (positions_in.dim() != 2 || positions_in.size(0) != x_in.size(0) ||
        positions_in.size(1) != static_cast<int64_t>(dims.size()) ||
        (positions_in.scalar_type() != at::kInt && positions_in.scalar_type() != at::kFloat)) {
        throw std::invalid_argument("positions must have shape (N, axes) and int32 or float32 dtype.");
    }
    if (frequencies_in.dim() != 1 || frequencies_in.size(0) != pairs || frequencies_in.scalar_type() != at::kDouble) {
        throw std::invalid_argument("frequencies must have shape (sum(dims) / 2,) and float64 dtype.");
    }
    require_device(x_in, "x");
    require_device(positions_in, "positions");
    require_device(frequencies_in, "frequencies");
    if (positions_in.device() != x_in.device() || frequencies_in.device() != x_in.device()) {
        throw std::invalid_argument("positions and frequencies must be on the device of x.");
    }
    const at::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.size(2) == 1 || x_in.stride(2) == 1 ? x_in : x_in.contiguous();
    const at::Tensor positions = unit_rows(positions_in);
    const at::Tensor frequencies = frequencies_in.contiguous();
    at::Tensor y = at::empty(x.sizes(), x.options());
    check_status(lattice_hip_rotary_positions(
        dtype, x.data_ptr(), row_stride(x), x.size(1) > 1 ? x.stride(1) : 0, row_count(x, "x"),
        static_cast<int>(x.size(1)), static_cast<int>(x.size(2)), positions.data_ptr(),
        positions.scalar_type() == at::kFloat, row_stride(positions), frequencies.data_ptr<double>(),
        static_cast<int>(dims.size()), dims.data(), interleaved, inverse, y.data_ptr(), current_stream(x)));
    return y;
}

// ------------------------------------------------------------ attention --

namespace {

struct Attention {
    lattice_attention args;
    at::Tensor q, k, v;
};

Attention attention_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
                       const at::Tensor& key_offsets, const c10::optional<at::Tensor>& key_lengths, int64_t left,
                       int64_t right, int64_t sinks, double scale) {
    if (q.dim() != 3 || k.dim() != 3 || v.dim() != 3) {
        throw std::invalid_argument("q, k and v must have shape (N, heads, dim).");
    }
    const int dtype = dtype_code(q, "q, k and v");
    require_row_values(q.size(1), q.size(2), "q, k and v");
    require_row_values(k.size(1), k.size(2), "q, k and v");
    if (k.sizes() != v.sizes()) throw std::invalid_argument("k and v must have the same shape.");
    if (q.size(2) != k.size(2)) throw std::invalid_argument("q, k and v must share the channels of a head.");
    if (q.size(2) < 1 || q.size(2) > 128) {
        throw std::invalid_argument("attention heads must have between 1 and 128 channels.");
    }
    if (q.size(1) < 1 || k.size(1) < 1 || q.size(1) % k.size(1) != 0) {
        throw std::invalid_argument("the number of heads must be a multiple of the number of key heads.");
    }
    if (left < 0 || right < 0 || sinks < 0) {
        throw std::invalid_argument("left, right and sinks must be non-negative.");
    }
    require_device(q, "q");
    require_same(k, q, "k");
    require_same(v, q, "v");
    if (offsets.dim() != 1 || offsets.size(0) < 1) {
        throw std::invalid_argument("offsets must have shape (B + 1,) and int32 dtype.");
    }
    require_index(offsets, q, offsets.size(0), "offsets must have shape (B + 1,) and int32 dtype.");
    require_index(key_offsets, q, offsets.size(0), "key_offsets must have the shape and dtype of offsets.");
    if (!offsets.is_contiguous() || !key_offsets.is_contiguous()) {
        throw std::invalid_argument("offsets must be contiguous.");
    }
    const int32_t* lengths = nullptr;
    if (key_lengths && key_lengths->defined()) {
        require_index(*key_lengths, q, offsets.size(0) - 1, "key_lengths must have shape (B,) and int32 dtype.");
        if (!key_lengths->is_contiguous()) throw std::invalid_argument("key_lengths must be contiguous.");
        lengths = ci32(*key_lengths);
    }
    Attention a{{}, pieces(q, q.size(1) / k.size(1)), pieces(k), pieces(v)};
    const auto head_stride = [](const at::Tensor& t) { return t.size(1) > 1 ? t.stride(1) : 0; };
    a.args.dtype = dtype;
    a.args.queries = row_count(q, "q");
    a.args.keys = row_count(k, "k");
    a.args.heads = static_cast<int>(q.size(1));
    a.args.kv_heads = static_cast<int>(k.size(1));
    a.args.dim = static_cast<int>(a.q.size(2));
    a.args.sequences = static_cast<int>(offsets.size(0) - 1);
    a.args.left = static_cast<int>(std::min(left, kMost));
    a.args.right = static_cast<int>(std::min(right, kMost));
    a.args.sinks = static_cast<int>(std::min(sinks, kMost));
    a.args.scale = static_cast<float>(scale);
    a.args.q = a.q.data_ptr();
    a.args.k = a.k.data_ptr();
    a.args.v = a.v.data_ptr();
    a.args.q_row_stride = row_stride(a.q);
    a.args.k_row_stride = row_stride(a.k);
    a.args.v_row_stride = row_stride(a.v);
    a.args.q_head_stride = head_stride(a.q);
    a.args.k_head_stride = head_stride(a.k);
    a.args.v_head_stride = head_stride(a.v);
    a.args.offsets = ci32(offsets);
    a.args.key_offsets = ci32(key_offsets);
    a.args.key_lengths = lengths;
    return a;
}

// A contiguous tensor on a 16-byte boundary.
at::Tensor whole_pieces(const at::Tensor& t) {
    const at::Tensor p = pieces(t);
    return p.is_contiguous() ? p : p.contiguous();
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& offsets,
    const at::Tensor& key_offsets, const c10::optional<at::Tensor>& key_lengths, int64_t left, int64_t right,
    int64_t sinks, double scale, bool keep) {
    refuse_tangents({q, k, v});
    const c10::OptionalDeviceGuard guard(q.is_cuda() ? c10::make_optional(q.device()) : c10::nullopt);
    const Attention a = attention_of(q, k, v, offsets, key_offsets, key_lengths, left, right, sinks, scale);
    at::Tensor out = at::empty(a.q.sizes(), q.options());
    at::Tensor lse, rest;
    if (keep) {
        lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
        if (q.scalar_type() != at::kFloat) rest = at::empty(a.q.sizes(), q.options());
    }
    const size_t bytes = lattice_hip_window_attention_workspace_bytes(&a.args);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    check_status(lattice_hip_window_attention(&a.args, out.data_ptr(), keep ? lse.data_ptr<float>() : nullptr,
                                              or_null(rest), or_null(ws), bytes, current_stream(q)));
    return {unpadded(out, q.size(2)), lse, rest};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> window_attention_grad(
    const at::Tensor& grad_out_in, const at::Tensor& out_in, const at::Tensor& lse,
    const c10::optional<at::Tensor>& rest, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& offsets, const at::Tensor& key_offsets, const c10::optional<at::Tensor>& key_lengths,
    int64_t left, int64_t right, int64_t sinks, double scale) {
    refuse_tangents({grad_out_in, q, k, v});
    const c10::OptionalDeviceGuard guard(q.is_cuda() ? c10::make_optional(q.device()) : c10::nullopt);
    const Attention a = attention_of(q, k, v, offsets, key_offsets, key_lengths, left, right, sinks, scale);
    require_same(grad_out_in, q, "the cotangent");
    require_same(out_in, q, "out");
    if (grad_out_in.sizes() != q.sizes() || out_in.sizes() != q.sizes()) {
        throw std::invalid_argument("the cotangent must match the output shape.");
    }
    if (lse.dim() != 2 || lse.size(0) != q.size(0) || lse.size(1) != q.size(1) || lse.scalar_type() != at::kFloat ||
        !lse.is_contiguous() || lse.device() != q.device()) {
        throw std::invalid_argument("lse must be that of the forward call.");
    }
    const at::Tensor grad_out = whole_pieces(grad_out_in), out = whole_pieces(out_in);
    if (rest && rest->defined() &&
        (rest->sizes() != a.q.sizes() || rest->scalar_type() != q.scalar_type() || !rest->is_contiguous() ||
         rest->device() != q.device())) {
        throw std::invalid_argument("rest must be that of the forward call.");
    }
    at::Tensor dq = at::empty(a.q.sizes(), q.options());
    at::Tensor dk = at::empty(a.k.sizes(), q.options()), dv = at::empty(a.k.sizes(), q.options());
    const size_t bytes = lattice_hip_window_attention_grad_workspace_bytes(&a.args);
    at::Tensor ws;
    if (bytes) ws = workspace(bytes, q);
    check_status(lattice_hip_window_attention_grad(&a.args, out.data_ptr(), data_or_null(rest),
                                                   lse.data_ptr<float>(), grad_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                                   or_null(ws), bytes, current_stream(q)));
    const int64_t dim = q.size(2);
    return {unpadded(dq, dim), unpadded(dk, dim), unpadded(dv, dim)};
}

}  // namespace lattice_native
