// Gradients of the windowed attention.
//
//   p_ij = exp(s_ij - lse_i),  dp_ij = do_i . v_j,  delta_i = do_i . o_i,
//   ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
//   dv_j = sum_i p_ij do_i;
// the sums over i run over every head that shares the key head.  Each sum has
// one owner that makes it in a fixed order: no atomics.  The scores are made
// twice, once for the queries' sums and once for the keys': seven products in
// place of five, but neither pass shares its sums with another block.

#include "attention_grad.h"

using namespace lattice;

extern "C" size_t lattice_hip_window_attention_grad_workspace_bytes(const lattice_attention* args) {
    if (attn_fault(args)) return 0;
    const GradLayout l = grad_layout(attn_bounded(*args));
    return aligned_bytes(l.states * sizeof(float2)) + aligned_bytes(l.past_values * sizeof(float)) +
           aligned_bytes(l.window_values * sizeof(float));
}

extern "C" int lattice_hip_window_attention_grad(const lattice_attention* args, const void* out, const void* out_rest,
                                                 const float* lse, const void* grad_out, void* grad_q, void* grad_k, void* grad_v,
                                                 void* workspace, size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE_ATTENTION(args);
    if (args->queries == 0 && args->keys == 0) return LATTICE_OK;
    LATTICE_REQUIRE(args->queries == 0 || (out && lse && grad_out && grad_q), "attention pointers must be non-null.");
    LATTICE_REQUIRE(args->keys == 0 || (grad_k && grad_v), "attention pointers must be non-null.");
    LATTICE_REQUIRE((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(out_rest) |
                     reinterpret_cast<uintptr_t>(grad_out)) %
                            16 ==
                        0,
                    "attention rows must lie on 16-byte boundaries.");
    const lattice_attention a = attn_bounded(*args);
    const GradLayout l = grad_layout(a);
    Workspace ws{static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
    float2* states = ws.take<float2>(l.states);
    FirstParts parts{nullptr, nullptr, l.first_tiles};
    parts.past = ws.take<float>(l.past_values);
    parts.window = ws.take<float>(l.window_values);
    LATTICE_REQUIRE(a.queries == 0 || (states && parts.past && parts.window),
                    "attention gradient workspace is too small.");
    hipStream_t stream = as_stream(stream_ptr);
    if (a.dtype == LATTICE_F32)
        return attend_grad<float>(a, l, out, out_rest, lse, grad_out, grad_q, grad_k, grad_v, states, parts, stream);
    if (a.dtype == LATTICE_F16)
        return attend_grad<_Float16>(a, l, out, out_rest, lse, grad_out, grad_q, grad_k, grad_v, states, parts, stream);
    return attend_grad<__bf16>(a, l, out, out_rest, lse, grad_out, grad_q, grad_k, grad_v, states, parts, stream);
}
