// Gradients of the windowed attention.
//
//   p_ij = exp(s_ij - lse_i),  dp_ij = do_i . v_j,  delta_i = do_i . o_i,
//   ds_ij = p_ij (dp_ij - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
//   dv_j = sum_i p_ij do_i;
// the sums over i run over every head that shares the key head.  Each sum is
// made by one owner in a fixed order: no atomics.

#include "attention.h"

namespace lattice {
namespace {

constexpr int kAttnBlock = 256;
constexpr int kAttnWaves = kAttnBlock / kWave;

// A wave a (query row, head); keeps delta for the keys' pass.
template <typename T>
__global__ void __launch_bounds__(kAttnBlock)
grad_query_rows(lattice_attention a, const T* __restrict__ out, const float* __restrict__ lse,
                const T* __restrict__ grad_out, T* __restrict__ grad_q, float* __restrict__ delta) {
    __shared__ AttnRowScratch scratch[kAttnWaves];
    const int wave = threadIdx.x / kWave;
    const long long item = static_cast<long long>(blockIdx.x) * kAttnWaves + wave;
    if (item >= static_cast<long long>(a.queries) * a.heads) return;
    const int row = static_cast<int>(item / a.heads), head = static_cast<int>(item % a.heads);
    const int e = query_rows(a).find(row, [](int start, int) { return static_cast<uint32_t>(start); });
    const AttnSequence s = attn_sequence(a, e);
    const float d = attn_delta(a, row, head, out, grad_out);
    if (lane_id() == 0) delta[item] = d;
    grad_query_row<T>(a, s, row - s.q0, head, lse, d, grad_out, grad_q, &scratch[wave]);
}

// A wave a (key row, key head).
template <typename T>
__global__ void __launch_bounds__(kAttnBlock)
grad_key_rows(lattice_attention a, const float* __restrict__ lse, const float* __restrict__ delta,
              const T* __restrict__ grad_out, T* __restrict__ grad_k, T* __restrict__ grad_v) {
    __shared__ AttnRowScratch scratch[kAttnWaves];
    const int wave = threadIdx.x / kWave;
    const long long item = static_cast<long long>(blockIdx.x) * kAttnWaves + wave;
    if (item >= static_cast<long long>(a.keys) * a.kv_heads) return;
    const int row = static_cast<int>(item / a.kv_heads), kv = static_cast<int>(item % a.kv_heads);
    const int e = key_rows(a).find(row, [](int start, int) { return static_cast<uint32_t>(start); });
    const AttnSequence s = attn_sequence(a, e);
    grad_key_row<T>(a, s, row - s.k0, kv, lse, delta, grad_out, grad_k, grad_v, &scratch[wave]);
}

template <typename T>
int attend_grad(const lattice_attention& a, const void* out, const float* lse, const void* grad_out, void* grad_q,
                void* grad_k, void* grad_v, float* delta, hipStream_t stream) {
    const T* dy = static_cast<const T*>(grad_out);
    if (a.queries) {
        grad_query_rows<T><<<grid_for(static_cast<long long>(a.queries) * a.heads, kAttnWaves, 1u << 30), kAttnBlock,
                             0, stream>>>(a, static_cast<const T*>(out), lse, dy, static_cast<T*>(grad_q), delta);
        LATTICE_LAUNCH_CHECK();
    }
    if (a.keys) {
        grad_key_rows<T><<<grid_for(static_cast<long long>(a.keys) * a.kv_heads, kAttnWaves, 1u << 30), kAttnBlock, 0,
                           stream>>>(a, lse, delta, dy, static_cast<T*>(grad_k), static_cast<T*>(grad_v));
        LATTICE_LAUNCH_CHECK();
    }
    return LATTICE_OK;
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" size_t lattice_hip_window_attention_grad_workspace_bytes(const lattice_attention* args) {
    if (attn_fault(args)) return 0;
    return aligned_bytes(static_cast<size_t>(args->queries) * args->heads * sizeof(float));
}

extern "C" int lattice_hip_window_attention_grad(const lattice_attention* args, const void* out, const float* lse,
                                                 const void* grad_out, void* grad_q, void* grad_k, void* grad_v,
                                                 void* workspace, size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE_ATTENTION(args);
    if (args->queries == 0 && args->keys == 0) return LATTICE_OK;
    LATTICE_REQUIRE(args->queries == 0 || (out && lse && grad_out && grad_q), "attention pointers must be non-null.");
    LATTICE_REQUIRE(args->keys == 0 || (grad_k && grad_v), "attention pointers must be non-null.");
    Workspace ws{static_cast<char*>(workspace), workspace_bytes};
    float* delta = ws.take<float>(static_cast<size_t>(args->queries) * args->heads);
    LATTICE_REQUIRE(args->queries == 0 || (workspace && delta), "attention gradient workspace is too small.");
    const lattice_attention a = attn_bounded(*args);
    hipStream_t stream = as_stream(stream_ptr);
    if (a.dtype == LATTICE_F32) return attend_grad<float>(a, out, lse, grad_out, grad_q, grad_k, grad_v, delta, stream);
    if (a.dtype == LATTICE_F16)
        return attend_grad<_Float16>(a, out, lse, grad_out, grad_q, grad_k, grad_v, delta, stream);
    return attend_grad<__bf16>(a, out, lse, grad_out, grad_q, grad_k, grad_v, delta, stream);
}
