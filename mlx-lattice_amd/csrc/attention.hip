// Attention over a sliding window with first keys that stay visible: the
// forward pass.
//
//   s_ij = scale q_i . k_j over the keys j that query i sees,
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),
// with the running maximum m and sum of one pass over the keys.

#include "attention.h"

namespace lattice {
namespace {

constexpr int kAttnBlock = 256;
constexpr int kAttnWaves = kAttnBlock / kWave;

// A wave a (query row, head).
template <typename T>
__global__ void __launch_bounds__(kAttnBlock)
attend_rows(lattice_attention a, T* __restrict__ out, float* __restrict__ lse) {
    __shared__ AttnRowScratch scratch[kAttnWaves];
    const int wave = threadIdx.x / kWave;
    const long long item = static_cast<long long>(blockIdx.x) * kAttnWaves + wave;
    if (item >= static_cast<long long>(a.queries) * a.heads) return;
    const int row = static_cast<int>(item / a.heads), head = static_cast<int>(item % a.heads);
    const int e = query_rows(a).find(row, [](int start, int) { return static_cast<long long>(start); });
    const AttnSequence s = attn_sequence(a, e);
    attend_row<T>(a, s, row - s.q0, head, out, lse, &scratch[wave]);
}

template <typename T>
int attend(const lattice_attention& a, void* out, float* lse, hipStream_t stream) {
    attend_rows<T><<<grid_for(static_cast<long long>(a.queries) * a.heads, kAttnWaves, 1u << 30), kAttnBlock, 0,
                     stream>>>(a, static_cast<T*>(out), lse);
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" size_t lattice_hip_window_attention_workspace_bytes(const lattice_attention* args) {
    return attn_fault(args) ? 0 : 0;
}

extern "C" int lattice_hip_window_attention(const lattice_attention* args, void* out, float* lse, void* workspace,
                                            size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE_ATTENTION(args);
    if (args->queries == 0) return LATTICE_OK;
    LATTICE_REQUIRE(out, "attention pointers must be non-null.");
    (void)workspace;
    (void)workspace_bytes;
    const lattice_attention a = attn_bounded(*args);
    hipStream_t stream = as_stream(stream_ptr);
    if (a.dtype == LATTICE_F32) return attend<float>(a, out, lse, stream);
    if (a.dtype == LATTICE_F16) return attend<_Float16>(a, out, lse, stream);
    return attend<__bf16>(a, out, lse, stream);
}
