// Kernels and launches of the windowed attention's gradients, for one type a
// translation unit.
#pragma once

#include "attention_tiles.h"

namespace lattice {

// Sums of the first keys, in tiles of 32, by key head: of the pairs past the
// window, which run to the end of a sequence, a part for each slot of
// kFirstRows of the sequence's (query, head) pairs; and of the pairs in it, a
// part for each sequence.  A part holds dk, then dv, in the registers' order.
struct FirstParts {
    float *past, *window;
    int tiles;  // 0: the keys' pass takes every pair by itself
    __device__ float* past_of(const lattice_attention& a, long long slot, int kv, int tile, int values) const {
        return past + ((slot * a.kv_heads + kv) * tiles + tile) * values;
    }
    __device__ float* window_of(const lattice_attention& a, int e, int kv, int tile, int values) const {
        return window + ((static_cast<long long>(e) * a.kv_heads + kv) * tiles + tile) * values;
    }
};
// Pairs of a slot.  (The parts of 60k rows of 4 heads of 64 over 2, one block a
// unit: 17.5 us, in slots of 1024 20.5, of 256 23.4; of 20k rows of 4 heads of
// 32, fp32: 17.6, 28.1 and 15.6; their sum grows with the number of slots.)
constexpr uint32_t kFirstRows = 512;

// Whether tiles of 128 of `rows` rows would leave units idle: below one block a
// unit the form for few rows is faster (156 blocks of heads of 64: 33 us for 38;
// 32 blocks, window 3556: 35 for 101), above it the other (312: 45 for 53).
inline bool grad_few(long long rows) { return rows < 128ll * 256; }

// What a call needs besides its outputs.
struct GradLayout {
    size_t states, past_values, window_values;
    int first_slots, first_tiles;
};
inline GradLayout grad_layout(const lattice_attention& a) {
    GradLayout l{static_cast<size_t>(a.queries) * a.heads, 0, 0, 0, 0};
    const long long pairs = static_cast<long long>(a.queries) * (a.heads / a.kv_heads);
    // The first keys' queries past the window are a pass of their own where
    // sequences are long: one block would walk all of a sequence.  In the form
    // for few rows its four waves do, and two launches are saved.
    const long long alone = grad_few(static_cast<long long>(a.keys) * a.kv_heads) ? 2048 : 512;
    if (a.sinks > 0 && a.sinks <= 128 && a.left < a.keys && pairs >= alone * std::max(1, a.sequences)) {
        l.first_slots = static_cast<int>(pairs / kFirstRows + a.sequences + 2);
        l.first_tiles = (a.sinks + 31) / 32;
        const size_t values = static_cast<size_t>(a.kv_heads) * l.first_tiles * 2 * attn_width(a.dim) * 32;
        l.past_values = l.first_slots * values;
        l.window_values = (a.sequences + 2) * values;
    }
    return l;
}

// The launches for rows of type T.
template <typename T>
int attend_grad(const lattice_attention& a, const GradLayout& l, const void* out, const void* out_rest,
                const float* lse, const void* grad_out, void* grad_q, void* grad_k, void* grad_v, float2* states,
                const FirstParts& parts, hipStream_t stream);

}  // namespace lattice
