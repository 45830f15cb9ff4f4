// What the windowed attention's kernels share: the sequence of a row or tile,
// what a query sees, and the row-by-row forms of the forward and backward
// pass, one wave a row.
#pragma once

#include "rows.h"

namespace lattice {

constexpr int kAttnBlock = 256;
constexpr int kAttnWaves = kAttnBlock / kWave;
constexpr int kAttnMaxDim = 128;
constexpr float kAttnLog2e = 1.44269504088896340736f;

// Row partition `offsets` [count + 1] of `rows` rows, with the rows before the
// first and after the last offset as sequences 0 and count + 1: every row is
// in one.  Values are clamped to the rows there are.
struct RowPartition {
    const int32_t* offsets;
    int count, rows;

    // Read whether needed or not, so that reads of several need not wait for
    // each other.
    __device__ int start(int e) const {
        const int at = min(max(offsets[min(max(e - 1, 0), count)], 0), rows);
        return e <= 0 ? 0 : e > count + 1 ? rows : at;
    }
    __device__ bool real(int e) const { return e >= 1 && e <= count; }

    // The last sequence whose first slot, slot_of(start) + sequence, is at
    // most `slot`; all lanes of the wave together, 64 probes a step.
    template <typename SlotOf>
    __device__ int find(uint32_t slot, SlotOf slot_of) const {
        int lo = 0, n = count + 2;
        while (n > 1) {
            const int step = (n + kWave - 1) / kWave;
            const int probe = lo + lane_id() * step;
            const bool at_most = lane_id() * step < n && slot_of(start(probe), probe) <= slot;
            // Lane 0 always holds: its sequence starts at or before the slot.
            const int held = max(1, static_cast<int>(__popcll(ballot(at_most))));
            lo += (held - 1) * step;
            n = min(step, n - (held - 1) * step);
        }
        return __builtin_amdgcn_readfirstlane(lo);
    }
};

// A sequence: its query rows q0 .. q0 + nq and key rows k0 .. k0 + nk; query i
// has position i + nk - nq.
struct AttnSequence {
    int q0, nq, k0, nk;
    __device__ int shift() const { return nk - nq; }
};

__device__ inline RowPartition query_rows(const lattice_attention& a) { return {a.offsets, a.sequences, a.queries}; }
__device__ inline RowPartition key_rows(const lattice_attention& a) { return {a.key_offsets, a.sequences, a.keys}; }

// Sequence e of either partition (queries and keys share the numbering).
__device__ inline AttnSequence attn_sequence(const lattice_attention& a, int e) {
    const RowPartition q = query_rows(a), k = key_rows(a);
    AttnSequence s;
    s.q0 = q.start(e);
    s.nq = max(0, q.start(e + 1) - s.q0);
    s.k0 = k.start(e);
    s.nk = max(0, k.start(e + 1) - s.k0);
    if (!q.real(e)) {
        s.nk = 0;
    } else if (a.key_lengths) {
        s.nk = min(s.nk, max(0, a.key_lengths[e - 1]));
    }
    return s;
}

// The keys that a position sees: 0 .. first, then lo .. lo + window.
struct AttnSeen {
    int first, lo, window;
    __device__ int total() const { return first + window; }
    __device__ int key(int t) const { return t < first ? t : lo + (t - first); }
};
__device__ inline AttnSeen attn_seen(const lattice_attention& a, int nk, int p) {
    const int hi = min(nk - 1, p + a.right);
    const int lo = max(0, p - a.left);
    if (hi < 0) return {0, 0, 0};
    return {min(a.sinks, lo), lo, max(0, hi - lo + 1)};
}

__device__ inline bool attn_visible(const lattice_attention& a, int nk, int p, int j) {
    return j < nk && j <= p + a.right && (j >= p - a.left || j < a.sinks);
}

// The queries that see key j, i in from .. to (exclusive).
__device__ inline int2 attn_seen_by(const lattice_attention& a, const AttnSequence& s, int j) {
    const int from = max(0, j - a.right - s.shift());
    const int to = j < a.sinks ? s.nq : min(s.nq, j + a.left - s.shift() + 1);
    return int2{from, max(from, to)};
}

__device__ inline float wave_sum(float v) {
    for (int step = 1; step < kWave; step *= 2) v += __shfl_xor(v, step);
    return v;
}
__device__ inline float wave_max(float v) {
    for (int step = 1; step < kWave; step *= 2) v = fmaxf(v, __shfl_xor(v, step));
    return v;
}
// Orders a wave's LDS accesses.
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Until the wave has what it read from LDS: before a copy, which takes no turn
// among its LDS accesses, overwrites what they read.
__device__ inline void wait_for_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <typename T>
__device__ inline float row_dot(const float* __restrict__ a, const T* __restrict__ b, int dim) {
    float sum = 0.0f;
    for (int d = 0; d < dim; ++d) sum += a[d] * static_cast<float>(b[d]);
    return sum;
}

// A wave's scratch for the row forms.
struct AttnRowScratch {
    float a[kAttnMaxDim], b[kAttnMaxDim], p[kWave], r[kWave];
};

template <typename T>
__device__ inline void stage_row(float* to, const T* from, int dim) {
    for (int d = lane_id(); d < dim; d += kWave) to[d] = static_cast<float>(from[d]);
}

// What a forward pass keeps for the gradient (NULL: nothing): log2 of each
// row's softmax sum, and what rounding took from out, in its type.
template <typename T>
struct AttnKept {
    float* lse;
    T* rest;
};
// An infinity leaves none.
template <typename T>
__device__ inline T rounding_rest(float value, T rounded) {
    const float rest = value - static_cast<float>(rounded);
    return static_cast<T>(fabsf(rest) < INFINITY ? rest : 0.0f);
}

// The forward pass of one query row and head, keys in order 64 at a time, one
// a lane, with the running maximum and sum; then a channel a lane.  A key that
// the row does not see is not read.
template <typename T>
__device__ inline void attend_row(const lattice_attention& a, const AttnSequence& s, int i, int head, T* out,
                                  const AttnKept<T>& kept, AttnRowScratch* scratch) {
    const int lane = lane_id();
    const int kv = static_cast<int>(static_cast<long long>(head) * a.kv_heads / a.heads);
    const long long row = static_cast<long long>(s.q0) + i;
    const T* q = static_cast<const T*>(a.q) + row * a.q_row_stride + head * a.q_head_stride;
    const T* k = static_cast<const T*>(a.k) + s.k0 * a.k_row_stride + kv * a.k_head_stride;
    const T* v = static_cast<const T*>(a.v) + s.k0 * a.v_row_stride + kv * a.v_head_stride;
    const AttnSeen seen = attn_seen(a, s.nk, i + s.shift());
    const int total = seen.total();
    wave_fence();
    stage_row(scratch->a, q, a.dim);
    wave_fence();
    const float scale = a.scale * kAttnLog2e;
    float top = -INFINITY, sum = 0.0f, acc[kAttnMaxDim / kWave] = {};
    for (int base = 0; base < total; base += kWave) {
        const int count = min(kWave, total - base);
        float x = -INFINITY;
        if (lane < count) x = row_dot(scratch->a, k + seen.key(base + lane) * a.k_row_stride, a.dim) * scale;
        const float next = fmaxf(top, wave_max(x));
        const float old = top == next ? 1.0f : exp2f(top - next);
        // Of -inf before any other score, no share (alone, 0 / 0 in the end).
        const float p = x != -INFINITY ? exp2f(x - next) : 0.0f;
        top = next;
        sum = sum * old + wave_sum(p);
        wave_fence();
        scratch->p[lane] = p;
        wave_fence();
#pragma unroll
        for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
            const int d = lane + c * kWave;
            if (d >= a.dim) continue;
            float add = 0.0f;
            for (int t = 0; t < count; ++t)
                add += scratch->p[t] * static_cast<float>(v[seen.key(base + t) * a.v_row_stride + d]);
            acc[c] = acc[c] * old + add;
        }
    }
    if (kept.lse && lane == 0) kept.lse[row * a.heads + head] = total ? top + log2f(sum) : INFINITY;
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
        const int d = lane + c * kWave;
        if (d >= a.dim) continue;
        const float value = total ? acc[c] / sum : 0.0f;
        const T rounded = static_cast<T>(value);
        out[(row * a.heads + head) * a.dim + d] = rounded;
        if (kept.rest) kept.rest[(row * a.heads + head) * a.dim + d] = rounding_rest(value, rounded);
    }
}

// grad_q of one query row and head.
template <typename T>
__device__ inline void grad_query_row(const lattice_attention& a, const AttnSequence& s, int i, int head,
                                      const float* lse, float delta, const T* grad_out, T* grad_q,
                                      AttnRowScratch* scratch) {
    const int lane = lane_id();
    const int kv = static_cast<int>(static_cast<long long>(head) * a.kv_heads / a.heads);
    const long long row = static_cast<long long>(s.q0) + i;
    const long long at = row * a.heads + head;
    const T* q = static_cast<const T*>(a.q) + row * a.q_row_stride + head * a.q_head_stride;
    const T* k = static_cast<const T*>(a.k) + s.k0 * a.k_row_stride + kv * a.k_head_stride;
    const T* v = static_cast<const T*>(a.v) + s.k0 * a.v_row_stride + kv * a.v_head_stride;
    const AttnSeen seen = attn_seen(a, s.nk, i + s.shift());
    const int total = seen.total();
    wave_fence();
    stage_row(scratch->a, q, a.dim);
    stage_row(scratch->b, grad_out + at * a.dim, a.dim);
    wave_fence();
    const float scale = a.scale * kAttnLog2e, log_sum = lse[at];
    float acc[kAttnMaxDim / kWave] = {};
    for (int base = 0; base < total; base += kWave) {
        const int count = min(kWave, total - base);
        float slope = 0.0f;
        if (lane < count) {
            const int j = seen.key(base + lane);
            const float p = exp2f(row_dot(scratch->a, k + j * a.k_row_stride, a.dim) * scale - log_sum);
            slope = p * (row_dot(scratch->b, v + j * a.v_row_stride, a.dim) - delta);
        }
        wave_fence();
        scratch->p[lane] = slope;
        wave_fence();
#pragma unroll
        for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
            const int d = lane + c * kWave;
            if (d >= a.dim) continue;
            for (int t = 0; t < count; ++t)
                acc[c] += scratch->p[t] * static_cast<float>(k[seen.key(base + t) * a.k_row_stride + d]);
        }
    }
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
        const int d = lane + c * kWave;
        if (d < a.dim) grad_q[at * a.dim + d] = static_cast<T>(acc[c] * a.scale);
    }
}

// grad_k and grad_v of one key row and key head: states holds (lse, delta) by
// key head, row and head, channels from_dim .. to_dim are written; over the
// queries that see it and the heads that share it, (query, head) pairs 64 at a
// time, one a lane.
template <typename T>
__device__ inline void grad_key_row(const lattice_attention& a, const AttnSequence& s, int j, int kv,
                                    const float* lse, const float2* states, const T* grad_out, T* grad_k, T* grad_v,
                                    AttnRowScratch* scratch, int from_dim = 0, int to_dim = kAttnMaxDim) {
    const int lane = lane_id();
    const int group = a.heads / a.kv_heads;
    const long long row = static_cast<long long>(s.k0) + j;
    const T* q = static_cast<const T*>(a.q) + s.q0 * a.q_row_stride + kv * group * a.q_head_stride;
    const T* k = static_cast<const T*>(a.k) + row * a.k_row_stride + kv * a.k_head_stride;
    const T* v = static_cast<const T*>(a.v) + row * a.v_row_stride + kv * a.v_head_stride;
    // The rows that see the key; rows past the sequence's keys see nothing.
    const int2 by = j < s.nk ? attn_seen_by(a, s, j) : int2{0, 0};
    const long long total = static_cast<long long>(by.y - by.x) * group;
    wave_fence();
    stage_row(scratch->a, k, a.dim);
    stage_row(scratch->b, v, a.dim);
    wave_fence();
    const float scale = a.scale * kAttnLog2e;
    float acc_k[kAttnMaxDim / kWave] = {}, acc_v[kAttnMaxDim / kWave] = {};
    for (long long base = 0; base < total; base += kWave) {
        const int count = static_cast<int>(min(static_cast<long long>(kWave), total - base));
        float p = 0.0f, slope = 0.0f;
        if (lane < count) {
            const long long i = by.x + (base + lane) / group;
            const int h = static_cast<int>((base + lane) % group);
            const long long at = (s.q0 + i) * a.heads + kv * group + h;
            p = exp2f(row_dot(scratch->a, q + i * a.q_row_stride + h * a.q_head_stride, a.dim) * scale - lse[at]);
            slope = p * (row_dot(scratch->b, grad_out + at * a.dim, a.dim) -
                         states[(static_cast<long long>(kv) * a.queries + s.q0 + i) * group + h].y);
        }
        wave_fence();
        scratch->p[lane] = p;
        scratch->r[lane] = slope;
        wave_fence();
        for (int t = 0; t < count; ++t) {
            const long long i = by.x + (base + t) / group;
            const int h = static_cast<int>((base + t) % group);
            const T* qi = q + i * a.q_row_stride + h * a.q_head_stride;
            const T* gi = grad_out + ((s.q0 + i) * a.heads + kv * group + h) * a.dim;
#pragma unroll
            for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
                const int d = lane + c * kWave;
                if (d >= a.dim) continue;
                acc_k[c] += scratch->r[t] * static_cast<float>(qi[d]);
                acc_v[c] += scratch->p[t] * static_cast<float>(gi[d]);
            }
        }
    }
    const long long at = (row * a.kv_heads + kv) * a.dim;
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
        const int d = lane + c * kWave;
        if (d >= a.dim || d < from_dim || d >= to_dim) continue;
        grad_k[at + d] = static_cast<T>(acc_k[c] * a.scale);
        grad_v[at + d] = static_cast<T>(acc_v[c]);
    }
}

// What every entry checks; NULL, or what is wrong.
inline const char* attn_fault(const lattice_attention* a) {
    if (!a) return "attention arguments must be non-null.";
    if (a->dtype != LATTICE_F32 && a->dtype != LATTICE_F16 && a->dtype != LATTICE_BF16)
        return "attention supports float32, float16 and bfloat16.";
    if (a->queries < 0 || a->keys < 0 || a->sequences < 0 || a->queries >= 1 << 29 || a->keys >= 1 << 29)
        return "attention takes up to 2^29 - 1 rows of queries and of keys.";
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0)
        return "the number of heads must be a multiple of the number of key heads.";
    if (static_cast<long long>(a->queries) * a->heads >= 1ll << 31 ||
        static_cast<long long>(a->keys) * a->kv_heads >= 1ll << 31)
        return "attention takes up to 2^31 - 1 rows of heads.";
    if (a->dim < 1 || a->dim > kAttnMaxDim) return "attention heads must have between 1 and 128 channels.";
    if (a->left < 0 || a->right < 0 || a->sinks < 0) return "left, right and sinks must be non-negative.";
    if (a->queries && (!a->q || !a->offsets || !a->key_offsets)) return "attention pointers must be non-null.";
    if (a->keys && (!a->k || !a->v || !a->key_offsets || !a->offsets)) return "attention pointers must be non-null.";
    const long long piece = 16 / (a->dtype == LATTICE_F32 ? 4 : 2);
    const long long strides[] = {a->q_row_stride, a->q_head_stride, a->k_row_stride,
                                 a->k_head_stride, a->v_row_stride, a->v_head_stride};
    for (long long s : strides)
        if (s < 0 || s % piece != 0) return "attention strides must be whole 16-byte pieces.";
    // Within a tile, places are counted in 32 bits: rows of a tile and the heads
    // of a group lie within 2^30 bytes.
    if (std::max({a->q_row_stride, a->k_row_stride, a->v_row_stride, static_cast<long long>(a->heads) * a->dim}) >=
        piece << 18)
        return "attention rows must be under 4 MiB apart.";
    if (a->q_head_stride >= (piece << 25) / (a->heads / a->kv_heads))
        return "the query heads of a key head must lie within 512 MiB.";
    if (a->dim % piece != 0) return "attention rows must be whole 16-byte pieces.";
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v)) %
        16 != 0)
        return "attention rows must lie on 16-byte boundaries.";
    return nullptr;
}

// left, right and sinks are bounded by the rows there are, so that positions
// stay far inside 32 bits.
inline lattice_attention attn_bounded(const lattice_attention& a) {
    lattice_attention b = a;
    const int most = a.queries + a.keys;
    b.left = std::min(b.left, most);
    b.right = std::min(b.right, most);
    b.sinks = std::min(b.sinks, a.keys);
    return b;
}

// Dynamic LDS past the 64 KiB that every kernel may use has to be allowed.
inline hipError_t allow_lds(const void* kernel, size_t bytes) {
    if (bytes <= 64 * 1024) return hipSuccess;
    return hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

#define LATTICE_REQUIRE_ATTENTION(args)                           \
    do {                                                          \
        if (const char* fault_ = ::lattice::attn_fault(args)) {   \
            ::lattice::set_error(fault_);                         \
            return LATTICE_ERROR_INVALID_ARGUMENT;                \
        }                                                         \
    } while (0)

}  // namespace lattice
