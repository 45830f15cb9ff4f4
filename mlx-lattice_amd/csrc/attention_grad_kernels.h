// Kernels of the windowed attention's gradients and their launches.
//
// grad_q is bound as the forward pass by the vector instructions between the
// products (an exponential, four others and two roundings a score; their pipe
// is busy 40 % of the time, the matrix cores 25); grad_k and grad_v by waits, with
// one or two waves a SIMD for the registers of their sums (vector 25 %, matrix
// cores 24, half of a wave's time in waits).  60,001 rows of 4 heads of 64 over
// 2, window 513, bf16: grad_q 89 us, grad_k and grad_v 113, the first keys' long
// sums 17 + 9; 20,000 rows of 4 heads of 32, window 128, fp32: 60, 65, 17 + 4
// (fp32 products have a sixteenth of the 16-bit rate: matrix cores 35 %; eight or
// nine short steps leave a block waiting for its copies, 45 % of a wave's time).
#pragma once

#include "attention_grad.h"

namespace lattice {
namespace {

// Slopes are rounded to the type before their products.  In half precision
// they are first scaled by a power of two that follows their size, since the
// gradients of a long row are far below the type's smallest normal number;
// the sums carry the scale and drop it at the end.
template <typename T>
struct SlopeScale {
    static constexpr bool kUsed = false;
    __device__ float factor() const { return 1.0f; }
};
__device__ inline float power_of_two(int exponent) { return __int_as_float((max(exponent, -126) + 127) << 23); }
template <>
struct SlopeScale<_Float16> {
    static constexpr bool kUsed = true;
    static constexpr int kNone = 100, kMost = 40;
    int exponent = kNone;
    __device__ float factor() const { return exponent == kNone ? 1.0f : power_of_two(exponent); }
    // Follows the wave's largest slope; the factor by which the sums so far
    // have to be scaled.  A column with a slope that is not finite is made
    // again by itself and has no say in the others' scale.
    __device__ float follow(float largest) {
        largest = largest < INFINITY ? largest : 0.0f;
        if (!__any(largest * power_of_two(exponent) > 32768.0f)) return 1.0f;
        largest = wave_max(largest);
        // The largest becomes 2^11 .. 2^12.
        const int next = min(kMost, 138 - (__float_as_int(largest) >> 23));
        const float change = exponent == kNone ? 1.0f : power_of_two(next - exponent);
        exponent = next;
        return change;
    }
};

// The power of two that scales the shares of half precision.
template <typename T> constexpr float kShareLog2 = 0.0f;
template <> constexpr float kShareLog2<_Float16> = 14.0f;

template <int BLOCKS>
__device__ inline void scale_sums(f32x16_attn (&acc)[BLOCKS], float factor) {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) acc[b] *= factor;
}

// Rounds slopes into the scale's range and adds their products to acc.
template <typename Tile, typename T, int BLOCKS>
__device__ inline void add_slopes(f32x16_attn (&acc)[BLOCKS], SlopeScale<T>& scale, const char* tile, int row0,
                                  f32x16_attn& ds) {
    if constexpr (SlopeScale<T>::kUsed) {
        float largest = fabsf(ds[0]);
#pragma unroll
        for (int r = 1; r < 16; ++r) largest = fmaxf(largest, fabsf(ds[r]));
        const float change = scale.follow(largest);
        if (change != 1.0f) scale_sums(acc, change);
        ds *= scale.factor();
    }
    add_columns<Tile, T>(acc, tile, row0, ds);
}

// Adds the waves' sums pairwise into the first wave's; `lds` holds half of the
// waves'.
template <int BLOCKS>
__device__ inline void join_waves(f32x16_attn (&acc)[BLOCKS], float* lds, int wave) {
    const int lane = lane_id();
    constexpr int kValues = BLOCKS * 16 * kWave;
#pragma unroll
    for (int active = kAttnWaves / 2; active > 0; active /= 2) {
        __syncthreads();
        if (wave >= active && wave < 2 * active) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    lds[(wave - active) * kValues + (b * 16 + r) * kWave + lane] = acc[b][r];
            }
        }
        __syncthreads();
        if (wave < active) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[b][r] += lds[wave * kValues + (b * 16 + r) * kWave + lane];
            }
        }
    }
    __syncthreads();
}
template <int DP> constexpr size_t kJoinBytes = kAttnWaves / 2 * (DP / 32) * 16 * kWave * sizeof(float);

// Stores column n of acc times `factor` into row n's `to` (dim channels);
// lanes without a row pass valid = false.
template <typename T, int BLOCKS>
__device__ inline void store_columns(const f32x16_attn (&acc)[BLOCKS], float factor, T* to, int dim, bool valid) {
    const int half = lane_id() >> 5;
    if (!valid) return;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * b + 8 * g + 4 * half;
            if (d >= dim) continue;
            RowVec<T, 4> v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v.set(i, acc[b][4 * g + i] * factor);
            v.store(to + d);
        }
    }
}

// Lanes (0 .. 31) whose column is not finite in either half.
__device__ inline uint32_t spoilt_columns(bool valid, bool finite) {
    const uint64_t spoilt = ballot(valid && !finite);
    return static_cast<uint32_t>(spoilt) | static_cast<uint32_t>(spoilt >> 32);
}

// (lse, delta) of a query row and head, where the keys' pass reads them: by key
// head, row and head, so that a tile's lie side by side.
__device__ inline long long query_state(const lattice_attention& a, uint32_t group, long long row, int head) {
    const uint32_t kv = head / group;
    return (static_cast<long long>(kv) * a.queries + row) * group + (head - kv * group);
}

// Adds the keys j0 .. of a tile to the sums of a wave's 32 rows.
template <typename T, int DP, int KT>
__device__ __forceinline__ void add_keys(const lattice_attention& a, int nk, const AttnOperand<T, DP>& q,
                                         const AttnOperand<T, DP>& d, const char* k_tile, float scale, float log_sum,
                                         float along, const AttnRows& w, const AttnMask& mask, int j0,
                                         f32x16_attn (&acc)[DP / 32], SlopeScale<T>& slopes) {
    typedef AttnTile<T, DP, KT> Tile;
    const char* v_tile = k_tile + Tile::kBytes;
#pragma unroll
    for (int row0 = 0; row0 < KT; row0 += 32) {
        const AttnView view = attn_view(a, nk, w.p_low, w.p_high, j0 + row0, 32);
        if (view == kSeesNone) continue;
        f32x16_attn p = tile_product<Tile, T, DP>(k_tile, row0, q, f32x16_attn{});
        f32x16_attn dp = tile_product<Tile, T, DP>(v_tile, row0, d, f32x16_attn{});
        if (view == kSeesSome) mask.apply(p, j0 + row0, j0 + row0 < a.sinks);
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = __builtin_amdgcn_exp2f(p[r] * scale - log_sum) * (dp[r] - along);
        add_slopes<Tile, T>(acc, slopes, k_tile, row0, dp);
    }
}

// The same, with the copy of the keys j_next .. (negative: none) into `next`
// under way: see attend_step.
template <typename T, int DP, int KT, typename Source>
__device__ __forceinline__ void grad_query_step(const lattice_attention& a, int nk, const Source& source, int j_next,
                                                char* __restrict__ next, const AttnOperand<T, DP>& q,
                                                const AttnOperand<T, DP>& d, const char* __restrict__ tile,
                                                float scale, float log_sum, float along, const AttnRows& w,
                                                const AttnMask& mask, int j0, f32x16_attn (&acc)[DP / 32],
                                                SlopeScale<T>& slopes) {
    if (j_next >= 0) source.copy(next, j_next, nk);
    add_keys<T, DP, KT>(a, nk, q, d, tile, scale, log_sum, along, w, mask, j0, acc, slopes);
}

// grad_q, laid out as the forward pass; keeps lse and delta for the keys' pass.
// FEW: 32 rows a block, whose tiles the waves take in turn, each with its own
// copies; their sums are joined.
template <typename T, int DP, int KT, bool FEW>
__global__ void __launch_bounds__(kAttnBlock, DP <= 64 || sizeof(T) == 2 ? 2 : 1)
grad_query_tiles(lattice_attention a, const T* __restrict__ out, const T* __restrict__ rest,
                 const float* __restrict__ lse, const T* __restrict__ grad_out, T* __restrict__ grad_q, float2* __restrict__ states) {
    typedef AttnTile<T, DP, KT> Tile;
    typedef AttnOperand<T, DP> Operand;
    constexpr int kBlocks = DP / 32;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int half = lane_id() >> 5;
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y;
    constexpr int kRows = FEW ? 32 : 32 * kAttnWaves;
    const AttnSlot t = attn_slot<kRows>(a, group, block_slot(1));
    const AttnSequence s = t.s;
    if (t.first >= t.rows) return;
    const float scale = exponent_scale(a);
    const AttnRows w = attn_rows(s, kv, group, t.first + (FEW ? 0 : 32 * wave));
    const long long row = static_cast<long long>(s.q0) + w.i;
    const long long at = row * a.heads + w.head;
    Operand q, d;
    q.load(static_cast<const T*>(a.q) + row * a.q_row_stride + w.head * a.q_head_stride, a.dim, w.valid,
           a.scale < 0.0f);
    d.load(grad_out + at * a.dim, a.dim, w.valid, false);
    float along = 0.0f;
    {
        Operand o;
        o.load(out + at * a.dim, a.dim, w.valid, false);
#pragma unroll
        for (int c = 0; c < Operand::kSteps; ++c) {
#pragma unroll
            for (int i = 0; i < Tile::kElems; ++i)
                along += static_cast<float>(o.f[c][i]) * static_cast<float>(d.f[c][i]);
        }
        if (rest) {
            // What rounding took from out would be a third of delta's error.
            o.load(rest + at * a.dim, a.dim, w.valid, false);
#pragma unroll
            for (int c = 0; c < Operand::kSteps; ++c) {
#pragma unroll
                for (int i = 0; i < Tile::kElems; ++i)
                    along += static_cast<float>(o.f[c][i]) * static_cast<float>(d.f[c][i]);
            }
        }
        along = halves_sum(along);
    }
    const float log_sum = w.valid ? lse[at] : INFINITY;
    if (w.valid && half == 0 && (!FEW || wave == 0))
        states[query_state(a, group, row, w.head)] = float2{log_sum, along};
    const AttnMask mask(a, s.nk, w.p);
    f32x16_attn acc[kBlocks] = {};
    SlopeScale<T> slopes;
    const int p_low = static_cast<int>(t.first / group) + s.shift();
    const int p_high = static_cast<int>((min(t.first + kRows, t.rows) - 1) / group) + s.shift();
    const AttnTiles tiles = attn_tiles<KT>(a, s.nk, p_low, p_high);
    constexpr int kThreads = FEW ? kWave : kAttnBlock, kStep = FEW ? kAttnWaves : 1;
    const KeyTiles<T, DP, KT, kThreads> source(a, s, kv, FEW ? lane_id() : threadIdx.x);
    if constexpr (!FEW) {
        if (tiles.count) source.copy(shared, tiles.tile(0) * KT, s.nk);
        wait_for_copies();
        __syncthreads();
    }
    for (int index = FEW ? wave : 0; index < tiles.count; index += kStep) {
        char* tile = shared + (FEW ? wave : index & 1) * 2 * Tile::kBytes;
        const int j0 = tiles.tile(index) * KT;
        if constexpr (FEW) {
            source.copy(tile, j0, s.nk);
            wait_for_copies();
            wave_fence();
            add_keys<T, DP, KT>(a, s.nk, q, d, tile, scale, log_sum, along, w, mask, j0, acc, slopes);
            wait_for_reads();
        } else {
            const int next = index + 1 < tiles.count ? tiles.tile(index + 1) * KT : -1;
            grad_query_step<T, DP, KT>(a, s.nk, source, next, shared + (~index & 1) * 2 * Tile::kBytes, q, d, tile,
                                       scale, log_sum, along, w, mask, j0, acc, slopes);
            wait_for_copies();
            __syncthreads();
        }
    }
    if constexpr (SlopeScale<T>::kUsed) scale_sums(acc, 1.0f / slopes.factor());
    if constexpr (FEW) {
        join_waves(acc, reinterpret_cast<float*>(shared), wave);
        if (wave != 0) return;
    }
    // A row that is not finite is made again from what it sees alone.
    uint32_t again = spoilt_columns(w.valid, finite_columns(acc, a.scale));
    store_columns(acc, a.scale, grad_q + at * a.dim, a.dim, w.valid && !(again >> (lane_id() & 31) & 1));
    while (again) {
        const int n = __ffs(again) - 1;
        again &= again - 1;
        grad_query_row<T>(a, s, __shfl(w.i, n), __shfl(w.head, n), lse, __shfl(along, n), grad_out, grad_q,
                          reinterpret_cast<AttnRowScratch*>(shared) + wave);
    }
}

// ROWS (query, head) pairs r0 .. of a sequence and key head in LDS: q and
// grad_out rows, and of each its lse (+inf past the rows there are, so that
// its shares are zero) less the shares' scale, -delta and position.
template <typename T, int DP, int ROWS>
struct QueryTile {
    typedef AttnTile<T, DP, ROWS> Tile;
    static constexpr int kBytes = 2 * Tile::kBytes + (ROWS * 12 + 127) / 128 * 128;

    __device__ static const float* states(const char* tile) {
        return reinterpret_cast<const float*>(tile + 2 * Tile::kBytes);
    }
};

// Copies them by THREADS threads.  A tile starts at a multiple of ROWS; where
// the heads of a group divide that, each starts with a group's first head and
// the places of its rows are the same but for the base.
template <typename T, int DP, int ROWS, int THREADS>
struct QueryTiles {
    typedef QueryTile<T, DP, ROWS> Queries;
    typedef typename Queries::Tile Tile;
    static constexpr int kCopies = Tile::copies(THREADS);
    const T *q, *grad_out;  // of the sequence's first query and the key head's first head
    const float2* states;
    long long q_stride, d_stride;
    int thread, wave, q_row, q_head, d_row, d_head, shift;
    GroupDivide by_group;
    bool aligned;
    int own_query;
    int q_offsets[kCopies], d_offsets[kCopies];

    // What a thread holds of the states until it stores them.
    struct State {
        float lse, delta;
        int position;
    };

    __device__ QueryTiles(const lattice_attention& a, const AttnSequence& s, int kv, uint32_t heads,
                          const float2* all_states, const T* all_grad_out, int of_thread)
        : by_group(heads) {
        constexpr int kSize = sizeof(T);
        thread = of_thread;
        wave = __builtin_amdgcn_readfirstlane(thread / kWave);
        const uint32_t group = heads;
        shift = s.shift();
        q_stride = a.q_row_stride;
        d_stride = static_cast<long long>(a.heads) * a.dim;
        q = static_cast<const T*>(a.q) + s.q0 * q_stride + static_cast<long long>(kv) * group * a.q_head_stride;
        grad_out = all_grad_out + s.q0 * d_stride + static_cast<long long>(kv) * group * a.dim;
        states = all_states + (static_cast<long long>(kv) * a.queries + s.q0) * group;
        q_row = static_cast<int>(a.q_row_stride) * kSize;
        q_head = static_cast<int>(a.q_head_stride) * kSize;
        d_row = a.heads * a.dim * kSize;
        d_head = a.dim * kSize;
        aligned = ROWS % group == 0;
        places(0);
    }
    __device__ void places(uint32_t h0) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const uint32_t n = h0 + Tile::template copy_row<THREADS>(i, thread);
            const int query = by_group(n), head = n - query * by_group.group;
            const int piece = Tile::template copy_piece<THREADS>(i, thread, d_head / 16);
            q_offsets[i] = query * q_row + head * q_head + piece;
            d_offsets[i] = query * d_row + head * d_head + piece;
        }
        own_query = by_group(h0 + thread);
    }
    // Starts the copies of pairs r0 .. of `rows`; rows past them hold other
    // rows or zeros, whose shares are zero.
    __device__ State copy(char* to, uint32_t r0, uint32_t rows) {
        const uint32_t group = by_group.group, i0 = by_group(r0), h0 = r0 - i0 * group;
        if (!aligned) places(h0);
        const uint32_t count = min(rows - r0, static_cast<uint32_t>(ROWS));
        // The range ends with the last query's last head.
        const int last = by_group(h0 + count - 1);
        Tile::template copy<THREADS>(to, q + i0 * q_stride,
                                     last * q_row + static_cast<int>(group - 1) * q_head + d_head, q_offsets, wave);
        Tile::template copy<THREADS>(to + Tile::kBytes, grad_out + i0 * d_stride,
                                     last * d_row + static_cast<int>(group) * d_head, d_offsets, wave);
        State state{INFINITY, 0.0f, static_cast<int>(i0) + own_query + shift};
        if (thread < count) {
            const float2 kept = states[r0 + thread];
            state.lse = kept.x;
            state.delta = kept.y;
        }
        return state;
    }
    __device__ void store(char* to, const State& state) const {
        if (thread >= ROWS) return;
        float* at = reinterpret_cast<float*>(to + 2 * Tile::kBytes);
        at[thread] = state.lse - kShareLog2<T>;
        at[ROWS + thread] = -state.delta;
        reinterpret_cast<int*>(at)[2 * ROWS + thread] = state.position;
    }
};

// Which positions of a tile a lane's key is seen from: lo .. hi; `below`,
// `above`: some tile's position is below some lane's lo, above some hi.
struct QueryMask {
    int lo, hi;
    bool below, above;
};

// Adds the queries of a tile to a wave's 32 keys.  (A form of its own for tiles
// without a mask costs more registers than it saves branches: 855 for 787 us at
// heads of 128, 133 for 121 at 64.)
template <typename T, int DP, int QT>
__device__ inline void add_queries(const char* tile, const AttnOperand<T, DP>& k, const AttnOperand<T, DP>& v,
                                   float scale, const QueryMask& mask, f32x16_attn (&acc_k)[DP / 32],
                                   f32x16_attn (&acc_v)[DP / 32], SlopeScale<T>& slopes) {
    typedef QueryTile<T, DP, QT> Queries;
    typedef typename Queries::Tile Tile;
    const int half = lane_id() >> 5;
    const char* d_tile = tile + Tile::kBytes;
    const float* states = Queries::states(tile);
#pragma unroll
    for (int part = 0; part < QT / 32; ++part) {
        f32x16_attn p = tile_product<Tile, T, DP>(tile, 32 * part, k, f32x16_attn{});
        // dp - delta.  The product may start from -delta; with one wave a SIMD
        // (heads of 128) that read would hold it up, and delta is added after.
        constexpr bool kFromDelta = DP < 128;
        f32x16_attn ds = {};
        if constexpr (kFromDelta) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 delta = *reinterpret_cast<const float4*>(states + QT + 32 * part + 8 * g + 4 * half);
                ds[4 * g] = delta.x;
                ds[4 * g + 1] = delta.y;
                ds[4 * g + 2] = delta.z;
                ds[4 * g + 3] = delta.w;
            }
        }
        ds = tile_product<Tile, T, DP>(d_tile, 32 * part, v, ds);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int row = 32 * part + 8 * g + 4 * half;
            if (mask.below || mask.above) {
                const int4 at = *reinterpret_cast<const int4*>(states + 2 * QT + row);
                const int position[4] = {at.x, at.y, at.z, at.w};
                // One end at a time where registers are left for the branches (8 heads of
                // 80: 122.5 -> 117.7 us; of 128: 782 -> 818).
                if constexpr (DP < 128) {
                    if (mask.below) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[4 * g + i] = position[i] < mask.lo ? -INFINITY : p[4 * g + i];
                    }
                    if (mask.above) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[4 * g + i] = position[i] > mask.hi ? -INFINITY : p[4 * g + i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (position[i] < mask.lo || position[i] > mask.hi) p[4 * g + i] = -INFINITY;
                }
            }
            const float4 lse = *reinterpret_cast<const float4*>(states + row);
            const float log_sum[4] = {lse.x, lse.y, lse.z, lse.w};
            float4 delta{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (!kFromDelta) delta = *reinterpret_cast<const float4*>(states + QT + row);
            const float along[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * g + i;
                p[r] = __builtin_amdgcn_exp2f(p[r] * scale - log_sum[i]);
                ds[r] = p[r] * (kFromDelta ? ds[r] : ds[r] + along[i]);
            }
        }
        add_columns<Tile, T>(acc_v, d_tile, 32 * part, p);
        add_slopes<Tile, T>(acc_k, slopes, tile, 32 * part, ds);
    }
}

// The same (none: nothing is added), with the copy of the queries r_next ..
// into `next` under way: see attend_step.  What it holds of their states.
template <typename T, int DP, int QT, typename Source>
__device__ __forceinline__ typename Source::State
grad_key_step(Source& source, bool more, uint32_t r_next, uint32_t rows, char* __restrict__ next,
              const char* __restrict__ tile, const AttnOperand<T, DP>& k, const AttnOperand<T, DP>& v, float scale,
              const QueryMask& mask, bool none, f32x16_attn (&acc_k)[DP / 32], f32x16_attn (&acc_v)[DP / 32],
              SlopeScale<T>& slopes) {
    typename Source::State state{};
    if (more) state = source.copy(next, r_next, rows);
    if (!none) add_queries<T, DP, QT>(tile, k, v, scale, mask, acc_k, acc_v, slopes);
    return state;
}

template <int DP> constexpr int kFirstValues = 2 * DP * 32;

template <int BLOCKS>
__device__ inline void store_part(float* to, const f32x16_attn (&acc_k)[BLOCKS], const f32x16_attn (&acc_v)[BLOCKS]) {
    const int lane = lane_id();
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            to[(b * 16 + r) * kWave + lane] = acc_k[b][r];
            to[((BLOCKS + b) * 16 + r) * kWave + lane] = acc_v[b][r];
        }
    }
}

// Two waves a SIMD leave 256 registers a lane: enough up to heads of 96 (25k
// rows of 8 heads of 80, window 330: 123 us, with one wave 228).  At 128 the
// sums alone take half of them and a second wave spills (8k rows of 16 heads,
// window 4096: 1735 us, with one wave 787; with the keys read from LDS 959).
template <typename T, int DP> constexpr int kKeyWaves = DP <= 64 || (DP <= 96 && sizeof(T) == 2) ? 2 : 1;

// The part of a slot: each wave takes every fourth tile of 32 pairs.
template <typename T, int DP, int WAVES>
__global__ void __launch_bounds__(kAttnBlock, WAVES)
grad_first_keys(lattice_attention a, const float2* __restrict__ states, const T* __restrict__ grad_out,
                FirstParts parts) {
    constexpr int QT = 32;
    constexpr int kBlocks = DP / 32;
    typedef QueryTile<T, DP, QT> Queries;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y, j0 = blockIdx.z * 32;
    const AttnSlot t = attn_slot<kFirstRows>(a, group, blockIdx.x);
    const AttnSequence s = t.s;
    const int j = j0 + (lane & 31);
    if (t.first >= t.rows || j0 >= min(a.sinks, s.nk)) return;
    const bool valid = j < s.nk;
    const long long row = static_cast<long long>(s.k0) + min(j, s.nk - 1);
    AttnOperand<T, DP> k, v;
    k.load(static_cast<const T*>(a.k) + row * a.k_row_stride + kv * a.k_head_stride, a.dim, valid,
           a.scale < 0.0f);
    v.load(static_cast<const T*>(a.v) + row * a.v_row_stride + kv * a.v_head_stride, a.dim, valid, false);
    const float scale = exponent_scale(a);
    f32x16_attn acc_k[kBlocks] = {}, acc_v[kBlocks] = {};
    SlopeScale<T> slopes;
    QueryTiles<T, DP, QT, kWave> source(a, s, kv, group, states, grad_out, lane);
    // From the first pair whose query lies past the window of key j0.
    const int i_from = max(0, j0 + a.left + 1 - s.shift());
    const uint32_t from = max(t.first, static_cast<uint32_t>(min(i_from, s.nq)) * group / QT * QT);
    const uint32_t to = min(t.first + kFirstRows, t.rows);
    char* tile = shared + wave * Queries::kBytes;
    const QueryMask mask{j + a.left + 1, INT_MAX, true, false};
    for (uint32_t base = from; base < to; base += QT * kAttnWaves) {
        const uint32_t r0 = base + QT * wave;
        if (r0 >= to) break;
        source.store(tile, source.copy(tile, r0, to));
        wait_for_copies();
        wave_fence();
        add_queries<T, DP, QT>(tile, k, v, scale, mask, acc_k, acc_v, slopes);
        wait_for_reads();
    }
    if constexpr (SlopeScale<T>::kUsed) scale_sums(acc_k, 1.0f / slopes.factor());
    join_waves(acc_k, reinterpret_cast<float*>(shared), wave);
    join_waves(acc_v, reinterpret_cast<float*>(shared), wave);
    if (wave == 0) store_part(parts.past_of(a, blockIdx.x, kv, blockIdx.z, kFirstValues<DP>), acc_k, acc_v);
}

// Adds the parts of 32 first keys and eight channels of a sequence and key
// head: 256 values of dk and as many of dv, which lie side by side in a part.
// Four groups of threads take a quarter of the slots each, in slot order, after
// the window's part; their sums are added in order.
constexpr int kJoinGroups = 4, kJoinBlock = kJoinGroups * kAttnBlock;
template <typename T, int DP>
__global__ void __launch_bounds__(kJoinBlock)
join_first_keys(lattice_attention a, const float* __restrict__ lse, const float2* __restrict__ states,
                const T* __restrict__ grad_out, FirstParts parts, T* __restrict__ grad_k, T* __restrict__ grad_v) {
    __shared__ AttnRowScratch scratch[kAttnWaves];
    __shared__ float2 sums[kJoinGroups - 1][kAttnBlock];
    __shared__ uint32_t spoilt;
    const uint32_t group = a.heads / a.kv_heads;
    const int e = blockIdx.x + 1, kv = blockIdx.y;
    const int tile = blockIdx.z / (DP / 8), eighth = blockIdx.z % (DP / 8), j0 = tile * 32, d0 = eighth * 8;
    const AttnSequence s = attn_sequence(a, e);
    const int keys = min(a.sinks, s.nk);
    if (j0 >= keys || d0 >= a.dim) return;
    const uint32_t quarter = threadIdx.x / kAttnBlock, thread = threadIdx.x % kAttnBlock;
    const int lane = lane_id(), wave = thread / kWave;
    const int j = j0 + (lane & 31);
    const uint32_t slot = s.q0 * group / kFirstRows + e, slots = (s.nq * group + kFirstRows - 1) / kFirstRows;
    const int of_k = eighth * kAttnBlock + thread, of_v = of_k + DP * 32;
    float sum_k = 0.0f, sum_v = 0.0f;
    if (quarter == 0) {
        const float* at = parts.window_of(a, e, kv, tile, kFirstValues<DP>);
        sum_k = at[of_k];
        sum_v = at[of_v];
    }
    constexpr int kAhead = 8;  // parts in flight
    const uint32_t share_slots = (slots + kJoinGroups - 1) / kJoinGroups;
    const uint32_t to = min(slots, (quarter + 1) * share_slots);
    for (uint32_t u = quarter * share_slots; u < to; u += kAhead) {
        float past_k[kAhead], past_v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const bool here = u + i < to;
            const float* past = parts.past_of(a, slot + (here ? u + i : 0), kv, tile, kFirstValues<DP>);
            past_k[i] = here ? past[of_k] : 0.0f;
            past_v[i] = here ? past[of_v] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            sum_k += past_k[i];
            sum_v += past_v[i];
        }
    }
    if (quarter > 0) sums[quarter - 1][thread] = float2{sum_k, sum_v};
    if (threadIdx.x == 0) spoilt = 0;
    __syncthreads();
    if (quarter == 0) {
#pragma unroll
        for (int g = 0; g < kJoinGroups - 1; ++g) {
            sum_k += sums[g][thread].x;
            sum_v += sums[g][thread].y;
        }
    }
    const float share = __builtin_amdgcn_exp2f(-kShareLog2<T>);
    sum_k *= a.scale * share;
    sum_v *= share;
    if (quarter == 0 && j < keys && !(fabsf(sum_k) < INFINITY && fabsf(sum_v) < INFINITY))
        atomicOr(&spoilt, 1u << (lane & 31));
    __syncthreads();
    if (quarter > 0) return;
    const uint32_t again = spoilt;
    if (j < keys && !(again >> (lane & 31) & 1)) {
        const int d = d0 + 4 * (lane >> 5) + wave;
        const long long to = ((static_cast<long long>(s.k0) + j) * a.kv_heads + kv) * a.dim + d;
        if (d < a.dim) {
            grad_k[to] = static_cast<T>(sum_k);
            grad_v[to] = static_cast<T>(sum_v);
        }
    }
    for (int n = wave; n < 32; n += kAttnWaves) {
        if (again >> n & 1)
            grad_key_row<T>(a, s, j0 + n, kv, lse, states, grad_out, grad_k, grad_v, &scratch[wave], d0, d0 + 8);
    }
}

// grad_k and grad_v: 128 keys a block, 32 a wave, over the tiles of (query,
// head) pairs that see them.  FEW: 32 keys a block, whose tiles the waves take in
// turn, each with its own copies; their sums are joined.
template <typename T, int DP, int QT, bool FEW, int WAVES>
__global__ void __launch_bounds__(kAttnBlock, WAVES)
grad_key_tiles(lattice_attention a, const float* __restrict__ lse, const float2* __restrict__ states,
               const T* __restrict__ grad_out, FirstParts parts, T* __restrict__ grad_k, T* __restrict__ grad_v) {
    constexpr int kBlocks = DP / 32;
    constexpr int kKeys = FEW ? 32 : 32 * kAttnWaves, kThreads = FEW ? kWave : kAttnBlock;
    typedef QueryTile<T, DP, QT> Queries;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y;
    const auto slot_of = [](int start, int e) { return static_cast<uint32_t>(start) / kKeys + e; };
    const uint32_t slot = block_slot(1);
    const int e = key_rows(a).find(slot, slot_of);
    const AttnSequence s = attn_sequence(a, e);
    const int owned = max(0, key_rows(a).start(e + 1) - s.k0);
    const int j0 = slot_first<kKeys>(slot, slot_of(s.k0, e), owned);
    if (j0 >= owned) return;
    const int j_wave = j0 + (FEW ? 0 : 32 * wave), j = j_wave + (lane & 31);
    const bool valid = j < s.nk;
    const long long row = static_cast<long long>(s.k0) + min(j, owned - 1);
    AttnOperand<T, DP> k, v;
    k.load(static_cast<const T*>(a.k) + row * a.k_row_stride + kv * a.k_head_stride, a.dim, valid,
           a.scale < 0.0f);
    v.load(static_cast<const T*>(a.v) + row * a.v_row_stride + kv * a.v_head_stride, a.dim, valid, false);
    const float scale = exponent_scale(a);
    f32x16_attn acc_k[kBlocks] = {}, acc_v[kBlocks] = {};
    SlopeScale<T> slopes;
    QueryTiles<T, DP, QT, kThreads> source(a, s, kv, group, states, grad_out, FEW ? lane : threadIdx.x);
    const uint32_t rows = s.nq * group;
    // The pairs whose window holds a key of the block.
    const int i_from = max(0, j0 - a.right - s.shift());
    const int i_to = min(s.nq, min(j0 + kKeys, s.nk) + a.left - s.shift());
    const bool any = j0 < s.nk && i_from < i_to;
    const uint32_t from = any ? i_from * group / QT : 0;
    const uint32_t window_to = any ? (i_to * group + QT - 1) / QT : 0;
    // Without a pass of their own, the first keys' other pairs follow.
    const int past_from = max(0, j0 + a.left + 1 - s.shift());
    const bool rest = parts.tiles == 0 && j0 < min(a.sinks, s.nk) && past_from < s.nq;
    const uint32_t past = rest ? past_from * group / QT : 0;
    const uint32_t past_to = rest ? (rows + QT - 1) / QT : 0;
    const int window_tiles = static_cast<int>(window_to - from);
    const int count = window_tiles + static_cast<int>(past_to - past);
    const auto first_row = [&](int index) {
        return (index < window_tiles ? from + index : past + (index - window_tiles)) * QT;
    };
    constexpr int kStep = FEW ? kAttnWaves : 1;
    if constexpr (!FEW) {
        if (count > 0) source.store(shared, source.copy(shared, first_row(0), rows));
        wait_for_copies();
        __syncthreads();
    }
    for (int index = FEW ? wave : 0; index < count; index += kStep) {
        char* tile = shared + (FEW ? wave : index & 1) * Queries::kBytes;
        const uint32_t r0 = first_row(index);
        // In the window, or past it: of the first keys alone.
        const bool outside = index >= window_tiles;
        const int lo = !outside ? j - a.right : j < a.sinks ? j + a.left + 1 : INT_MAX;
        const int hi = outside ? INT_MAX : j + a.left;
        const int p_low = static_cast<int>(source.by_group(r0)) + s.shift();
        const int p_high = static_cast<int>(source.by_group(min(r0 + QT, rows) - 1)) + s.shift();
        const bool none = outside ? j_wave >= a.sinks || p_high <= j_wave + a.left
                                  : p_high < j_wave - a.right || p_low > j_wave + 31 + a.left;
        const QueryMask mask{lo, hi, outside || p_low < j_wave + 31 - a.right, !outside && p_high > j_wave + a.left};
        if constexpr (FEW) {
            source.store(tile, source.copy(tile, r0, rows));
            wait_for_copies();
            wave_fence();
            if (!none) add_queries<T, DP, QT>(tile, k, v, scale, mask, acc_k, acc_v, slopes);
            wait_for_reads();
        } else {
            char* next = shared + (~index & 1) * Queries::kBytes;
            const bool more = index + 1 < count;
            const auto state = grad_key_step<T, DP, QT>(source, more, more ? first_row(index + 1) : 0, rows, next, tile,
                                                        k, v, scale, mask, none, acc_k, acc_v, slopes);
            if (more) source.store(next, state);
            wait_for_copies();
            __syncthreads();
        }
    }
    if constexpr (SlopeScale<T>::kUsed) scale_sums(acc_k, 1.0f / slopes.factor());
    if constexpr (FEW) {
        join_waves(acc_k, reinterpret_cast<float*>(shared), wave);
        join_waves(acc_v, reinterpret_cast<float*>(shared), wave);
        if (wave != 0) return;
    }
    const int first_keys = parts.tiles ? min(a.sinks, s.nk) : 0;
    if (j_wave < first_keys) store_part(parts.window_of(a, e, kv, j_wave / 32, kFirstValues<DP>), acc_k, acc_v);
    // Keys past the sequence's get zeros; a key whose sums are not finite is
    // made again from the queries that see it alone.
    const float share = __builtin_amdgcn_exp2f(-kShareLog2<T>);
    const float slope = a.scale * share;
    const bool finite = finite_columns(acc_k, slope) && finite_columns(acc_v, share);
    uint32_t again = spoilt_columns(valid && j >= first_keys, finite);
    const bool mine = j < owned && j >= first_keys && !(again >> (lane & 31) & 1);
    const long long at = (row * a.kv_heads + kv) * a.dim;
    if (!valid) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc_k[b] = acc_v[b] = f32x16_attn{};
    }
    store_columns(acc_k, slope, grad_k + at, a.dim, mine);
    store_columns(acc_v, share, grad_v + at, a.dim, mine);
    while (again) {
        const int n = __ffs(again) - 1;
        again &= again - 1;
        grad_key_row<T>(a, s, j_wave + n, kv, lse, states, grad_out, grad_k, grad_v,
                        reinterpret_cast<AttnRowScratch*>(shared) + wave);
    }
}

template <typename T, int DP, bool FEW>
int launch_grad_query(const lattice_attention& a, const T* out, const T* rest, const float* lse, const T* grad_out,
                      T* grad_q, float2* states, hipStream_t stream) {
    constexpr int kTile = sizeof(T) == 2 && !FEW ? 64 : 32, kRows = FEW ? 32 : 32 * kAttnWaves;
    constexpr size_t kLds = std::max({(FEW ? kAttnWaves : 2) * size_t{2} * AttnTile<T, DP, kTile>::kBytes,
                                      FEW ? kJoinBytes<DP> : 0, kAttnWaves * sizeof(AttnRowScratch)});
    static_assert(kLds <= 160 * 1024);
    const auto kernel = grad_query_tiles<T, DP, kTile, FEW>;
    LATTICE_HIP_TRY(allow_lds(reinterpret_cast<const void*>(kernel), kLds));
    const long long slots = static_cast<long long>(a.queries) * (a.heads / a.kv_heads) / kRows + a.sequences + 2;
    kernel<<<slot_grid(slots, a.kv_heads, 1), kAttnBlock, kLds, stream>>>(a, out, rest, lse, grad_out,
                                                                                        grad_q, states);
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T, int DP, bool FEW>
int launch_grad_keys(const lattice_attention& a, const float* lse, const float2* states, const T* grad_out,
                     const FirstParts& parts, T* grad_k, T* grad_v, hipStream_t stream) {
    constexpr int kTile = sizeof(T) == 2 && !FEW ? 64 : 32, kKeys = FEW ? 32 : 32 * kAttnWaves;
    constexpr size_t kLds = std::max({(FEW ? kAttnWaves : 2) * size_t{QueryTile<T, DP, kTile>::kBytes},
                                      FEW ? kJoinBytes<DP> : 0, kAttnWaves * sizeof(AttnRowScratch)});
    static_assert(kLds <= 160 * 1024);
    const auto kernel = grad_key_tiles<T, DP, kTile, FEW, FEW ? 1 : kKeyWaves<T, DP>>;
    LATTICE_HIP_TRY(allow_lds(reinterpret_cast<const void*>(kernel), kLds));
    const long long slots = a.keys / kKeys + a.sequences + 2;
    kernel<<<slot_grid(slots, a.kv_heads, 1), kAttnBlock, kLds, stream>>>(a, lse, states, grad_out,
                                                                                        parts, grad_k, grad_v);
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T, int DP>
int launch_grad(const lattice_attention& a, const GradLayout& l, const T* out, const T* rest, const float* lse,
                const T* grad_out, T* grad_q, T* grad_k, T* grad_v, float2* states, const FirstParts& parts, hipStream_t stream) {
    if (a.queries) {
        const int rc = grad_few(static_cast<long long>(a.queries) * a.heads)
                           ? launch_grad_query<T, DP, true>(a, out, rest, lse, grad_out, grad_q, states, stream)
                           : launch_grad_query<T, DP, false>(a, out, rest, lse, grad_out, grad_q, states, stream);
        if (rc != LATTICE_OK) return rc;
    }
    if (a.keys == 0) return LATTICE_OK;
    if (l.first_tiles) {
        constexpr size_t kLds = std::max<size_t>(kAttnWaves * QueryTile<T, DP, 32>::kBytes, kJoinBytes<DP>);
        static_assert(kLds <= 160 * 1024);
        const auto kernel = grad_first_keys<T, DP, kKeyWaves<T, DP>>;
        LATTICE_HIP_TRY(allow_lds(reinterpret_cast<const void*>(kernel), kLds));
        kernel<<<dim3(l.first_slots, a.kv_heads, l.first_tiles), kAttnBlock, kLds, stream>>>(a, states, grad_out,
                                                                                            parts);
        LATTICE_LAUNCH_CHECK();
    }
    const int rc = grad_few(static_cast<long long>(a.keys) * a.kv_heads)
                       ? launch_grad_keys<T, DP, true>(a, lse, states, grad_out, parts, grad_k, grad_v, stream)
                       : launch_grad_keys<T, DP, false>(a, lse, states, grad_out, parts, grad_k, grad_v, stream);
    if (rc != LATTICE_OK) return rc;
    if (l.first_tiles && a.sequences) {
        join_first_keys<T, DP><<<dim3(a.sequences, a.kv_heads, l.first_tiles * (DP / 8)), kJoinBlock, 0, stream>>>(
            a, lse, states, grad_out, parts, grad_k, grad_v);
        LATTICE_LAUNCH_CHECK();
    }
    return LATTICE_OK;
}

}  // namespace

template <typename T>
int attend_grad(const lattice_attention& a, const GradLayout& l, const void* out, const void* out_rest,
                const float* lse, const void* grad_out, void* grad_q, void* grad_k, void* grad_v, float2* states,
                const FirstParts& parts, hipStream_t stream) {
    const T* o = static_cast<const T*>(out);
    const T* rest = sizeof(T) == 4 ? nullptr : static_cast<const T*>(out_rest);
    const T* dy = static_cast<const T*>(grad_out);
    T* dq = static_cast<T*>(grad_q);
    T* dk = static_cast<T*>(grad_k);
    T* dv = static_cast<T*>(grad_v);
    if (a.dim <= 32) return launch_grad<T, 32>(a, l, o, rest, lse, dy, dq, dk, dv, states, parts, stream);
    if (a.dim <= 64) return launch_grad<T, 64>(a, l, o, rest, lse, dy, dq, dk, dv, states, parts, stream);
    if (a.dim <= 96) return launch_grad<T, 96>(a, l, o, rest, lse, dy, dq, dk, dv, states, parts, stream);
    return launch_grad<T, 128>(a, l, o, rest, lse, dy, dq, dk, dv, states, parts, stream);
}

}  // namespace lattice
