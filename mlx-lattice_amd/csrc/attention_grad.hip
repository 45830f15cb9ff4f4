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

#include "attention_tiles.h"

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
template <>
struct SlopeScale<_Float16> {
    static constexpr bool kUsed = true;
    int exponent = kNone;
    static constexpr int kNone = 1000;
    static constexpr int kMost = 40;
    __device__ float factor() const { return exponent == kNone ? 1.0f : ldexpf(1.0f, exponent); }
    // Follows the wave's largest slope; the factor by which the sums so far
    // have to be scaled.
    __device__ float follow(float largest) {
        if (exponent != kNone && !__any(ldexpf(largest, exponent) > 32768.0f)) return 1.0f;
        largest = wave_max(largest);
        if (!(largest > 0.0f) || largest == INFINITY) return 1.0f;
        // The largest becomes 2^11 .. 2^12.
        const int next = min(kMost, 12 - (__float_as_int(largest) >> 23 & 255) + 126);
        const float change = exponent == kNone ? 1.0f : ldexpf(1.0f, next - exponent);
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

// Whether the column's channels below dim are finite.
template <int BLOCKS>
__device__ inline bool finite_columns(const f32x16_attn (&acc)[BLOCKS], float factor, int dim) {
    bool finite = true;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            finite = finite && (32 * b + result_row(r) >= dim || fabsf(acc[b][r] * factor) < INFINITY);
    }
    return finite;
}

// Lanes (0 .. 31) whose column is not finite in either half.
__device__ inline uint32_t spoilt_columns(bool valid, bool finite) {
    const uint64_t spoilt = ballot(valid && !finite);
    return static_cast<uint32_t>(spoilt) | static_cast<uint32_t>(spoilt >> 32);
}

// grad_q, laid out as the forward pass; keeps delta for the keys' pass.
template <typename T, int DP, int KT>
__global__ void __launch_bounds__(kAttnBlock, DP <= 64 || sizeof(T) == 2 ? 2 : 1)
grad_query_tiles(lattice_attention a, const T* __restrict__ out, const float* __restrict__ lse,
                 const T* __restrict__ grad_out, T* __restrict__ grad_q, float* __restrict__ delta) {
    typedef AttnTile<T, DP, KT> Tile;
    typedef AttnOperand<T, DP> Operand;
    constexpr int kBlocks = DP / 32;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int half = lane_id() >> 5;
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y;
    const AttnSlot t = attn_slot<32 * kAttnWaves>(a, group, blockIdx.x);
    const AttnSequence s = t.s;
    if (t.first >= t.rows) return;
    const float scale = fabsf(a.scale) * kAttnLog2e;
    const AttnRows w = attn_rows(s, kv, group, t.first + 32 * wave);
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
        along += other_half(along);
    }
    if (w.valid && half == 0) delta[at] = along;
    const float log_sum = w.valid ? lse[at] : INFINITY;
    f32x16_attn acc[kBlocks] = {};
    SlopeScale<T> slopes;
    const int p_low = static_cast<int>(t.first / group) + s.shift();
    const int p_high = static_cast<int>((min(t.first + 32 * kAttnWaves, t.rows) - 1) / group) + s.shift();
    const AttnTiles tiles = attn_tiles<KT>(a, s.nk, p_low, p_high);
    const T* keys = static_cast<const T*>(a.k) + s.k0 * a.k_row_stride + kv * a.k_head_stride;
    const T* values = static_cast<const T*>(a.v) + s.k0 * a.v_row_stride + kv * a.v_head_stride;
    const int pieces = a.dim * static_cast<int>(sizeof(T)) / 16;
    const auto copy = [&](int index) {
        const int j0 = tiles.tile(index) * KT;
        char* to = shared + (index & 1) * 2 * Tile::kBytes;
        Tile::template load<kAttnBlock>(to, keys + j0 * a.k_row_stride, a.k_row_stride, s.nk - j0, pieces,
                                        threadIdx.x);
        Tile::template load<kAttnBlock>(to + Tile::kBytes, values + j0 * a.v_row_stride, a.v_row_stride, s.nk - j0,
                                        pieces, threadIdx.x);
    };
    if (tiles.count) copy(0);
    __syncthreads();
    for (int index = 0; index < tiles.count; ++index) {
        if (index + 1 < tiles.count) copy(index + 1);
        const int j0 = tiles.tile(index) * KT;
        const char* k_tile = shared + (index & 1) * 2 * Tile::kBytes;
        const char* v_tile = k_tile + Tile::kBytes;
        const bool none = j0 > w.p_high + a.right || (j0 + KT - 1 < w.p_low - a.left && j0 >= a.sinks);
        const bool all = j0 + KT <= s.nk && j0 + KT - 1 <= w.p_low + a.right &&
                         (j0 >= w.p_high - a.left || j0 + KT <= a.sinks);
        if (!none) {
#pragma unroll
            for (int part = 0; part < KT / 32; ++part) {
                f32x16_attn p = tile_product<Tile, T, DP>(k_tile, 32 * part, q);
                f32x16_attn dp = tile_product<Tile, T, DP>(v_tile, 32 * part, d);
                if (!all) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!attn_visible(a, s.nk, w.p, j0 + 32 * part + result_row(r))) p[r] = -INFINITY;
                }
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    dp[r] = __builtin_amdgcn_exp2f(p[r] * scale - log_sum) * (dp[r] - along);
                add_slopes<Tile, T>(acc, slopes, k_tile, 32 * part, dp);
            }
        }
        __syncthreads();
    }
    // A row that is not finite is made again from what it sees alone.
    const float factor = a.scale / slopes.factor();
    uint32_t again = spoilt_columns(w.valid, finite_columns(acc, factor, a.dim));
    store_columns(acc, factor, grad_q + at * a.dim, a.dim, w.valid && !(again >> (lane_id() & 31) & 1));
    while (again) {
        const int n = __ffs(again) - 1;
        again &= again - 1;
        grad_query_row<T>(a, s, __shfl(w.i, n), __shfl(w.head, n), lse, __shfl(along, n), grad_out, grad_q,
                          reinterpret_cast<AttnRowScratch*>(shared) + wave);
    }
}

// The (query, head) pairs r0 .. r0 + ROWS of a sequence and key head, staged
// in LDS: q and grad_out rows, and of each its lse (+inf past the rows there
// are, so that its shares are zero), delta and position.
template <typename T, int DP, int ROWS>
struct QueryTile {
    typedef AttnTile<T, DP, ROWS> Tile;
    static constexpr int kStateBytes = ROWS * 12;
    static constexpr int kBytes = 2 * Tile::kBytes + (kStateBytes + 127) / 128 * 128;

    // What a thread holds of the states until it stores them.
    struct State {
        float lse, delta;
        int position;
    };

    template <int THREADS>
    __device__ static State load(char* to, const lattice_attention& a, const AttnSequence& s, int kv, uint32_t group,
                                 uint32_t r0, uint32_t rows, const float* lse, const float* delta, const T* grad_out,
                                 int pieces, int thread) {
        const uint32_t i0 = r0 / group, h0 = r0 - i0 * group;
        const long long first = static_cast<long long>(s.q0) + i0;
        const int count = static_cast<int>(min(rows - r0, static_cast<uint32_t>(ROWS)));
        copy<THREADS>(to, static_cast<const T*>(a.q) + first * a.q_row_stride + kv * group * a.q_head_stride,
                      a.q_row_stride, a.q_head_stride, h0, group, count, pieces, thread);
        copy<THREADS>(to + Tile::kBytes, grad_out + (first * a.heads + kv * group) * a.dim,
                      static_cast<long long>(a.heads) * a.dim, a.dim, h0, group, count, pieces, thread);
        State state{INFINITY, 0.0f, 0};
        if (thread < ROWS) {
            const uint32_t n = h0 + thread, i = n / group;
            state.position = static_cast<int>(i0 + i) + s.shift();
            if (thread < count) {
                const long long at = (first + i) * a.heads + kv * group + (n - i * group);
                state.lse = lse[at];
                state.delta = delta[at];
            }
        }
        return state;
    }
    __device__ static void store(char* to, const State& state, int thread) {
        if (thread >= ROWS) return;
        float* states = reinterpret_cast<float*>(to + 2 * Tile::kBytes);
        states[thread] = state.lse;
        states[ROWS + thread] = state.delta;
        reinterpret_cast<int*>(states)[2 * ROWS + thread] = state.position;
    }
    __device__ static const float* states(const char* tile) {
        return reinterpret_cast<const float*>(tile + 2 * Tile::kBytes);
    }

  private:
    // Tile::load for rows n = h0 .. of (n / group, n % group).
    template <int THREADS>
    __device__ static void copy(char* to, const T* from, long long row_stride, long long head_stride, uint32_t h0,
                                uint32_t group, int rows, int pieces, int thread) {
        constexpr int kRange = 1 << 30;
        const __amdgpu_buffer_rsrc_t rsrc =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(from), 0, kRange, 0x00020000);
        const int row_bytes = static_cast<int>(row_stride * static_cast<long long>(sizeof(T)));
        const int head_bytes = static_cast<int>(head_stride * static_cast<long long>(sizeof(T)));
        const int wave = __builtin_amdgcn_readfirstlane(thread / kWave);
#pragma unroll
        for (int i = 0; i < Tile::kBytes / (THREADS * 16); ++i) {
            const int first = (i * (THREADS / kWave) + wave) * kWave;
            const int at = first + lane_id();
            const int row = at / Tile::kPieces;
            const int piece = (at % Tile::kPieces) ^ Tile::mix(row);
            const uint32_t n = h0 + row;
            const int query = group == 1 ? n : n / group;
            const int head = n - query * group;
            const int offset = row < rows && piece < pieces ? query * row_bytes + head * head_bytes + piece * 16
                                                            : kRange;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rsrc, (__attribute__((address_space(3))) void*)(to + first * 16), 16, offset, 0, 0, 0);
        }
    }
};

// Adds the queries of a tile to a wave's 32 keys; `masked`: a lane's key is
// seen from the positions lo .. hi alone.
template <typename T, int DP, int QT>
__device__ inline void add_queries(const char* tile, const AttnOperand<T, DP>& k, const AttnOperand<T, DP>& v,
                                   float scale, int lo, int hi, bool masked, f32x16_attn (&acc_k)[DP / 32],
                                   f32x16_attn (&acc_v)[DP / 32], SlopeScale<T>& slopes) {
    typedef QueryTile<T, DP, QT> Queries;
    typedef typename Queries::Tile Tile;
    const int half = lane_id() >> 5;
    const char* d_tile = tile + Tile::kBytes;
    const float* states = Queries::states(tile);
#pragma unroll
    for (int part = 0; part < QT / 32; ++part) {
        f32x16_attn p = tile_product<Tile, T, DP>(tile, 32 * part, k);
        f32x16_attn ds = tile_product<Tile, T, DP>(d_tile, 32 * part, v);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int row = 32 * part + 8 * g + 4 * half;
            if (masked) {
                const int4 at = *reinterpret_cast<const int4*>(states + 2 * QT + row);
                const int position[4] = {at.x, at.y, at.z, at.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (position[i] < lo || position[i] > hi) p[4 * g + i] = -INFINITY;
            }
            const float4 lse = *reinterpret_cast<const float4*>(states + row);
            const float4 delta = *reinterpret_cast<const float4*>(states + QT + row);
            const float log_sum[4] = {lse.x, lse.y, lse.z, lse.w};
            const float along[4] = {delta.x, delta.y, delta.z, delta.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * g + i;
                p[r] = __builtin_amdgcn_exp2f(p[r] * scale - (log_sum[i] - kShareLog2<T>));
                ds[r] = p[r] * (ds[r] - along[i]);
            }
        }
        add_columns<Tile, T>(acc_v, d_tile, 32 * part, p);
        add_slopes<Tile, T>(acc_k, slopes, tile, 32 * part, ds);
    }
}

// Sums of the first keys over the queries past their windows, which run to
// the end of a sequence: [slot][key head][tile of 32 first keys], each dk then
// dv, in the registers' order.
struct FirstParts {
    float* sums;
    int slots, tiles;  // tiles 0: the keys' pass takes every pair by itself
};
constexpr uint32_t kFirstRows = 4096;  // (query, head) pairs a slot
template <int DP> constexpr int kFirstValues = 2 * DP * 32;

template <typename T, int DP>
__global__ void __launch_bounds__(kAttnBlock)
grad_first_keys(lattice_attention a, const float* __restrict__ lse, const float* __restrict__ delta,
                const T* __restrict__ grad_out, FirstParts parts) {
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
    const long long row = static_cast<long long>(s.k0) + j;
    const bool valid = j < s.nk;
    AttnOperand<T, DP> k, v;
    k.load(static_cast<const T*>(a.k) + row * a.k_row_stride + kv * a.k_head_stride, a.dim, valid, a.scale < 0.0f);
    v.load(static_cast<const T*>(a.v) + row * a.v_row_stride + kv * a.v_head_stride, a.dim, valid, false);
    const float scale = fabsf(a.scale) * kAttnLog2e;
    f32x16_attn acc_k[kBlocks] = {}, acc_v[kBlocks] = {};
    SlopeScale<T> slopes;
    const int pieces = a.dim * static_cast<int>(sizeof(T)) / 16;
    // The first pair whose query lies past the window of key j0.
    const int i_from = max(0, j0 + a.left + 1 - s.shift());
    const uint32_t from = max(t.first, min(static_cast<uint32_t>(i_from), static_cast<uint32_t>(s.nq)) * group / QT * QT);
    const uint32_t to = min(t.first + kFirstRows, t.rows);
    char* tile = shared + wave * Queries::kBytes;
    for (uint32_t base = from; base < to; base += QT * kAttnWaves) {
        const uint32_t r0 = base + QT * wave;
        __syncthreads();
        if (r0 < to) {
            const auto state = Queries::template load<kWave>(tile, a, s, kv, group, r0, to, lse, delta, grad_out,
                                                             pieces, lane);
            Queries::store(tile, state, lane);
        }
        __syncthreads();
        if (r0 < to) {
            const int p_low = static_cast<int>(r0 / group) + s.shift();
            add_queries<T, DP, QT>(tile, k, v, scale, j + a.left + 1, INT_MAX, p_low <= j0 + 31 + a.left, acc_k,
                                   acc_v, slopes);
        }
    }
    scale_sums(acc_k, 1.0f / slopes.factor());
    // The waves' sums are added in wave order.
    float* sums = reinterpret_cast<float*>(shared);
    for (int u = 1; u < kAttnWaves; ++u) {
        __syncthreads();
        if (wave == u) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    sums[(b * 16 + r) * kWave + lane] = acc_k[b][r];
                    sums[((kBlocks + b) * 16 + r) * kWave + lane] = acc_v[b][r];
                }
            }
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    acc_k[b][r] += sums[(b * 16 + r) * kWave + lane];
                    acc_v[b][r] += sums[((kBlocks + b) * 16 + r) * kWave + lane];
                }
            }
        }
    }
    if (wave != 0) return;
    float* mine = parts.sums + ((static_cast<long long>(blockIdx.x) * a.kv_heads + kv) * parts.tiles + blockIdx.z) *
                                   kFirstValues<DP>;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            mine[(b * 16 + r) * kWave + lane] = acc_k[b][r];
            mine[((kBlocks + b) * 16 + r) * kWave + lane] = acc_v[b][r];
        }
    }
}

// grad_k and grad_v: 128 keys a block, 32 a wave, over the tiles of (query,
// head) pairs that see them.
template <typename T, int DP, int QT>
__global__ void __launch_bounds__(kAttnBlock, DP <= 64 ? 2 : 1)
grad_key_tiles(lattice_attention a, const float* __restrict__ lse, const float* __restrict__ delta,
               const T* __restrict__ grad_out, FirstParts parts, T* __restrict__ grad_k, T* __restrict__ grad_v) {
    constexpr int kBlocks = DP / 32;
    constexpr int kKeys = 32 * kAttnWaves;
    typedef QueryTile<T, DP, QT> Queries;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y;
    const auto slot_of = [](int start, int e) { return static_cast<uint32_t>(start) / kKeys + e; };
    const int e = key_rows(a).find(blockIdx.x, slot_of);
    const AttnSequence s = attn_sequence(a, e);
    const int owned = max(0, key_rows(a).start(e + 1) - s.k0);
    const int j0 = static_cast<int>(blockIdx.x - slot_of(s.k0, e)) * kKeys;
    if (j0 >= owned) return;
    const int j_wave = j0 + 32 * wave, j = j_wave + (lane & 31);
    const bool valid = j < s.nk;
    const long long row = static_cast<long long>(s.k0) + min(j, owned - 1);
    AttnOperand<T, DP> k, v;
    k.load(static_cast<const T*>(a.k) + row * a.k_row_stride + kv * a.k_head_stride, a.dim, valid, a.scale < 0.0f);
    v.load(static_cast<const T*>(a.v) + row * a.v_row_stride + kv * a.v_head_stride, a.dim, valid, false);
    const float scale = fabsf(a.scale) * kAttnLog2e;
    f32x16_attn acc_k[kBlocks] = {}, acc_v[kBlocks] = {};
    SlopeScale<T> slopes;
    const int pieces = a.dim * static_cast<int>(sizeof(T)) / 16;
    const uint32_t rows = s.nq * group;
    // The pairs whose window holds a key of the block.
    const int i_from = max(0, j0 - a.right - s.shift());
    const int i_to = min(s.nq, min(j0 + kKeys, s.nk) - 1 + a.left - s.shift() + 1);
    const bool any = j0 < s.nk && i_from < i_to;
    const uint32_t from = any ? i_from * group / QT : 0;
    const uint32_t window_to = any ? (i_to * group + QT - 1) / QT : 0;
    // Without a pass of their own, the first keys' other pairs follow.
    const bool rest = parts.tiles == 0 && j0 < min(a.sinks, s.nk);
    const int rest_from = max(0, j0 + a.left + 1 - s.shift());
    const uint32_t more = rest && rest_from < s.nq ? rest_from * group / QT : 0;
    const uint32_t more_to = rest && rest_from < s.nq ? (rows + QT - 1) / QT : 0;
    const int window_tiles = static_cast<int>(window_to - from);
    const int count = window_tiles + static_cast<int>(more_to - more);
    const auto first_row = [&](int index) {
        return (index < window_tiles ? from + index : more + (index - window_tiles)) * QT;
    };
    if (count > 0) {
        const auto state = Queries::template load<kAttnBlock>(shared, a, s, kv, group, first_row(0), rows, lse, delta,
                                                              grad_out, pieces, threadIdx.x);
        Queries::store(shared, state, threadIdx.x);
    }
    __syncthreads();
    for (int index = 0; index < count; ++index) {
        char* next = shared + ((index + 1) & 1) * Queries::kBytes;
        typename Queries::State state;
        if (index + 1 < count)
            state = Queries::template load<kAttnBlock>(next, a, s, kv, group, first_row(index + 1), rows, lse, delta,
                                                       grad_out, pieces, threadIdx.x);
        const char* tile = shared + (index & 1) * Queries::kBytes;
        const uint32_t r0 = first_row(index);
        const int p_low = static_cast<int>(r0 / group) + s.shift();
        const int p_high = static_cast<int>((min(r0 + QT, rows) - 1) / group) + s.shift();
        // In the window, or past it: of the first keys alone.
        const bool past = index >= window_tiles;
        const int lo = !past ? j - a.right : j < a.sinks ? j + a.left + 1 : INT_MAX;
        const int hi = past ? INT_MAX : j + a.left;
        const bool none = past ? j_wave >= a.sinks || p_high <= j_wave + a.left
                               : p_high < j_wave - a.right || p_low > j_wave + 31 + a.left;
        const bool all = !past && j_wave + 31 <= p_low + a.right && j_wave >= p_high - a.left;
        if (!none) add_queries<T, DP, QT>(tile, k, v, scale, lo, hi, !all, acc_k, acc_v, slopes);
        if (index + 1 < count) Queries::store(next, state, threadIdx.x);
        __syncthreads();
    }
    scale_sums(acc_k, 1.0f / slopes.factor());
    if (parts.tiles && j_wave < min(a.sinks, s.nk)) {
        // The parts of the first keys, in slot order; each holds the pairs of
        // one slot of the sequence's queries.
        const auto part_of = [group](int start, int e) { return start * group / kFirstRows + e; };
        const uint32_t slots = (rows + kFirstRows - 1) / kFirstRows;
        for (uint32_t u = 0; u < slots; ++u) {
            const float* sums =
                parts.sums + ((static_cast<long long>(part_of(s.q0, e)) + u) * a.kv_heads + kv) * parts.tiles *
                                 kFirstValues<DP> +
                j_wave / 32 * static_cast<long long>(kFirstValues<DP>);
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (j >= a.sinks) continue;
                    acc_k[b][r] += sums[(b * 16 + r) * kWave + lane];
                    acc_v[b][r] += sums[((kBlocks + b) * 16 + r) * kWave + lane];
                }
            }
        }
    }
    // Keys past the sequence's get zeros; a key whose sums are not finite is
    // made again from the queries that see it alone.
    const bool here = j < owned;
    const float share = __builtin_amdgcn_exp2f(-kShareLog2<T>);
    const float slope = a.scale * share;
    const bool finite =
        finite_columns(acc_k, slope, a.dim) && finite_columns(acc_v, share, a.dim);
    uint32_t again = spoilt_columns(valid, finite);
    const bool mine = here && !(again >> (lane & 31) & 1);
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
        grad_key_row<T>(a, s, j_wave + n, kv, lse, delta, grad_out, grad_k, grad_v,
                        reinterpret_cast<AttnRowScratch*>(shared) + wave);
    }
}

// What a call needs besides its outputs.
struct GradLayout {
    size_t deltas;
    int first_slots, first_tiles;
    size_t first_values;
};
inline GradLayout grad_layout(const lattice_attention& a) {
    GradLayout l{static_cast<size_t>(a.queries) * a.heads, 0, 0, 0};
    const long long pairs = static_cast<long long>(a.queries) * (a.heads / a.kv_heads);
    // The first keys' queries past the window are a pass of their own where
    // sequences are long: one block would walk all of a sequence.
    if (a.sinks > 0 && a.sinks <= 128 && a.left < a.keys && pairs >= 512ll * std::max(1, a.sequences)) {
        l.first_slots = static_cast<int>(pairs / kFirstRows + a.sequences + 2);
        l.first_tiles = (a.sinks + 31) / 32;
        const int dp = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128;
        l.first_values = static_cast<size_t>(l.first_slots) * a.kv_heads * l.first_tiles * 2 * dp * 32;
    }
    return l;
}

template <typename T, int DP>
int launch_grad(const lattice_attention& a, const GradLayout& l, const T* out, const float* lse, const T* grad_out,
                T* grad_q, T* grad_k, T* grad_v, float* delta, float* first, hipStream_t stream) {
    constexpr int kTile = sizeof(T) == 2 ? 64 : 32;
    const int group = a.heads / a.kv_heads;
    if (a.queries) {
        constexpr size_t kLds = std::max<size_t>(4 * AttnTile<T, DP, kTile>::kBytes,
                                                 kAttnWaves * sizeof(AttnRowScratch));
        const auto kernel = grad_query_tiles<T, DP, kTile>;
        LATTICE_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
        const long long slots = static_cast<long long>(a.queries) * group / (32 * kAttnWaves) + a.sequences + 2;
        kernel<<<dim3(static_cast<unsigned>(slots), a.kv_heads), kAttnBlock, kLds, stream>>>(a, out, lse, grad_out,
                                                                                            grad_q, delta);
        LATTICE_LAUNCH_CHECK();
    }
    if (a.keys == 0) return LATTICE_OK;
    const FirstParts parts{first, l.first_slots, l.first_tiles};
    if (l.first_tiles) {
        constexpr size_t kLds = std::max<size_t>(kAttnWaves * QueryTile<T, DP, 32>::kBytes,
                                                 kFirstValues<DP> * sizeof(float));
        static_assert(kLds <= 160 * 1024);
        const auto kernel = grad_first_keys<T, DP>;
        LATTICE_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                            hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
        kernel<<<dim3(l.first_slots, a.kv_heads, l.first_tiles), kAttnBlock, kLds, stream>>>(a, lse, delta, grad_out,
                                                                                            parts);
        LATTICE_LAUNCH_CHECK();
    }
    constexpr size_t kLds =
        std::max<size_t>(2 * QueryTile<T, DP, kTile>::kBytes, kAttnWaves * sizeof(AttnRowScratch));
    static_assert(kLds <= 160 * 1024);
    const auto kernel = grad_key_tiles<T, DP, kTile>;
    LATTICE_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    const long long slots = a.keys / (32 * kAttnWaves) + a.sequences + 2;
    kernel<<<dim3(static_cast<unsigned>(slots), a.kv_heads), kAttnBlock, kLds, stream>>>(a, lse, delta, grad_out, parts,
                                                                                        grad_k, grad_v);
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T>
int attend_grad(const lattice_attention& a, const GradLayout& l, const void* out, const float* lse,
                const void* grad_out, void* grad_q, void* grad_k, void* grad_v, float* delta, float* first,
                hipStream_t stream) {
    const T* o = static_cast<const T*>(out);
    const T* dy = static_cast<const T*>(grad_out);
    T* dq = static_cast<T*>(grad_q);
    T* dk = static_cast<T*>(grad_k);
    T* dv = static_cast<T*>(grad_v);
    if (a.dim <= 32) return launch_grad<T, 32>(a, l, o, lse, dy, dq, dk, dv, delta, first, stream);
    if (a.dim <= 64) return launch_grad<T, 64>(a, l, o, lse, dy, dq, dk, dv, delta, first, stream);
    return launch_grad<T, 128>(a, l, o, lse, dy, dq, dk, dv, delta, first, stream);
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" size_t lattice_hip_window_attention_grad_workspace_bytes(const lattice_attention* args) {
    if (attn_fault(args)) return 0;
    const GradLayout l = grad_layout(attn_bounded(*args));
    return aligned_bytes(l.deltas * sizeof(float)) + aligned_bytes(l.first_values * sizeof(float));
}

extern "C" int lattice_hip_window_attention_grad(const lattice_attention* args, const void* out, const float* lse,
                                                 const void* grad_out, void* grad_q, void* grad_k, void* grad_v,
                                                 void* workspace, size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE_ATTENTION(args);
    if (args->queries == 0 && args->keys == 0) return LATTICE_OK;
    LATTICE_REQUIRE(args->queries == 0 || (out && lse && grad_out && grad_q), "attention pointers must be non-null.");
    LATTICE_REQUIRE(args->keys == 0 || (grad_k && grad_v), "attention pointers must be non-null.");
    LATTICE_REQUIRE((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(grad_out)) % 16 == 0,
                    "attention rows must lie on 16-byte boundaries.");
    const lattice_attention a = attn_bounded(*args);
    const GradLayout l = grad_layout(a);
    Workspace ws{static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
    float* delta = ws.take<float>(l.deltas);
    float* first = ws.take<float>(l.first_values);
    LATTICE_REQUIRE(a.queries == 0 || (workspace && delta && (first || !l.first_values)),
                    "attention gradient workspace is too small.");
    hipStream_t stream = as_stream(stream_ptr);
    if (a.dtype == LATTICE_F32)
        return attend_grad<float>(a, l, out, lse, grad_out, grad_q, grad_k, grad_v, delta, first, stream);
    if (a.dtype == LATTICE_F16)
        return attend_grad<_Float16>(a, l, out, lse, grad_out, grad_q, grad_k, grad_v, delta, first, stream);
    return attend_grad<__bf16>(a, l, out, lse, grad_out, grad_q, grad_k, grad_v, delta, first, stream);
}
