// Attention over an 8-bit cache.
//
//   s_ij = scale 2^(ek_b) q_i . ck_j,  o_i = sum_j exp(s_ij - m_i) 2^(ev_b) cv_j / sum_j exp(s_ij - m_i)
// over the tokens j (of block b) that query i sees, in one pass with the running
// maximum m and sum.
//
// A wave holds tiles of 16 (query, head) pairs of the heads that share a key
// head and walks blocks of 32 tokens.  Products are 16 x 16 x 32: their operand
// of 8 values a lane is 8 codes, widened in registers on their way from memory,
// with no LDS between.  The scores are made transposed (rows: tokens, columns:
// pairs) from two products whose token rows are chosen so that a lane ends with
// the scores of 8 successive tokens of one pair; that is the right operand of
// the second product as it stands, and the values, which lie with a block's
// tokens innermost, are its left operand as they stand.  So a lane's softmax
// needs its neighbours only where the maximum moves.
//
// Codes are exact in bfloat16 and half precision.  The keys' power of two goes
// into the factor of the scores, the values' into the shares; shares of half
// precision are relative to a running power of two of (share times scale), so
// that neither blocks of large nor of small values leave the type's range.
// float32 queries and shares are three bfloat16 terms each (24 bits).
#pragma once

#include "cache_attention.h"

namespace lattice {
namespace {

template <typename T> struct CacheMath {
    typedef T Operand;
    static constexpr int kTerms = 1;
};
template <> struct CacheMath<float> {
    typedef __bf16 Operand;
    static constexpr int kTerms = 3;
};

template <typename O> struct CacheOperand;
template <> struct CacheOperand<__bf16> {
    typedef bf16x8_attn Frag;
    typedef bf16x2_cache Pair;
    __device__ static f32x4_attn product(Frag a, Frag b, f32x4_attn c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct CacheOperand<_Float16> {
    typedef f16x8_attn Frag;
    typedef f16x2_cache Pair;
    __device__ static f32x4_attn product(Frag a, Frag b, f32x4_attn c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

// The operand of 8 codes.
template <typename Code, typename O>
__device__ inline typename CacheOperand<O>::Frag widen(uint2 w) {
    struct Four {
        typename CacheOperand<O>::Pair p[4];
    } f;
    Code::values(w.x, f.p);
    Code::values(w.y, f.p + 2);
    return __builtin_bit_cast(typename CacheOperand<O>::Frag, f);
}

// 8 values as the terms of an operand, each what the ones before leave.
template <typename T>
struct CacheTerms {
    typedef typename CacheMath<T>::Operand O;
    typedef typename CacheOperand<O>::Frag Frag;
    static constexpr int kTerms = CacheMath<T>::kTerms;
    Frag f[kTerms];
    __device__ void set(const float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float rest = x[i];
#pragma unroll
            for (int t = 0; t < kTerms; ++t) {
                f[t][i] = static_cast<O>(rest);
                if (t + 1 < kTerms) rest -= static_cast<float>(f[t][i]);
            }
        }
    }
    __device__ f32x4_attn product(Frag a, f32x4_attn c) const {
#pragma unroll
        for (int t = kTerms - 1; t >= 0; --t) c = CacheOperand<O>::product(a, f[t], c);
        return c;
    }
};

// A block's codes as a lane holds them: of two rows of keys, and of DP / 16
// channels of values.
template <int DP>
struct CacheCodes {
    uint2 k[2][DP / 32], v[DP / 16];
    int key_exponent, value_exponent;
};

// The channels that a lane gives to step `c` of the first product: 16 bytes a
// load serve two steps, a rest of 32 channels 8 bytes one.
template <int DP>
__device__ constexpr int key_channel(int c, int g) {
    return c < DP / 64 * 2 ? 64 * (c / 2) + 16 * g + 8 * (c & 1) : DP / 64 * 64 + 8 * g;
}

template <int DP>
struct CacheReader {
    const uint8_t *keys, *values;
    const int8_t *key_exponents, *value_exponents;
    int key_place, value_place;

    __device__ CacheReader(const lattice_cache& c, int sequence, int kv) {
        const long long at = (static_cast<long long>(sequence) * c.kv_heads + kv) * c.blocks;
        keys = static_cast<const uint8_t*>(c.keys) + at * kCacheBlock * DP;
        values = static_cast<const uint8_t*>(c.values) + at * kCacheBlock * DP;
        key_exponents = c.key_exponents + at;
        value_exponents = c.value_exponents + at;
        const int n = lane_id() & 15, g = lane_id() >> 4;
        key_place = (8 * (n >> 2) + (n & 3)) * DP;
        value_place = n * kCacheBlock + 8 * g;
    }
    __device__ void load(CacheCodes<DP>& to, int block) const {
        const uint8_t* k = keys + static_cast<long long>(block) * (kCacheBlock * DP);
        const uint8_t* v = values + static_cast<long long>(block) * (kCacheBlock * DP);
        const int g = lane_id() >> 4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const uint4 w = *reinterpret_cast<const uint4*>(k + key_place + 4 * i * DP + 64 * c + 16 * g);
                to.k[i][2 * c] = uint2{w.x, w.y};
                to.k[i][2 * c + 1] = uint2{w.z, w.w};
            }
            if constexpr (DP % 64 != 0)
                to.k[i][DP / 32 - 1] =
                    *reinterpret_cast<const uint2*>(k + key_place + 4 * i * DP + DP / 64 * 64 + 8 * g);
        }
#pragma unroll
        for (int t = 0; t < DP / 16; ++t)
            to.v[t] = *reinterpret_cast<const uint2*>(v + value_place + 16 * t * kCacheBlock);
        to.key_exponent = key_exponents[block];
        to.value_exponent = value_exponents[block];
    }
};

// A share is exp2(score - top), where top is the running maximum and may lag
// behind the scores by kLag powers of two.  Shares times 2^(e - unit + kFill) go
// into the second product: at most 2^(kUnitLag + kFill), where the running unit
// lags.  In half precision, which loses bits below 2^-14, they fill the range:
// a product keeps all bits down to 2^-26 of the largest.
constexpr float kCacheLag = 8.0f;
template <typename T> struct CacheRange {
    static constexpr int kFill = 0, kUnitLag = 8;
};
template <> struct CacheRange<_Float16> {
    static constexpr int kFill = 13, kUnitLag = 2;
};
constexpr int kCacheNoUnit = -(1 << 20);

// What a pair sees.
struct CacheRow {
    int i, head;  // query of its sequence, head
    int lo, hi;   // the window's tokens
    bool valid;
};

template <typename T, int DP, int R>
struct CacheState {
    f32x4_attn acc[R][DP / 16];
    float top[R], sum[R];
    int unit[R];  // acc is in units of 2^unit

    __device__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) acc[r][t] = f32x4_attn{};
            top[r] = -3.0e38f;
            sum[r] = 0.0f;
            unit[r] = kCacheNoUnit;
        }
    }
    __device__ void rescale(int r, float factor) {
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) acc[r][t] *= factor;
    }
};

// Over the four lanes of a pair.
__device__ inline float pair_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float pair_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// 2^e, zero far below.
__device__ inline float bounded_power(int e) { return e < -126 ? 0.0f : power_of_two(min(e, 126)); }

// Adds the tokens j0 .. j0 + 31 to the wave's pairs; `masked`: some are not seen
// by some pair.
template <typename T, typename Code, int DP, int R>
__device__ inline void attend_codes(CacheState<T, DP, R>& state, const CacheTerms<T> (&q)[R][DP / 32],
                                    const CacheCodes<DP>& codes, const CacheRow (&rows)[R], float scale, int sinks,
                                    int nk, int j0, bool masked) {
    typedef typename CacheMath<T>::Operand O;
    typedef typename CacheOperand<O>::Frag Frag;
    const int g = lane_id() >> 4;
    f32x4_attn s[R][2];
#pragma unroll
    for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = f32x4_attn{};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            const Frag k = widen<Code, O>(codes.k[i][c]);
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][i] = q[r][c].product(k, s[r][i]);
        }
    }
    const int key_exponent = max(codes.key_exponent, kCacheLeast);
    const int value_exponent = max(codes.value_exponent, kCacheLeast);
    // Positive, so that -inf stays -inf.
    const float factor = fmaxf(scale * power_of_two(key_exponent), FLT_MIN);
    CacheTerms<T> p[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = s[r][e / 4][e % 4];
        if (masked) {
            const int j = j0 + 8 * g;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool seen = j + e <= rows[r].hi && (j + e >= rows[r].lo || j + e < sinks);
                x[e] = seen ? x[e] : -INFINITY;
            }
        }
        float most = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) most = fmaxf(most, x[e]);
        most *= factor;
        if (__any(most > state.top[r] + kCacheLag)) {
            const float next = fmaxf(state.top[r], pair_max(most));
            const float old = __builtin_amdgcn_exp2f(state.top[r] - next);
            state.rescale(r, old);
            state.sum[r] *= old;
            state.top[r] = next;
        }
        // The largest share times the block's power of two.
        if (__any(most - state.top[r] + static_cast<float>(value_exponent) >
                  static_cast<float>(state.unit[r] + CacheRange<T>::kUnitLag))) {
            const float size = pair_max(most) - state.top[r] + static_cast<float>(value_exponent);
            const int next = max(state.unit[r], static_cast<int>(ceilf(fmaxf(size, -512.0f))));
            state.rescale(r, bounded_power(state.unit[r] - next));
            state.unit[r] = next;
        }
        const float share = bounded_power(value_exponent - state.unit[r] + CacheRange<T>::kFill);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_amdgcn_exp2f(x[e] * factor - state.top[r]);
            sum += x[e];
            x[e] *= share;
        }
        state.sum[r] += sum;
        p[r].set(x);
    }
    // Bytes behind the last token stand for nothing.
    const int behind = nk - (j0 + 8 * g);
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        uint2 w = codes.v[t];
        if (masked && behind < 8) {
            const uint64_t keep = behind <= 0 ? 0 : ~0ull >> 8 * (8 - behind);
            w.x &= static_cast<uint32_t>(keep);
            w.y &= static_cast<uint32_t>(keep >> 32);
        }
        const Frag v = widen<Code, O>(w);
#pragma unroll
        for (int r = 0; r < R; ++r) state.acc[r][t] = p[r].product(v, state.acc[r][t]);
    }
}

// One (query, head) pair from the definition, 64 tokens at a time: for results
// that are not finite, since a product over a block carries a zero share of what
// a pair does not see.  Only what it sees is read.
template <typename T, typename Code>
__device__ inline void attend_pair(const CacheCall& call, const CacheSequence& s, int sequence, int i, int head,
                                   T* out, AttnRowScratch* scratch) {
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int lane = lane_id();
    const int width = cache_width(c);
    const int kv = static_cast<int>(static_cast<long long>(head) * c.kv_heads / a.heads);
    const long long at = (static_cast<long long>(sequence) * c.kv_heads + kv) * c.blocks;
    const uint8_t* keys = static_cast<const uint8_t*>(c.keys) + at * kCacheBlock * width;
    const uint8_t* values = static_cast<const uint8_t*>(c.values) + at * kCacheBlock * width;
    const long long row = static_cast<long long>(s.q0) + i;
    const int p = i + s.shift();
    const int hi = min(s.nk - 1, p + a.right), lo = max(0, p - a.left);
    const int first = hi < 0 ? 0 : min(min(a.sinks, lo), hi + 1), total = hi < 0 ? 0 : first + max(0, hi - lo + 1);
    wave_fence();
    stage_row(scratch->a, static_cast<const T*>(a.q) + row * a.q_row_stride + head * a.q_head_stride, c.dim);
    wave_fence();
    float top = -INFINITY, sum = 0.0f, acc[kAttnMaxDim / kWave] = {};
    for (int base = 0; base < total; base += kWave) {
        const int count = min(kWave, total - base);
        const auto token = [&](int t) { return t < first ? t : lo + (t - first); };
        float x = -INFINITY;
        if (lane < count) {
            const int j = token(base + lane);
            const uint8_t* k = keys + static_cast<long long>(j) * width;
            float dot = 0.0f;
            for (int d = 0; d < c.dim; ++d) dot += scratch->a[d] * Code::value(k[d]);
            const int e = c.key_exponents[at + j / kCacheBlock];
            x = dot * power_of_two(max(e, kCacheLeast)) * (a.scale * kAttnLog2e);
        }
        const float next = fmaxf(top, wave_max(x));
        const float old = top == next ? 1.0f : exp2f(top - next);
        // Of -inf before any other score, no share (alone, 0 / 0 in the end).
        const float share = x != -INFINITY ? exp2f(x - next) : 0.0f;
        top = next;
        sum = sum * old + wave_sum(share);
        wave_fence();
        scratch->p[lane] = share;
        wave_fence();
#pragma unroll
        for (int b = 0; b < kAttnMaxDim / kWave; ++b) {
            const int d = lane + b * kWave;
            if (d >= c.dim) continue;
            float add = 0.0f;
            for (int t = 0; t < count; ++t) {
                const int j = token(base + t), block = j / kCacheBlock;
                const uint8_t code =
                    values[(static_cast<long long>(block) * width + d) * kCacheBlock + j % kCacheBlock];
                const int e = c.value_exponents[at + block];
                add += scratch->p[t] * (Code::value(code) * power_of_two(max(e, kCacheLeast)));
            }
            acc[b] = acc[b] * old + add;
        }
    }
#pragma unroll
    for (int b = 0; b < kAttnMaxDim / kWave; ++b) {
        const int d = lane + b * kWave;
        if (d < c.dim) out[(row * a.heads + head) * c.dim + d] = static_cast<T>(total ? acc[b] / sum : 0.0f);
    }
}

// The rows of sequence `s` that a wave has: R tiles of 16 pairs from `first` on.
template <int R>
__device__ inline void cache_rows(CacheRow (&rows)[R], const CacheCall& call, const CacheSequence& s, int kv,
                                  uint32_t first) {
    const uint32_t group = call.args.heads / call.cache.kv_heads;
    const uint32_t count = s.nq * group;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t pair = first + 16 * r + (lane_id() & 15), in = min(pair, count - 1);
        rows[r].i = in / group;
        rows[r].head = kv * group + in % group;
        rows[r].valid = pair < count;
        const int p = rows[r].i + s.shift();
        rows[r].lo = p - call.args.left;
        rows[r].hi = min(s.nk - 1, p + call.args.right);
    }
}

// The blocks that positions p_low .. p_high see: those of the first tokens that
// lie before the window's, then the window's.
__device__ inline AttnTiles cache_blocks(const lattice_cache_attention& a, int nk, int p_low, int p_high) {
    const int hi = min(nk - 1, p_high + a.right);
    if (hi < 0) return {0, 0, 0};
    const int from = max(0, p_low - a.left) / kCacheBlock;
    const int first = min((min(a.sinks, hi + 1) + kCacheBlock - 1) / kCacheBlock, from);
    return {first, from, first + max(0, hi / kCacheBlock - from + 1)};
}

// SHARE: the block's waves have the same R tiles of pairs and take turns at the
// blocks of tokens; their parts are joined in LDS.  Otherwise each has R tiles
// of its own.
template <typename T, typename Code, int DP, int R, bool SHARE>
__global__ void __launch_bounds__(kAttnBlock)
cache_attend(CacheCall call, int splits, CachePart part, T* __restrict__ out) {
    constexpr int kTiles = DP / 16;
    constexpr int kRows = 16 * R;
    constexpr int kValues = R * kTiles * 4 * kWave;  // sums of a wave
    __shared__ AttnRowScratch scratch[kAttnWaves];
    __shared__ float2 states[SHARE ? kAttnWaves * kRows : 1];
    __shared__ float sums[SHARE ? kAttnWaves / 2 * kValues : 1];
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const int n = lane & 15, g = lane >> 4;
    const uint32_t group = a.heads / c.kv_heads;
    const int kv = blockIdx.y, split = block_part(splits);
    constexpr int kSlot = SHARE ? kRows : kRows * kAttnWaves;
    const RowPartition partition{a.offsets, c.sequences, a.queries};
    const auto slot_of = [group](int start, int e) { return start * group / kSlot + e; };
    const uint32_t slot = block_slot(splits);
    const int e = partition.find(slot, slot_of);
    const CacheSequence s = cache_sequence(partition, a.lengths, c.blocks * kCacheBlock, e);
    const uint32_t count = s.nq * group;
    const uint32_t start = slot_first<kSlot>(slot, slot_of(s.q0, e), count);
    const uint32_t first = start + (SHARE ? 0 : wave * kRows);
    if (start >= count) return;
    if (!SHARE && first >= count) return;

    CacheRow rows[R];
    cache_rows<R>(rows, call, s, kv, first);
    CacheTerms<T> q[R][DP / 32];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* row = static_cast<const T*>(a.q) + (static_cast<long long>(s.q0) + rows[r].i) * a.q_row_stride +
                       rows[r].head * a.q_head_stride;
        constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
#pragma unroll
        for (int k = 0; k < DP / 32; ++k) {
            float x[8];
#pragma unroll
            for (int h = 0; h < 8 / kPiece; ++h) {
                const int channel = key_channel<DP>(k, g) + h * kPiece;
                RowVec<T, kPiece> in;
                const bool here = rows[r].valid && channel < c.dim;
                if (here) in = RowVec<T, kPiece>::load(row + channel);
#pragma unroll
                for (int j = 0; j < kPiece; ++j) {
                    const float value = here ? in.at(j) : 0.0f;
                    x[h * kPiece + j] = a.scale < 0.0f ? -value : value;
                }
            }
            q[r][k].set(x);
        }
    }
    const float scale = fabsf(a.scale) * kAttnLog2e;
    const int p_low = static_cast<int>(first / group) + s.shift();
    const int p_high = static_cast<int>((min(first + kRows, count) - 1) / group) + s.shift();
    CacheState<T, DP, R> state;
    state.clear();
    if (partition.real(e)) {
        const AttnTiles blocks = cache_blocks(a, s.nk, p_low, p_high);
        const CacheReader<DP> reader(c, e - 1, kv);
        const int parts = SHARE ? splits * kAttnWaves : 1, mine = SHARE ? split * kAttnWaves + wave : 0;
        const int from = static_cast<int>(static_cast<long long>(blocks.count) * mine / parts);
        const int to = static_cast<int>(static_cast<long long>(blocks.count) * (mine + 1) / parts);
        CacheCodes<DP> codes;
        if (from < to) reader.load(codes, blocks.tile(from));
        for (int index = from; index < to; ++index) {
            const CacheCodes<DP> now = codes;
            if (index + 1 < to) reader.load(codes, blocks.tile(index + 1));
            const int j0 = blocks.tile(index) * kCacheBlock, end = j0 + kCacheBlock;
            const bool all = end <= s.nk && end - 1 <= p_low + a.right && (j0 >= p_high - a.left || end <= a.sinks);
            attend_codes<T, Code, DP, R>(state, q, now, rows, scale, a.sinks, s.nk, j0, !all);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        state.sum[r] = pair_sum(state.sum[r]);
        // To units of one, in two steps of normal numbers.
        const int half = (state.unit[r] - CacheRange<T>::kFill) / 2;
        state.rescale(r, bounded_power(half));
        state.rescale(r, bounded_power(state.unit[r] - CacheRange<T>::kFill - half));
    }
    if constexpr (SHARE) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (g == 0) states[wave * kRows + 16 * r + n] = float2{state.top[r], state.sum[r]};
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = -3.0e38f, sum = 0.0f;
            for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, states[w * kRows + 16 * r + n].x);
            for (int w = 0; w < kAttnWaves; ++w) {
                const float2 other = states[w * kRows + 16 * r + n];
                sum += other.y * __builtin_amdgcn_exp2f(other.x - top);
            }
            state.rescale(r, __builtin_amdgcn_exp2f(state.top[r] - top));
            state.top[r] = top;
            state.sum[r] = sum;
        }
#pragma unroll
        for (int active = kAttnWaves / 2; active > 0; active /= 2) {
            __syncthreads();
            if (wave >= active && wave < 2 * active) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        *reinterpret_cast<f32x4_attn*>(sums + (wave - active) * kValues +
                                                       ((r * kTiles + t) * kWave + lane) * 4) = state.acc[r][t];
                }
            }
            __syncthreads();
            if (wave < active) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        state.acc[r][t] += *reinterpret_cast<const f32x4_attn*>(
                            sums + wave * kValues + ((r * kTiles + t) * kWave + lane) * 4);
                }
            }
        }
        if (wave != 0) return;
    }
    const long long items = static_cast<long long>(a.queries) * a.heads;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long long at = (static_cast<long long>(s.q0) + rows[r].i) * a.heads + rows[r].head;
        if (splits > 1) {
            if (!rows[r].valid) continue;
            const long long row = split * items + at;
            if (g == 0) part.states[row] = float2{state.top[r], state.sum[r]};
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int d = 16 * t + 4 * g;
                if (d < c.dim) *reinterpret_cast<f32x4_attn*>(part.values + row * c.dim + d) = state.acc[r][t];
            }
            continue;
        }
        const bool sees = rows[r].hi >= max(0, rows[r].lo) || (a.sinks > 0 && rows[r].hi >= 0);
        const float inv = sees ? 1.0f / state.sum[r] : 0.0f;
        uint32_t largest = 0;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                state.acc[r][t][i] *= inv;
                // The bits of magnitudes are ordered, NaN above infinity.
                largest = max(largest, __float_as_uint(state.acc[r][t][i]) & 0x7fffffffu);
            }
        }
        const uint64_t spoilt = ballot(rows[r].valid && largest >= 0x7f800000u);
        uint32_t again = static_cast<uint32_t>(spoilt | spoilt >> 16 | spoilt >> 32 | spoilt >> 48) & 0xffffu;
        if (rows[r].valid && !(again >> n & 1)) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const int d = 16 * t + 4 * g;
                if (d >= c.dim) continue;
                RowVec<T, 4> v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v.set(i, state.acc[r][t][i]);
                v.store(out + at * c.dim + d);
            }
        }
        while (again) {
            const int which = __ffs(again) - 1;
            again &= again - 1;
            attend_pair<T, Code>(call, s, e - 1, __shfl(rows[r].i, which), __shfl(rows[r].head, which), out,
                                 &scratch[wave]);
        }
    }
}

// Joins the parts (at most 64) of a pair: a wave a (query, head).
template <typename T, typename Code>
__global__ void __launch_bounds__(kAttnBlock)
cache_join(CacheCall call, int splits, CachePart part, T* __restrict__ out) {
    __shared__ AttnRowScratch scratch[kAttnWaves];
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int wave = threadIdx.x / kWave, lane = lane_id();
    const long long items = static_cast<long long>(a.queries) * a.heads;
    const long long at = static_cast<long long>(blockIdx.x) * kAttnWaves + wave;
    if (at >= items) return;
    const float2 state = lane < splits ? part.states[lane * items + at] : float2{-3.0e38f, 0.0f};
    const float top = wave_max(state.x);
    const float factor = __builtin_amdgcn_exp2f(state.x - top);
    const float sum = wave_sum(state.y * factor);
    float acc[kAttnMaxDim / kWave] = {};
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
        const float share = __shfl(factor, z);
#pragma unroll
        for (int b = 0; b < kAttnMaxDim / kWave; ++b) {
            const int d = min(lane + b * kWave, c.dim - 1);
            acc[b] += part.values[(z * items + at) * c.dim + d] * share;
        }
    }
    bool finite = sum > 0.0f;
#pragma unroll
    for (int b = 0; b < kAttnMaxDim / kWave; ++b) {
        acc[b] /= sum;
        finite = finite && fabsf(acc[b]) < INFINITY;
    }
    // Rows that see nothing, and those that are not finite.
    if (__any(!finite)) {
        const int row = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
        const RowPartition partition{a.offsets, c.sequences, a.queries};
        const int e = partition.find(row, [](int start, int) { return static_cast<uint32_t>(start); });
        const CacheSequence s = cache_sequence(partition, a.lengths, c.blocks * kCacheBlock, e);
        attend_pair<T, Code>(call, s, e - 1, row - s.q0, head, out, &scratch[wave]);
        return;
    }
#pragma unroll
    for (int b = 0; b < kAttnMaxDim / kWave; ++b) {
        const int d = lane + b * kWave;
        if (d < c.dim) out[at * c.dim + d] = static_cast<T>(acc[b]);
    }
}

template <typename T, typename Code, int DP>
int launch_cache_attend(const CacheCall& call, const CacheLayout& l, const CachePart& part, T* out,
                        hipStream_t stream) {
    const dim3 grid = slot_grid(l.slots, call.cache.kv_heads, l.splits);
#define LATTICE_CACHE_ATTEND(TILES, SHARE) \
    cache_attend<T, Code, DP, TILES, SHARE><<<grid, kAttnBlock, 0, stream>>>(call, l.splits, part, out)
    if (l.share) {
        LATTICE_CACHE_ATTEND(1, true);
    } else {
        LATTICE_CACHE_ATTEND(2, false);
    }
#undef LATTICE_CACHE_ATTEND
    LATTICE_LAUNCH_CHECK();
    if (l.splits > 1) {
        cache_join<T, Code><<<grid_for(static_cast<long long>(call.args.queries) * call.args.heads, kAttnWaves,
                                       1u << 30), kAttnBlock, 0, stream>>>(call, l.splits, part, out);
        LATTICE_LAUNCH_CHECK();
    }
    return LATTICE_OK;
}

template <typename T, typename Code>
int launch_cache_code(const CacheCall& call, const CacheLayout& l, const CachePart& part, void* out,
                      hipStream_t stream) {
    T* o = static_cast<T*>(out);
    const int dim = call.cache.dim;
    if (dim <= 32) return launch_cache_attend<T, Code, 32>(call, l, part, o, stream);
    if (dim <= 64) return launch_cache_attend<T, Code, 64>(call, l, part, o, stream);
    if (dim <= 96) return launch_cache_attend<T, Code, 96>(call, l, part, o, stream);
    return launch_cache_attend<T, Code, 128>(call, l, part, o, stream);
}

template <typename T>
int launch_cache(const CacheCall& call, const CacheLayout& l, const CachePart& part, void* out, hipStream_t stream) {
    if (call.cache.code == LATTICE_CODE_E4M3) return launch_cache_code<T, CodeE4m3>(call, l, part, out, stream);
    return launch_cache_code<T, CodeInt8>(call, l, part, out, stream);
}

}  // namespace
}  // namespace lattice
