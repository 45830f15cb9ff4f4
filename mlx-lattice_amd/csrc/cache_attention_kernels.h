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
// float32 queries and shares are three bfloat16 terms each (24 bits).  In the
// 16-bit types shares are rounded to the operand's type, half a step at most and
// to either side, as window_attention rounds its own; their sum is of the
// unrounded ones.  A second term would be a second product with the values.  So a
// result is off by two roundings, this and its own: by 0.0024 of the results'
// norm in bfloat16 and 0.00029 in half precision, 0.0017 and 0.00021 being the
// result's own, and over long averages less (0.00023).
//
// Single tokens are bound by memory: a byte a value is read, once.  One query of
// 16 heads over 4 key heads of 128 channels, 32 caches of 32768 tokens, some 24
// thousand filled, in half precision: 164 us, 5.07 TB/s, where a copy reaches
// 5.23.  Small calls are bound by latency: 6.2 us for 4 caches in a window of
// 512.  Chunks are bound by the matrix cores and the exponentials and widenings
// beside them: 2 x 2048 causal queries of 16 heads of 128 channels over 16384
// tokens in bfloat16 take 540 to 560 us from card to card, 890 to 925 TFLOP/s,
// where a product of 8192 x 8192 x 8192 reaches 1207; the matrix cores work 0.36
// of the time, the vector units 0.48, mostly in turn.
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
struct CacheKeys {
    uint2 w[2][DP / 32];
    int exponent;
};
template <int DP>
struct CacheValues {
    uint2 w[DP / 16];
    int exponent;
};

// The channels that a lane gives to step `c` of the first product.  WIDE: 16
// bytes a load serve two steps, a rest of 32 channels 8 bytes one.
template <int DP, bool WIDE>
__device__ constexpr int key_channel(int c, int g) {
    return !WIDE ? 32 * c + 8 * g : c < DP / 64 * 2 ? 64 * (c / 2) + 16 * g + 8 * (c & 1) : DP / 64 * 64 + 8 * g;
}
// The token of row `n` of the first product's half `i`: a lane ends with the
// scores of tokens 8 g .. 8 g + 7.
__device__ constexpr int key_token(int i, int n) { return 8 * (n >> 2) + 4 * i + (n & 3); }

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
        key_place = key_token(0, n) * DP;
        value_place = n * kCacheBlock + 8 * g;
    }
    __device__ void load(CacheKeys<DP>& to, int block) const {
        const uint8_t* k = keys + static_cast<long long>(block) * (kCacheBlock * DP);
        const int g = lane_id() >> 4;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) {
                const uint4 w = *reinterpret_cast<const uint4*>(k + key_place + 4 * i * DP + 64 * c + 16 * g);
                to.w[i][2 * c] = uint2{w.x, w.y};
                to.w[i][2 * c + 1] = uint2{w.z, w.w};
            }
            if constexpr (DP % 64 != 0)
                to.w[i][DP / 32 - 1] =
                    *reinterpret_cast<const uint2*>(k + key_place + 4 * i * DP + DP / 64 * 64 + 8 * g);
        }
        to.exponent = key_exponents[block];
    }
    __device__ void load(CacheValues<DP>& to, int block) const {
        const uint8_t* v = values + static_cast<long long>(block) * (kCacheBlock * DP);
#pragma unroll
        for (int t = 0; t < DP / 16; ++t)
            to.w[t] = *reinterpret_cast<const uint2*>(v + value_place + 16 * t * kCacheBlock);
        to.exponent = value_exponents[block];
    }
};

// What goes into the second product is 2^(score - top + e - unit + kFill), e the
// exponent of the block's values: top and unit are running maxima of the scores
// and of (score - top + e).  They move where the eight of a lane add up to more
// than kMost, so that nothing is compared on the way.  In half precision, which
// loses bits below 2^-14, they fill the range: a product keeps all bits down to
// 2^-25 of the largest.
template <typename T> struct CacheRange {
    static constexpr int kFill = 0;
    static constexpr float kMost = 2048.0f;
};
template <> struct CacheRange<_Float16> {
    static constexpr int kFill = 12;
    static constexpr float kMost = 40000.0f;
};
// The power of two that is taken into the exponent is no less, so that sums of
// shares are not lost where a block's values are next to nothing.
constexpr int kCacheLeastShift = -60;
constexpr int kCacheNoUnit = -(1 << 20);
// A row's top starts far below every score but above -inf, so that what is
// masked (-inf) has a share of zero.
constexpr float kCacheFloor = -3.0e38f;

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
    int unit[R];  // sums are in units of 2^top, acc in units of 2^(top + unit); once closed, acc is their quotient

    __device__ void clear() {
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) acc[r][t] = f32x4_attn{};
            top[r] = kCacheFloor;
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

// 2^e for e up to 127, zero below -126 (the bits of zero).
__device__ inline float bounded_power(int e) { return power_of_two(max(e, -127)); }

// Bytes of tokens behind the last stand for nothing: those of a lane's eight
// that are kept of a block's first `count`.
__device__ inline uint64_t kept_bytes(int count) {
    const int mine = count - 8 * (lane_id() >> 4);
    return mine <= 0 ? 0 : mine >= 8 ? ~0ull : ~0ull >> 8 * (8 - mine);
}
__device__ inline uint2 cut_bytes(uint2 w, uint64_t keep) {
    return uint2{w.x & static_cast<uint32_t>(keep), w.y & static_cast<uint32_t>(keep >> 32)};
}

// The scores of a block's tokens, before any scale, 8 tokens a lane; key(i, c)
// gives the first product's left operand.
template <typename T, int DP, int R, typename Keys>
__device__ inline void cache_scores(f32x4_attn (&s)[R][2], const CacheTerms<T> (&q)[R][DP / 32], const Keys& key) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r][0] = s[r][1] = f32x4_attn{};
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const auto k = key(i, c);
#pragma unroll
            for (int r = 0; r < R; ++r) s[r][i] = q[r][c].product(k, s[r][i]);
        }
    }
}

// 8 shares of a pair and their sum, whose exponent was lowered by `shift` less.
struct CacheShares {
    float y[8], sum;
    int wanted, shift;

    template <typename T, int DP, int R>
    __device__ void make(const CacheState<T, DP, R>& state, int r, const f32x4_attn (&s)[2], float factor,
                         int value_exponent) {
        wanted = value_exponent - state.unit[r] + CacheRange<T>::kFill;
        shift = max(wanted, kCacheLeastShift);
        const float base = static_cast<float>(shift) - state.top[r];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 4][e % 4], factor, base));
        sum = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
    }
};

// What tokens j0 .. j0 + 31 some pair does not see has no share.
template <int R>
__device__ inline void hide_scores(f32x4_attn (&s)[R][2], const CacheRow (&rows)[R], int sinks, int j0) {
    const int j = j0 + 8 * (lane_id() >> 4);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool seen = j + e <= rows[r].hi && (j + e >= rows[r].lo || j + e < sinks);
            s[r][e / 4][e % 4] = seen ? s[r][e / 4][e % 4] : -INFINITY;
        }
    }
}

// Moves a row's maxima to what its scores ask for.
template <typename T, int DP, int R>
__device__ inline void move_maxima(CacheState<T, DP, R>& state, int r, const f32x4_attn (&s)[2], float factor,
                                   int value_exponent) {
    float most = s[0][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) most = fmaxf(most, s[e / 4][e % 4]);
    most = pair_max(most * factor);
    const float top = fmaxf(state.top[r], most);
    const float down = fminf(top - state.top[r], 1024.0f);
    const float size = fmaxf(most - top + static_cast<float>(value_exponent), -512.0f);
    const int unit = max(state.unit[r] - static_cast<int>(down), static_cast<int>(ceilf(size)));
    state.sum[r] *= __builtin_amdgcn_exp2f(state.top[r] - top);
    state.rescale(r, __builtin_amdgcn_exp2f(state.top[r] - top + static_cast<float>(state.unit[r] - unit)));
    state.top[r] = top;
    state.unit[r] = unit;
}

// The shares of the wave's pairs as the second product's operand.  One test a
// block tells whether a maximum has to move.
template <typename T, int DP, int R>
__device__ inline void cache_shares(CacheTerms<T> (&p)[R], CacheState<T, DP, R>& state, const f32x4_attn (&s)[R][2],
                                    float factor, int value_exponent) {
    CacheShares x[R];
    for (int tries = 0;; ++tries) {
        bool moves = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            x[r].make(state, r, s[r], factor, value_exponent);
            moves = moves || x[r].sum > CacheRange<T>::kMost;
        }
        if (!__any(moves) || tries > 0) break;
#pragma unroll
        for (int r = 0; r < R; ++r) move_maxima<T, DP, R>(state, r, s[r], factor, value_exponent);
    }
    bool low = false;
#pragma unroll
    for (int r = 0; r < R; ++r) low = low || x[r].wanted < kCacheLeastShift;
    if (__any(low)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float rest = bounded_power(x[r].wanted - x[r].shift);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[r].y[e] *= rest;
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        state.sum[r] += x[r].sum * bounded_power(-x[r].shift);
        p[r].set(x[r].y);
    }
}

// acc += values times shares; value(t) gives the second product's left operand.
template <typename T, int DP, int R, typename Values>
__device__ inline void add_cache_values(CacheState<T, DP, R>& state, const CacheTerms<T> (&p)[R],
                                        const Values& value) {
#pragma unroll
    for (int t = 0; t < DP / 16; ++t) {
        const auto v = value(t);
#pragma unroll
        for (int r = 0; r < R; ++r) state.acc[r][t] = p[r].product(v, state.acc[r][t]);
    }
}

// One (query, head) pair from the definition, 64 tokens at a time: for results
// that are not finite, since a product over a block carries a zero share of what
// a pair does not see.  Only what it sees is read.  Slow: a wave takes its
// pairs one after the other, a channel of a token at a time.  One NaN that the
// queries above see, or that lies just ahead of a window, makes 55 us (in a window
// of 1000) 16 ms, and four pairs over 24 thousand tokens take 10 ms.
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
        // Averages, as close_state has them.
        const float before = sum * old;
        top = next;
        sum = before + wave_sum(share);
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f, kept = before * inv;
        wave_fence();
        scratch->p[lane] = share * inv;
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
                add += scratch->p[t] * Code::value(code) * power_of_two(max(e, kCacheLeast));
            }
            acc[b] = acc[b] * kept + add;
        }
    }
#pragma unroll
    for (int b = 0; b < kAttnMaxDim / kWave; ++b) {
        const int d = lane + b * kWave;
        if (d < c.dim) out[(row * a.heads + head) * c.dim + d] = static_cast<T>(total && sum == 0.0f ? NAN : acc[b]);
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

// The queries of the wave's pairs, negated where the scale is negative.
template <typename T, int DP, int R, bool WIDE>
__device__ inline void cache_queries(CacheTerms<T> (&q)[R][DP / 32], const CacheCall& call, const CacheSequence& s,
                                     const CacheRow (&rows)[R]) {
    const lattice_cache_attention& a = call.args;
    constexpr int kPiece = 16 / static_cast<int>(sizeof(T));
    const int g = lane_id() >> 4;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* row = static_cast<const T*>(a.q) + (static_cast<long long>(s.q0) + rows[r].i) * a.q_row_stride +
                       rows[r].head * a.q_head_stride;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k) {
            float x[8];
#pragma unroll
            for (int h = 0; h < 8 / kPiece; ++h) {
                const int channel = key_channel<DP, WIDE>(k, g) + h * kPiece;
                RowVec<T, kPiece> in;
                const bool here = rows[r].valid && channel < call.cache.dim;
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
}

// Whether positions p_low .. p_high see all of a block of tokens from j0 on.
struct CacheView {
    int to, from, first;
    __device__ CacheView(const lattice_cache_attention& a, int nk, int p_low, int p_high)
        : to(min(nk, p_low + a.right + 1) - kCacheBlock), from(p_high - a.left), first(a.sinks - kCacheBlock) {}
    __device__ bool all(int j0) const { return j0 <= to && (j0 >= from || j0 <= first); }
};

// The factor of a block's scores, positive, so that -inf stays -inf.
__device__ inline float cache_factor(float scale, int key_exponent) {
    return fmaxf(scale * power_of_two(max(key_exponent, kCacheLeast)), 0x1p-149f);
}

// Sums over the four lanes of a pair, and averages of the values: divided before
// the power of two comes back, since a sum of values near the type's end is past
// it where their average is not.  What sees nothing has zeros.
template <typename T, int DP, int R>
__device__ inline void close_state(CacheState<T, DP, R>& state) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        state.sum[r] = pair_sum(state.sum[r]);
        state.rescale(r, state.sum[r] != 0.0f ? 1.0f / state.sum[r] : 0.0f);
        // In two steps of normal numbers.
        const int unit = state.unit[r] - CacheRange<T>::kFill;
        state.rescale(r, bounded_power(unit / 2));
        state.rescale(r, bounded_power(unit - unit / 2));
    }
}

// Writes the wave's results.  One that is not finite is made again from its
// definition.
template <typename T, typename Code, int DP, int R>
__device__ inline void write_pairs(const CacheCall& call, const CacheSequence& s, int sequence,
                                   const CacheRow (&rows)[R], CacheState<T, DP, R>& state, T* out,
                                   AttnRowScratch* scratch) {
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int n = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long long at = (static_cast<long long>(s.q0) + rows[r].i) * a.heads + rows[r].head;
        const bool sees = rows[r].hi >= max(0, rows[r].lo) || (a.sinks > 0 && rows[r].hi >= 0);
        // Without any share, all scores are -inf.
        uint32_t largest = sees && state.sum[r] == 0.0f ? 0x7f800000u : 0;
#pragma unroll
        for (int t = 0; t < DP / 16; ++t) {
            // The bits of magnitudes are ordered, NaN above infinity.
#pragma unroll
            for (int i = 0; i < 4; ++i) largest = max(largest, __float_as_uint(state.acc[r][t][i]) & 0x7fffffffu);
        }
        const uint64_t spoilt = ballot(rows[r].valid && largest >= 0x7f800000u);
        uint32_t again = static_cast<uint32_t>(spoilt | spoilt >> 16 | spoilt >> 32 | spoilt >> 48) & 0xffffu;
        if (rows[r].valid && !(again >> n & 1)) {
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
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
            attend_pair<T, Code>(call, s, sequence, __shfl(rows[r].i, which), __shfl(rows[r].head, which), out,
                                 scratch);
        }
    }
}

// For few queries: the block's waves have the same R tiles of pairs and take
// each its share of the blocks of tokens, codes straight from memory to
// registers; their parts are joined in LDS.
template <typename T, typename Code, int DP, int R>
__global__ void __launch_bounds__(kAttnBlock, 2)
cache_attend_few(CacheCall call, int splits, CachePart part, T* __restrict__ out) {
    typedef typename CacheMath<T>::Operand O;
    constexpr int kTiles = DP / 16;
    constexpr int kRows = 16 * R;
    constexpr int kValues = R * kTiles * 4 * kWave;  // sums of a wave
    __shared__ AttnRowScratch scratch;
    __shared__ float2 states[kAttnWaves * kRows];
    __shared__ float sums[kAttnWaves / 2 * kValues];
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const int n = lane & 15, g = lane >> 4;
    const uint32_t group = a.heads / c.kv_heads;
    const int kv = blockIdx.x % c.kv_heads, split = block_part(splits);
    const RowPartition partition{a.offsets, c.sequences, a.queries};
    const auto slot_of = [group](int start, int e) { return start * group / kRows + e; };
    const uint32_t slot = cache_place(c.kv_heads, splits);
    const CacheSequence s = find_cache_sequence(partition, a.lengths, c.blocks * kCacheBlock, slot, slot_of);
    const uint32_t count = s.nq * group;
    const uint32_t first = slot_first<kRows>(slot, slot_of(s.q0, s.index), count);
    if (first >= count) return;

    const int p_low = static_cast<int>(first / group) + s.shift();
    const int p_high = static_cast<int>((min(first + kRows, count) - 1) / group) + s.shift();
    const AttnTiles blocks = s.real ? cache_blocks(a, s.nk, p_low, p_high) : AttnTiles{0, 0, 0};
    const CacheReader<DP> reader(c, s.index - 1, kv);
    const int parts = splits * kAttnWaves, mine = split * kAttnWaves + wave;
    const int from = static_cast<int>(static_cast<long long>(blocks.count) * mine / parts);
    const int to = static_cast<int>(static_cast<long long>(blocks.count) * (mine + 1) / parts);
    // Codes are read into the registers that the block before has left, the first
    // ones before the queries are.
    CacheKeys<DP> keys;
    CacheValues<DP> values;
    if (from < to) {
        reader.load(keys, blocks.tile(from));
        reader.load(values, blocks.tile(from));
    }
    CacheRow rows[R];
    cache_rows<R>(rows, call, s, kv, first);
    CacheTerms<T> q[R][DP / 32];
    cache_queries<T, DP, R, true>(q, call, s, rows);
    const float scale = fabsf(a.scale) * kAttnLog2e;
    const CacheView view(a, s.nk, p_low, p_high);
    CacheState<T, DP, R> state;
    state.clear();
    for (int index = from; index < to; ++index) {
        const int next = blocks.tile(min(index + 1, to - 1));
        const int j0 = blocks.tile(index) * kCacheBlock;
        f32x4_attn scores[R][2];
        cache_scores<T, DP, R>(scores, q, [&](int i, int k) { return widen<Code, O>(keys.w[i][k]); });
        const float factor = cache_factor(scale, keys.exponent);
        reader.load(keys, next);
        CacheTerms<T> p[R];
        if (!view.all(j0)) {
            hide_scores<R>(scores, rows, a.sinks, j0);
            const uint64_t keep = kept_bytes(s.nk - j0);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) values.w[t] = cut_bytes(values.w[t], keep);
        }
        cache_shares<T, DP, R>(p, state, scores, factor, max(values.exponent, kCacheLeast));
        add_cache_values<T, DP, R>(state, p, [&](int t) { return widen<Code, O>(values.w[t]); });
        reader.load(values, next);
    }
    close_state<T, DP, R>(state);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (g == 0) states[wave * kRows + 16 * r + n] = float2{state.top[r], state.sum[r]};
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float top = kCacheFloor, sum = 0.0f;
        for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, states[w * kRows + 16 * r + n].x);
        for (int w = 0; w < kAttnWaves; ++w) {
            const float2 other = states[w * kRows + 16 * r + n];
            sum += other.y * __builtin_amdgcn_exp2f(other.x - top);
        }
        const float mine = state.sum[r] * __builtin_amdgcn_exp2f(state.top[r] - top);
        state.rescale(r, sum != 0.0f ? mine / sum : 0.0f);
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
    if (splits == 1) {
        write_pairs<T, Code, DP, R>(call, s, s.index - 1, rows, state, out, &scratch);
        return;
    }
    const long long items = static_cast<long long>(a.queries) * a.heads;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (!rows[r].valid) continue;
        const long long row =
            split * items + (static_cast<long long>(s.q0) + rows[r].i) * a.heads + rows[r].head;
        if (g == 0) part.states[row] = float2{state.top[r], state.sum[r]};
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int d = 16 * t + 4 * g;
            if (d < c.dim) *reinterpret_cast<f32x4_attn*>(part.values + row * c.dim + d) = state.acc[r][t];
        }
    }
}

// Blocks of tokens as operands in LDS, 16 bytes a lane each, written as they are
// read: DP / 16 of a block's keys, or of its values.
template <typename T, typename Code, int DP>
struct CacheStage {
    typedef typename CacheMath<T>::Operand O;
    typedef typename CacheOperand<O>::Frag Frag;
    static constexpr int kFrags = DP / 16;
    static constexpr int kBytes = kFrags * kWave * 16;
    static_assert(kFrags % kAttnWaves == 0);
    static constexpr int kMine = kFrags / kAttnWaves;  // operands that a wave makes
    struct Codes {
        uint2 w[kMine];
    };

    const uint8_t* base;
    uint32_t place[kMine];

    // The keys or the values of `codes`.
    __device__ CacheStage(const void* codes, long long at, bool values, int wave)
        : base(static_cast<const uint8_t*>(codes) + at * kCacheBlock * DP) {
        const int n = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            const int f = wave + kAttnWaves * k;
            place[k] = values ? (16 * f + n) * kCacheBlock + 8 * g
                              : key_token(f / (DP / 32), n) * DP + key_channel<DP, false>(f % (DP / 32), g);
        }
    }
    // Starts the reads of a block's codes.
    __device__ void load(Codes& to, int block) const {
        const uint8_t* from = base + static_cast<long long>(block) * (kCacheBlock * DP);
#pragma unroll
        for (int k = 0; k < kMine; ++k) to.w[k] = *reinterpret_cast<const uint2*>(from + place[k]);
    }
    // Tokens from `count` on stand for nothing (values).
    __device__ static void cut(Codes& codes, int count) {
        const uint64_t keep = kept_bytes(count);
#pragma unroll
        for (int k = 0; k < kMine; ++k) codes.w[k] = cut_bytes(codes.w[k], keep);
    }
    // Widens a block's codes into `to`.
    __device__ static void write(char* to, const Codes& from, int wave) {
#pragma unroll
        for (int k = 0; k < kMine; ++k) {
            *reinterpret_cast<Frag*>(to + ((wave + kAttnWaves * k) * kWave + lane_id()) * 16) =
                widen<Code, O>(from.w[k]);
        }
    }
    __device__ static Frag operand(const char* from, int f) {
        return *reinterpret_cast<const Frag*>(from + (f * kWave + lane_id()) * 16);
    }
};

// For many queries: each wave has R tiles of pairs of its own; a block of tokens
// is widened once for the four, into LDS.  A step makes the shares of one block
// while the scores of the next are on their way through the matrix cores, then
// adds the block's values while the codes of the next are widened.
template <typename T, typename Code, int DP, int R>
__global__ void __launch_bounds__(kAttnBlock, 2)
cache_attend_many(CacheCall call, T* __restrict__ out) {
    typedef CacheStage<T, Code, DP> Stage;
    constexpr int kRows = 16 * R;
    __shared__ AttnRowScratch scratch[kAttnWaves];
    __shared__ __align__(16) char staged[4 * Stage::kBytes];
    const lattice_cache& c = call.cache;
    const lattice_cache_attention& a = call.args;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t group = a.heads / c.kv_heads;
    const int kv = blockIdx.x % c.kv_heads;
    constexpr int kSlot = kRows * kAttnWaves;
    const RowPartition partition{a.offsets, c.sequences, a.queries};
    const auto slot_of = [group](int start, int e) { return start * group / kSlot + e; };
    const uint32_t slot = cache_place(c.kv_heads, 1);
    const CacheSequence s = find_cache_sequence(partition, a.lengths, c.blocks * kCacheBlock, slot, slot_of);
    const uint32_t count = s.nq * group;
    const uint32_t start = slot_first<kSlot>(slot, slot_of(s.q0, s.index), count);
    if (start >= count) return;
    // A wave behind the last pair repeats it, unwritten.
    const uint32_t first = start + wave * kRows, mine = min(first, count - 1);

    CacheRow rows[R];
    cache_rows<R>(rows, call, s, kv, first);
    CacheTerms<T> q[R][DP / 32];
    cache_queries<T, DP, R, false>(q, call, s, rows);
    const float scale = fabsf(a.scale) * kAttnLog2e;
    const int p_low = static_cast<int>(mine / group) + s.shift();
    const int p_high = static_cast<int>((min(mine + kRows, count) - 1) / group) + s.shift();
    CacheState<T, DP, R> state;
    state.clear();
    const AttnTiles blocks = s.real
                                 ? cache_blocks(a, s.nk, static_cast<int>(start / group) + s.shift(),
                                                static_cast<int>((min(start + kSlot, count) - 1) / group) + s.shift())
                                 : AttnTiles{0, 0, 0};
    if (blocks.count > 0) {
        const long long at = (static_cast<long long>(s.index - 1) * c.kv_heads + kv) * c.blocks;
        const Stage keys(c.keys, at, false, wave), values(c.values, at, true, wave);
        const int8_t *key_exponents = c.key_exponents + at, *value_exponents = c.value_exponents + at;
        const CacheView view(a, s.nk, p_low, p_high);
        const int last = blocks.tile(blocks.count - 1);
        const auto after = [&](int tile) {
            return tile == last ? last : tile + 1 == blocks.first ? blocks.from : tile + 1;
        };
        const auto key_half = [&](int index) { return staged + (index & 1) * Stage::kBytes; };
        const auto value_half = [&](int index) { return staged + (2 + (index & 1)) * Stage::kBytes; };
        typename Stage::Codes k_codes, v_codes;
        const auto cut = [&](int tile) {
            const int tokens = s.nk - tile * kCacheBlock;
            if (tokens < kCacheBlock) Stage::cut(v_codes, tokens);
        };
        // Ready are the first two blocks' keys and the first's values, on their way
        // the third's keys and the second's values.
        int tile = blocks.tile(0), next = after(tile), second = after(next);
        keys.load(k_codes, tile);
        values.load(v_codes, tile);
        int key_exponent = key_exponents[tile], value_exponent = value_exponents[tile];
        int next_key_exponent = key_exponents[next], next_value_exponent = value_exponents[next];
        Stage::write(key_half(0), k_codes, wave);
        cut(tile);
        Stage::write(value_half(0), v_codes, wave);
        keys.load(k_codes, next);
        values.load(v_codes, next);
        Stage::write(key_half(1), k_codes, wave);
        keys.load(k_codes, second);
        __syncthreads();
        f32x4_attn scores[R][2];
        cache_scores<T, DP, R>(scores, q, [&](int i, int k) {
            return Stage::operand(key_half(0), i * (DP / 32) + k);
        });
        for (int index = 0; index < blocks.count; ++index) {
            const int j0 = tile * kCacheBlock;
            const int third = after(second);
            __syncthreads();
            // What lay there was last read before the barrier; long before the next
            // one it is written.
            Stage::write(key_half(index), k_codes, wave);
            cut(next);
            Stage::write(value_half(index + 1), v_codes, wave);
            keys.load(k_codes, third);
            values.load(v_codes, second);
            const int second_key_exponent = key_exponents[second], second_value_exponent = value_exponents[second];
            if (!view.all(j0)) hide_scores<R>(scores, rows, a.sinks, j0);
            f32x4_attn following[R][2];
            const char* key_now = key_half(index + 1);
            cache_scores<T, DP, R>(following, q, [&](int i, int k) {
                return Stage::operand(key_now, i * (DP / 32) + k);
            });
            CacheTerms<T> p[R];
            cache_shares<T, DP, R>(p, state, scores, cache_factor(scale, key_exponent),
                                   max(value_exponent, kCacheLeast));
            const char* value_now = value_half(index);
            add_cache_values<T, DP, R>(state, p, [&](int t) { return Stage::operand(value_now, t); });
            tile = next;
            next = second;
            second = third;
            key_exponent = next_key_exponent;
            value_exponent = next_value_exponent;
            next_key_exponent = second_key_exponent;
            next_value_exponent = second_value_exponent;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                scores[r][0] = following[r][0];
                scores[r][1] = following[r][1];
            }
        }
    }
    close_state<T, DP, R>(state);
    write_pairs<T, Code, DP, R>(call, s, s.index - 1, rows, state, out, &scratch[wave]);
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
    const float2 state = lane < splits ? part.states[lane * items + at] : float2{kCacheFloor, 0.0f};
    const float top = wave_max(state.x);
    const float mine = state.y * __builtin_amdgcn_exp2f(state.x - top);
    const float sum = wave_sum(mine), factor = sum != 0.0f ? mine / sum : 0.0f;
    // Each half of the wave has every second part, a lane four channels.
    const int half = lane >> 5, d = (lane & 31) * 4;
    const float* values = part.values + at * c.dim + min(d, c.dim - 4);
    f32x4_attn acc{};
#pragma unroll 8
    for (int z0 = 0; z0 < splits; z0 += 2) {
        // Both halves go around together: a lane that has left has no factor to give.
        const int z = min(z0 + half, splits - 1);
        const float share = __shfl(factor, z);
        acc += *reinterpret_cast<const f32x4_attn*>(values + z * items * c.dim) * (z0 + half < splits ? share : 0.0f);
    }
    bool finite = sum > 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        acc[i] += __shfl_xor(acc[i], 32);
        finite = finite && fabsf(acc[i]) < INFINITY;
    }
    // Rows that see nothing, and those that are not finite.
    if (__any(!finite)) {
        const int row = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
        const RowPartition partition{a.offsets, c.sequences, a.queries};
        const CacheSequence s =
            find_cache_sequence(partition, a.lengths, c.blocks * kCacheBlock, row,
                                [](int start, int) { return static_cast<uint32_t>(start); });
        attend_pair<T, Code>(call, s, s.index - 1, row - s.q0, head, out, &scratch[wave]);
        return;
    }
    if (half == 0 && d < c.dim) {
        RowVec<T, 4> v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v.set(i, acc[i]);
        v.store(out + at * c.dim + d);
    }
}

template <typename T, typename Code, int DP>
int launch_cache_attend(const CacheCall& call, const CacheLayout& l, const CachePart& part, T* out,
                        hipStream_t stream) {
    // Key heads next to each other: a die's L2 has few of them, and the blocks of
    // a unit are of unequal sequences (537 us, 550 slot by slot, for the chunks above).
    const dim3 grid = cache_grid(l.slots, call.cache.kv_heads, l.splits);
    const auto few = [&](auto kernel) { kernel<<<grid, kAttnBlock, 0, stream>>>(call, l.splits, part, out); };
    if (!l.share) {
        if constexpr (cache_many<T>(DP)) cache_attend_many<T, Code, DP, 2><<<grid, kAttnBlock, 0, stream>>>(call, out);
    } else if (l.tiles == 1) {
        few(cache_attend_few<T, Code, DP, 1>);
    } else if (l.tiles == 2) {
        few(cache_attend_few<T, Code, DP, 2>);
    } else if (cache_most_tiles<T>(DP) > 2) {
        few(cache_attend_few<T, Code, DP, cache_most_tiles<T>(DP)>);
    }
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
