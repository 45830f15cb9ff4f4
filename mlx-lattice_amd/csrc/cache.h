// A cache of keys and values in 8 bits: its codes, its sequences and what every
// entry checks.
#pragma once

#include "attention_tiles.h"

namespace lattice {

constexpr int kCacheBlock = 32;        // tokens that share an exponent
constexpr int kCacheLeast = -126;      // the least exponent: 2^e is a normal number
constexpr int kCacheLongest = 1 << 29;  // lengths are clamped to it, so that positions stay inside 32 bits

// 2^e for e in -126 .. 127.
__device__ inline float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// 2^-e for e in -126 .. 127, the last of which is below the normal numbers.
__device__ inline float inverse_power(int e) {
    return __uint_as_float(e < 127 ? static_cast<uint32_t>(127 - e) << 23 : 1u << 22);
}

typedef __bf16 bf16x2_cache __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_cache __attribute__((ext_vector_type(2)));

// What a code type does: the exponent that holds a magnitude, codes from
// values, and values (whole in any of the operand types: codes have at most 7
// significant bits) from codes.
struct CodeE4m3 {
    // 448 = 1.75 * 2^8.
    static constexpr int kShift = 9;
    static constexpr uint32_t kMostMantissa = 0x600000;

    static constexpr bool kHasNan = true;

    // Codes of one, two or four values times `factor`, the first in the lowest
    // byte; what is not finite becomes NaN.
    template <int N>
    __device__ static uint32_t codes(const float (&x)[N], float factor) {
        int out = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * factor, x[N > 1 ? 1 : 0] * factor, 0, false);
        if constexpr (N == 4) out = __builtin_amdgcn_cvt_pk_fp8_f32(x[2] * factor, x[3] * factor, out, true);
        return static_cast<uint32_t>(out) & (N == 4 ? ~0u : N == 2 ? 0xffffu : 0xffu);
    }
    __device__ static float value(uint8_t c) { return __builtin_amdgcn_cvt_f32_fp8(c, 0); }
    // The values of four codes.
    __device__ static void values(uint32_t w, bf16x2_cache* v) {
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    }
    __device__ static void values(uint32_t w, f16x2_cache* v) {
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
    }
};
struct CodeInt8 {
    static constexpr int kShift = 7;
    static constexpr uint32_t kMostMantissa = 0x7e0000;  // 127 = 1.984375 * 2^6

    static constexpr bool kHasNan = false;

    // As above, of products from -127 to 127: 1.5 2^23 more has the rounded
    // product in its low bits.
    template <int N>
    __device__ static uint32_t codes(const float (&x)[N], float factor) {
        uint32_t w[4] = {};
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __float_as_uint(__builtin_fmaf(x[i], factor, 12582912.0f));
        if constexpr (N == 1) return w[0] & 0xffu;
        const uint32_t low = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400u);
        if constexpr (N == 2) return low;
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w[3], w[2], 0x0c0c0400u), low, 0x05040100u);
    }
    __device__ static float value(uint8_t c) { return static_cast<float>(static_cast<int8_t>(c)); }
    __device__ static void values(uint32_t w, bf16x2_cache* v) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            v[i] = bf16x2_cache{static_cast<__bf16>(value(w >> 16 * i & 0xff)),
                                static_cast<__bf16>(value(w >> (16 * i + 8) & 0xff))};
    }
    // 1024 + (c + 128) has the bits 0x6400 | (c + 128) in half precision.
    __device__ static void values(uint32_t w, f16x2_cache* v) {
        const uint32_t biased = w ^ 0x80808080u;
        const f16x2_cache bias{static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
        v[0] = __builtin_bit_cast(f16x2_cache, __builtin_amdgcn_perm(0x64646464u, biased, 0x04010400u)) - bias;
        v[1] = __builtin_bit_cast(f16x2_cache, __builtin_amdgcn_perm(0x64646464u, biased, 0x04030402u)) - bias;
    }
};

// The exponent of a block whose largest magnitude is `most`.
template <typename Code>
__device__ inline int block_exponent(float most) {
    const uint32_t bits = __float_as_uint(most);
    const int e = static_cast<int>(bits >> 23) - 126 - Code::kShift + ((bits & 0x7fffffu) > Code::kMostMantissa);
    return max(e, kCacheLeast);
}

// A sequence: its rows q0 .. q0 + nq, the last of `length` tokens, of which the
// cache has `nk`; row i is token i + shift.
struct CacheSequence {
    int index;  // as RowPartition counts
    bool real;
    int q0, nq, nk, length;
    __device__ int shift() const { return length - nq; }
};
__device__ inline CacheSequence cache_sequence(const RowPartition& rows, int capacity, int e, int from, int to,
                                               int length) {
    CacheSequence s;
    s.index = e;
    s.real = rows.real(e);
    s.q0 = from;
    s.nq = max(0, to - from);
    s.length = s.real ? min(max(length, 0), kCacheLongest) : 0;
    s.nk = min(s.length, capacity);
    return s;
}
// The last sequence whose first slot is at most `slot`, as RowPartition finds it;
// all lanes of the wave together.  Up to 61 sequences are a read of the offsets
// and lengths, which does not wait for the search: 0.2 of the 6.2 us in which one
// token of 32 sequences is written.
template <typename SlotOf>
__device__ inline CacheSequence find_cache_sequence(const RowPartition& rows, const int32_t* lengths, int capacity,
                                                    uint32_t slot, SlotOf slot_of) {
    if (rows.count + 3 <= kWave) {
        const int lane = lane_id(), at = rows.start(lane), length = rows.real(lane) ? lengths[lane - 1] : 0;
        const bool at_most = lane < rows.count + 2 && slot_of(at, lane) <= slot;
        const int e = max(1, static_cast<int>(__popcll(ballot(at_most)))) - 1;
        return cache_sequence(rows, capacity, e, __builtin_amdgcn_readlane(at, e),
                              __builtin_amdgcn_readlane(at, e + 1), __builtin_amdgcn_readlane(length, e));
    }
    const int e = rows.find(slot, slot_of);
    return cache_sequence(rows, capacity, e, rows.start(e), rows.start(e + 1), rows.real(e) ? lengths[e - 1] : 0);
}

// Places, slots or blocks of tokens, of `groups` blocks of threads each, next to
// each other; those past 2^22 blocks of threads go on along z, above `parts`.
inline dim3 cache_grid(long long places, uint32_t groups, int parts) {
    const long long x = std::min<long long>(places, (1 << 22) / groups);
    return dim3(static_cast<unsigned>(x) * groups, 1, static_cast<unsigned>((places + x - 1) / x * parts));
}
__device__ inline uint32_t cache_place(uint32_t groups, uint32_t parts) {
    return blockIdx.x / groups + gridDim.x / groups * (parts == 1 ? blockIdx.z : blockIdx.z / parts);
}

__host__ __device__ inline int cache_width(const lattice_cache& c) { return (c.dim + 31) / 32 * 32; }

// What every entry checks; NULL, or what is wrong.
inline const char* cache_fault(const lattice_cache* c) {
    if (!c) return "cache arguments must be non-null.";
    if (c->code != LATTICE_CODE_E4M3 && c->code != LATTICE_CODE_INT8) return "caches hold e4m3 or int8 codes.";
    if (c->sequences < 0 || c->kv_heads < 1 || c->blocks < 0) return "cache shapes must be positive.";
    if (c->sequences >= 1 << 24 || c->kv_heads >= 1 << 16 || c->blocks >= 1 << 23)
        return "caches have under 2^24 sequences, 2^16 key heads and 2^28 tokens.";
    if (c->dim < 1 || c->dim > kAttnMaxDim) return "cache heads must have between 1 and 128 channels.";
    if (c->sequences == 0 || c->blocks == 0) return nullptr;
    if (!c->keys || !c->values || !c->key_exponents || !c->value_exponents) return "cache pointers must be non-null.";
    if ((reinterpret_cast<uintptr_t>(c->keys) | reinterpret_cast<uintptr_t>(c->values)) % 16 != 0)
        return "cache codes must lie on 16-byte boundaries.";
    return nullptr;
}

#define LATTICE_REQUIRE_CACHE(cache)                              \
    do {                                                          \
        if (const char* fault_ = ::lattice::cache_fault(cache)) { \
            ::lattice::set_error(fault_);                         \
            return LATTICE_ERROR_INVALID_ARGUMENT;                \
        }                                                         \
    } while (0)

}  // namespace lattice
