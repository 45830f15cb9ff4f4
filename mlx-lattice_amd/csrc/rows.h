// Element types and vectors of the row operators (layer norm, dropout, rotary
// positions, attention): loads widen to fp32, stores round once, to nearest
// even.
#pragma once

#include <hip/hip_bf16.h>

#include <algorithm>
#include <initializer_list>

#include "lattice_common.h"

namespace lattice {

typedef unsigned int u32x2_row_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4_row_t __attribute__((ext_vector_type(4)));

// The unsigned type of BYTES bytes that a vector is moved as.
template <int BYTES> struct RowBits;
template <> struct RowBits<2> { typedef uint16_t type; };
template <> struct RowBits<4> { typedef uint32_t type; };
template <> struct RowBits<8> { typedef u32x2_row_t type; };
template <> struct RowBits<16> { typedef u32x4_row_t type; };

// V consecutive elements of T (at most 16 bytes), aligned to their size.
template <typename T, int V>
struct RowVec {
    typedef typename RowBits<static_cast<int>(sizeof(T)) * V>::type Bits;
    T e[V];

    __device__ static RowVec load(const T* p) {
        return __builtin_bit_cast(RowVec, *reinterpret_cast<const Bits*>(p));
    }
    __device__ void store(T* p) const { *reinterpret_cast<Bits*>(p) = __builtin_bit_cast(Bits, *this); }
    // Streamed past the caches, for results that are not read back soon.
    __device__ void store_through(T* p) const {
        __builtin_nontemporal_store(__builtin_bit_cast(Bits, *this), reinterpret_cast<Bits*>(p));
    }
    __device__ float at(int i) const { return static_cast<float>(e[i]); }
    __device__ void set(int i, float v) { e[i] = static_cast<T>(v); }
};

// The widest vector, up to 16 bytes, that divides `channels` and fits the
// alignment of every address and row stride (in elements).
template <typename T>
inline int row_vector(long long channels, std::initializer_list<const void*> addresses,
                      std::initializer_list<long long> strides) {
    int v = 16 / static_cast<int>(sizeof(T));
    for (; v > 1; v /= 2) {
        bool fits = channels % v == 0;
        for (const void* a : addresses) fits = fits && reinterpret_cast<uintptr_t>(a) % (v * sizeof(T)) == 0;
        for (long long s : strides) fits = fits && s % v == 0;
        if (fits) break;
    }
    return v;
}

}  // namespace lattice
