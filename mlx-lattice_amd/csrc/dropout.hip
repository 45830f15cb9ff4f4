// Dropout from a counter-based generator.
//
// Element e is kept when its 32-bit word reaches a threshold; the word is word
// e % 4 of Philox 4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011) over the counter (e / 4, offset) and
// the key `seed`.  The mask is a function of (seed, offset, e), so it is never
// stored: the gradient makes it again.
//
// Bound by memory where the residual is read with the values (6 bytes a value
// in half precision); the generator's twenty 32 x 32 -> 64 products for four
// values come near that bound otherwise (one v_mad_u64_u32 a product, a quarter of
// the issue rate).  A lane takes V consecutive values, V / 4 counters, in
// 16-byte moves.  400,000 x 128 fp16 with a residual: 52 us (5.9 TB/s, part of
// it from the Infinity Cache), its gradient 44 us (4.7 TB/s).

#include "rows.h"

namespace lattice {
namespace {

constexpr int kDropoutBlock = 256;

struct PhiloxWords {
    uint32_t w[4];
};

__device__ inline PhiloxWords philox(uint64_t number, uint64_t offset, uint64_t seed) {
    uint32_t c0 = static_cast<uint32_t>(number), c1 = static_cast<uint32_t>(number >> 32);
    uint32_t c2 = static_cast<uint32_t>(offset), c3 = static_cast<uint32_t>(offset >> 32);
    uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u;
        const uint64_t b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
        c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
        c1 = static_cast<uint32_t>(b);
        c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
        c3 = static_cast<uint32_t>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// V (4 or 8) consecutive values a lane; a threshold of 2^32 keeps none.  A
// dropped value is replaced, not multiplied by zero: an infinity or a NaN
// that is dropped leaves no trace.
template <typename T, int V, bool ALIGNED>
__global__ void __launch_bounds__(kDropoutBlock)
dropout_values(const T* __restrict__ x, const T* __restrict__ residual, long long count, uint64_t seed,
               uint64_t offset, uint64_t threshold, float scale, T* __restrict__ y) {
    typedef RowVec<T, V> Vec;
    const long long step = static_cast<long long>(gridDim.x) * kDropoutBlock * V;
    for (long long e = (static_cast<long long>(blockIdx.x) * kDropoutBlock + threadIdx.x) * V; e < count; e += step) {
        const bool whole = ALIGNED && e + V <= count;
        Vec a, r, out;
        if (whole) {
            a = Vec::load(x + e);
            if (residual) r = Vec::load(residual + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (e + j < count) {
                    a.e[j] = x[e + j];
                    if (residual) r.e[j] = residual[e + j];
                }
            }
        }
#pragma unroll
        for (int c = 0; c < V / 4; ++c) {
            const PhiloxWords words = philox(static_cast<uint64_t>(e) / 4 + c, offset, seed);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float kept = words.w[j] >= threshold ? a.at(4 * c + j) * scale : 0.0f;
                out.set(4 * c + j, residual ? r.at(4 * c + j) + kept : kept);
            }
        }
        if (whole) {
            out.store(y + e);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (e + j < count) y[e + j] = out.e[j];
        }
    }
}

template <typename T>
int dropout_of(const void* x, const void* residual, long long count, uint64_t seed, uint64_t offset,
               uint64_t threshold, float scale, void* y, hipStream_t stream) {
    constexpr int kMost = 16 / sizeof(T);
    const uintptr_t bits = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
                           reinterpret_cast<uintptr_t>(y);
    const T* in = static_cast<const T*>(x);
    const T* res = static_cast<const T*>(residual);
    T* out = static_cast<T*>(y);
    if (bits % 16 == 0) {
        dropout_values<T, kMost, true><<<grid_for(count, kDropoutBlock * kMost, 1u << 16), kDropoutBlock, 0, stream>>>(
            in, res, count, seed, offset, threshold, scale, out);
    } else {
        dropout_values<T, 4, false><<<grid_for(count, kDropoutBlock * 4, 1u << 16), kDropoutBlock, 0, stream>>>(
            in, res, count, seed, offset, threshold, scale, out);
    }
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" int lattice_hip_dropout(int dtype, const void* x, const void* residual, long long count, uint64_t seed,
                                   uint64_t offset, uint64_t threshold, float scale, void* y, void* stream_ptr) {
    LATTICE_REQUIRE(dtype == LATTICE_F32 || dtype == LATTICE_F16 || dtype == LATTICE_BF16,
                    "dropout supports float32, float16 and bfloat16.");
    LATTICE_REQUIRE(count >= 0, "the number of values must be non-negative.");
    LATTICE_REQUIRE(threshold <= 1ull << 32, "the threshold must be at most 2^32.");
    if (count == 0) return LATTICE_OK;
    LATTICE_REQUIRE(x && y, "dropout pointers must be non-null.");
    hipStream_t stream = as_stream(stream_ptr);
    if (dtype == LATTICE_F32) return dropout_of<float>(x, residual, count, seed, offset, threshold, scale, y, stream);
    if (dtype == LATTICE_F16)
        return dropout_of<_Float16>(x, residual, count, seed, offset, threshold, scale, y, stream);
    return dropout_of<__bf16>(x, residual, count, seed, offset, threshold, scale, y, stream);
}
