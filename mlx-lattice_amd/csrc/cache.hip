// Writing rows into a cache of 8-bit codes, and reading it back.
//
//   e' = max(e of the block's earlier tokens, least e with max|x| <= most 2^e),
//   earlier codes: round(c 2^(e - e')), new codes: round(x 2^-e').
//
// A power of two as the scale makes every step exact but the last rounding, so
// that codes do not depend on how the quotient is computed; recoding e4m3 is
// exact but for its subnormals.
//
// A block of threads has one block of tokens of a key head, keys or values: it
// alone reads and writes those bytes.  Rows are read with 16-byte loads,
// reduced to the exponent, encoded into the block's image in LDS and merged
// into its pieces of 16 bytes.

#include "cache.h"

namespace lattice {
namespace {

constexpr int kCacheThreads = 256;
constexpr int kCacheImage = kCacheBlock * kAttnMaxDim;  // most bytes of a block

__device__ inline float threads_max(float v, float* shared) {
    v = wave_max(v);
    if (lane_id() == 0) shared[threadIdx.x / kWave] = v;
    __syncthreads();
    float most = shared[0];
    for (int w = 1; w < kCacheThreads / kWave; ++w) most = fmaxf(most, shared[w]);
    return most;
}

struct CacheSource {
    const void* rows;
    long long row_stride, head_stride;
};

// The place in a block's image of a token's channel.
__device__ inline int image_place(bool values, int width, int token, int channel) {
    return values ? channel * kCacheBlock + token : token * width + channel;
}

template <typename Code>
__device__ inline uint32_t recode(uint32_t word, float factor) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        out |= static_cast<uint32_t>(Code::code(Code::value(word >> 8 * i & 0xff) * factor)) << 8 * i;
    return out;
}

// Slots: of 32 rows and two more a sequence, enough for the blocks its rows
// touch.
__device__ inline uint32_t write_slot(int start, int e) { return static_cast<uint32_t>(start) / kCacheBlock + 2u * e; }

template <typename T, int V, typename Code>
__global__ void __launch_bounds__(kCacheThreads)
cache_write_blocks(lattice_cache c, CacheSource keys, CacheSource vals, int rows, const int32_t* __restrict__ offsets,
                   const int32_t* __restrict__ lengths) {
    typedef RowVec<T, V> Vec;
    constexpr int kHeld = kAttnMaxDim / (8 * V);  // vectors of a row that a thread holds, of 8 threads
    __shared__ float shared[kCacheThreads / kWave];
    __shared__ __align__(16) uint8_t image[kCacheImage];
    const uint32_t slot = block_slot(2);
    const bool values = block_part(2) != 0;
    const int head = blockIdx.y;
    const RowPartition partition{offsets, c.sequences, rows};
    const int e = partition.find(slot, write_slot);
    if (!partition.real(e)) return;
    const CacheSequence s = cache_sequence(partition, lengths, c.blocks * kCacheBlock, e);
    const int first = max(s.shift(), 0);
    const long long block = first / kCacheBlock + static_cast<long long>(slot - write_slot(s.q0, e));
    if (block >= c.blocks) return;
    const int lo = static_cast<int>(block) * kCacheBlock;
    const int begin = max(first, lo) - lo, end = min(s.nk - lo, kCacheBlock);
    if (begin >= end) return;

    const int width = cache_width(c);
    const long long at = (static_cast<long long>(e - 1) * c.kv_heads + head) * c.blocks + block;
    uint8_t* codes = static_cast<uint8_t*>(values ? c.values : c.keys) + at * kCacheBlock * width;
    int8_t* exponent = (values ? c.value_exponents : c.key_exponents) + at;
    const CacheSource& source = values ? vals : keys;

    const int token = threadIdx.x / 8, part = threadIdx.x % 8;
    const bool fresh = token >= begin && token < end;
    float x[kHeld][V];
    float most = 0.0f;
    const T* row = static_cast<const T*>(source.rows) +
                   (static_cast<long long>(s.q0) + (lo + token - s.shift())) * source.row_stride +
                   head * source.head_stride;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int channel = (part + 8 * k) * V;
        Vec in;
        const bool here = fresh && channel < c.dim;
        if (here) in = Vec::load(row + channel);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            x[k][j] = here ? in.at(j) : 0.0f;
            const float size = fabsf(x[k][j]);
            most = fmaxf(most, size < INFINITY ? size : 0.0f);
        }
    }
    const int before = max(static_cast<int>(*exponent), kCacheLeast);
    most = threads_max(most, shared);
    int next = block_exponent<Code>(most);
    if (begin > 0) next = max(next, before);
    const float factor = power_of_two(-next), moved = power_of_two(max(before - next, kCacheLeast));
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int channel = (part + 8 * k) * V;
        if (!fresh || channel >= width) continue;
#pragma unroll
        for (int j = 0; j < V; ++j)
            image[image_place(values, width, token, channel + j)] = Code::code(x[k][j] * factor);
    }
    __syncthreads();
    if (threadIdx.x == 0) *exponent = static_cast<int8_t>(next);
    // The image's pieces of 16 bytes: a token's channels, or a channel's tokens.
    for (int piece = threadIdx.x; piece < kCacheBlock * width / 16; piece += kCacheThreads) {
        uint4* to = reinterpret_cast<uint4*>(codes) + piece;
        const uint4 made = reinterpret_cast<const uint4*>(image)[piece];
        const uint32_t words[4] = {made.x, made.y, made.z, made.w};
        const int from = values ? 16 * (piece & 1) : 16 * piece / width;  // the first byte's token
        const int step = values ? 1 : 0;
        const int last = from + 15 * step;
        if (from >= end || (last < begin && before == next)) continue;
        if (from >= begin && last < end) {
            *to = made;
            continue;
        }
        const uint4 held = *to;
        const uint32_t old[4] = {held.x, held.y, held.z, held.w};
        uint32_t out[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t again = before == next ? old[w] : recode<Code>(old[w], moved);
            out[w] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = from + (4 * w + i) * step;
                const uint32_t word = t < begin ? again : t < end ? words[w] : old[w];
                out[w] |= word & 0xffu << 8 * i;
            }
        }
        *to = uint4{out[0], out[1], out[2], out[3]};
    }
}

// A block of tokens of a key head: keys as they lie, values by way of LDS.
template <typename T, int V, typename Code>
__global__ void __launch_bounds__(kCacheThreads)
cache_read_blocks(lattice_cache c, const int32_t* __restrict__ lengths, T* __restrict__ k, T* __restrict__ v) {
    typedef RowVec<T, V> Vec;
    __shared__ __align__(16) uint8_t image[kCacheImage];
    const int block = blockIdx.x % c.blocks, head = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const int width = cache_width(c);
    for (long long s = blockIdx.x / c.blocks; s < c.sequences; s += gridDim.x / c.blocks) {
        const int lo = block * kCacheBlock;
        const int filled = min(max(lengths[s], 0) - lo, kCacheBlock);
        const long long at = (s * c.kv_heads + head) * c.blocks + block;
        const uint4* codes =
            reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(values ? c.values : c.keys) + at * kCacheBlock * width);
        const float factor =
            power_of_two(max(static_cast<int>((values ? c.value_exponents : c.key_exponents)[at]), kCacheLeast));
        __syncthreads();
        if (filled > 0) {
            for (int piece = threadIdx.x; piece < kCacheBlock * width / 16; piece += kCacheThreads)
                reinterpret_cast<uint4*>(image)[piece] = codes[piece];
        }
        __syncthreads();
        T* out = (values ? v : k) + ((s * c.blocks * kCacheBlock + lo) * c.kv_heads + head) * c.dim;
        const int vectors = c.dim / V;
        for (int i = threadIdx.x; i < kCacheBlock * vectors; i += kCacheThreads) {
            const int token = i / vectors, channel = i % vectors * V;
            Vec row;
#pragma unroll
            for (int j = 0; j < V; ++j)
                row.set(j, token < filled
                               ? Code::value(image[image_place(values, width, token, channel + j)]) * factor
                               : 0.0f);
            row.store(out + static_cast<long long>(token) * c.kv_heads * c.dim + channel);
        }
    }
}

template <typename T, typename Code>
int write_of(const lattice_cache& c, const CacheSource& k, const CacheSource& v, int rows, const int32_t* offsets,
             const int32_t* lengths, hipStream_t stream) {
    constexpr int kMost = 16 / sizeof(T);
    const int vector = row_vector<T>(c.dim, {k.rows, v.rows},
                                     {k.row_stride, k.head_stride, v.row_stride, v.head_stride});
    const long long slots = static_cast<long long>(rows) / kCacheBlock + 2ll * (c.sequences + 2);
    const dim3 grid = slot_grid(slots, c.kv_heads, 2);
    if (vector == kMost) {
        cache_write_blocks<T, kMost, Code><<<grid, kCacheThreads, 0, stream>>>(c, k, v, rows, offsets, lengths);
    } else {
        cache_write_blocks<T, 1, Code><<<grid, kCacheThreads, 0, stream>>>(c, k, v, rows, offsets, lengths);
    }
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T, typename Code>
int read_of(const lattice_cache& c, const int32_t* lengths, void* k, void* v, hipStream_t stream) {
    constexpr int kMost = 16 / sizeof(T);
    // Blocks of threads below 2^22 along x; the rest of the sequences follow in
    // their loops.
    const int together = static_cast<int>(std::max(1ll, std::min<long long>(c.sequences, (1ll << 22) / c.blocks)));
    const dim3 grid(static_cast<unsigned>(together) * c.blocks, c.kv_heads, 2);
    T *keys = static_cast<T*>(k), *values = static_cast<T*>(v);
    if (row_vector<T>(c.dim, {k, v}, {}) == kMost) {
        cache_read_blocks<T, kMost, Code><<<grid, kCacheThreads, 0, stream>>>(c, lengths, keys, values);
    } else {
        cache_read_blocks<T, 1, Code><<<grid, kCacheThreads, 0, stream>>>(c, lengths, keys, values);
    }
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename Code>
int write_code(const lattice_cache& c, int dtype, const CacheSource& k, const CacheSource& v, int rows,
               const int32_t* offsets, const int32_t* lengths, hipStream_t stream) {
    if (dtype == LATTICE_F32) return write_of<float, Code>(c, k, v, rows, offsets, lengths, stream);
    if (dtype == LATTICE_F16) return write_of<_Float16, Code>(c, k, v, rows, offsets, lengths, stream);
    return write_of<__bf16, Code>(c, k, v, rows, offsets, lengths, stream);
}

template <typename Code>
int read_code(const lattice_cache& c, int dtype, const int32_t* lengths, void* k, void* v, hipStream_t stream) {
    if (dtype == LATTICE_F32) return read_of<float, Code>(c, lengths, k, v, stream);
    if (dtype == LATTICE_F16) return read_of<_Float16, Code>(c, lengths, k, v, stream);
    return read_of<__bf16, Code>(c, lengths, k, v, stream);
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" int lattice_hip_cache_write(const lattice_cache* cache, int dtype, const void* k, long long k_row_stride,
                                       long long k_head_stride, const void* v, long long v_row_stride,
                                       long long v_head_stride, int rows, const int32_t* offsets,
                                       const int32_t* lengths, void* stream_ptr) {
    LATTICE_REQUIRE_CACHE(cache);
    LATTICE_REQUIRE(dtype == LATTICE_F32 || dtype == LATTICE_F16 || dtype == LATTICE_BF16,
                    "cache rows must be float32, float16 or bfloat16.");
    LATTICE_REQUIRE(rows >= 0 && rows < 1 << 29, "caches take up to 2^29 - 1 rows at once.");
    LATTICE_REQUIRE(k_row_stride >= 0 && k_head_stride >= 0 && v_row_stride >= 0 && v_head_stride >= 0,
                    "cache row strides must be non-negative.");
    if (rows == 0 || cache->sequences == 0 || cache->blocks == 0) return LATTICE_OK;
    LATTICE_REQUIRE(k && v && offsets && lengths, "cache row pointers must be non-null.");
    const CacheSource keys{k, k_row_stride, k_head_stride}, values{v, v_row_stride, v_head_stride};
    hipStream_t stream = as_stream(stream_ptr);
    if (cache->code == LATTICE_CODE_E4M3)
        return write_code<CodeE4m3>(*cache, dtype, keys, values, rows, offsets, lengths, stream);
    return write_code<CodeInt8>(*cache, dtype, keys, values, rows, offsets, lengths, stream);
}

extern "C" int lattice_hip_cache_read(const lattice_cache* cache, int dtype, const int32_t* lengths, void* k, void* v,
                                      void* stream_ptr) {
    LATTICE_REQUIRE_CACHE(cache);
    LATTICE_REQUIRE(dtype == LATTICE_F32 || dtype == LATTICE_F16 || dtype == LATTICE_BF16,
                    "cache rows must be float32, float16 or bfloat16.");
    if (cache->sequences == 0 || cache->blocks == 0) return LATTICE_OK;
    LATTICE_REQUIRE(k && v && lengths, "cache row pointers must be non-null.");
    hipStream_t stream = as_stream(stream_ptr);
    if (cache->code == LATTICE_CODE_E4M3) return read_code<CodeE4m3>(*cache, dtype, lengths, k, v, stream);
    return read_code<CodeInt8>(*cache, dtype, lengths, k, v, stream);
}
