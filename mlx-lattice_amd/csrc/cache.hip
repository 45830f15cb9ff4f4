// Writing rows into a cache of 8-bit codes, and reading it back.
//
//   e' = max(e of the block's earlier tokens, least e with max|x| <= most 2^e),
//   earlier codes: round(c 2^(e - e')), new codes: round(x 2^-e').
//
// A power of two as the scale makes every step exact but the last rounding, so
// that codes do not depend on how the quotient is computed; recoding e4m3 is
// exact but for its subnormals.
//
// Bound by memory: writing reads 2 to 4 bytes a value and writes one, reading the
// other way round.  A wave has one block of tokens of a key head, keys or values:
// it alone reads and writes those bytes.  A lane holds some successive tokens of
// some successive channels, 16 bytes of a row a load, so that keys are encoded
// along its channels and values along its tokens, and either is stored as it
// lies, with no exchange but the maximum's; LDS in between, as at first, took 57
// us where this takes 47.  Blocks of threads that follow each other have the
// heads of one block of tokens, whose rows lie together.
//
// 30001 rows of 8 key heads of 128 channels, keys and values: 61 us from float32
// (5.0 TB/s), 47 from half precision to int8 (3.9 TB/s; 120004 rows 4.5).  8-byte
// loads, with more tokens a lane, take 61 us.  One token of 32 sequences: 6.2 us,
// the launch and four reads that wait for each other.  Reading 65536 tokens of 4
// key heads of 128 channels to bfloat16: 31 us (5.9 TB/s, codes partly from the
// last cache), 41 with nothing cached; heads of 32 channels at the same rate.

#include "cache.h"

namespace lattice {
namespace {

constexpr int kCacheThreads = 256;

struct CacheSource {
    const void* rows;
    long long row_stride, head_stride;
};

template <typename Code>
__device__ inline uint32_t recode(uint32_t word, float factor) {
    const float x[4] = {Code::value(word & 0xff), Code::value(word >> 8 & 0xff), Code::value(word >> 16 & 0xff),
                        Code::value(word >> 24)};
    return Code::codes(x, factor);
}

// Codes of values, some of which are not finite if `odd`: an infinity has the
// code of largest size, NaN its own or zero.
template <typename Code, int N>
__device__ inline uint32_t encode(const float (&x)[N], float factor, bool odd) {
    if constexpr (!Code::kHasNan) {
        if (odd) {
            float y[N];
#pragma unroll
            for (int i = 0; i < N; ++i) y[i] = x[i] == x[i] ? __builtin_amdgcn_fmed3f(x[i] * factor, -127.0f, 127.0f) : 0.0f;
            return Code::codes(y, 1.0f);
        }
    }
    return Code::codes(x, factor);
}

// Slots: of 32 rows and two more a sequence, enough for the blocks its rows
// touch.
__device__ inline uint32_t write_slot(int start, int e) { return static_cast<uint32_t>(start) / kCacheBlock + 2u * e; }

// Blocks of threads for the keys and values of all heads.
__host__ __device__ inline uint32_t head_groups(int kv_heads) {
    return (2u * kv_heads + kCacheThreads / kWave - 1) / (kCacheThreads / kWave);
}

inline bool cache_fits(const lattice_cache& c, long long places) {
    return places < 1ll << 31 && places * head_groups(c.kv_heads) < 1ll << 36;
}

// N bytes as they are moved.
template <int N> struct CacheBytes {
    alignas(N < 4 ? 4 : N) uint32_t w[(N + 3) / 4];
    __device__ static CacheBytes load(const uint8_t* p) {
        CacheBytes b;
        if constexpr (N >= 4) {
            typedef typename RowBits<N>::type Bits;
            *reinterpret_cast<Bits*>(b.w) = *reinterpret_cast<const Bits*>(p);
        } else {
            b.w[0] = N == 2 ? *reinterpret_cast<const uint16_t*>(p) : *p;
        }
        return b;
    }
    __device__ void store(uint8_t* p) const {
        if constexpr (N >= 4) {
            typedef typename RowBits<N>::type Bits;
            *reinterpret_cast<Bits*>(p) = *reinterpret_cast<const Bits*>(w);
        } else if constexpr (N == 2) {
            *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(w[0]);
        } else {
            *p = static_cast<uint8_t>(w[0]);
        }
    }
};

// The largest magnitude of rows' values, infinite or NaN if one of them is: the
// bits of magnitudes are ordered.
template <typename T, int V>
struct Magnitude {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    uint32_t bits = 0;
    __device__ void add(const RowVec<T, V>& v) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < V; ++j) bits = max(bits, __float_as_uint(v.e[j]) & 0x7fffffffu);
        } else if constexpr (V == 1) {
            bits = max(bits, __builtin_bit_cast(uint16_t, v.e[0]) & 0x7fffu);
        } else {
            struct Words {
                uint32_t w[V / 2];
            };
            const Words words = __builtin_bit_cast(Words, v);
#pragma unroll
            for (int j = 0; j < V / 2; ++j)
                bits = __builtin_bit_cast(
                    uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, bits),
                                                        __builtin_bit_cast(u16x2, words.w[j] & 0x7fff7fffu)));
        }
    }
    __device__ float value() const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(bits);
        } else {
            return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(max(bits & 0xffffu, bits >> 16))));
        }
    }
};

// How a wave's lanes hold a block of 32 tokens of DP channels, V of them a load:
// kAcross lanes a row, kTokens successive tokens and kGroups vectors of channels a
// lane.
template <int DP, int V>
struct CacheHold {
    static constexpr int kVectors = DP / V;
    static constexpr int kAcross = kVectors > 32 ? 64 : kVectors > 16 ? 32 : kVectors > 8 ? 16 : kVectors > 4 ? 8 : 4;
    static constexpr int kGroups = (kVectors + kAcross - 1) / kAcross;
    static constexpr int kTokens = kAcross / 2;  // 32 tokens over 64 / kAcross lanes
};

template <typename T, int V, typename Code, int DP>
__global__ void __launch_bounds__(kCacheThreads)
cache_write_blocks(lattice_cache c, CacheSource keys, CacheSource vals, int rows, const int32_t* __restrict__ offsets,
                   const int32_t* __restrict__ lengths) {
    typedef RowVec<T, V> Vec;
    typedef CacheHold<DP, V> Hold;
    constexpr int kTokens = Hold::kTokens, kGroups = Hold::kGroups;
    // The heads of a slot next to each other, as they lie in its rows.
    const uint32_t groups = head_groups(c.kv_heads);
    const uint32_t slot = cache_place(groups, 1);
    const int task = blockIdx.x % groups * (kCacheThreads / kWave) + threadIdx.x / kWave;
    const RowPartition partition{offsets, c.sequences, rows};
    const CacheSequence s = find_cache_sequence(partition, lengths, c.blocks * kCacheBlock, slot, write_slot);
    if (!s.real || task >= 2 * c.kv_heads) return;
    const bool values = task & 1;
    const int head = task >> 1;
    const int first = max(s.shift(), 0);
    const long long block = first / kCacheBlock + static_cast<long long>(slot - write_slot(s.q0, s.index));
    if (block >= c.blocks) return;
    const int lo = static_cast<int>(block) * kCacheBlock;
    const int begin = max(first, lo) - lo, end = min(s.nk - lo, kCacheBlock);
    if (begin >= end) return;

    const long long at = (static_cast<long long>(s.index - 1) * c.kv_heads + head) * c.blocks + block;
    uint8_t* codes = static_cast<uint8_t*>(values ? c.values : c.keys) + at * kCacheBlock * DP;
    int8_t* exponent = (values ? c.value_exponents : c.key_exponents) + at;
    const CacheSource& source = values ? vals : keys;
    const int before = max(static_cast<int>(*exponent), kCacheLeast);
    const int lane = lane_id();
    const int token0 = lane / Hold::kAcross * kTokens, channel0 = lane % Hold::kAcross * V;
    const T* from = static_cast<const T*>(source.rows) +
                    (static_cast<long long>(s.q0) + (lo + token0 - s.shift())) * source.row_stride +
                    head * source.head_stride + channel0;
    Vec in[kTokens][kGroups];
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
        const bool fresh = token0 + t >= begin && token0 + t < end;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int channel = channel0 + g * Hold::kAcross * V;
#pragma unroll
            for (int j = 0; j < V; ++j) in[t][g].set(j, 0.0f);
            if (fresh && channel < c.dim) in[t][g] = Vec::load(from + t * source.row_stride + g * Hold::kAcross * V);
        }
    }
    // A lane's tokens of a channel lie together among the values; those that are
    // not all new are merged into what is there.
    constexpr int kBytes = kTokens > 16 ? 16 : kTokens, kParts = kTokens / kBytes;
    const bool whole = token0 >= begin && token0 + kTokens <= end;
    CacheBytes<kBytes> held[kGroups][V][kParts] = {};
    if (values && !whole && token0 < end) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const int channel = channel0 + g * Hold::kAcross * V + j;
                if (channel >= DP) continue;
#pragma unroll
                for (int part = 0; part < kParts; ++part)
                    held[g][j][part] =
                        CacheBytes<kBytes>::load(codes + channel * kCacheBlock + token0 + part * kBytes);
            }
        }
    }
    Magnitude<T, V> largest;
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) largest.add(in[t][g]);
    }
    float most = largest.value();
    const bool odd = __any(!(most < INFINITY));
    if (odd) {  // of what is finite
        most = 0.0f;
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float size = fabsf(in[t][g].at(j));
                    most = fmaxf(most, size < INFINITY ? size : 0.0f);
                }
            }
        }
    }
    int next = block_exponent<Code>(wave_max(most));
    if (begin > 0) next = max(next, before);
    const bool moves = begin > 0 && next != before;
    const float factor = inverse_power(next), moved = power_of_two(max(before - next, kCacheLeast));
    if (lane == 0) *exponent = static_cast<int8_t>(next);
    if (!values) {
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            const int token = token0 + t;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int channel = channel0 + g * Hold::kAcross * V;
                if (channel >= DP || token >= end || (token < begin && !moves)) continue;
                uint8_t* to = codes + token * DP + channel;
                CacheBytes<V> out;
                if (token < begin) {
                    out = CacheBytes<V>::load(to);
#pragma unroll
                    for (int w = 0; w < (V + 3) / 4; ++w) out.w[w] = recode<Code>(out.w[w], moved);
                } else {
#pragma unroll
                    for (int w = 0; w < (V + 3) / 4; ++w) {
                        float x[V < 4 ? V : 4];
#pragma unroll
                        for (int i = 0; i < (V < 4 ? V : 4); ++i) x[i] = in[t][g].at(4 * w + i);
                        out.w[w] = encode<Code>(x, factor, odd);
                    }
                }
                out.store(to);
            }
        }
        return;
    }
    const bool some = token0 < end && (moves || token0 + kTokens > begin);
    if (!some) return;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int channel = channel0 + g * Hold::kAcross * V + j;
            if (channel >= DP) continue;
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                uint8_t* to = codes + channel * kCacheBlock + token0 + part * kBytes;
                CacheBytes<kBytes> out;
#pragma unroll
                for (int w = 0; w < (kBytes + 3) / 4; ++w) {
                    float x[kBytes < 4 ? kBytes : 4];
#pragma unroll
                    for (int i = 0; i < (kBytes < 4 ? kBytes : 4); ++i)
                        x[i] = in[part * kBytes + 4 * w + i][g].at(j);
                    out.w[w] = encode<Code>(x, factor, odd);
                }
                if (!whole) {
#pragma unroll
                    for (int w = 0; w < (kBytes + 3) / 4; ++w) {
                        const uint32_t old = held[g][j][part].w[w];
                        const uint32_t again = moves ? recode<Code>(old, moved) : old;
                        uint32_t merged = 0;
#pragma unroll
                        for (int i = 0; i < (kBytes < 4 ? kBytes : 4); ++i) {
                            const int token = token0 + part * kBytes + 4 * w + i;
                            const uint32_t word = token < begin ? again : token < end ? out.w[w] : old;
                            merged |= word & 0xffu << 8 * i;
                        }
                        out.w[w] = merged;
                    }
                }
                out.store(to);
            }
        }
    }
}

// The value of a lane's byte i, tokens or channels, of codes as they are moved.
template <typename Code, int N>
__device__ inline float value_of(const CacheBytes<N>& b, int i) {
    return Code::value(static_cast<uint8_t>(b.w[i / 4] >> 8 * (i % 4)));
}

// The inverse, of the same lanes: what is behind a sequence's last token is zero.
template <typename T, int V, typename Code, int DP>
__global__ void __launch_bounds__(kCacheThreads)
cache_read_blocks(lattice_cache c, const int32_t* __restrict__ lengths, T* __restrict__ k, T* __restrict__ v) {
    typedef RowVec<T, V> Vec;
    typedef CacheHold<DP, V> Hold;
    constexpr int kTokens = Hold::kTokens, kGroups = Hold::kGroups;
    // The heads of a block next to each other, as they lie in its rows.
    const uint32_t groups = head_groups(c.kv_heads);
    const uint32_t place = cache_place(groups, 1);
    const int task = blockIdx.x % groups * (kCacheThreads / kWave) + threadIdx.x / kWave;
    const long long s = place / c.blocks;
    const int block = place % c.blocks;
    if (s >= c.sequences || task >= 2 * c.kv_heads) return;
    const bool values = task >= c.kv_heads;
    const int head = values ? task - c.kv_heads : task;
    const int lo = block * kCacheBlock;
    const int filled = min(max(lengths[s], 0) - lo, kCacheBlock);
    const long long at = (s * c.kv_heads + head) * c.blocks + block;
    const uint8_t* codes = static_cast<const uint8_t*>(values ? c.values : c.keys) + at * kCacheBlock * DP;
    const float factor =
        power_of_two(max(static_cast<int>((values ? c.value_exponents : c.key_exponents)[at]), kCacheLeast));
    const int lane = lane_id();
    const int token0 = lane / Hold::kAcross * kTokens, channel0 = lane % Hold::kAcross * V;
    T* out = (values ? v : k) + ((s * c.blocks * kCacheBlock + lo + token0) * c.kv_heads + head) * c.dim;
    const long long stride = static_cast<long long>(c.kv_heads) * c.dim;
    if (!values) {
        CacheBytes<V> in[kTokens][kGroups] = {};
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int channel = channel0 + g * Hold::kAcross * V;
                if (token0 + t < filled && channel < c.dim)
                    in[t][g] = CacheBytes<V>::load(codes + (token0 + t) * DP + channel);
            }
        }
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int channel = channel0 + g * Hold::kAcross * V;
                Vec row;
#pragma unroll
                for (int j = 0; j < V; ++j) row.set(j, value_of<Code>(in[t][g], j) * factor);
                if (channel < c.dim) row.store(out + t * stride + channel);
            }
        }
        return;
    }
    constexpr int kBytes = kTokens > 16 ? 16 : kTokens, kParts = kTokens / kBytes;
    CacheBytes<kBytes> in[kGroups][V][kParts] = {};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int channel = channel0 + g * Hold::kAcross * V + j;
#pragma unroll
            for (int part = 0; part < kParts; ++part)
                if (token0 + part * kBytes < filled && channel < c.dim)
                    in[g][j][part] = CacheBytes<kBytes>::load(codes + channel * kCacheBlock + token0 + part * kBytes);
        }
    }
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            const int channel = channel0 + g * Hold::kAcross * V;
            Vec row;
#pragma unroll
            for (int j = 0; j < V; ++j)
                row.set(j, token0 + t < filled ? value_of<Code>(in[g][j][t / kBytes], t % kBytes) * factor : 0.0f);
            if (channel < c.dim) row.store(out + t * stride + channel);
        }
    }
}

long long write_slots(const lattice_cache& c, int rows) {
    return rows / kCacheBlock + 2ll * (c.sequences + 2);
}

template <typename T, int V, typename Code>
void launch_write(const lattice_cache& c, const CacheSource& k, const CacheSource& v, int rows,
                  const int32_t* offsets, const int32_t* lengths, hipStream_t stream) {
    const dim3 grid = cache_grid(write_slots(c, rows), head_groups(c.kv_heads), 1);
    const auto launch = [&](auto kernel) {
        kernel<<<grid, kCacheThreads, 0, stream>>>(c, k, v, rows, offsets, lengths);
    };
    switch (cache_width(c)) {
        case 32: return launch(cache_write_blocks<T, V, Code, 32>);
        case 64: return launch(cache_write_blocks<T, V, Code, 64>);
        case 96: return launch(cache_write_blocks<T, V, Code, 96>);
        default: return launch(cache_write_blocks<T, V, Code, 128>);
    }
}

template <typename T, typename Code>
int write_of(const lattice_cache& c, const CacheSource& k, const CacheSource& v, int rows, const int32_t* offsets,
             const int32_t* lengths, hipStream_t stream) {
    constexpr int kMost = 16 / sizeof(T);
    const int vector = row_vector<T>(c.dim, {k.rows, v.rows},
                                     {k.row_stride, k.head_stride, v.row_stride, v.head_stride});
    if (vector == kMost) {
        launch_write<T, kMost, Code>(c, k, v, rows, offsets, lengths, stream);
    } else {
        launch_write<T, 1, Code>(c, k, v, rows, offsets, lengths, stream);
    }
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T, int V, typename Code>
void launch_read(const lattice_cache& c, const int32_t* lengths, T* k, T* v, hipStream_t stream) {
    const dim3 grid = cache_grid(1ll * c.sequences * c.blocks, head_groups(c.kv_heads), 1);
    const auto launch = [&](auto kernel) { kernel<<<grid, kCacheThreads, 0, stream>>>(c, lengths, k, v); };
    switch (cache_width(c)) {
        case 32: return launch(cache_read_blocks<T, V, Code, 32>);
        case 64: return launch(cache_read_blocks<T, V, Code, 64>);
        case 96: return launch(cache_read_blocks<T, V, Code, 96>);
        default: return launch(cache_read_blocks<T, V, Code, 128>);
    }
}

template <typename T, typename Code>
int read_of(const lattice_cache& c, const int32_t* lengths, void* k, void* v, hipStream_t stream) {
    constexpr int kMost = 16 / sizeof(T);
    T *keys = static_cast<T*>(k), *values = static_cast<T*>(v);
    if (row_vector<T>(c.dim, {k, v}, {}) == kMost) {
        launch_read<T, kMost, Code>(c, lengths, keys, values, stream);
    } else {
        launch_read<T, 1, Code>(c, lengths, keys, values, stream);
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
    LATTICE_REQUIRE(cache_fits(*cache, write_slots(*cache, rows)), "the cache has too many sequences and heads.");
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
    LATTICE_REQUIRE(cache_fits(*cache, 1ll * cache->sequences * cache->blocks),
                    "the cache has too many sequences and heads.");
    hipStream_t stream = as_stream(stream_ptr);
    if (cache->code == LATTICE_CODE_E4M3) return read_code<CodeE4m3>(*cache, dtype, lengths, k, v, stream);
    return read_code<CodeInt8>(*cache, dtype, lengths, k, v, stream);
}
