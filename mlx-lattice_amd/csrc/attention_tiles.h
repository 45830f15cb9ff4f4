// Tiles of the windowed attention's matrix-core kernels: 32 x 32 products
// (v_mfma_f32_32x32x16 for 16-bit types, 32x32x2 for fp32) over rows staged in
// LDS.
//
// A product's result holds, in lane L = 32 h + n and register r, row
// 8 (r / 4) + 4 h + r % 4 of column n.  The scores are made transposed (rows:
// keys, columns: queries), so that a lane holds the scores of one query: the
// softmax runs within a lane but for one exchange between the halves, and a
// lane's registers are, in the order they lie, the right operand of the next
// product, whose left operand is read in the same order of rows.
#pragma once

#include <cfloat>

#include "attention.h"

namespace lattice {

typedef float f32x16_attn __attribute__((ext_vector_type(16)));
typedef float f32x4_attn __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_attn __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_attn __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_attn __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_attn __attribute__((ext_vector_type(4)));
typedef short i16x4_attn __attribute__((__vector_size__(4 * sizeof(short))));

// Frag: the 16 bytes a lane gives to the products over KSTEP channels (or
// rows); half h holds values 8 h .. 8 h + 7 of 16 (fp32: 4 h .. 4 h + 3 of 8,
// one at a time).
template <typename T> struct AttnMath;
template <> struct AttnMath<_Float16> {
    typedef f16x8_attn Frag;
    static constexpr int kStep = 16;
    __device__ static f32x16_attn product(Frag a, Frag b, f32x16_attn c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct AttnMath<__bf16> {
    typedef bf16x8_attn Frag;
    static constexpr int kStep = 16;
    __device__ static f32x16_attn product(Frag a, Frag b, f32x16_attn c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct AttnMath<float> {
    typedef f32x4_attn Frag;
    static constexpr int kStep = 8;
    __device__ static f32x16_attn product(Frag a, Frag b, f32x16_attn c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// Kernels are made for heads of up to DP = 32, 64, 96 and 128 channels; a
// tile's rows lie a power of two apart.
inline int attn_width(int dim) { return (dim + 31) / 32 * 32; }
template <int DP> constexpr int kTileDim = DP == 96 ? 128 : DP;

// ROWS rows of DP channels (zeros past the channels there are) in LDS, in
// 16-byte pieces.  LDS serves 256 bytes a cycle from 64 banks: 16 lanes that
// read a piece each of 16 rows, or 32 that read 64 bytes of each of 4 rows
// (four neighbours, for a transposed operand).  A row's pieces are permuted by
// an exclusive or with bits of the row, so that either falls on all banks.
template <typename T, int DP, int ROWS>
struct AttnTile {
    typedef typename AttnMath<T>::Frag Frag;
    static constexpr int kRowBytes = kTileDim<DP> * static_cast<int>(sizeof(T));
    static constexpr int kPieces = kRowBytes / 16;
    static constexpr int kBytes = ROWS * kRowBytes;
    static constexpr int kElems = 16 / static_cast<int>(sizeof(T));

    __device__ static int mix(int row) {
        const int quad = row >> 2 & 3;
        return kPieces >= 16 ? (row & 3) << 2 | quad : kPieces == 8 ? (row >> 1 & 1) << 2 | quad : quad;
    }
    __device__ static int place(int row, int piece) { return row * kRowBytes + ((piece ^ mix(row)) << 4); }

    // Copies by the waves of THREADS threads: the row and piece of copy i.
    static constexpr int kRange = 1 << 30;
    static constexpr int copies(int threads) { return kBytes / (threads * 16); }
    template <int THREADS>
    __device__ static int copy_row(int i, int thread) {
        return ((i * (THREADS / kWave) + thread / kWave) * kWave + lane_id()) / kPieces;
    }
    // A piece past the head's lies outside every range and reads as zeros.
    template <int THREADS>
    __device__ static int copy_piece(int i, int thread, int pieces) {
        const int at = (i * (THREADS / kWave) + thread / kWave) * kWave + lane_id();
        const int piece = (at % kPieces) ^ mix(at / kPieces);
        return piece < pieces ? piece * 16 : kRange;
    }
    // Starts the copies of offsets[i] of `from`; past `range` bytes they give
    // zeros.  The memory counter tells when they are done.
    template <int THREADS>
    __device__ static void copy(char* to, const T* from, int range, const int* offsets, int wave) {
        const __amdgpu_buffer_rsrc_t rsrc =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(from), 0, range, 0x00020000);
#pragma unroll
        for (int i = 0; i < copies(THREADS); ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rsrc, (__attribute__((address_space(3))) void*)(to + (i * (THREADS / kWave) + wave) * kWave * 16), 16,
                offsets[i], 0, 0, 0);
    }

    // Left (or right) operand of a product over channels: row `row`, channels
    // step * kStep on, the half's share.
    __device__ static Frag row_frag(const char* tile, int row, int step, int half) {
        return *reinterpret_cast<const Frag*>(tile + place(row, step * 2 + half));
    }
};

// Until the copies that this wave started are in LDS.
__device__ inline void wait_for_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Transposed operand of a product over rows: channel 32 block + L % 32 of the
// tile's rows in the order in which a lane's registers 8 step .. 8 step + 7
// hold them: rows 16 step + 4 h + 0 .. 3 and 16 step + 8 + 4 h + 0 .. 3.
template <typename Tile, typename T>
__device__ inline typename AttnMath<T>::Frag column_frag(const char* tile, int step, int block) {
    static_assert(sizeof(T) == 2);
    const int lane = lane_id();
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int piece = 4 * block + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const char* at = tile + ((lane & 1) << 3) + step * 16 * Tile::kRowBytes;
    typedef __attribute__((address_space(3))) i16x4_attn* Local;
    struct Pair {
        i16x4_attn a, b;
    };
    const Pair both{__builtin_amdgcn_ds_read_tr16_b64_v4i16((Local)(at + Tile::place(row, piece))),
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((Local)(at + Tile::place(row + 8, piece)))};
    return __builtin_bit_cast(typename AttnMath<T>::Frag, both);
}

// acc[block] += (columns 32 block + n of the tile's 32 rows from `row0`)
// times x, the registers of a product's result over those rows.
template <typename Tile, typename T, int BLOCKS>
__device__ inline void add_columns(f32x16_attn (&acc)[BLOCKS], const char* tile, int row0, const f32x16_attn& x) {
    if constexpr (sizeof(T) == 2) {
        typedef typename AttnMath<T>::Frag Frag;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            Frag b;
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = static_cast<T>(x[8 * half + i]);
#pragma unroll
            for (int block = 0; block < BLOCKS; ++block)
                acc[block] = AttnMath<T>::product(column_frag<Tile, T>(tile, row0 / 16 + half, block), b, acc[block]);
        }
    } else {
        const int lane = lane_id();
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = row0 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
#pragma unroll
            for (int block = 0; block < BLOCKS; ++block) {
                const float a = *reinterpret_cast<const float*>(
                    tile + Tile::place(row, 8 * block + ((lane & 31) >> 2)) + ((lane & 3) << 2));
                acc[block] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, x[r], acc[block], 0, 0, 0);
            }
        }
    }
}

// The keys and values of a sequence and key head, copied KT rows at a time
// into two tiles one after the other.
template <typename T, int DP, int KT, int THREADS>
struct KeyTiles {
    typedef AttnTile<T, DP, KT> Tile;
    static constexpr int kCopies = Tile::copies(THREADS);
    const T *keys, *values;
    long long k_stride, v_stride;
    int row_bytes, wave;
    int k_offsets[kCopies], v_offsets[kCopies];

    __device__ KeyTiles(const lattice_attention& a, const AttnSequence& s, int kv, int thread) {
        keys = static_cast<const T*>(a.k) + s.k0 * a.k_row_stride + kv * a.k_head_stride;
        values = static_cast<const T*>(a.v) + s.k0 * a.v_row_stride + kv * a.v_head_stride;
        k_stride = a.k_row_stride;
        v_stride = a.v_row_stride;
        row_bytes = a.dim * static_cast<int>(sizeof(T));
        wave = __builtin_amdgcn_readfirstlane(thread / kWave);
        constexpr int kSize = sizeof(T);
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int row = Tile::template copy_row<THREADS>(i, thread);
            const int piece = Tile::template copy_piece<THREADS>(i, thread, row_bytes / 16);
            k_offsets[i] = row * static_cast<int>(k_stride) * kSize + piece;
            v_offsets[i] = row * static_cast<int>(v_stride) * kSize + piece;
        }
    }
    // Rows j0 .. of the sequence's nk; the range ends with the last of them.
    __device__ void copy(char* to, int j0, int nk) const {
        const int last = min(nk - j0, KT) - 1;
        constexpr int kSize = sizeof(T);
        Tile::template copy<THREADS>(to, keys + j0 * k_stride, last * static_cast<int>(k_stride) * kSize + row_bytes,
                                     k_offsets, wave);
        Tile::template copy<THREADS>(to + Tile::kBytes, values + j0 * v_stride,
                                     last * static_cast<int>(v_stride) * kSize + row_bytes, v_offsets, wave);
    }
};

// The operand of a wave's 32 rows (row L % 32 at `row`), kept in registers;
// zeros past `dim`.
template <typename T, int DP>
struct AttnOperand {
    typedef typename AttnMath<T>::Frag Frag;
    static constexpr int kSteps = DP / AttnMath<T>::kStep;
    Frag f[kSteps];

    __device__ void load(const T* row, int dim, bool valid, bool negate) {
        const int half = lane_id() >> 5;
        constexpr int kShare = AttnMath<T>::kStep / 2;
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
        const Words signs = Words{} + (!negate ? 0u : sizeof(T) == 2 ? 0x80008000u : 0x80000000u);
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            const int d = (2 * c + half) * kShare;
            Words words{};
            if (valid && d < dim) words = *reinterpret_cast<const Words*>(row + d);
            f[c] = __builtin_bit_cast(Frag, words ^ signs);
        }
    }
};

// The scale of the scores in the exponent.  Positive, so that the -inf of a
// key that is not seen stays -inf: the sign goes into one operand of the scores
// (a.scale < 0), and a scale of zero becomes the smallest normal number, whose
// product with a score below 1e30 vanishes beside every exponent.
__device__ inline float exponent_scale(const lattice_attention& a) {
    const float size = fabsf(a.scale);
    return (size < FLT_MIN ? FLT_MIN : size) * kAttnLog2e;
}

// c + rows row0 .. row0 + 31 of the tile times the operand's rows.
template <typename Tile, typename T, int DP>
__device__ inline f32x16_attn tile_product(const char* tile, int row0, const AttnOperand<T, DP>& b, f32x16_attn c) {
    const int lane = lane_id();
#pragma unroll
    for (int step = 0; step < AttnOperand<T, DP>::kSteps; ++step)
        c = AttnMath<T>::product(Tile::row_frag(tile, row0 + (lane & 31), step, lane >> 5), b.f[step], c);
    return c;
}

// The maximum and sum over both halves of a wave, in both.
__device__ inline float2 both_halves(float v) {
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return float2{__uint_as_float(halves[0]), __uint_as_float(halves[1])};
}
__device__ inline float halves_max(float v) {
    const float2 both = both_halves(v);
    return fmaxf(both.x, both.y);
}
__device__ inline float halves_sum(float v) {
    const float2 both = both_halves(v);
    return both.x + both.y;
}

// Row of a result's register r.
__device__ inline int result_row(int r) { return 8 * (r / 4) + 4 * (lane_id() >> 5) + r % 4; }

// Whether a column's sums times `factor` are finite (channels past a head's
// are zeros, or as infinite as the others).
template <int BLOCKS>
__device__ inline bool finite_columns(const f32x16_attn (&acc)[BLOCKS], float factor) {
    uint32_t largest = 0;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            // The bits of magnitudes are ordered, NaN above infinity.
            const uint32_t bits = __float_as_uint(acc[b][r] * factor) & 0x7fffffffu;
            largest = max(largest, bits);
        }
    }
    return largest < 0x7f800000u;
}

// What a lane's query sees: lo <= j <= hi, or a first key (j <= hi).
struct AttnMask {
    int lo, hi, sinks;
    __device__ AttnMask(const lattice_attention& a, int nk, int p)
        : lo(p - a.left), hi(min(nk - 1, p + a.right)), sinks(a.sinks) {}
    // The scores of keys j0 + result_row(r); `first`: some are first keys.  Most
    // tiles cross one end of the window, and each end has its own test.
    __device__ void apply(f32x16_attn& x, int j0, bool first) const {
        const int j = j0 + 4 * (lane_id() >> 5);
        const int most = hi - j, least = lo - j;
        if (__any(most < kLastRow)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) hide(x, r, row(r) > most);
        }
        if (first) {
            const int firsts = sinks - j;
#pragma unroll
            for (int r = 0; r < 16; ++r) hide(x, r, row(r) < least && row(r) >= firsts);
        }
        if (!first && __any(least > 0)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) hide(x, r, row(r) < least);
        }
    }

   private:
    static constexpr int kLastRow = 27;
    __device__ static constexpr int row(int r) { return 8 * (r / 4) + r % 4; }
    // In order: 16 tests at once would take more scalar registers than there are.
    __device__ static void hide(f32x16_attn& x, int r, bool hidden) {
        x[r] = hidden ? -INFINITY : x[r];
        if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
};

// How the positions p_low .. p_high see the keys j0 .. j0 + count.
enum AttnView { kSeesNone, kSeesSome, kSeesAll };
__device__ inline AttnView attn_view(const lattice_attention& a, int nk, int p_low, int p_high, int j0, int count) {
    const int end = j0 + count;
    if (j0 >= nk || j0 > p_high + a.right || (end <= p_low - a.left && j0 >= a.sinks)) return kSeesNone;
    const bool all = end <= nk && end - 1 <= p_low + a.right && (j0 >= p_high - a.left || end <= a.sinks);
    return all ? kSeesAll : kSeesSome;
}

// r / group, with one product for the division.
struct GroupDivide {
    uint32_t group, magic;
    __device__ explicit GroupDivide(uint32_t g) : group(g), magic(g > 1 ? 0xffffffffu / g + 1 : 0) {}
    __device__ uint32_t operator()(uint32_t r) const {
        if (group == 1) return r;
        const uint32_t q = __umulhi(r, magic);
        return q * group > r ? q - 1 : q;
    }
};

// The tiles of KT keys that a range of positions sees: first those of the
// first keys that lie before the window's, then the window's.
struct AttnTiles {
    int first, from, count;
    __device__ int tile(int t) const { return t < first ? t : from + (t - first); }
};
template <int KT>
__device__ inline AttnTiles attn_tiles(const lattice_attention& a, int nk, int p_low, int p_high) {
    const int hi = min(nk - 1, p_high + a.right);
    if (hi < 0) return {0, 0, 0};
    const int from = max(0, p_low - a.left) / KT;
    const int first = min((min(a.sinks, hi + 1) + KT - 1) / KT, from);
    return {first, from, first + max(0, hi / KT - from + 1)};
}

// What a wave's 32 rows are: row L % 32 of the tile.
struct AttnRows {
    int i, head, p;      // query of the sequence, head, position
    bool valid;
    int p_low, p_high;   // of all 32 rows
};
__device__ inline AttnRows attn_rows(const AttnSequence& s, int kv, uint32_t group, uint32_t first) {
    const uint32_t rows = s.nq * group;
    const uint32_t r = first + (lane_id() & 31);
    const uint32_t in = min(r, rows - 1);
    AttnRows w;
    w.i = in / group;
    w.head = kv * group + in % group;
    w.p = w.i + s.shift();
    w.valid = r < rows;
    w.p_low = __builtin_amdgcn_readfirstlane(w.i) + s.shift();
    w.p_high = __builtin_amdgcn_readlane(w.i, 31) + s.shift();
    return w;
}

// A launch takes fewer than 2^32 threads along x: slots past 2^22 go on along
// z, above its own `parts`.
inline dim3 slot_grid(long long slots, int kv_heads, int parts) {
    const long long x = std::min(slots, 1ll << 22);
    return dim3(static_cast<unsigned>(x), kv_heads, static_cast<unsigned>((slots + x - 1) / x * parts));
}
__device__ inline uint32_t block_slot(uint32_t parts) {
    return blockIdx.x + gridDim.x * (parts == 1 ? blockIdx.z : blockIdx.z / parts);
}
__device__ inline int block_part(uint32_t parts) { return parts == 1 ? 0 : blockIdx.z % parts; }

// The first of `rows` rows of a slot of M, where the sequence's slots begin at
// `start`: `rows` itself, none, where the slot is not the sequence's.  Offsets
// that decrease can lead the search to a sequence that starts past the slot.
template <int M>
__device__ inline uint32_t slot_first(uint32_t slot, uint32_t start, uint32_t rows) {
    const uint32_t tile = slot - start;
    return tile < (rows + M - 1) / M ? tile * M : rows;
}

// Which sequence, tile of M rows and key head a block has.
struct AttnSlot {
    AttnSequence s;
    uint32_t rows, first;  // (query, head) pairs: of the sequence, before the tile's
};
template <int M>
__device__ inline AttnSlot attn_slot(const lattice_attention& a, uint32_t group, uint32_t slot) {
    // Sequence e has the slots from start / M + e on: enough for its tiles.
    const auto slot_of = [group](int start, int e) { return start * group / M + e; };
    const int e = query_rows(a).find(slot, slot_of);
    AttnSlot t;
    t.s = attn_sequence(a, e);
    t.rows = t.s.nq * group;
    t.first = slot_first<M>(slot, slot_of(t.s.q0, e), t.rows);
    return t;
}

}  // namespace lattice
