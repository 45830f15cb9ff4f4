// Attention over a sliding window with first keys that stay visible: the
// forward pass.
//
//   s_ij = scale q_i . k_j over the keys j that query i sees,
//   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),
// with the running maximum m and sum of one pass over the keys.
//
// The rows of a tile are (query, head) pairs of the heads that share a key
// head, so that each key is staged once for all of them and the band of keys
// that a tile sees is as narrow as may be.  A wave holds 32 rows: q as the right
// operand in registers, the scores transposed, so that a lane has one row's and
// the softmax needs one exchange between two lanes a step.
//
// Shares are rounded to the rows' type for the second product, as q, k and v
// are; maximum, sums and results are fp32.  That is one more rounding of a
// row's result, which does not grow with the number of keys (error against
// float64 2.9e-4 in half precision and 2.4e-3 in bfloat16, of which the result's
// own rounding makes 2.1e-4 and 1.7e-3).
//
// Bound, by the counters, by the vector instructions of the softmax (eight a
// score): their pipe is busy 62 % of the time at heads of 32 and 47 % at 64,
// beside 13 and 19 % of the matrix cores; neighbouring tiles of rows, which lie
// on different dies, each read their keys beyond the L2 (846 MB at 120,000 rows
// of heads of 32, 6.6 TB/s).  At heads of 128 both pipes are busy about evenly
// (42 and 45 %, two waves a SIMD), few queries wait for the keys.  120,000 rows
// of 8 heads of 32, window 257, fp16: 127 us (249 TFLOP/s).  16,384 causal rows
// of 16 heads of 128 over 4, window 4096, bf16: 534 us under the profiler, 518
// without (931 TFLOP/s; a library product of 8192^3 1191); fp32: 4.9 ms (98 of
// 154).  One query of 16 heads of 128 over 4 against 32 caches of 24,000 keys,
// fp16: 298 us (5.5 TB/s); fp32: 831 (4.0).

#include "attention_tiles.h"

namespace lattice {
namespace {

// The part of a softmax over some of a row's keys: the sum over them of
// exp2(x - top), and of that times v.
struct AttnPart {
    float* values;  // [splits][queries * heads][dim]
    float2* states;  // [splits][queries * heads]: (top, sum)
};

// A row's top starts far below every score but above -inf, so that what is
// masked (-inf) has a share of zero.
constexpr float kAttnFloor = -3.0e38f;
// Shares are exp2(score - top), where top is the running maximum less kBase and
// may lag behind the scores by kLag powers of two more before the sums are
// scaled down to a new one: shares stay within 2^(kBase + kLag).  In half
// precision, where a share below 2^-14 loses bits and one below 2^-25 is lost
// (the sum of shares is not rounded), they fill the type's range instead: a
// share keeps all bits down to 2^-25 of the largest and some down to 2^-36, so
// that a tail of 2^24 equal keys is right to half a rounding of the result.
template <typename T> struct ShareRange {
    static constexpr float kBase = 0.0f, kLag = 8.0f;
};
template <> struct ShareRange<_Float16> {
    static constexpr float kBase = 11.0f, kLag = 4.0f;
};

template <typename T, int DP>
struct AttnState {
    static constexpr int kBlocks = DP / 32;
    f32x16_attn acc[kBlocks];
    float top, sum;

    __device__ void clear() {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[b] = f32x16_attn{};
        top = kAttnFloor;
        sum = 0.0f;
    }
    __device__ void rescale(float factor) {
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[b] *= factor;
        sum *= factor;
    }
};

// Adds the keys j0 .. j0 + 32 PARTS, rows row0 .. of a tile, to the sums of the
// wave's 32 rows; `masked`: some of them are not seen by some row.
template <int PARTS, typename T, int DP, int KT>
__device__ inline void attend_keys(AttnState<T, DP>& state, const AttnOperand<T, DP>& q, const char* keys,
                                   const char* values, int row0, float scale, const AttnMask& mask, int j0,
                                   bool masked) {
    typedef AttnTile<T, DP, KT> Tile;
    f32x16_attn s[PARTS];
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
        s[part] = tile_product<Tile, T, DP>(keys, row0 + 32 * part, q, f32x16_attn{});
    if (masked) {
#pragma unroll
        for (int part = 0; part < PARTS; ++part) mask.apply(s[part], j0 + 32 * part, j0 < mask.sinks);
    }
    float most = s[0][0];
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, s[part][r]);
    }
    most = halves_max(most) * scale;
    typedef ShareRange<T> Range;
    if (__any(most > state.top + (Range::kBase + Range::kLag))) {
        const float next = fmaxf(state.top, most - Range::kBase);
        state.rescale(__builtin_amdgcn_exp2f(state.top - next));
        state.top = next;
    }
    float sum = 0.0f;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[part][r] = __builtin_amdgcn_exp2f(s[part][r] * scale - state.top);
            sum += s[part][r];
        }
    }
    state.sum += sum;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) add_columns<Tile, T>(state.acc, values, row0 + 32 * part, s[part]);
}

// A tile of KT keys: 32 at a time, those that some row sees; in one step for
// heads of 96 and 128, whose sums leave registers for two waves a SIMD either
// way.  (120k rows of heads of 32, window 257: 131 us, 171 in one step; 60k rows
// of heads of 64, window 513: 67 and 74; 16k causal rows of heads of 128, window
// 4096: 612 and 572.  A form of each, by what the rows see, costs registers:
// 143, 74, 612.)
template <typename T, int DP, int KT>
__device__ inline void attend_tile(const lattice_attention& a, AttnState<T, DP>& state, const AttnOperand<T, DP>& q,
                                   const char* keys, const char* values, float scale, int nk, const AttnRows& w,
                                   const AttnMask& mask, int j0) {
    const AttnView view = attn_view(a, nk, w.p_low, w.p_high, j0, KT);
    if (view == kSeesNone) return;
    if constexpr (KT > 32 && DP >= 96) {
        attend_keys<KT / 32, T, DP, KT>(state, q, keys, values, 0, scale, mask, j0, view == kSeesSome);
    } else {
        for (int row0 = 0; row0 < KT; row0 += 32) {
            const AttnView part = attn_view(a, nk, w.p_low, w.p_high, j0 + row0, 32);
            if (part != kSeesNone)
                attend_keys<1, T, DP, KT>(state, q, keys, values, row0, scale, mask, j0 + row0, part == kSeesSome);
        }
    }
}

// Writes the wave's rows: the result, or a part of it (splits > 1).  A result
// that is not finite is made again row by row: products over a tile carry a
// zero share of what a row does not see, which spoils the row if that is not
// finite.
template <typename T, int DP>
__device__ inline void write_rows(const lattice_attention& a, const AttnSequence& s, const AttnRows& w,
                                  AttnState<T, DP>& state, bool partial, int split, const AttnPart& part, T* out,
                                  const AttnKept<T>& kept, AttnRowScratch* scratch) {
    const int half = lane_id() >> 5;
    const float sum = halves_sum(state.sum);
    const long long at = (static_cast<long long>(s.q0) + w.i) * a.heads + w.head;
    if (partial) {
        if (!w.valid) return;
        const long long row = static_cast<long long>(split) * a.queries * a.heads + at;
        if (half == 0) part.states[row] = float2{state.top, sum};
#pragma unroll
        for (int b = 0; b < AttnState<T, DP>::kBlocks; ++b) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * b + 8 * g + 4 * half;
                if (d >= a.dim) continue;
                RowVec<float, 4> v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v.e[i] = state.acc[b][4 * g + i];
                v.store(part.values + row * a.dim + d);
            }
        }
        return;
    }
    const bool sees = attn_seen(a, s.nk, w.p).total() > 0;
    const float inv = sees ? 1.0f / sum : 0.0f;
#pragma unroll
    for (int b = 0; b < AttnState<T, DP>::kBlocks; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) state.acc[b][r] *= inv;
    }
    const uint64_t spoilt = ballot(w.valid && !finite_columns(state.acc, 1.0f));
    uint32_t again = static_cast<uint32_t>(spoilt) | static_cast<uint32_t>(spoilt >> 32);
    if (w.valid && !(again >> (lane_id() & 31) & 1)) {
        if (kept.lse && half == 0) kept.lse[at] = sees ? state.top + __builtin_amdgcn_logf(sum) : INFINITY;
#pragma unroll
        for (int b = 0; b < AttnState<T, DP>::kBlocks; ++b) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * b + 8 * g + 4 * half;
                if (d >= a.dim) continue;
                RowVec<T, 4> v;
#pragma unroll
                for (int i = 0; i < 4; ++i) v.set(i, state.acc[b][4 * g + i]);
                v.store(out + at * a.dim + d);
                if (!kept.rest) continue;
                RowVec<T, 4> rest;
#pragma unroll
                for (int i = 0; i < 4; ++i) rest.e[i] = rounding_rest(state.acc[b][4 * g + i], v.e[i]);
                rest.store(kept.rest + at * a.dim + d);
            }
        }
    }
    while (again) {
        const int n = __ffs(again) - 1;
        again &= again - 1;
        attend_row<T>(a, s, __shfl(w.i, n), __shfl(w.head, n), out, kept, scratch);
    }
}

// The first of `count` tiles (at most 2^24) that split `split` of at most 64 has.
__device__ inline int split_tile(int count, int split, int splits) {
    return splits == 1 ? count * split : static_cast<int>(static_cast<uint32_t>(count) * split / splits);
}

// Starts the copy of tile `index` + 1 (below `to`) into `next` and adds tile
// `index`, which lies in `tile`.  That the two do not overlap lets the reads of
// one pass the copies of the other: without the qualifiers the compiler waits
// for all copies before it reads a transposed operand.
template <typename T, int DP, int KT, typename Source>
__device__ __forceinline__ void attend_step(const lattice_attention& a, AttnState<T, DP>& state,
                                            const AttnOperand<T, DP>& q, const Source& source,
                                            const AttnTiles& tiles, int index, int to, char* __restrict__ next,
                                            const char* __restrict__ tile, float scale, int nk, const AttnRows& w,
                                            const AttnMask& mask) {
    if (index + 1 < to) source.copy(next, tiles.tile(index + 1) * KT, nk);
    attend_tile<T, DP, KT>(a, state, q, tile, tile + AttnTile<T, DP, KT>::kBytes, scale, nk, w, mask,
                           tiles.tile(index) * KT);
}

// 128 rows a block, 32 a wave, over tiles of KT keys that the waves share.
// Double-buffered: a tile is copied to LDS while the one before is used.
template <typename T, int DP, int KT>
__global__ void __launch_bounds__(kAttnBlock, 2)
attend_tiles(lattice_attention a, int splits, AttnPart part, T* __restrict__ out, AttnKept<T> kept) {
    typedef AttnTile<T, DP, KT> Tile;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y, split = block_part(splits);
    const AttnSlot t = attn_slot<32 * kAttnWaves>(a, group, block_slot(splits));
    const AttnSequence s = t.s;
    if (t.first >= t.rows) return;
    const float scale = exponent_scale(a);
    const AttnRows w = attn_rows(s, kv, group, t.first + 32 * wave);
    AttnOperand<T, DP> q;
    q.load(static_cast<const T*>(a.q) + (static_cast<long long>(s.q0) + w.i) * a.q_row_stride +
               w.head * a.q_head_stride,
           a.dim, w.valid, a.scale < 0.0f);
    const AttnMask mask(a, s.nk, w.p);
    AttnState<T, DP> state;
    state.clear();
    const int p_low = static_cast<int>(t.first / group) + s.shift();
    const int p_high = static_cast<int>((min(t.first + 32 * kAttnWaves, t.rows) - 1) / group) + s.shift();
    const AttnTiles tiles = attn_tiles<KT>(a, s.nk, p_low, p_high);
    const int from = split_tile(tiles.count, split, splits), to = split_tile(tiles.count, split + 1, splits);
    const KeyTiles<T, DP, KT, kAttnBlock> source(a, s, kv, threadIdx.x);
    if (from < to) source.copy(shared + (from & 1) * 2 * Tile::kBytes, tiles.tile(from) * KT, s.nk);
    wait_for_copies();
    __syncthreads();
    for (int index = from; index < to; ++index) {
        attend_step<T, DP, KT>(a, state, q, source, tiles, index, to, shared + (~index & 1) * 2 * Tile::kBytes,
                               shared + (index & 1) * 2 * Tile::kBytes, scale, s.nk, w, mask);
        wait_for_copies();
        __syncthreads();
    }
    write_rows<T, DP>(a, s, w, state, splits > 1, split, part, out, kept,
                      reinterpret_cast<AttnRowScratch*>(shared) + wave);
}

// Waves a block for few queries: two tiles a wave fit the LDS of a unit.
template <typename T, int DP> constexpr int few_waves() { return kTileDim<DP> * static_cast<int>(sizeof(T)) <= 256 ? 8 : 4; }

// 32 rows a block, for few queries: each wave takes its own tiles
// of KT keys, with no wait for the others, and the waves' parts are joined in
// LDS.
template <typename T, int DP, int KT, int kFewWaves>
__global__ void __launch_bounds__(kFewWaves * kWave)
attend_few(lattice_attention a, int splits, AttnPart part, T* __restrict__ out, AttnKept<T> kept) {
    typedef AttnTile<T, DP, KT> Tile;
    constexpr int kBlocks = AttnState<T, DP>::kBlocks;
    extern __shared__ __align__(128) char shared[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t group = a.heads / a.kv_heads;
    const int kv = blockIdx.y, split = block_part(splits);
    const AttnSlot t = attn_slot<32>(a, group, block_slot(splits));
    const AttnSequence s = t.s;
    if (t.first >= t.rows) return;
    const float scale = exponent_scale(a);
    const AttnRows w = attn_rows(s, kv, group, t.first);
    AttnOperand<T, DP> q;
    q.load(static_cast<const T*>(a.q) + (static_cast<long long>(s.q0) + w.i) * a.q_row_stride +
               w.head * a.q_head_stride,
           a.dim, w.valid, a.scale < 0.0f);
    const AttnMask mask(a, s.nk, w.p);
    AttnState<T, DP> state;
    state.clear();
    const AttnTiles tiles = attn_tiles<KT>(a, s.nk, w.p_low, w.p_high);
    const int from = split_tile(tiles.count, split, splits), to = split_tile(tiles.count, split + 1, splits);
    const KeyTiles<T, DP, KT, kWave> source(a, s, kv, lane_id());
    char* mine = shared + wave * 2 * Tile::kBytes;
    for (int index = from + wave; index < to; index += kFewWaves) {
        const int j0 = tiles.tile(index) * KT;
        source.copy(mine, j0, s.nk);
        wait_for_copies();
        wave_fence();
        attend_tile<T, DP, KT>(a, state, q, mine, mine + Tile::kBytes, scale, s.nk, w, mask, j0);
        wait_for_reads();
    }
    // Every wave's sums to the largest maximum, then pairwise into the first
    // wave's.
    const int lane = lane_id();
    state.sum = halves_sum(state.sum);
    __syncthreads();
    float2* states = reinterpret_cast<float2*>(shared);
    float* sums = reinterpret_cast<float*>(shared + kFewWaves * 32 * sizeof(float2));
    if (lane < 32) states[wave * 32 + lane] = float2{state.top, state.sum};
    __syncthreads();
    float top = kAttnFloor, sum = 0.0f;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) top = fmaxf(top, states[v * 32 + (lane & 31)].x);
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) {
        const float2 other = states[v * 32 + (lane & 31)];
        sum += other.y * __builtin_amdgcn_exp2f(other.x - top);
    }
    state.rescale(__builtin_amdgcn_exp2f(state.top - top));
    constexpr int kValues = kBlocks * 16 * kWave;
#pragma unroll
    for (int active = kFewWaves / 2; active > 0; active /= 2) {
        if (active < kFewWaves / 2) __syncthreads();
        if (wave >= active && wave < 2 * active) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    sums[(wave - active) * kValues + (b * 16 + r) * kWave + lane] = state.acc[b][r];
            }
        }
        __syncthreads();
        if (wave < active) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) state.acc[b][r] += sums[wave * kValues + (b * 16 + r) * kWave + lane];
            }
        }
    }
    __syncthreads();
    if (wave != 0) return;
    state.top = top;
    state.sum = lane < 32 ? sum : 0.0f;  // write_rows adds the halves
    write_rows<T, DP>(a, s, w, state, splits > 1, split, part, out, kept,
                      reinterpret_cast<AttnRowScratch*>(shared));
}

// Joins the parts (at most 64) of a row: a wave a (query row, head).
template <typename T>
__global__ void __launch_bounds__(kAttnBlock)
join_parts(lattice_attention a, int splits, AttnPart part, T* __restrict__ out, AttnKept<T> kept) {
    __shared__ AttnRowScratch scratch[kAttnWaves];
    const int wave = threadIdx.x / kWave, lane = lane_id();
    const long long items = static_cast<long long>(a.queries) * a.heads;
    const long long at = static_cast<long long>(blockIdx.x) * kAttnWaves + wave;
    if (at >= items) return;
    const float2 state = lane < splits ? part.states[lane * items + at] : float2{kAttnFloor, 0.0f};
    const float top = wave_max(state.x);
    const float factor = __builtin_amdgcn_exp2f(state.x - top);
    const float sum = wave_sum(state.y * factor);
    float acc[kAttnMaxDim / kWave] = {};
#pragma unroll 4
    for (int z = 0; z < splits; ++z) {
        const float share = __shfl(factor, z);
#pragma unroll
        for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
            const int d = min(lane + c * kWave, a.dim - 1);
            acc[c] += part.values[(z * items + at) * a.dim + d] * share;
        }
    }
    bool finite = sum > 0.0f;
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
        acc[c] /= sum;
        finite = finite && fabsf(acc[c]) < INFINITY;
    }
    // Rows that see nothing, and those that are not finite.
    if (__any(!finite)) {
        const int row = static_cast<int>(at / a.heads), head = static_cast<int>(at % a.heads);
        const int e = query_rows(a).find(row, [](int start, int) { return static_cast<uint32_t>(start); });
        const AttnSequence s = attn_sequence(a, e);
        attend_row<T>(a, s, row - s.q0, head, out, kept, &scratch[wave]);
        return;
    }
    if (kept.lse && lane == 0) kept.lse[at] = top + log2f(sum);
#pragma unroll
    for (int c = 0; c < kAttnMaxDim / kWave; ++c) {
        const int d = lane + c * kWave;
        if (d >= a.dim) continue;
        const T rounded = static_cast<T>(acc[c]);
        out[at * a.dim + d] = rounded;
        if (kept.rest) kept.rest[at * a.dim + d] = rounding_rest(acc[c], rounded);
    }
}

// How a call is laid out: rows a tile, tiles of rows at most, and into how
// many blocks the keys of a tile of rows are split.
struct AttnLayout {
    bool few;
    long long slots;
    int splits;
};
inline AttnLayout attn_layout(const lattice_attention& a) {
    const int group = a.heads / a.kv_heads;
    const long long pairs = static_cast<long long>(a.queries) * group;
    const int sequences = std::max(1, a.sequences);
    // The keys that a block sees, were the rows spread evenly over the sequences.
    const auto seen_by = [&](int m) {
        const long long span = static_cast<long long>(a.left) + a.right + std::min(m, a.queries) + a.sinks;
        return std::min<long long>(span, (static_cast<long long>(a.keys) + sequences - 1) / sequences);
    };
    AttnLayout l;
    // Few rows a sequence leave three of four waves of a large tile idle; few
    // rows in all leave units idle where there are too few keys to split (2.9k
    // rows fp32, 4 heads of 128, window 414: 58 us, in large tiles 148; 256 rows
    // of 8 heads against 8k keys: 38, split in large tiles 35).
    l.few = pairs <= 32ll * sequences || (pairs * a.kv_heads < 128ll * 256 && seen_by(128) < 2048);
    const int m = l.few ? 32 : 128;
    l.slots = pairs / m + a.sequences + 2;
    // Blocks that have rows.
    const long long busy =
        std::max<long long>((pairs + m - 1) / m, std::min<long long>(sequences, a.queries)) * a.kv_heads;
    const long long seen = seen_by(m);
    // Two blocks a compute unit, each with at least 512 keys.
    const long long wanted = std::min<long long>((512 + busy - 1) / busy, seen / 512);
    l.splits = static_cast<int>(std::max<long long>(1, std::min<long long>(wanted, 64)));
    return l;
}

template <typename T, int DP>
int launch_attend(const lattice_attention& a, const AttnLayout& l, const AttnPart& part, T* out,
                  const AttnKept<T>& kept, hipStream_t stream) {
    // Tiles twice as large are no faster (120k rows of heads of 32: 132 us for 127).
    constexpr int kTile = sizeof(T) == 2 ? 64 : 32;
    typedef AttnTile<T, DP, kTile> Tile;
    const dim3 grid = slot_grid(l.slots, a.kv_heads, l.splits);
    if (l.few) {
        constexpr int kFew = 32, kFewWaves = few_waves<T, DP>();
        constexpr size_t kLds =
            std::max<size_t>(kFewWaves * 2 * AttnTile<T, DP, kFew>::kBytes,
                             kFewWaves * 32 * sizeof(float2) + kFewWaves / 2 * DP / 32 * 16 * kWave * sizeof(float));
        static_assert(kLds >= sizeof(AttnRowScratch) && kLds <= 160 * 1024);
        const auto kernel = attend_few<T, DP, kFew, kFewWaves>;
        LATTICE_HIP_TRY(allow_lds(reinterpret_cast<const void*>(kernel), kLds));
        kernel<<<grid, kFewWaves * kWave, kLds, stream>>>(a, l.splits, part, out, kept);
    } else {
        constexpr size_t kLds = std::max<size_t>(4 * Tile::kBytes, kAttnWaves * sizeof(AttnRowScratch));
        static_assert(kLds <= 160 * 1024);
        const auto kernel = attend_tiles<T, DP, kTile>;
        LATTICE_HIP_TRY(allow_lds(reinterpret_cast<const void*>(kernel), kLds));
        kernel<<<grid, kAttnBlock, kLds, stream>>>(a, l.splits, part, out, kept);
    }
    LATTICE_LAUNCH_CHECK();
    if (l.splits > 1) {
        join_parts<T><<<grid_for(static_cast<long long>(a.queries) * a.heads, kAttnWaves, 1u << 30), kAttnBlock, 0,
                        stream>>>(a, l.splits, part, out, kept);
        LATTICE_LAUNCH_CHECK();
    }
    return LATTICE_OK;
}

template <typename T>
int attend(const lattice_attention& a, const AttnLayout& l, const AttnPart& part, void* out, float* lse,
           void* rest, hipStream_t stream) {
    const AttnKept<T> kept{lse, sizeof(T) == 4 ? nullptr : static_cast<T*>(rest)};
    T* o = static_cast<T*>(out);
    if (a.dim <= 32) return launch_attend<T, 32>(a, l, part, o, kept, stream);
    if (a.dim <= 64) return launch_attend<T, 64>(a, l, part, o, kept, stream);
    if (a.dim <= 96) return launch_attend<T, 96>(a, l, part, o, kept, stream);
    return launch_attend<T, 128>(a, l, part, o, kept, stream);
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" size_t lattice_hip_window_attention_workspace_bytes(const lattice_attention* args) {
    if (attn_fault(args) || args->queries == 0) return 0;
    const lattice_attention a = attn_bounded(*args);
    const AttnLayout l = attn_layout(a);
    if (l.splits == 1) return 0;
    const size_t rows = static_cast<size_t>(l.splits) * a.queries * a.heads;
    return aligned_bytes(rows * a.dim * sizeof(float)) + aligned_bytes(rows * sizeof(float2));
}

extern "C" int lattice_hip_window_attention(const lattice_attention* args, void* out, float* lse, void* out_rest,
                                            void* workspace, size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE_ATTENTION(args);
    if (args->queries == 0) return LATTICE_OK;
    LATTICE_REQUIRE(out, "attention pointers must be non-null.");
    const lattice_attention a = attn_bounded(*args);
    const AttnLayout l = attn_layout(a);
    AttnPart part{nullptr, nullptr};
    if (l.splits > 1) {
        Workspace ws{static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
        const size_t rows = static_cast<size_t>(l.splits) * a.queries * a.heads;
        part.values = ws.take<float>(rows * a.dim);
        part.states = ws.take<float2>(rows);
        LATTICE_REQUIRE(part.values && part.states, "attention workspace is too small.");
    }
    hipStream_t stream = as_stream(stream_ptr);
    if (a.dtype == LATTICE_F32) return attend<float>(a, l, part, out, lse, out_rest, stream);
    if (a.dtype == LATTICE_F16) return attend<_Float16>(a, l, part, out, lse, out_rest, stream);
    return attend<__bf16>(a, l, part, out, lse, out_rest, stream);
}
