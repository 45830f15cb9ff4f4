// Rotary positions of several axes.
//
// The first channels of a head are cut into a section per axis; pair i of
// section a, (u, v), is turned by t = position_a * frequency_i:
//   u' = u cos t - v sin t,  v' = u sin t + v cos t,
// and by -t for the gradient, which is the transpose.
//
// Bound by memory: x is read and y written once.  A block takes some rows and
// first makes the cosines and sines that all heads of a row share in LDS, each
// once.  The angle is position * frequency / (2 pi) turns in float64, reduced
// to half a turn there: in float32 a coordinate of 10^5 would leave it wrong by
// a hundredth of a radian.  Then a lane moves a 16-byte piece of a head; its
// partners, which lie at any channel distance (an axis has any even number of
// channels), come from the wave's copy of the piece in LDS.
//
// 200,000 rows of 16 heads of 32, bf16, out of rows of 24: 102 us (4.0 TB/s).
// 60,001 rows of 6 heads of 64, fp32: 48 us (3.9).  Both read and write each
// value once, and waves spend 71 % of their time in waits; the partners' reads of
// single channels conflict in LDS (two of three cycles in use; LDS is in use 25
// and 12 % of the time, the vector pipe 35 and 30).

#include "rows.h"

namespace lattice {
namespace {

constexpr int kRotaryBlock = 256;
constexpr int kRotaryWaves = kRotaryBlock / kWave;
constexpr int kRotaryAxes = 4;
constexpr int kRotaryMaxDim = 1024;
constexpr int kRotaryUnroll = 4;

struct RotaryAxes {
    int axes, pairs, interleaved;
    int dims[kRotaryAxes];
};

struct RotaryPositions {
    const void* values;
    long long stride;
    int is_float;
    __device__ double at(long long row, int axis) const {
        return is_float ? static_cast<double>(static_cast<const float*>(values)[row * stride + axis])
                        : static_cast<double>(static_cast<const int32_t*>(values)[row * stride + axis]);
    }
};

// Channel c of a head: the pair it belongs to (-1: copied), its partner's
// channel, and the sign of the partner's part.
struct RotaryChannel {
    int pair, partner;
    float sign;
};
__device__ inline RotaryChannel rotary_channel(const RotaryAxes& axes, int c) {
    int start = 0;
    for (int a = 0; a < axes.axes; ++a) {
        const int width = axes.dims[a];
        if (c < start + width) {
            const int i = c - start, half = width / 2;
            if (axes.interleaved) return {start / 2 + i / 2, c ^ 1, i & 1 ? 1.0f : -1.0f};
            return i < half ? RotaryChannel{start / 2 + i, c + half, -1.0f}
                            : RotaryChannel{start / 2 + i - half, c - half, 1.0f};
        }
        start += width;
    }
    return {-1, c, 0.0f};
}

// (cos, sin) of every pair of `count` rows from `first`.
__device__ inline void rotary_table(float2* table, const RotaryAxes& axes, const RotaryPositions& positions,
                                    const double* frequencies, long long first, int count, float sign) {
    constexpr double kPerTurn = 0.15915494309189533577;  // 1 / (2 pi)
    for (int i = threadIdx.x; i < count * axes.pairs; i += kRotaryBlock) {
        const int row = i / axes.pairs, pair = i - row * axes.pairs;
        int axis = 0, end = axes.dims[0] / 2;
        while (pair >= end && axis + 1 < axes.axes) end += axes.dims[++axis] / 2;
        const double turns = positions.at(first + row, axis) * (frequencies[pair] * kPerTurn);
        float s, c;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
        table[i] = float2{c, sign * s};
    }
}

// x rows of dim = chunks * V channels, chunks <= 64.  A lane has a piece of a
// row and walks the row's heads, so that its cosines and sines stay in
// registers; the waves that are left over share the heads.
template <typename T, int V>
__global__ void __launch_bounds__(kRotaryBlock)
rotary_rows(const T* __restrict__ x, long long x_row, long long x_head, int rows, int heads, int dim,
            RotaryPositions positions, const double* __restrict__ frequencies, RotaryAxes axes, float sign,
            int block_rows, T* __restrict__ y) {
    typedef RowVec<T, V> Vec;
    extern __shared__ float2 table[];
    __shared__ __align__(16) T stage[kRotaryWaves][kRotaryUnroll][kWave * V];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = lane_id();
    const int chunks = dim / V;
    const int wave_rows = kWave / chunks;
    const int sub = lane / chunks, c0 = (lane - sub * chunks) * V;
    int from[V], pair[V];
    float turn[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const RotaryChannel ch = rotary_channel(axes, c0 + j);
        pair[j] = ch.pair;
        from[j] = sub * dim + ch.partner;
        turn[j] = ch.sign;
    }
    for (long long first = static_cast<long long>(blockIdx.x) * block_rows; first < rows;
         first += static_cast<long long>(gridDim.x) * block_rows) {
        const int count = static_cast<int>(min(static_cast<long long>(block_rows), rows - first));
        rotary_table(table, axes, positions, frequencies, first, count, sign);
        __syncthreads();
        const int groups = (count + wave_rows - 1) / wave_rows;
        const int shares = max(1, kRotaryWaves / groups);  // waves a group of rows
        for (int unit = wave; unit < groups * shares; unit += kRotaryWaves) {
            const int row = unit / shares * wave_rows + sub;
            const bool live = sub < wave_rows && row < count;
            float cosine[V], sine[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 t = live && pair[j] >= 0 ? table[row * axes.pairs + pair[j]] : float2{1.0f, 0.0f};
                cosine[j] = t.x;
                sine[j] = turn[j] * t.y;
            }
            const T* in = x + (first + row) * x_row + c0;
            T* out = y + (first + row) * heads * dim + c0;
            // Neighbouring heads, which share lines, together.
            const int share = (heads + shares - 1) / shares;
            const int end = min(heads, (unit % shares + 1) * share);
            for (int base = unit % shares * share; base < end; base += kRotaryUnroll) {
                Vec v[kRotaryUnroll];
#pragma unroll
                for (int u = 0; u < kRotaryUnroll; ++u) {
                    const int head = base + u;
                    if (live && head < end) v[u] = Vec::load(in + head * x_head);
                }
#pragma unroll
                for (int u = 0; u < kRotaryUnroll; ++u)
                    if (live && base + u < end) v[u].store(&stage[wave][u][lane * V]);
                // The wave alone reads what it wrote, in order.
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int u = 0; u < kRotaryUnroll; ++u) {
                    const int head = base + u;
                    if (!live || head >= end) continue;
                    Vec turned;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float other = static_cast<float>(stage[wave][u][from[j]]);
                        turned.set(j, v[u].at(j) * cosine[j] + other * sine[j]);
                        // Channels past the axes are copied, whatever they hold.
                        if (pair[j] < 0) turned.e[j] = v[u].e[j];
                    }
                    turned.store(out + head * dim);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        __syncthreads();
    }
}

// Any dim and alignment: a lane a channel, its partner read from x.
template <typename T>
__global__ void __launch_bounds__(kRotaryBlock)
rotary_channels(const T* __restrict__ x, long long x_row, long long x_head, int rows, int heads, int dim,
                RotaryPositions positions, const double* __restrict__ frequencies, RotaryAxes axes, float sign,
                int block_rows, T* __restrict__ y) {
    extern __shared__ float2 table[];
    const long long width = static_cast<long long>(heads) * dim;
    for (long long first = static_cast<long long>(blockIdx.x) * block_rows; first < rows;
         first += static_cast<long long>(gridDim.x) * block_rows) {
        const int count = static_cast<int>(min(static_cast<long long>(block_rows), rows - first));
        rotary_table(table, axes, positions, frequencies, first, count, sign);
        __syncthreads();
        for (long long i = threadIdx.x; i < count * width; i += kRotaryBlock) {
            const int row = static_cast<int>(i / width);
            const int at = static_cast<int>(i - row * width);
            const int head = at / dim;
            const RotaryChannel ch = rotary_channel(axes, at - head * dim);
            const T* in = x + (first + row) * x_row + head * x_head;
            T out = in[at - head * dim];
            if (ch.pair >= 0) {
                const float2 t = table[row * axes.pairs + ch.pair];
                out = static_cast<T>(static_cast<float>(out) * t.x +
                                     ch.sign * (static_cast<float>(in[ch.partner]) * t.y));
            }
            y[first * width + i] = out;
        }
        __syncthreads();
    }
}

template <typename T>
int rotary_of(const void* x, long long x_row, long long x_head, int rows, int heads, int dim,
              const RotaryPositions& positions, const double* frequencies, const RotaryAxes& axes, float sign,
              void* y, hipStream_t stream) {
    constexpr int kMost = 16 / sizeof(T);
    const T* in = static_cast<const T*>(x);
    T* out = static_cast<T*>(y);
    // A table of about 512 pairs a block, fewer where that leaves units idle.
    const int block_rows = static_cast<int>(std::max<long long>(
        1, std::min<long long>(std::max(1, 512 / std::max(1, axes.pairs)), (rows + 1023ll) / 1024)));
    // A launch takes fewer than 2^32 threads; far fewer blocks fill the chip.
    const unsigned grid = grid_for(rows, block_rows, 1u << 22);
    // Working out a lane's eight channels of a 16-bit type is worth more than
    // an even end: blocks that stay (five a unit) take 101 us over 200k rows of
    // 16 heads of 32, a block for every table 107; with four channels (fp32)
    // there is less to gain and the even end counts.
    const unsigned resident = sizeof(T) == 2 ? std::min(grid, 256u * 5u) : grid;
    const size_t lds = static_cast<size_t>(block_rows) * axes.pairs * sizeof(float2);
    if (row_vector<T>(dim, {x, y}, {x_row, x_head}) == kMost && dim / kMost <= kWave) {
        rotary_rows<T, kMost><<<resident, kRotaryBlock, lds, stream>>>(in, x_row, x_head, rows, heads, dim, positions,
                                                                   frequencies, axes, sign, block_rows, out);
    } else {
        rotary_channels<T><<<grid, kRotaryBlock, lds, stream>>>(in, x_row, x_head, rows, heads, dim, positions,
                                                                frequencies, axes, sign, block_rows, out);
    }
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" int lattice_hip_rotary_positions(int dtype, const void* x, long long x_row_stride, long long x_head_stride,
                                            int rows, int heads, int dim, const void* positions, int float_positions,
                                            long long position_stride, const double* frequencies, int axes,
                                            const int32_t* dims, int interleaved, int inverse, void* y,
                                            void* stream_ptr) {
    LATTICE_REQUIRE(dtype == LATTICE_F32 || dtype == LATTICE_F16 || dtype == LATTICE_BF16,
                    "rotary positions support float32, float16 and bfloat16.");
    LATTICE_REQUIRE(rows >= 0 && heads > 0 && dim > 0 && dim <= kRotaryMaxDim,
                    "rotary heads must have between 1 and 1024 channels.");
    LATTICE_REQUIRE(static_cast<long long>(heads) * dim < 1ll << 31, "rotary rows take up to 2^31 - 1 values.");
    LATTICE_REQUIRE(x_row_stride >= 0 && x_head_stride >= 0 && position_stride >= 0,
                    "rotary strides must be non-negative.");
    LATTICE_REQUIRE(axes >= 1 && axes <= kRotaryAxes && dims, "rotary positions need between 1 and 4 axes.");
    RotaryAxes sections{axes, 0, interleaved != 0, {0, 0, 0, 0}};
    for (int a = 0; a < axes; ++a) {
        LATTICE_REQUIRE(dims[a] >= 0 && dims[a] % 2 == 0 && dims[a] <= kRotaryMaxDim,
                        "rotary dims must be even and non-negative.");
        sections.dims[a] = dims[a];
        sections.pairs += dims[a] / 2;
    }
    LATTICE_REQUIRE(2 * sections.pairs <= dim, "rotary dims must fit the head.");
    if (rows == 0) return LATTICE_OK;
    LATTICE_REQUIRE(x && y && positions && (frequencies || sections.pairs == 0),
                    "rotary pointers must be non-null.");
    const RotaryPositions at{positions, position_stride, float_positions != 0};
    const float sign = inverse ? -1.0f : 1.0f;
    hipStream_t stream = as_stream(stream_ptr);
    if (dtype == LATTICE_F32)
        return rotary_of<float>(x, x_row_stride, x_head_stride, rows, heads, dim, at, frequencies, sections, sign, y,
                                stream);
    if (dtype == LATTICE_F16)
        return rotary_of<_Float16>(x, x_row_stride, x_head_stride, rows, heads, dim, at, frequencies, sections, sign,
                                   y, stream);
    return rotary_of<__bf16>(x, x_row_stride, x_head_stride, rows, heads, dim, at, frequencies, sections, sign, y,
                             stream);
}
