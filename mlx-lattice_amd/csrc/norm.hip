// Layer norm of feature rows and its gradients.
//
//   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  h = (x - mu) r,
//   y = h w + b;
//   g = dy w,  dx = r (g - mean_c g - h mean_c(g h)),
//   dw = sum_n dy h,  db = sum_n dy.
//
// Bound by memory: the forward reads x and writes y once, the gradient reads
// dy and x and writes dx once; a few operations a value.  A group of G lanes
// (a power of two up to 64) holds a row in registers, K vectors of V values a
// lane, so that the squares are summed about the mean (no cancellation of
// large sums) without a second read; several narrow rows share a wave.  The
// weight's and bias's sums stay in the registers of the lanes that own the
// channels over all the rows a block walks, then go through LDS to one partial
// row per block, and a second launch adds the partials in a fixed order.
// Rows wider than 256 vectors take a block each and are read again from the
// caches.
//
// 400,000 x 128 fp16: forward 40 us (5.1 TB/s of the 5.4 that a copy of that
// size reaches), gradient 64 us (4.8 TB/s; 64 bytes of sums a lane cost it some
// of its waves), the partials' sum 4 us.  20,000 x 32 fp32: 3.5 us, a launch.
// The gradient of wider rows has fewer blocks, a partial row each: 51 M values
// in rows of 512, 1000 and 2048, bf16: 113, 149 and 222 us (2.7, 2.0 and 1.4
// TB/s), the forward pass 42, 43 and 65.

#include "rows.h"

namespace lattice {
namespace {

constexpr int kNormBlock = 256;
constexpr int kNormHeld = 4;       // most vectors of a row that a lane holds
constexpr int kNormPartials = 1024;  // most blocks that sum a weight gradient

// Sum over the `group` lanes (a power of two) that share a row.
__device__ inline float group_sum(float v, int group) {
    for (int step = 1; step < group; step *= 2) v += __shfl_xor(v, step);
    return v;
}

// Sum over the block, returned to every thread.
__device__ inline float block_sum(float v, float* shared) {
    v = group_sum(v, kWave);
    __syncthreads();
    if (lane_id() == 0) shared[threadIdx.x / kWave] = v;
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < kNormBlock / kWave; ++w) total += shared[w];
    return total;
}

__device__ inline int active_count(const int32_t* active_rows, int rows) {
    return active_rows ? max(0, min(active_rows[0], rows)) : rows;
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kNormBlock)
layer_norm_rows(const T* __restrict__ x, long long x_stride, int rows, int channels, int group,
                const T* __restrict__ weight, const T* __restrict__ bias, float eps,
                const int32_t* __restrict__ active_rows, T* __restrict__ y, float2* __restrict__ statistics) {
    typedef RowVec<T, V> Vec;
    const int active = active_count(active_rows, rows);
    const int lane = threadIdx.x & (group - 1);
    const int per_block = kNormBlock / group;
    const float inv = 1.0f / static_cast<float>(channels);
    Vec w[K], b[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (lane + k * group) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            w[k].set(j, 1.0f);
            b[k].set(j, 0.0f);
        }
        if (c < channels && weight) w[k] = Vec::load(weight + c);
        if (c < channels && bias) b[k] = Vec::load(bias + c);
    }
    for (long long first = static_cast<long long>(blockIdx.x) * per_block; first < rows;
         first += static_cast<long long>(gridDim.x) * per_block) {
        const long long row = first + threadIdx.x / group;
        const bool live = row < active;
        float v[K][V];
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (lane + k * group) * V;
            Vec in;
            if (live && c < channels) in = Vec::load(x + row * x_stride + c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[k][j] = live && c < channels ? in.at(j) : 0.0f;
                sum += v[k][j];
            }
        }
        const float mean = group_sum(sum, group) * inv;
        float square = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if ((lane + k * group) * V >= channels) continue;
#pragma unroll
            for (int j = 0; j < V; ++j) square += (v[k][j] - mean) * (v[k][j] - mean);
        }
        const float rstd = 1.0f / sqrtf(group_sum(square, group) * inv + eps);
        if (row >= rows) continue;
        if (statistics && lane == 0) statistics[row] = live ? float2{mean, rstd} : float2{0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (lane + k * group) * V;
            if (c >= channels) continue;
            Vec out;
#pragma unroll
            for (int j = 0; j < V; ++j)
                out.set(j, live ? (v[k][j] - mean) * rstd * w[k].at(j) + b[k].at(j) : 0.0f);
            out.store(y + row * channels + c);
        }
    }
}

// One block a row, read three times.
template <typename T, int V>
__global__ void __launch_bounds__(kNormBlock)
layer_norm_wide(const T* __restrict__ x, long long x_stride, int rows, int channels, const T* __restrict__ weight,
                const T* __restrict__ bias, float eps, const int32_t* __restrict__ active_rows, T* __restrict__ y,
                float2* __restrict__ statistics) {
    typedef RowVec<T, V> Vec;
    __shared__ float shared[kNormBlock / kWave];
    const int active = active_count(active_rows, rows);
    const float inv = 1.0f / static_cast<float>(channels);
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const bool live = row < active;
        const T* in = x + row * x_stride;
        float mean = 0.0f, rstd = 0.0f;
        if (live) {
            float sum = 0.0f;
            for (int c = threadIdx.x * V; c < channels; c += kNormBlock * V) {
                const Vec a = Vec::load(in + c);
#pragma unroll
                for (int j = 0; j < V; ++j) sum += a.at(j);
            }
            mean = block_sum(sum, shared) * inv;
            float square = 0.0f;
            for (int c = threadIdx.x * V; c < channels; c += kNormBlock * V) {
                const Vec a = Vec::load(in + c);
#pragma unroll
                for (int j = 0; j < V; ++j) square += (a.at(j) - mean) * (a.at(j) - mean);
            }
            rstd = 1.0f / sqrtf(block_sum(square, shared) * inv + eps);
        }
        if (statistics && threadIdx.x == 0) statistics[row] = float2{mean, rstd};
        for (int c = threadIdx.x * V; c < channels; c += kNormBlock * V) {
            Vec out;
#pragma unroll
            for (int j = 0; j < V; ++j) out.set(j, 0.0f);
            if (live) {
                const Vec a = Vec::load(in + c);
                Vec w, b;
                if (weight) w = Vec::load(weight + c);
                if (bias) b = Vec::load(bias + c);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    out.set(j, (a.at(j) - mean) * rstd * (weight ? w.at(j) : 1.0f) + (bias ? b.at(j) : 0.0f));
            }
            out.store(y + row * channels + c);
        }
    }
}

// grad_x, and this block's sums of dy h and dy over its rows in
// partials[block][2][channels] (NULL: grad_x alone).
template <typename T, int V, int K>
__global__ void __launch_bounds__(kNormBlock)
layer_norm_grad_rows(const T* __restrict__ dy, long long dy_stride, const T* __restrict__ x, long long x_stride,
                     int rows, int channels, int group, const T* __restrict__ weight,
                     const float2* __restrict__ statistics, const int32_t* __restrict__ active_rows,
                     T* __restrict__ grad_x, float* __restrict__ partials) {
    typedef RowVec<T, V> Vec;
    __shared__ float shared[2 * V * kNormBlock];
    const int active = active_count(active_rows, rows);
    const int lane = threadIdx.x & (group - 1);
    const int per_block = kNormBlock / group;
    const float inv = 1.0f / static_cast<float>(channels);
    float sum_w[K][V] = {}, sum_b[K][V] = {};
    Vec w[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (lane + k * group) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) w[k].set(j, 1.0f);
        if (c < channels && weight) w[k] = Vec::load(weight + c);
    }
    for (long long first = static_cast<long long>(blockIdx.x) * per_block; first < rows;
         first += static_cast<long long>(gridDim.x) * per_block) {
        const long long row = first + threadIdx.x / group;
        const bool live = row < active;
        const float2 stat = live ? statistics[row] : float2{0.0f, 0.0f};
        float h[K][V], g[K][V];
        float along_g = 0.0f, along_h = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (lane + k * group) * V;
            const bool here = live && c < channels;
            Vec a, d;
            if (here) {
                a = Vec::load(x + row * x_stride + c);
                d = Vec::load(dy + row * dy_stride + c);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float slope = here ? d.at(j) : 0.0f;
                h[k][j] = here ? (a.at(j) - stat.x) * stat.y : 0.0f;
                g[k][j] = slope * w[k].at(j);
                sum_w[k][j] += slope * h[k][j];
                sum_b[k][j] += slope;
                along_g += g[k][j];
                along_h += g[k][j] * h[k][j];
            }
        }
        along_g = group_sum(along_g, group) * inv;
        along_h = group_sum(along_h, group) * inv;
        if (row >= rows) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (lane + k * group) * V;
            if (c >= channels) continue;
            Vec out;
#pragma unroll
            for (int j = 0; j < V; ++j)
                out.set(j, live ? stat.y * (g[k][j] - along_g - h[k][j] * along_h) : 0.0f);
            out.store(grad_x + row * channels + c);
        }
    }
    if (!partials) return;
    float* mine = partials + static_cast<long long>(blockIdx.x) * 2 * channels;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < V; ++j) {
            shared[j * kNormBlock + threadIdx.x] = sum_w[k][j];
            shared[(V + j) * kNormBlock + threadIdx.x] = sum_b[k][j];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 2 * V * group; i += kNormBlock) {
            const int value = i / group;  // V sums of dy h, then V of dy
            const int at = i & (group - 1);
            const int c = (at + k * group) * V + value % V;
            if (c >= channels) continue;
            float sum = 0.0f;
            for (int r = 0; r < per_block; ++r) sum += shared[value * kNormBlock + r * group + at];
            mine[(value / V) * static_cast<long long>(channels) + c] = sum;
        }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kNormBlock)
layer_norm_grad_wide(const T* __restrict__ dy, long long dy_stride, const T* __restrict__ x, long long x_stride,
                     int rows, int channels, const T* __restrict__ weight, const float2* __restrict__ statistics,
                     const int32_t* __restrict__ active_rows, T* __restrict__ grad_x) {
    typedef RowVec<T, V> Vec;
    __shared__ float shared[kNormBlock / kWave];
    const int active = active_count(active_rows, rows);
    const float inv = 1.0f / static_cast<float>(channels);
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const bool live = row < active;
        const float2 stat = live ? statistics[row] : float2{0.0f, 0.0f};
        float along_g = 0.0f, along_h = 0.0f;
        if (live) {
            for (int c = threadIdx.x * V; c < channels; c += kNormBlock * V) {
                const Vec a = Vec::load(x + row * x_stride + c), d = Vec::load(dy + row * dy_stride + c);
                Vec w;
                if (weight) w = Vec::load(weight + c);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float g = d.at(j) * (weight ? w.at(j) : 1.0f);
                    along_g += g;
                    along_h += g * ((a.at(j) - stat.x) * stat.y);
                }
            }
            along_g = block_sum(along_g, shared) * inv;
            along_h = block_sum(along_h, shared) * inv;
        }
        for (int c = threadIdx.x * V; c < channels; c += kNormBlock * V) {
            Vec out;
#pragma unroll
            for (int j = 0; j < V; ++j) out.set(j, 0.0f);
            if (live) {
                const Vec a = Vec::load(x + row * x_stride + c), d = Vec::load(dy + row * dy_stride + c);
                Vec w;
                if (weight) w = Vec::load(weight + c);
#pragma unroll
                for (int j = 0; j < V; ++j)
                    out.set(j, stat.y * (d.at(j) * (weight ? w.at(j) : 1.0f) - along_g -
                                         (a.at(j) - stat.x) * stat.y * along_h));
            }
            out.store(grad_x + row * channels + c);
        }
    }
}

// The column sums of wide rows: a thread a channel, a grid row a share of the
// rows.
template <typename T>
__global__ void __launch_bounds__(kNormBlock)
layer_norm_grad_columns(const T* __restrict__ dy, long long dy_stride, const T* __restrict__ x, long long x_stride,
                        int rows, int channels, const float2* __restrict__ statistics,
                        const int32_t* __restrict__ active_rows, float* __restrict__ partials) {
    const int active = active_count(active_rows, rows);
    const int c = blockIdx.x * kNormBlock + threadIdx.x;
    if (c >= channels) return;
    float sum_w = 0.0f, sum_b = 0.0f;
    for (long long row = blockIdx.y; row < active; row += gridDim.y) {
        const float2 stat = statistics[row];
        const float slope = static_cast<float>(dy[row * dy_stride + c]);
        sum_w += slope * ((static_cast<float>(x[row * x_stride + c]) - stat.x) * stat.y);
        sum_b += slope;
    }
    float* mine = partials + static_cast<long long>(blockIdx.y) * 2 * channels;
    mine[c] = sum_w;
    mine[channels + c] = sum_b;
}

// partials [count][2][channels] -> grad_weight and grad_bias: 16 columns a
// block, 64 slices of the partials added in slice order.
constexpr int kFinishBlock = 1024, kFinishSlices = kFinishBlock / 16;
template <typename T>
__global__ void __launch_bounds__(kFinishBlock)
layer_norm_grad_finish(const float* __restrict__ partials, int count, int channels, T* __restrict__ grad_weight,
                       T* __restrict__ grad_bias) {
    __shared__ float shared[kFinishSlices][17];
    const int at = threadIdx.x & 15, slice = threadIdx.x >> 4;
    const long long columns = 2ll * channels;
    for (long long first = blockIdx.x * 16ll; first < columns; first += gridDim.x * 16ll) {
        const long long column = first + at;
        float sum = 0.0f;
        if (column < columns) {
            // Four chains of additions keep four reads in flight.
            float chain[4] = {};
            int i = slice;
            for (; i + 3 * kFinishSlices < count; i += 4 * kFinishSlices) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    chain[u] += partials[(i + static_cast<long long>(kFinishSlices) * u) * columns + column];
            }
            for (; i < count; i += kFinishSlices) chain[0] += partials[static_cast<long long>(i) * columns + column];
            sum = (chain[0] + chain[1]) + (chain[2] + chain[3]);
        }
        shared[slice][at] = sum;
        __syncthreads();
        if (slice == 0 && column < columns) {
            for (int s = 1; s < kFinishSlices; ++s) sum += shared[s][at];
            if (column < channels) {
                if (grad_weight) grad_weight[column] = static_cast<T>(sum);
            } else if (grad_bias) {
                grad_bias[column - channels] = static_cast<T>(sum);
            }
        }
        __syncthreads();
    }
}
// A launch takes fewer than 2^32 threads.
inline unsigned finish_blocks(int channels) { return grid_for(2ll * channels, 16, 1u << 20); }

// Lanes and vectors a lane for rows of `vectors` vectors.
struct NormShape {
    int group, held;  // held 0: a block a row
};
inline NormShape norm_shape(int vectors) {
    if (vectors > kWave * kNormHeld) return {kNormBlock, 0};
    int group = 1;
    while (group < vectors && group < kWave) group *= 2;
    const int held = (vectors + group - 1) / group;
    return {group, held == 3 ? 4 : held};
}

// Vectors of 16, 4 and one element's bytes are instantiated.
template <typename T>
int norm_vector(int channels, std::initializer_list<const void*> addresses,
                std::initializer_list<long long> strides) {
    const int v = row_vector<T>(channels, addresses, strides);
    const int most = 16 / static_cast<int>(sizeof(T)), word = 4 / static_cast<int>(sizeof(T));
    return v == most ? v : v >= word ? word : 1;
}

inline int norm_partials(int rows, int channels, int per_block) {
    const long long blocks = (static_cast<long long>(rows) + per_block - 1) / per_block;
    // Wide rows: no more partials than a quarter of a million sums.
    const long long cap = std::max<long long>(64, std::min<long long>(kNormPartials, (1ll << 18) / channels));
    return static_cast<int>(std::max<long long>(1, std::min(blocks, cap)));
}

template <typename T, int V>
int launch_norm(const T* x, long long x_stride, int rows, int channels, const T* weight, const T* bias, float eps,
                const int32_t* active_rows, T* y, float2* statistics, hipStream_t stream) {
    const NormShape shape = norm_shape(channels / V);
#define LATTICE_NORM_ROWS(K)                                                                                     \
    layer_norm_rows<T, V, K><<<grid_for(rows, kNormBlock / shape.group, 4096), kNormBlock, 0, stream>>>(         \
        x, x_stride, rows, channels, shape.group, weight, bias, eps, active_rows, y, statistics)
    switch (shape.held) {
        case 1: LATTICE_NORM_ROWS(1); break;
        case 2: LATTICE_NORM_ROWS(2); break;
        case 4: LATTICE_NORM_ROWS(4); break;
        default:
            layer_norm_wide<T, V><<<grid_for(rows, 1, 4096), kNormBlock, 0, stream>>>(
                x, x_stride, rows, channels, weight, bias, eps, active_rows, y, statistics);
    }
#undef LATTICE_NORM_ROWS
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T, int V>
int launch_norm_grad(const T* dy, long long dy_stride, const T* x, long long x_stride, int rows, int channels,
                     const T* weight, const float2* statistics, const int32_t* active_rows, T* grad_x,
                     T* grad_weight, T* grad_bias, float* partials, hipStream_t stream) {
    const NormShape shape = norm_shape(channels / V);
    const int per_block = shape.held ? kNormBlock / shape.group : 1;
    const int blocks = norm_partials(rows, channels, per_block);
#define LATTICE_NORM_ROWS(K)                                                                                  \
    layer_norm_grad_rows<T, V, K><<<partials ? blocks : grid_for(rows, per_block, 4096), kNormBlock, 0, stream>>>( \
        dy, dy_stride, x, x_stride, rows, channels, shape.group, weight, statistics, active_rows, grad_x, partials)
    switch (shape.held) {
        case 1: LATTICE_NORM_ROWS(1); break;
        case 2: LATTICE_NORM_ROWS(2); break;
        case 4: LATTICE_NORM_ROWS(4); break;
        default:
            layer_norm_grad_wide<T, V><<<grid_for(rows, 1, 4096), kNormBlock, 0, stream>>>(
                dy, dy_stride, x, x_stride, rows, channels, weight, statistics, active_rows, grad_x);
            if (partials) {
                LATTICE_LAUNCH_CHECK();
                layer_norm_grad_columns<T>
                    <<<dim3((channels + kNormBlock - 1) / kNormBlock, blocks), kNormBlock, 0, stream>>>(
                        dy, dy_stride, x, x_stride, rows, channels, statistics, active_rows, partials);
            }
    }
#undef LATTICE_NORM_ROWS
    LATTICE_LAUNCH_CHECK();
    if (partials) {
        layer_norm_grad_finish<T><<<finish_blocks(channels), kFinishBlock, 0, stream>>>(partials, blocks, channels,
                                                                               grad_weight, grad_bias);
        LATTICE_LAUNCH_CHECK();
    }
    return LATTICE_OK;
}

template <typename T>
int norm_of(const void* x, long long x_stride, int rows, int channels, const void* weight, const void* bias,
            float eps, const int32_t* active_rows, void* y, float* statistics, hipStream_t stream) {
    const T* in = static_cast<const T*>(x);
    const T* w = static_cast<const T*>(weight);
    const T* b = static_cast<const T*>(bias);
    T* out = static_cast<T*>(y);
    float2* stats = reinterpret_cast<float2*>(statistics);
    constexpr int kMost = 16 / sizeof(T), kWord = 4 / sizeof(T);
    const int v = norm_vector<T>(channels, {x, weight, bias, y}, {x_stride});
    if (v == kMost) return launch_norm<T, kMost>(in, x_stride, rows, channels, w, b, eps, active_rows, out, stats, stream);
    if constexpr (kWord > 1) {
        if (v == kWord)
            return launch_norm<T, kWord>(in, x_stride, rows, channels, w, b, eps, active_rows, out, stats, stream);
    }
    return launch_norm<T, 1>(in, x_stride, rows, channels, w, b, eps, active_rows, out, stats, stream);
}

template <typename T>
int norm_grad_of(const void* grad_y, long long dy_stride, const void* x, long long x_stride, int rows, int channels,
                 const void* weight, const float* statistics, const int32_t* active_rows, void* grad_x,
                 void* grad_weight, void* grad_bias, float* partials, hipStream_t stream) {
    const T* dy = static_cast<const T*>(grad_y);
    const T* in = static_cast<const T*>(x);
    const T* w = static_cast<const T*>(weight);
    T* dx = static_cast<T*>(grad_x);
    T* dw = static_cast<T*>(grad_weight);
    T* db = static_cast<T*>(grad_bias);
    const float2* stats = reinterpret_cast<const float2*>(statistics);
    constexpr int kMost = 16 / sizeof(T), kWord = 4 / sizeof(T);
    const int v = norm_vector<T>(channels, {grad_y, x, weight, grad_x}, {dy_stride, x_stride});
    if (v == kMost)
        return launch_norm_grad<T, kMost>(dy, dy_stride, in, x_stride, rows, channels, w, stats, active_rows, dx, dw,
                                          db, partials, stream);
    if constexpr (kWord > 1) {
        if (v == kWord)
            return launch_norm_grad<T, kWord>(dy, dy_stride, in, x_stride, rows, channels, w, stats, active_rows, dx,
                                              dw, db, partials, stream);
    }
    return launch_norm_grad<T, 1>(dy, dy_stride, in, x_stride, rows, channels, w, stats, active_rows, dx, dw, db,
                                  partials, stream);
}

}  // namespace
}  // namespace lattice

using namespace lattice;

extern "C" int lattice_hip_layer_norm(int dtype, const void* x, long long x_stride, int rows, int channels,
                                      const void* weight, const void* bias, float eps, const int32_t* active_rows,
                                      void* y, float* statistics, void* stream_ptr) {
    LATTICE_REQUIRE(dtype == LATTICE_F32 || dtype == LATTICE_F16 || dtype == LATTICE_BF16,
                    "layer norm supports float32, float16 and bfloat16.");
    LATTICE_REQUIRE(rows >= 0 && channels > 0 && x_stride >= 0, "layer norm shapes must be positive.");
    LATTICE_REQUIRE(channels < 1 << 30, "layer norm takes up to 2^30 - 1 channels.");
    LATTICE_REQUIRE(eps >= 0.0f, "eps must be non-negative.");
    if (rows == 0) return LATTICE_OK;
    LATTICE_REQUIRE(x && y, "layer norm pointers must be non-null.");
    hipStream_t stream = as_stream(stream_ptr);
    if (dtype == LATTICE_F32)
        return norm_of<float>(x, x_stride, rows, channels, weight, bias, eps, active_rows, y, statistics, stream);
    if (dtype == LATTICE_F16)
        return norm_of<_Float16>(x, x_stride, rows, channels, weight, bias, eps, active_rows, y, statistics, stream);
    return norm_of<__bf16>(x, x_stride, rows, channels, weight, bias, eps, active_rows, y, statistics, stream);
}

extern "C" size_t lattice_hip_layer_norm_grad_workspace_bytes(int rows, int channels) {
    if (rows <= 0 || channels <= 0) return 0;
    // The most blocks any vector width gives: one row a block.
    return static_cast<size_t>(norm_partials(rows, channels, 1)) * 2 * channels * sizeof(float);
}

extern "C" int lattice_hip_layer_norm_grad(int dtype, const void* grad_y, long long grad_y_stride, const void* x,
                                           long long x_stride, int rows, int channels, const void* weight,
                                           const float* statistics, const int32_t* active_rows, void* grad_x,
                                           void* grad_weight, void* grad_bias, void* workspace,
                                           size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE(dtype == LATTICE_F32 || dtype == LATTICE_F16 || dtype == LATTICE_BF16,
                    "layer norm supports float32, float16 and bfloat16.");
    LATTICE_REQUIRE(rows >= 0 && channels > 0 && x_stride >= 0 && grad_y_stride >= 0,
                    "layer norm shapes must be positive.");
    LATTICE_REQUIRE(channels < 1 << 30, "layer norm takes up to 2^30 - 1 channels.");
    const bool sums = grad_weight || grad_bias;
    LATTICE_REQUIRE(rows == 0 || (grad_y && x && statistics && grad_x), "layer norm pointers must be non-null.");
    LATTICE_REQUIRE(!sums || rows == 0 ||
                        (workspace && workspace_bytes >= lattice_hip_layer_norm_grad_workspace_bytes(rows, channels)),
                    "layer norm gradient workspace is too small.");
    hipStream_t stream = as_stream(stream_ptr);
    float* partials = sums ? static_cast<float*>(workspace) : nullptr;
    if (rows == 0) {
        if (!sums) return LATTICE_OK;
        // No partials: the sums are zero.
        const unsigned blocks = finish_blocks(channels);
        if (dtype == LATTICE_F32) {
            layer_norm_grad_finish<float><<<blocks, kFinishBlock, 0, stream>>>(
                nullptr, 0, channels, static_cast<float*>(grad_weight), static_cast<float*>(grad_bias));
        } else {  // zero has the same bits in both 16-bit types
            layer_norm_grad_finish<_Float16><<<blocks, kFinishBlock, 0, stream>>>(
                nullptr, 0, channels, static_cast<_Float16*>(grad_weight), static_cast<_Float16*>(grad_bias));
        }
        LATTICE_LAUNCH_CHECK();
        return LATTICE_OK;
    }
    if (dtype == LATTICE_F32)
        return norm_grad_of<float>(grad_y, grad_y_stride, x, x_stride, rows, channels, weight, statistics, active_rows,
                                   grad_x, grad_weight, grad_bias, partials, stream);
    if (dtype == LATTICE_F16)
        return norm_grad_of<_Float16>(grad_y, grad_y_stride, x, x_stride, rows, channels, weight, statistics,
                                      active_rows, grad_x, grad_weight, grad_bias, partials, stream);
    return norm_grad_of<__bf16>(grad_y, grad_y_stride, x, x_stride, rows, channels, weight, statistics, active_rows,
                                grad_x, grad_weight, grad_bias, partials, stream);
}
