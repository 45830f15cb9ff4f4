// The junction of two parts of a block: a part's result, normed if asked for,
// times a gate and a scale, is added to the residual stream, and the sum is
// normed for the next part.
//
//   norm(z) = (z - mu) r,  mu = mean_c z,  r = 1 / sqrt(mean_c (z - mu)^2 + eps)   (rms: mu = 0)
//   u = norm(x) wp + bp  or  x,   f = scale gate,
//   h = residual + f u  (rounded: what the stream holds),   n = norm(h),   y = n w + b;
//   g = dy w,   t = dh + r (g - mean_c g - n mean_c(g n))   (rms: without mean_c g)
//   d residual = t,  dw = sum dy n,  db = sum dy,  d gate = scale sum t u,
//   k = f t wp,   dx = rp (k - mean_c k - m mean_c(k m)), m = norm(x);   without the first norm dx = f t,
//   d wp = sum f t m,  d bp = sum f t.
//
// Bound by memory: the forward pass reads two arrays and writes two, the
// gradients read four (three where neither gate nor first norm need x) and
// write two.  A power of two of threads, of a wave's lanes or of a block's waves,
// holds a row in registers, 16 bytes a thread, and reads the next row while it
// computes one: 160 us without that, 125 with, for the gradients below.  Sums go
// across lanes without LDS (102 us with, 86 without, for the forward pass of
// 400000 rows of 128 channels in bfloat16 with the first norm).  The vectors'
// sums stay in the registers of the lanes that own the channels over all rows a
// block walks, then go to one partial row a block, and a second launch adds those
// in a fixed order.  Rows wider than a block holds are read again from the
// caches, and their vectors' sums take a pass of their own.
//
// 400000 rows of 128 channels, half precision, with a gate: forward 76 us (5.4
// TB/s), gradients 125 us (4.9 TB/s) and 4 for the vectors' sums.  25013 rows of
// 1000 channels, float32, both norms: 74 us (5.4), 140 (4.3) and 5.  6250 rows of
// 8192 channels, half precision: 162 and 371 us, as rows that no block holds 406
// and 763.

#include "rows.h"

namespace lattice {
namespace {

constexpr int kJoinBlock = 256;
constexpr int kJoinWidest = 512;     // most threads a row
constexpr int kJoinHeld = 2;         // most vectors of a row that a thread holds
constexpr int kJoinMost = 16 / 2 * kJoinWidest * kJoinHeld;  // most channels that a block holds
constexpr int kJoinPartials = 1024;  // most blocks that sum the vectors' gradients
constexpr int kJoinBlocks = 4096;    // most blocks that walk the rows otherwise
constexpr int kJoinSums = 5;         // weight, bias, gate, post weight, post bias

struct JoinGrads {
    const void *sum, *grad_sum, *grad_normed;
    void *grad_x, *grad_residual;
    void* vectors[kJoinSums];  // NULL: not wanted
};

// The sum over `lanes` lanes, a power of two, next to each other.
template <int CONTROL>
__device__ inline float lane_moved(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CONTROL, 0xf, 0xf, true));
}
__device__ inline float lanes_sum(float v, int lanes) {
    if (lanes >= 2) v += lane_moved<0xb1>(v);    // of pairs: 1, 0, 3, 2
    if (lanes >= 4) v += lane_moved<0x4e>(v);    // of fours: 2, 3, 0, 1
    if (lanes >= 8) v += lane_moved<0x141>(v);   // eights mirrored: their fours are equal
    if (lanes >= 16) v += lane_moved<0x140>(v);  // sixteens mirrored
    if (lanes >= 32) {
        const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    }
    if (lanes >= 64) {
        const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
    }
    return v;
}

// The sum over a row's `group` threads: a power of two of a wave's lanes, or of
// a block's waves.
__device__ inline float2 lanes_sum(float2 v, int lanes) { return {lanes_sum(v.x, lanes), lanes_sum(v.y, lanes)}; }
__device__ inline void add_to(float& v, float more) { v += more; }
__device__ inline void add_to(float2& v, float2 more) {
    v.x += more.x;
    v.y += more.y;
}
template <typename F>
__device__ inline F row_sum(F v, int group, F* shared) {
    v = lanes_sum(v, min(group, kWave));
    if (group <= kWave) return v;
    const int wave = threadIdx.x / kWave, waves = group / kWave, from = wave & -waves;
    __syncthreads();
    if (lane_id() == 0) shared[wave] = v;
    __syncthreads();
    v = shared[from];
    for (int w = 1; w < waves; ++w) add_to(v, shared[from + w]);
    return v;
}

__device__ inline int active_count(const lattice_residual_norm& a) {
    return a.active_rows ? max(0, min(a.active_rows[0], a.rows)) : a.rows;
}

template <typename T, int V>
__device__ inline RowVec<T, V> vector_or(const void* from, int c, int channels, float value) {
    RowVec<T, V> v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.set(j, value);
    if (from && c < channels) v = RowVec<T, V>::load(static_cast<const T*>(from) + c);
    return v;
}

// The sum of a row's values (rms: 0) and 1 / deviation.  The mean is taken away
// with one rounding.
struct RowStatistics {
    float sum, inv, root;
    __device__ float mean() const { return sum * inv; }
    __device__ float away(float v) const { return __builtin_fmaf(-inv, sum, v); }
};

// Of the values that a row's threads hold; places past its channels hold zeros.
template <int V, int K>
__device__ inline RowStatistics row_statistics(const float (&v)[K][V], int channels, int first, int stride, int group,
                                               bool rms, float eps, float* shared) {
    RowStatistics s{0.0f, 1.0f / static_cast<float>(channels), 0.0f};
    if (!rms) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) sum += v[k][j];
        }
        s.sum = row_sum(sum, group, shared);
    }
    float square = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (first + k * stride >= channels) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) square += s.away(v[k][j]) * s.away(v[k][j]);
    }
    s.root = 1.0f / sqrtf(row_sum(square, group, shared) * s.inv + eps);
    return s;
}

template <typename T, int V, int K, int BLOCK, bool POST>
__global__ void __launch_bounds__(BLOCK)
residual_norm_rows(lattice_residual_norm a, int group, T* __restrict__ sum, T* __restrict__ normed,
                   float4* __restrict__ statistics) {
    typedef RowVec<T, V> Vec;
    __shared__ float shared[BLOCK / kWave];
    const int active = active_count(a), channels = a.channels;
    const int lane = threadIdx.x & (group - 1), first = lane * V, stride = group * V;
    const int per_block = BLOCK / group;
    Vec w[K], b[K], gate[K], post_w[K], post_b[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = first + k * stride;
        w[k] = vector_or<T, V>(a.weight, c, channels, 1.0f);
        b[k] = vector_or<T, V>(a.bias, c, channels, 0.0f);
        gate[k] = vector_or<T, V>(a.gate, c, channels, 1.0f);
        if constexpr (POST) {
            post_w[k] = vector_or<T, V>(a.post_weight, c, channels, 1.0f);
            post_b[k] = vector_or<T, V>(a.post_bias, c, channels, 0.0f);
        }
    }
    // A row's vectors are read while the one before is computed, where registers
    // hold both.
    constexpr bool kAhead = K == 1;
    struct Held {
        Vec part[K], rest[K];
    };
    const auto load = [&](long long row, Held& r) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = first + k * stride;
            r.part[k] = r.rest[k] = Vec{};
            if (row >= active || c >= channels) continue;
            r.part[k] = Vec::load(static_cast<const T*>(a.x) + row * a.x_stride + c);
            r.rest[k] = Vec::load(static_cast<const T*>(a.residual) + row * a.residual_stride + c);
        }
    };
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    Held next;
    if constexpr (kAhead) load(static_cast<long long>(blockIdx.x) * per_block + threadIdx.x / group, next);
    for (long long start = static_cast<long long>(blockIdx.x) * per_block; start < a.rows; start += step) {
        const long long row = start + threadIdx.x / group;
        const bool live = row < active;
        Held held;
        if constexpr (kAhead) {
            held = next;
            load(row + step, next);
        } else {
            load(row, held);
        }
        float u[K][V], h[K][V];
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                u[k][j] = held.part[k].at(j);
                h[k][j] = held.rest[k].at(j);
            }
        }
        RowStatistics post{0.0f, 0.0f, 0.0f};
        if constexpr (POST) {
            post = row_statistics<V, K>(u, channels, first, stride, group, a.rms, a.eps, shared);
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    u[k][j] = post.away(u[k][j]) * post.root * post_w[k].at(j) + post_b[k].at(j);
            }
        }
        Vec out[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool here = live && first + k * stride < channels;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                out[k].set(j, here ? h[k][j] + a.scale * gate[k].at(j) * u[k][j] : 0.0f);
                h[k][j] = out[k].at(j);
            }
        }
        const RowStatistics stat = row_statistics<V, K>(h, channels, first, stride, group, a.rms, a.eps, shared);
        if (row >= a.rows) continue;
        if (statistics && lane == 0)
            statistics[row] = live ? float4{stat.mean(), stat.root, post.mean(), post.root}
                                   : float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = first + k * stride;
            if (c >= channels) continue;
            out[k].store(sum + row * channels + c);
#pragma unroll
            for (int j = 0; j < V; ++j)
                out[k].set(j, live ? stat.away(h[k][j]) * stat.root * w[k].at(j) + b[k].at(j) : 0.0f);
            out[k].store(normed + row * channels + c);
        }
    }
}

// One value of the junction, for rows that no block holds.
template <typename T, bool POST>
struct JoinChannel {
    float w, b, gate, post_w, post_b;
    __device__ static float of(const void* from, int c, float value) {
        return from ? static_cast<float>(static_cast<const T*>(from)[c]) : value;
    }
    __device__ JoinChannel(const lattice_residual_norm& a, int c)
        : w(of(a.weight, c, 1.0f)),
          b(of(a.bias, c, 0.0f)),
          gate(of(a.gate, c, 1.0f)),
          post_w(POST ? of(a.post_weight, c, 1.0f) : 1.0f),
          post_b(POST ? of(a.post_bias, c, 0.0f) : 0.0f) {}
    // u of x.
    __device__ float part(float x, float2 post) const {
        return POST ? (x - post.x) * post.y * post_w + post_b : x;
    }
};

// Statistics of a row of memory.
template <typename T>
__device__ inline float2 wide_statistics(const T* row, int channels, bool rms, float eps, float* shared) {
    const float inv = 1.0f / static_cast<float>(channels);
    float mean = 0.0f;
    if (!rms) {
        float sum = 0.0f;
        for (int c = threadIdx.x; c < channels; c += kJoinBlock) sum += static_cast<float>(row[c]);
        mean = row_sum(sum, kJoinBlock, shared) * inv;
    }
    float square = 0.0f;
    for (int c = threadIdx.x; c < channels; c += kJoinBlock) {
        const float away = static_cast<float>(row[c]) - mean;
        square += away * away;
    }
    return float2{mean, 1.0f / sqrtf(row_sum(square, kJoinBlock, shared) * inv + eps)};
}

// A block a row; a thread reads of `sum` only what it wrote itself.
template <typename T, bool POST>
__global__ void __launch_bounds__(kJoinBlock)
residual_norm_wide(lattice_residual_norm a, T* sum, T* __restrict__ normed, float4* __restrict__ statistics) {
    __shared__ float shared[kJoinBlock / kWave];
    const int active = active_count(a), channels = a.channels;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const bool live = row < active;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* residual = static_cast<const T*>(a.residual) + row * a.residual_stride;
        T *h = sum + row * channels, *y = normed + row * channels;
        float2 post{0.0f, 0.0f}, stat{0.0f, 0.0f};
        if (live) {
            if constexpr (POST) post = wide_statistics(x, channels, a.rms, a.eps, shared);
            for (int c = threadIdx.x; c < channels; c += kJoinBlock) {
                const JoinChannel<T, POST> at(a, c);
                h[c] = static_cast<T>(static_cast<float>(residual[c]) +
                                      a.scale * at.gate * at.part(static_cast<float>(x[c]), post));
            }
            stat = wide_statistics(static_cast<const T*>(h), channels, a.rms, a.eps, shared);
        }
        if (statistics && threadIdx.x == 0) statistics[row] = float4{stat.x, stat.y, post.x, post.y};
        for (int c = threadIdx.x; c < channels; c += kJoinBlock) {
            const JoinChannel<T, POST> at(a, c);
            if (!live) h[c] = static_cast<T>(0.0f);
            y[c] = static_cast<T>(live ? (static_cast<float>(h[c]) - stat.x) * stat.y * at.w + at.b : 0.0f);
        }
    }
}

// grad_x and grad_residual, and this block's sums over its rows in
// partials[block][kJoinSums][channels] (NULL: none are wanted).
template <typename T, int V, int K, int BLOCK, bool POST>
__global__ void __launch_bounds__(BLOCK)
residual_norm_grad_rows(lattice_residual_norm a, JoinGrads g, int group, const float4* __restrict__ statistics,
                        float* __restrict__ partials) {
    typedef RowVec<T, V> Vec;
    constexpr int kSums = POST ? 5 : 3;
    __shared__ float2 shared[BLOCK / kWave];
    __shared__ float columns[V * BLOCK];
    const int active = active_count(a), channels = a.channels;
    const int lane = threadIdx.x & (group - 1), first = lane * V, stride = group * V;
    const int per_block = BLOCK / group;
    const float inv = 1.0f / static_cast<float>(channels);
    const bool reads_x = POST || g.vectors[2];
    Vec w[K], gate[K], post_w[K], post_b[K];
    float sums[kSums][K][V] = {};
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = first + k * stride;
        w[k] = vector_or<T, V>(a.weight, c, channels, 1.0f);
        gate[k] = vector_or<T, V>(a.gate, c, channels, 1.0f);
        if constexpr (POST) {
            post_w[k] = vector_or<T, V>(a.post_weight, c, channels, 1.0f);
            post_b[k] = vector_or<T, V>(a.post_bias, c, channels, 0.0f);
        }
    }
    // A row's vectors are read while the one before is computed, where registers
    // hold both.
    constexpr bool kAhead = K == 1;
    struct Held {
        float4 stat;
        Vec in[K], dy[K], dh[K], part[K];
    };
    const auto load = [&](long long row, Held& r) {
        const bool live = row < active;
        r.stat = live ? statistics[row] : float4{0.0f, 0.0f, 0.0f, 0.0f};
        const long long at = row * channels;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = first + k * stride;
            r.in[k] = r.dy[k] = r.dh[k] = r.part[k] = Vec{};
            if (!live || c >= channels) continue;
            r.in[k] = Vec::load(static_cast<const T*>(g.sum) + at + c);
            if (g.grad_normed) r.dy[k] = Vec::load(static_cast<const T*>(g.grad_normed) + at + c);
            if (g.grad_sum) r.dh[k] = Vec::load(static_cast<const T*>(g.grad_sum) + at + c);
            if (reads_x) r.part[k] = Vec::load(static_cast<const T*>(a.x) + row * a.x_stride + c);
        }
    };
    const long long step = static_cast<long long>(gridDim.x) * per_block;
    Held next;
    if constexpr (kAhead) load(static_cast<long long>(blockIdx.x) * per_block + threadIdx.x / group, next);
    for (long long start = static_cast<long long>(blockIdx.x) * per_block; start < a.rows; start += step) {
        const long long row = start + threadIdx.x / group;
        const bool live = row < active;
        Held held;
        if constexpr (kAhead) {
            held = next;
            load(row + step, next);
        } else {
            load(row, held);
        }
        const float4 stat = held.stat;
        const long long at = row * channels;
        float n[K][V], slope[K][V], t[K][V], m[K][V];
        float2 along{0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool here = live && first + k * stride < channels;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = held.dy[k].at(j);
                n[k][j] = here ? (held.in[k].at(j) - stat.x) * stat.y : 0.0f;
                t[k][j] = held.dh[k].at(j);
                m[k][j] = held.part[k].at(j);
                slope[k][j] = d * w[k].at(j);
                sums[0][k][j] += d * n[k][j];
                sums[1][k][j] += d;
                along.x += slope[k][j];
                along.y += slope[k][j] * n[k][j];
            }
        }
        along = row_sum(along, group, shared);
        if (a.rms) along.x = 0.0f;
        float2 back{0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const bool here = live && first + k * stride < channels;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                t[k][j] += here ? stat.y * (slope[k][j] - along.x * inv - n[k][j] * (along.y * inv)) : 0.0f;
                if constexpr (POST) {
                    m[k][j] = here ? (m[k][j] - stat.z) * stat.w : 0.0f;
                    sums[2][k][j] += t[k][j] * (m[k][j] * post_w[k].at(j) + post_b[k].at(j));
                    const float du = a.scale * gate[k].at(j) * t[k][j];
                    sums[3][k][j] += du * m[k][j];
                    sums[4][k][j] += du;
                    slope[k][j] = du * post_w[k].at(j);
                    back.x += slope[k][j];
                    back.y += slope[k][j] * m[k][j];
                } else {
                    sums[2][k][j] += t[k][j] * m[k][j];
                    slope[k][j] = a.scale * gate[k].at(j) * t[k][j];
                }
            }
        }
        if constexpr (POST) {
            back = row_sum(back, group, shared);
            if (a.rms) back.x = 0.0f;
        }
        if (row >= a.rows) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = first + k * stride;
            if (c >= channels) continue;
            Vec dx, dr;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                dr.set(j, t[k][j]);
                dx.set(j, POST ? stat.w * (slope[k][j] - back.x * inv - m[k][j] * (back.y * inv)) : slope[k][j]);
            }
            dr.store(static_cast<T*>(g.grad_residual) + at + c);
            dx.store(static_cast<T*>(g.grad_x) + at + c);
        }
    }
    if (!partials) return;
    float* mine = partials + static_cast<long long>(blockIdx.x) * kJoinSums * channels;
#pragma unroll
    for (int which = 0; which < kSums; ++which) {
        if (!g.vectors[which]) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < V; ++j) columns[j * BLOCK + threadIdx.x] = sums[which][k][j];
            __syncthreads();
            // `columns` holds V rows of per_block groups.
            for (int i = threadIdx.x; i < V * group; i += BLOCK) {
                const int j = i / group, owner = i & (group - 1), c = (owner + k * group) * V + j;
                if (c >= channels) continue;
                float sum = 0.0f;
                for (int r = 0; r < per_block; ++r) sum += columns[j * BLOCK + r * group + owner];
                mine[which * static_cast<long long>(channels) + c] = sum;
            }
        }
    }
}

// A block a row, in passes; keeps the means that its sums take, for the vectors'
// gradients: (mean g, mean g n, mean k, mean k m).
template <typename T, bool POST>
__global__ void __launch_bounds__(kJoinBlock)
residual_norm_grad_wide(lattice_residual_norm a, JoinGrads g, const float4* __restrict__ statistics,
                        float2* __restrict__ means) {
    __shared__ float2 shared[kJoinBlock / kWave];
    const int active = active_count(a), channels = a.channels;
    const float inv = 1.0f / static_cast<float>(channels);
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const bool live = row < active;
        const float4 stat = statistics[row];
        const float2 post{stat.z, stat.w};
        const long long at = row * channels;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const T* h = static_cast<const T*>(g.sum) + at;
        const T* dy = g.grad_normed ? static_cast<const T*>(g.grad_normed) + at : nullptr;
        const T* dh = g.grad_sum ? static_cast<const T*>(g.grad_sum) + at : nullptr;
        T *dx = static_cast<T*>(g.grad_x) + at, *dr = static_cast<T*>(g.grad_residual) + at;
        float2 along{0.0f, 0.0f}, back{0.0f, 0.0f};
        if (live && dy) {
            for (int c = threadIdx.x; c < channels; c += kJoinBlock) {
                const float slope = static_cast<float>(dy[c]) * JoinChannel<T, POST>(a, c).w;
                along.x += slope;
                along.y += slope * ((static_cast<float>(h[c]) - stat.x) * stat.y);
            }
            along = row_sum(along, kJoinBlock, shared);
        }
        along = a.rms ? float2{0.0f, along.y * inv} : float2{along.x * inv, along.y * inv};
        if (means && threadIdx.x == 0) means[row] = along;
        const auto stream = [&](const JoinChannel<T, POST>& v, int c) {
            const float n = (static_cast<float>(h[c]) - stat.x) * stat.y;
            const float slope = dy ? static_cast<float>(dy[c]) * v.w : 0.0f;
            return (dh ? static_cast<float>(dh[c]) : 0.0f) + stat.y * (slope - along.x - n * along.y);
        };
        if (POST && live) {
            for (int c = threadIdx.x; c < channels; c += kJoinBlock) {
                const JoinChannel<T, POST> v(a, c);
                const float slope = a.scale * v.gate * stream(v, c) * v.post_w;
                back.x += slope;
                back.y += slope * ((static_cast<float>(x[c]) - post.x) * post.y);
            }
            back = row_sum(back, kJoinBlock, shared);
            back = a.rms ? float2{0.0f, back.y * inv} : float2{back.x * inv, back.y * inv};
        }
        for (int c = threadIdx.x; c < channels; c += kJoinBlock) {
            const JoinChannel<T, POST> v(a, c);
            const float t = live ? stream(v, c) : 0.0f;
            float slope = a.scale * v.gate * t;
            if (POST && live)
                slope = post.y * (slope * v.post_w - back.x - (static_cast<float>(x[c]) - post.x) * post.y * back.y);
            dr[c] = static_cast<T>(t);
            dx[c] = static_cast<T>(slope);
        }
    }
}

// The vectors' sums of wide rows: a thread a channel, a grid row a share of the
// rows.
template <typename T, bool POST>
__global__ void __launch_bounds__(kJoinBlock)
residual_norm_grad_columns(lattice_residual_norm a, JoinGrads g, const float4* __restrict__ statistics,
                           const float2* __restrict__ means, float* __restrict__ partials) {
    const int active = active_count(a), channels = a.channels;
    const int c = blockIdx.x * kJoinBlock + threadIdx.x;
    if (c >= channels) return;
    const JoinChannel<T, POST> v(a, c);
    const bool reads_x = POST || g.vectors[2];
    float sums[kJoinSums] = {};
    for (long long row = blockIdx.y; row < active; row += gridDim.y) {
        const float4 stat = statistics[row];
        const float2 along = means[row];
        const long long at = row * channels + c;
        const float n = (static_cast<float>(static_cast<const T*>(g.sum)[at]) - stat.x) * stat.y;
        const float dy = g.grad_normed ? static_cast<float>(static_cast<const T*>(g.grad_normed)[at]) : 0.0f;
        const float dh = g.grad_sum ? static_cast<float>(static_cast<const T*>(g.grad_sum)[at]) : 0.0f;
        const float x = reads_x ? static_cast<float>(static_cast<const T*>(a.x)[row * a.x_stride + c]) : 0.0f;
        const float t = dh + stat.y * (dy * v.w - along.x - n * along.y);
        const float du = a.scale * v.gate * t;
        sums[0] += dy * n;
        sums[1] += dy;
        sums[2] += t * v.part(x, float2{stat.z, stat.w});
        sums[3] += POST ? du * ((x - stat.z) * stat.w) : 0.0f;
        sums[4] += POST ? du : 0.0f;
    }
    float* mine = partials + static_cast<long long>(blockIdx.y) * kJoinSums * channels;
#pragma unroll
    for (int which = 0; which < (POST ? 5 : 3); ++which)
        if (g.vectors[which]) mine[which * static_cast<long long>(channels) + c] = sums[which];
}

// partials [count][kJoinSums][channels] -> the vectors' gradients: 16 columns a
// block, 64 slices of the partials added in slice order.
constexpr int kFinishBlock = 1024, kFinishSlices = kFinishBlock / 16;
template <typename T>
__global__ void __launch_bounds__(kFinishBlock)
residual_norm_grad_finish(const float* __restrict__ partials, int count, int channels, float scale, JoinGrads g) {
    __shared__ float shared[kFinishSlices][17];
    const int at = threadIdx.x & 15, slice = threadIdx.x >> 4;
    T* out = static_cast<T*>(g.vectors[blockIdx.y]);
    if (!out) return;
    const long long row = static_cast<long long>(kJoinSums) * channels;
    for (long long first = blockIdx.x * 16ll; first < channels; first += gridDim.x * 16ll) {
        const long long c = first + at;
        float sum = 0.0f;
        if (c < channels) {
            const float* column = partials + blockIdx.y * static_cast<long long>(channels) + c;
            // Four chains of additions keep four reads in flight.
            float chain[4] = {};
            int i = slice;
            for (; i + 3 * kFinishSlices < count; i += 4 * kFinishSlices) {
#pragma unroll
                for (int u = 0; u < 4; ++u) chain[u] += column[(i + kFinishSlices * u) * row];
            }
            for (; i < count; i += kFinishSlices) chain[0] += column[i * row];
            sum = (chain[0] + chain[1]) + (chain[2] + chain[3]);
        }
        shared[slice][at] = sum;
        __syncthreads();
        if (slice == 0 && c < channels) {
            for (int s = 1; s < kFinishSlices; ++s) sum += shared[s][at];
            out[c] = static_cast<T>(blockIdx.y == 2 ? sum * scale : sum);
        }
        __syncthreads();
    }
}

// Threads a row and vectors a thread for rows of `vectors` vectors.
struct JoinShape {
    int group, held;  // held 0: rows that no block holds
    int block() const { return std::max(group, kJoinBlock); }
};
inline JoinShape join_shape(int vectors) {
    if (vectors > kJoinWidest * kJoinHeld) return {kJoinBlock, 0};
    int group = 1;
    while (group < vectors && group < kJoinWidest) group *= 2;
    return {group, (vectors + group - 1) / group};
}

// Vectors of 16, 4 and one element's bytes are instantiated.
template <typename T>
int join_vector(const lattice_residual_norm& a, std::initializer_list<const void*> more) {
    int v = row_vector<T>(a.channels, {a.x, a.residual, a.weight, a.bias, a.gate, a.post_weight, a.post_bias},
                          {a.x_stride, a.residual_stride});
    v = std::min(v, row_vector<T>(a.channels, more, {}));
    const int most = 16 / static_cast<int>(sizeof(T)), word = 4 / static_cast<int>(sizeof(T));
    return v == most ? v : v >= word ? word : 1;
}

// Blocks of `threads` that sum the vectors' gradients, of `per_block` rows at a
// time: what is resident, more while their partial rows stay under half a
// million sums.  1024 channels in float32 take 121 us with 512 blocks and 126
// with 1024 (25000 rows), 2048 in float16 134 with 512 and 216 with 256.  Rows
// that no block holds: two million sums, or 32 rows of them.
inline int join_partials(int rows, int channels, int per_block, int threads) {
    const long long blocks = (static_cast<long long>(rows) + per_block - 1) / per_block;
    const long long cap = channels > kJoinMost
                              ? std::max(32, (1 << 21) / channels)
                              : std::max(kJoinPartials / 2 * kJoinBlock / threads,
                                         std::min(kJoinPartials, (1 << 19) / channels));
    return static_cast<int>(std::max<long long>(1, std::min(blocks, cap)));
}

inline bool join_sums(const JoinGrads& g) {
    for (const void* v : g.vectors)
        if (v) return true;
    return false;
}

template <typename T, int V, bool POST>
int launch_join(const lattice_residual_norm& a, T* sum, T* normed, float4* statistics, hipStream_t stream) {
    const JoinShape shape = join_shape(a.channels / V);
    if (shape.held) {
        const auto kernel = shape.held == 2               ? residual_norm_rows<T, V, 2, kJoinWidest, POST>
                            : shape.group == kJoinWidest ? residual_norm_rows<T, V, 1, kJoinWidest, POST>
                                                         : residual_norm_rows<T, V, 1, kJoinBlock, POST>;
        kernel<<<grid_for(a.rows, shape.block() / shape.group, kJoinBlocks), shape.block(), 0, stream>>>(
            a, shape.group, sum, normed, statistics);
    } else {
        residual_norm_wide<T, POST><<<grid_for(a.rows, 1, 4096), kJoinBlock, 0, stream>>>(a, sum, normed, statistics);
    }
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

template <typename T, int V, bool POST>
int launch_join_grad(const lattice_residual_norm& a, const JoinGrads& g, const float4* statistics, float* partials,
                     float2* means, hipStream_t stream) {
    const JoinShape shape = join_shape(a.channels / V);
    const int per_block = shape.held ? shape.block() / shape.group : 1;
    const int blocks = join_partials(a.rows, a.channels, per_block, shape.held ? shape.block() : kJoinBlock);
    if (shape.held) {
        const auto kernel = shape.held == 2               ? residual_norm_grad_rows<T, V, 2, kJoinWidest, POST>
                            : shape.group == kJoinWidest ? residual_norm_grad_rows<T, V, 1, kJoinWidest, POST>
                                                         : residual_norm_grad_rows<T, V, 1, kJoinBlock, POST>;
        kernel<<<partials ? blocks : grid_for(a.rows, per_block, kJoinBlocks), shape.block(), 0, stream>>>(
            a, g, shape.group, statistics, partials);
    } else {
        residual_norm_grad_wide<T, POST>
            <<<grid_for(a.rows, 1, 4096), kJoinBlock, 0, stream>>>(a, g, statistics, partials ? means : nullptr);
        if (partials) {
            LATTICE_LAUNCH_CHECK();
            residual_norm_grad_columns<T, POST>
                <<<dim3((a.channels + kJoinBlock - 1) / kJoinBlock, blocks), kJoinBlock, 0, stream>>>(
                    a, g, statistics, means, partials);
        }
    }
    LATTICE_LAUNCH_CHECK();
    if (partials) {
        residual_norm_grad_finish<T><<<dim3(grid_for(a.channels, 16, 1u << 16), kJoinSums), kFinishBlock, 0, stream>>>(
            partials, blocks, a.channels, a.scale, g);
        LATTICE_LAUNCH_CHECK();
    }
    return LATTICE_OK;
}

template <typename T, int V>
int join_post(const lattice_residual_norm& a, T* sum, T* normed, float4* statistics, hipStream_t stream) {
    return a.post_norm ? launch_join<T, V, true>(a, sum, normed, statistics, stream)
                       : launch_join<T, V, false>(a, sum, normed, statistics, stream);
}
template <typename T>
int join_of(const lattice_residual_norm& a, void* sum, void* normed, float* statistics, hipStream_t stream) {
    T *h = static_cast<T*>(sum), *y = static_cast<T*>(normed);
    float4* stats = reinterpret_cast<float4*>(statistics);
    constexpr int kMost = 16 / sizeof(T), kWord = 4 / sizeof(T);
    const int v = join_vector<T>(a, {sum, normed});
    if (v == kMost) return join_post<T, kMost>(a, h, y, stats, stream);
    if constexpr (kWord > 1) {
        if (v == kWord) return join_post<T, kWord>(a, h, y, stats, stream);
    }
    return join_post<T, 1>(a, h, y, stats, stream);
}

template <typename T, int V>
int join_grad_post(const lattice_residual_norm& a, const JoinGrads& g, const float4* statistics, float* partials,
                   float2* means, hipStream_t stream) {
    return a.post_norm ? launch_join_grad<T, V, true>(a, g, statistics, partials, means, stream)
                       : launch_join_grad<T, V, false>(a, g, statistics, partials, means, stream);
}
template <typename T>
int join_grad_of(const lattice_residual_norm& a, const JoinGrads& g, const float* statistics, float* partials,
                 float2* means, hipStream_t stream) {
    const float4* stats = reinterpret_cast<const float4*>(statistics);
    constexpr int kMost = 16 / sizeof(T), kWord = 4 / sizeof(T);
    // What is not read does not count: not the residual nor the bias, x with the
    // first norm or for the gate.
    lattice_residual_norm read = a;
    read.residual = read.bias = nullptr;
    read.residual_stride = 0;
    if (!a.post_norm && !g.vectors[2]) {
        read.x = nullptr;
        read.x_stride = 0;
    }
    const int v = join_vector<T>(read, {g.sum, g.grad_sum, g.grad_normed, g.grad_x, g.grad_residual});
    if (v == kMost) return join_grad_post<T, kMost>(a, g, stats, partials, means, stream);
    if constexpr (kWord > 1) {
        if (v == kWord) return join_grad_post<T, kWord>(a, g, stats, partials, means, stream);
    }
    return join_grad_post<T, 1>(a, g, stats, partials, means, stream);
}

// What every entry checks; NULL, or what is wrong.
const char* join_fault(const lattice_residual_norm* a) {
    if (!a) return "residual norm arguments must be non-null.";
    if (a->dtype != LATTICE_F32 && a->dtype != LATTICE_F16 && a->dtype != LATTICE_BF16)
        return "residual norm supports float32, float16 and bfloat16.";
    if (a->rows < 0 || a->channels < 1 || a->x_stride < 0 || a->residual_stride < 0)
        return "residual norm shapes must be positive.";
    // A launch takes fewer than 2^32 threads.
    if (a->channels >= 1 << 26) return "residual norm takes up to 2^26 - 1 channels.";
    if (!(a->eps >= 0.0f)) return "eps must be non-negative.";
    if (a->rows > 0 && (!a->x || !a->residual)) return "residual norm pointers must be non-null.";
    return nullptr;
}

// No rows: the vectors' gradients are zero.
template <typename T>
int join_grad_empty(const lattice_residual_norm& a, const JoinGrads& g, hipStream_t stream) {
    residual_norm_grad_finish<T><<<dim3(grid_for(a.channels, 16, 1u << 16), kJoinSums), kFinishBlock, 0, stream>>>(
        nullptr, 0, a.channels, 0.0f, g);
    LATTICE_LAUNCH_CHECK();
    return LATTICE_OK;
}

}  // namespace
}  // namespace lattice

using namespace lattice;

#define LATTICE_REQUIRE_JOIN(args)                   \
    do {                                             \
        if (const char* fault_ = join_fault(args)) { \
            set_error(fault_);                       \
            return LATTICE_ERROR_INVALID_ARGUMENT;   \
        }                                            \
    } while (0)

extern "C" int lattice_hip_residual_norm(const lattice_residual_norm* args, void* sum, void* normed,
                                         float* statistics, void* stream_ptr) {
    LATTICE_REQUIRE_JOIN(args);
    if (args->rows == 0) return LATTICE_OK;
    LATTICE_REQUIRE(sum && normed, "residual norm pointers must be non-null.");
    LATTICE_REQUIRE(reinterpret_cast<uintptr_t>(statistics) % 16 == 0,
                    "residual norm statistics must lie on 16-byte boundaries.");
    hipStream_t stream = as_stream(stream_ptr);
    if (args->dtype == LATTICE_F32) return join_of<float>(*args, sum, normed, statistics, stream);
    if (args->dtype == LATTICE_F16) return join_of<_Float16>(*args, sum, normed, statistics, stream);
    return join_of<__bf16>(*args, sum, normed, statistics, stream);
}

extern "C" size_t lattice_hip_residual_norm_grad_workspace_bytes(int rows, int channels) {
    if (rows <= 0 || channels <= 0) return 0;
    // The most blocks any vector width gives: one row a block.
    return aligned_bytes(static_cast<size_t>(join_partials(rows, channels, 1, kJoinBlock)) * kJoinSums * channels * sizeof(float)) +
           aligned_bytes(static_cast<size_t>(rows) * sizeof(float2));
}

extern "C" int lattice_hip_residual_norm_grad(const lattice_residual_norm* args, const void* sum,
                                              const float* statistics, const void* grad_sum, const void* grad_normed,
                                              void* grad_x, void* grad_residual, void* grad_weight, void* grad_bias,
                                              void* grad_gate, void* grad_post_weight, void* grad_post_bias,
                                              void* workspace, size_t workspace_bytes, void* stream_ptr) {
    LATTICE_REQUIRE_JOIN(args);
    const JoinGrads g{sum, grad_sum, grad_normed, grad_x, grad_residual,
                      {grad_weight, grad_bias, grad_gate, grad_post_weight, grad_post_bias}};
    LATTICE_REQUIRE(args->rows == 0 || (sum && statistics && grad_x && grad_residual),
                    "residual norm pointers must be non-null.");
    LATTICE_REQUIRE(reinterpret_cast<uintptr_t>(statistics) % 16 == 0,
                    "residual norm statistics must lie on 16-byte boundaries.");
    LATTICE_REQUIRE(args->post_norm || (!grad_post_weight && !grad_post_bias),
                    "without post_norm there are no gradients of its vectors.");
    hipStream_t stream = as_stream(stream_ptr);
    if (args->rows == 0) {
        if (!join_sums(g)) return LATTICE_OK;
        // Zero has the same bits in both 16-bit types.
        return args->dtype == LATTICE_F32 ? join_grad_empty<float>(*args, g, stream)
                                          : join_grad_empty<_Float16>(*args, g, stream);
    }
    float* partials = nullptr;
    float2* means = nullptr;
    if (join_sums(g)) {
        Workspace ws{static_cast<char*>(workspace), workspace ? workspace_bytes : 0};
        partials = ws.take<float>(static_cast<size_t>(join_partials(args->rows, args->channels, 1, kJoinBlock)) * kJoinSums *
                                  args->channels);
        means = ws.take<float2>(args->rows);
        LATTICE_REQUIRE(partials && means, "residual norm gradient workspace is too small.");
    }
    if (args->dtype == LATTICE_F32) return join_grad_of<float>(*args, g, statistics, partials, means, stream);
    if (args->dtype == LATTICE_F16) return join_grad_of<_Float16>(*args, g, statistics, partials, means, stream);
    return join_grad_of<__bf16>(*args, g, statistics, partials, means, stream);
}
