// Group norm with an activation over channels-last features, with means over the positions and the channels of a sample's group:
//     h = (x - mean) r,  r = (mean((x - mean)^2) + eps)^-1/2;   z = h w + b + residual;   y = act(z)
// and the gradient, with dz = dy act'(z):
//     dw = sum dz h,  db = sum dz,  dresidual = dz;   dx = r (dz w - mean(dz w) - h mean(dz w h))
//
// A thread has a vector of channels (16 bytes where the rows allow it) and walks positions, so that the loads of a warp lie next to one
// another and its sums are those of fixed channels.  Variances are sums of squares about the thread's first element, joined over threads
// as n_i (mean_i - mean)^2 + M_i: no difference of large numbers, however far the mean is from zero.
//
// Samples that fit a CTA's shared memory are read once (`held`): CTAs walk over samples.  Larger ones take two passes, the second of
// which finds in L2 what the first has left there; it runs from the end backwards.
#include <algorithm>

#include "seq_common.cuh"

namespace dcn {
namespace seq {
namespace {

constexpr int64_t kMostChannels = 8192;
constexpr int kHeldBytes = 96 * 1024;            // of a sample's tensors, so that two CTAs share an SM

struct GnormArgs {
    const void *x, *weight, *bias, *residual, *dy;
    void *y, *dx, *dresidual;
    float *stats;                                // [samples][groups][2]
    float *partial;                              // forward [samples][splits][groups][2], backward [samples][splits][channels][2]
    float *sums;                                 // backward [samples][groups][2]
    int64_t samples, positions, split_positions;
    int channels, groups, per_group, vectors, act, wide_weights, splits;
    float eps, inv;                              // 1 / elements of a group
};

template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int c, int wide, float none) {
    if (w == nullptr) return none;
    if (wide) {
        Pack<float, 1> p;
        p.get(static_cast<const float*>(w) + c);
        return p.at(0);
    }
    Pack<T, 1> p;
    p.get(static_cast<const T*>(w) + c);
    return p.at(0);
}

__device__ __forceinline__ float activate(float z, int act) {
    if (act == DCN_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (act == DCN_ACT_SILU) {
        float s, rest;
        logistic(z, s, rest);
        return z * s;
    }
    return z;
}
__device__ __forceinline__ float activate_gradient(float z, float dy, int act) {
    if (act == DCN_ACT_RELU) return z > 0.0f ? dy : (z != z ? z : 0.0f);
    if (act == DCN_ACT_SILU) {
        float s, rest;
        logistic(z, s, rest);
        return dy * (s * fmaf(z, rest, 1.0f));
    }
    return dy;
}

// How the vectors of a row of channels lie over the threads: rows of threads where a row of vectors is shorter than the CTA, blocks of
// columns where it is longer.
struct Grid {
    int rows, row, col, blocks;                  // row -1: no part
    __device__ __forceinline__ Grid(int vectors) {
        const int n = blockDim.x;
        if (vectors <= n) {
            rows = n / vectors, row = threadIdx.x / vectors, col = threadIdx.x % vectors, blocks = 1;
            if (row >= rows) row = -1;
        } else {
            rows = 1, row = 0, col = threadIdx.x, blocks = (vectors + n - 1) / n;
        }
    }
};

// Mean and sum of squares about it from `n` entries (count, mean, sum) of which a warp reads e, e + 32, ...
template <typename F>
__device__ __forceinline__ void join(int n, F&& entry, float& mean, float& sq, float& count) {
    const int lane = threadIdx.x & 31;
    float c = 0.0f, s = 0.0f;
    for (int i = lane; i < n; i += 32) {
        float ci, mi, qi;
        entry(i, ci, mi, qi);
        c += ci, s = fmaf(ci, mi, s);
    }
    count = warp_sum(c);
    mean = count > 0.0f ? warp_sum(s) / count : 0.0f;
    float q = 0.0f;
    for (int i = lane; i < n; i += 32) {
        float ci, mi, qi;
        entry(i, ci, mi, qi);
        const float d = mi - mean;
        q += ci > 0.0f ? fmaf(ci * d, d, qi) : 0.0f;
    }
    sq = warp_sum(q);
}

// Sums of one thread's column over its positions, from its first element on
template <int V>
struct Moments {
    float first[V], s[V], q[V];
    int n = 0;
    template <typename T>
    __device__ __forceinline__ void add(const Pack<T, V>& p) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float v = p.at(e);
            if (n == 0) first[e] = v, s[e] = 0.0f, q[e] = 0.0f;
            const float d = v - first[e];
            s[e] += d, q[e] = fmaf(d, d, q[e]);
        }
        ++n;
    }
    __device__ __forceinline__ void put(float* mean, float* sq, float& count) const {
        count = (float)n;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float m = n > 0 ? s[e] / (float)n : 0.0f;
            mean[e] = n > 0 ? first[e] + m : 0.0f;
            sq[e] = n > 0 ? fmaxf(q[e] - s[e] * m, 0.0f) : 0.0f;
        }
    }
};

// Means and sums of every group from the threads' own ones in shared memory: entries [row][channel]
__device__ __forceinline__ void join_groups(const GnormArgs& a, int rows, const float* counts, const float* means, const float* sqs,
                                            float* out, bool finish) {
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    for (int g = warp; g < a.groups; g += warps) {
        float mean, sq, count;
        join(rows * a.per_group, [&](int i, float& c, float& m, float& q) {
            const int r = i / a.per_group, ch = g * a.per_group + i % a.per_group;
            c = counts[r], m = means[r * a.channels + ch], q = sqs[r * a.channels + ch];
        }, mean, sq, count);
        if ((threadIdx.x & 31) == 0) {
            out[2 * g] = mean;
            out[2 * g + 1] = finish ? rsqrtf(fmaf(sq, a.inv, a.eps)) : sq;
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void apply_vector(const GnormArgs& a, const Pack<T, V>& x, int64_t at, int c0, const float* stats) {
    Pack<T, V> res, y;
    if (a.residual != nullptr) res.get(static_cast<const T*>(a.residual) + at);
    float f[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = c0 + e, g = c / a.per_group;
        const float h = (x.at(e) - stats[2 * g]) * stats[2 * g + 1];
        float z = fmaf(h, weight_at<T>(a.weight, c, a.wide_weights, 1.0f), weight_at<T>(a.bias, c, a.wide_weights, 0.0f));
        if (a.residual != nullptr) z += res.at(e);
        f[e] = activate(z, a.act);
    }
    y.set(f);
    y.put(static_cast<T*>(a.y) + at);
}

// ---- samples that a CTA holds ---------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_held_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    const int mine = (int)((a.positions + grid.rows - 1) / grid.rows) * grid.blocks;     // vectors of a thread
    Raw<sizeof(T) * V>* const held = reinterpret_cast<Raw<sizeof(T) * V>*>(smem);
    float* const means = reinterpret_cast<float*>(smem + ((size_t)mine * blockDim.x * sizeof(T) * V + 15) / 16 * 16);
    float* const sqs = means + grid.rows * a.channels;
    float* const stats = sqs + grid.rows * a.channels;
    float* const counts = stats + 2 * a.groups;
    pdl_wait();
    for (int64_t sample = blockIdx.x; sample < a.samples; sample += gridDim.x) {
        const int64_t base = sample * a.positions * a.channels;
        int k = 0;
        for (int b = 0; b < grid.blocks; ++b) {
            const int col = grid.col + b * blockDim.x;
            if (grid.row < 0 || col >= a.vectors) continue;
            Moments<V> m;
            for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                Pack<T, V> x;
                x.get(static_cast<const T*>(a.x) + base + p * a.channels + col * V);
                m.add(x);
                held[(size_t)k * blockDim.x + threadIdx.x] = x.raw;
            }
            float mean[V], sq[V], count;
            m.put(mean, sq, count);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                means[grid.row * a.channels + col * V + e] = mean[e];
                sqs[grid.row * a.channels + col * V + e] = sq[e];
            }
            if (col == 0) counts[grid.row] = count;
        }
        __syncthreads();
        join_groups(a, grid.rows, counts, means, sqs, stats, true);
        __syncthreads();
        if (a.stats != nullptr)
            for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) a.stats[sample * 2 * a.groups + i] = stats[i];
        k = 0;
        for (int b = 0; b < grid.blocks; ++b) {
            const int col = grid.col + b * blockDim.x;
            if (grid.row < 0 || col >= a.vectors) continue;
            for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                Pack<T, V> x;
                x.raw = held[(size_t)k * blockDim.x + threadIdx.x];
                apply_vector<T, V>(a, x, base + p * a.channels + col * V, col * V, stats);
            }
        }
        __syncthreads();
    }
}

// ---- two passes -----------------------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_sums_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    float* const means = reinterpret_cast<float*>(smem);
    float* const sqs = means + grid.rows * a.channels;
    float* const counts = sqs + grid.rows * a.channels;
    pdl_wait();
    const int64_t sample = blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    const T* const x = static_cast<const T*>(a.x) + sample * a.positions * a.channels;
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x;
        if (grid.row < 0 || col >= a.vectors) continue;
        Moments<V> m;
        int64_t p = begin + grid.row;
        for (; p + 3 * grid.rows < end; p += 4 * grid.rows) {
            Pack<T, V> v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i].get(x + (p + i * grid.rows) * a.channels + col * V);
#pragma unroll
            for (int i = 0; i < 4; ++i) m.add(v[i]);
        }
        for (; p < end; p += grid.rows) {
            Pack<T, V> v;
            v.get(x + p * a.channels + col * V);
            m.add(v);
        }
        float mean[V], sq[V], count;
        m.put(mean, sq, count);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            means[grid.row * a.channels + col * V + e] = mean[e];
            sqs[grid.row * a.channels + col * V + e] = sq[e];
        }
        if (col == 0) counts[grid.row] = count;
    }
    __syncthreads();
    join_groups(a, grid.rows, counts, means, sqs, a.partial + (int64_t)blockIdx.x * 2 * a.groups, false);
}

template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_apply_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    float* const stats = reinterpret_cast<float*>(smem);
    const Grid grid(a.vectors);
    const int64_t block = gridDim.x - 1 - blockIdx.x, sample = block / a.splits;
    const int split = (int)(block % a.splits);
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    pdl_wait();
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    const float* const partial = a.partial + sample * a.splits * 2 * a.groups;
    for (int g = warp; g < a.groups; g += warps) {
        float mean, sq, count;
        join(a.splits, [&](int i, float& c, float& m, float& q) {
            const int64_t from = i * a.split_positions;
            c = (float)((min(from + a.split_positions, a.positions) - from) * a.per_group);
            m = gload(partial + (int64_t)i * 2 * a.groups + 2 * g), q = gload(partial + (int64_t)i * 2 * a.groups + 2 * g + 1);
        }, mean, sq, count);
        if ((threadIdx.x & 31) == 0) stats[2 * g] = mean, stats[2 * g + 1] = rsqrtf(fmaf(sq, a.inv, a.eps));
    }
    __syncthreads();
    if (a.stats != nullptr && split == 0)
        for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) a.stats[sample * 2 * a.groups + i] = stats[i];
    const int64_t base = sample * a.positions * a.channels;
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x;
        if (grid.row < 0 || col >= a.vectors) continue;
        for (int64_t p = begin + grid.row; p < end; p += grid.rows) {
            Pack<T, V> x;
            x.get(static_cast<const T*>(a.x) + base + p * a.channels + col * V);
            apply_vector<T, V>(a, x, base + p * a.channels + col * V, col * V, stats);
        }
    }
}

// ---- gradients ------------------------------------------------------------------------------------------------------------
// dz and h of a vector
template <typename T, int V>
__device__ __forceinline__ void gradients_of(const GnormArgs& a, const Pack<T, V>& x, const Pack<T, V>& dy, const Pack<T, V>& res, int c0,
                                             const float* stats, float (&dz)[V], float (&h)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = c0 + e, g = c / a.per_group;
        h[e] = (x.at(e) - stats[2 * g]) * stats[2 * g + 1];
        float z = fmaf(h[e], weight_at<T>(a.weight, c, a.wide_weights, 1.0f), weight_at<T>(a.bias, c, a.wide_weights, 0.0f));
        if (a.residual != nullptr) z += res.at(e);
        dz[e] = activate_gradient(z, dy.at(e), a.act);
    }
}

template <typename T, int V>
struct Loads {
    Pack<T, V> x, dy, res;
    __device__ __forceinline__ void get(const GnormArgs& a, int64_t at) {
        x.get(static_cast<const T*>(a.x) + at);
        dy.get(static_cast<const T*>(a.dy) + at);
        if (a.residual != nullptr) res.get(static_cast<const T*>(a.residual) + at);
    }
};

template <typename T, int V>
__device__ __forceinline__ void put_gradients(const GnormArgs& a, const Loads<T, V>& v, int64_t at, int c0, const float* stats,
                                              const float* sums) {
    float dz[V], h[V], dx[V];
    gradients_of<T, V>(a, v.x, v.dy, v.res, c0, stats, dz, h);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = c0 + e, g = c / a.per_group;
        const float dh = dz[e] * weight_at<T>(a.weight, c, a.wide_weights, 1.0f);
        dx[e] = stats[2 * g + 1] * (dh - sums[2 * g] * a.inv - h[e] * (sums[2 * g + 1] * a.inv));
    }
    Pack<T, V> o;
    if (a.dx != nullptr) o.set(dx), o.put(static_cast<T*>(a.dx) + at);
    if (a.dresidual != nullptr) o.set(dz), o.put(static_cast<T*>(a.dresidual) + at);
}

// Channels' sums of dz and dz h over the rows of threads, from shared memory [row][channel][2], to `out` [channel][2], and the groups'
// sums of them times w to `sums` [group][2] (may be null)
template <typename T>
__device__ __forceinline__ void join_channels(const GnormArgs& a, int rows, float* entries, float* out, bool add, float* sums) {
    for (int i = threadIdx.x; i < 2 * a.channels; i += blockDim.x) {
        float s = 0.0f;
        for (int r = 0; r < rows; ++r) s += entries[r * 2 * a.channels + i];
        entries[i] = s;
        if (out != nullptr) out[i] = add ? out[i] + s : s;
    }
    if (sums == nullptr) return;
    __syncthreads();
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    for (int g = warp; g < a.groups; g += warps) {
        float s = 0.0f, q = 0.0f;
        for (int i = threadIdx.x & 31; i < a.per_group; i += 32) {
            const int c = g * a.per_group + i;
            const float w = weight_at<T>(a.weight, c, a.wide_weights, 1.0f);
            s = fmaf(entries[2 * c], w, s), q = fmaf(entries[2 * c + 1], w, q);
        }
        s = warp_sum(s), q = warp_sum(q);
        if ((threadIdx.x & 31) == 0) sums[2 * g] = s, sums[2 * g + 1] = q;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_held_backward_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    const int mine = (int)((a.positions + grid.rows - 1) / grid.rows) * grid.blocks;
    const int kinds = a.residual != nullptr ? 3 : 2;
    Raw<sizeof(T) * V>* const held = reinterpret_cast<Raw<sizeof(T) * V>*>(smem);
    float* const entries = reinterpret_cast<float*>(smem + ((size_t)mine * kinds * blockDim.x * sizeof(T) * V + 15) / 16 * 16);
    float* const stats = entries + grid.rows * 2 * a.channels;
    float* const sums = stats + 2 * a.groups;
    float* const total = sums + 2 * a.groups;    // [channels][2] of all the CTA's samples
    for (int i = threadIdx.x; i < 2 * a.channels; i += blockDim.x) total[i] = 0.0f;
    pdl_wait();
    for (int64_t sample = blockIdx.x; sample < a.samples; sample += gridDim.x) {
        const int64_t base = sample * a.positions * a.channels;
        for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) stats[i] = gload(a.stats + sample * 2 * a.groups + i);
        __syncthreads();
        int k = 0;
        for (int b = 0; b < grid.blocks; ++b) {
            const int col = grid.col + b * blockDim.x;
            if (grid.row < 0 || col >= a.vectors) continue;
            float s[V] = {}, q[V] = {};
            for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                Loads<T, V> v;
                v.get(a, base + p * a.channels + col * V);
                float dz[V], h[V];
                gradients_of<T, V>(a, v.x, v.dy, v.res, col * V, stats, dz, h);
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] += dz[e], q[e] = fmaf(dz[e], h[e], q[e]);
                held[(size_t)(kinds * k) * blockDim.x + threadIdx.x] = v.x.raw;
                held[(size_t)(kinds * k + 1) * blockDim.x + threadIdx.x] = v.dy.raw;
                if (kinds == 3) held[(size_t)(kinds * k + 2) * blockDim.x + threadIdx.x] = v.res.raw;
            }
#pragma unroll
            for (int e = 0; e < V; ++e) {
                entries[(grid.row * a.channels + col * V + e) * 2] = s[e];
                entries[(grid.row * a.channels + col * V + e) * 2 + 1] = q[e];
            }
        }
        __syncthreads();
        join_channels<T>(a, grid.rows, entries, total, true, sums);
        __syncthreads();
        k = 0;
        if (a.dx != nullptr || a.dresidual != nullptr)
            for (int b = 0; b < grid.blocks; ++b) {
                const int col = grid.col + b * blockDim.x;
                if (grid.row < 0 || col >= a.vectors) continue;
                for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                    Loads<T, V> v;
                    v.x.raw = held[(size_t)(kinds * k) * blockDim.x + threadIdx.x];
                    v.dy.raw = held[(size_t)(kinds * k + 1) * blockDim.x + threadIdx.x];
                    if (kinds == 3) v.res.raw = held[(size_t)(kinds * k + 2) * blockDim.x + threadIdx.x];
                    put_gradients<T, V>(a, v, base + p * a.channels + col * V, col * V, stats, sums);
                }
            }
        __syncthreads();
    }
    if (a.partial != nullptr)
        for (int i = threadIdx.x; i < 2 * a.channels; i += blockDim.x) a.partial[(int64_t)blockIdx.x * 2 * a.channels + i] = total[i];
}

template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_sums_backward_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    float* const entries = reinterpret_cast<float*>(smem);
    float* const stats = entries + grid.rows * 2 * a.channels;
    pdl_wait();
    const int64_t sample = blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    const int64_t base = sample * a.positions * a.channels;
    for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) stats[i] = gload(a.stats + sample * 2 * a.groups + i);
    __syncthreads();
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x;
        if (grid.row < 0 || col >= a.vectors) continue;
        float s[V] = {}, q[V] = {};
        for (int64_t p = begin + grid.row; p < end; p += grid.rows) {
            Loads<T, V> v;
            v.get(a, base + p * a.channels + col * V);
            float dz[V], h[V];
            gradients_of<T, V>(a, v.x, v.dy, v.res, col * V, stats, dz, h);
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += dz[e], q[e] = fmaf(dz[e], h[e], q[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            entries[(grid.row * a.channels + col * V + e) * 2] = s[e];
            entries[(grid.row * a.channels + col * V + e) * 2 + 1] = q[e];
        }
    }
    __syncthreads();
    join_channels<T>(a, grid.rows, entries, a.partial + (int64_t)blockIdx.x * 2 * a.channels, false, nullptr);
}

// A sample's group sums from its splits' channel sums
template <typename T>
__global__ void __launch_bounds__(256) gnorm_join_kernel(const GnormArgs a) {
    pdl_wait();
    const int64_t sample = blockIdx.x;
    const float* const partial = a.partial + sample * a.splits * 2 * a.channels;
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5;
    for (int g = blockIdx.y * warps + warp; g < a.groups; g += gridDim.y * warps) {
        float s = 0.0f, q = 0.0f;
        for (int i = threadIdx.x & 31; i < a.per_group * a.splits; i += 32) {
            const int c = g * a.per_group + i % a.per_group, split = i / a.per_group;
            const float w = weight_at<T>(a.weight, c, a.wide_weights, 1.0f);
            const float* const p = partial + ((int64_t)split * a.channels + c) * 2;
            s = fmaf(gload(p), w, s), q = fmaf(gload(p + 1), w, q);
        }
        s = warp_sum(s), q = warp_sum(q);
        if ((threadIdx.x & 31) == 0) a.sums[(sample * a.groups + g) * 2] = s, a.sums[(sample * a.groups + g) * 2 + 1] = q;
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_apply_backward_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    float* const stats = reinterpret_cast<float*>(smem);
    float* const sums = stats + 2 * a.groups;
    const Grid grid(a.vectors);
    const int64_t block = gridDim.x - 1 - blockIdx.x, sample = block / a.splits;
    const int split = (int)(block % a.splits);
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    pdl_wait();
    for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) {
        stats[i] = gload(a.stats + sample * 2 * a.groups + i);
        sums[i] = gload(a.sums + sample * 2 * a.groups + i);
    }
    __syncthreads();
    const int64_t base = sample * a.positions * a.channels;
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x;
        if (grid.row < 0 || col >= a.vectors) continue;
        for (int64_t p = begin + grid.row; p < end; p += grid.rows) {
            const int64_t at = base + p * a.channels + col * V;
            Loads<T, V> v;
            v.get(a, at);
            put_gradients<T, V>(a, v, at, col * V, stats, sums);
        }
    }
}

// dw and db: sums of n partial ones [n][channels][2], in a fixed order
template <typename T>
__global__ void __launch_bounds__(1024) gnorm_weights_kernel(const float* partial, int64_t n, int channels, void* dw, void* db, int wide) {
    __shared__ float s[32][33], q[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    pdl_wait();
    float a = 0.0f, b = 0.0f;
    if (c < channels)
        for (int64_t i = threadIdx.y; i < n; i += 32) a += gload(partial + (i * channels + c) * 2), b += gload(partial + (i * channels + c) * 2 + 1);
    s[threadIdx.x][threadIdx.y] = a, q[threadIdx.x][threadIdx.y] = b;
    __syncthreads();
    a = warp_sum(s[threadIdx.y][threadIdx.x]), b = warp_sum(q[threadIdx.y][threadIdx.x]);
    const int mine = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && mine < channels) {
        if (db != nullptr) {
            if (wide) static_cast<float*>(db)[mine] = a;
            else static_cast<T*>(db)[mine] = from_float<T>(a);
        }
        if (dw != nullptr) {
            if (wide) static_cast<float*>(dw)[mine] = b;
            else static_cast<T*>(dw)[mine] = from_float<T>(b);
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int check_gnorm(const dcn_gnorm* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype) || (p->weight_dtype != DCN_SEQ_F32 && p->weight_dtype != p->dtype) || p->act < DCN_ACT_NONE || p->act > DCN_ACT_SILU)
        return DCN_ERR_UNSUPPORTED;
    if (p->samples < 0 || p->positions < 0 || p->channels < 1 || p->groups < 1 || p->channels % p->groups != 0 || !(p->eps >= 0.0f))
        return DCN_ERR_SHAPE;
    if (p->channels > kMostChannels || p->samples >= 1ll << 31 || p->positions >= 1ll << 31) return DCN_ERR_LIMIT;
    if (p->samples > 0 && p->positions > (1ll << 62) / p->samples / p->channels) return DCN_ERR_LIMIT;
    return DCN_OK;
}

// How a call runs, by its sizes alone
struct Plan {
    int v;                                       // elements of a vector, if the pointers allow it
    int threads, rows, blocks, splits;
    int64_t split_positions, ctas;
    bool held;
    size_t smem;
};

Plan plan_of(const dcn_gnorm* p, int v, bool backward, bool residual) {
    Plan r = {};
    const int e = elem_bytes(p->dtype), c = (int)p->channels;
    r.v = v;
    const int vectors = c / v;
    const int64_t all = (int64_t)vectors * p->positions;
    const int kinds = backward ? (residual ? 3 : 2) : 1;
    auto lay = [&](int threads) {
        r.threads = threads;
        r.rows = vectors <= threads ? threads / vectors : 1;
        r.blocks = vectors <= threads ? 1 : (vectors + threads - 1) / threads;
    };
    // held: four vectors a thread or more, 64 to 512 threads
    int threads = 64;
    while (threads < 512 && threads * 4 < all) threads *= 2;
    if (vectors > threads / 2 && vectors <= 512) threads = (vectors + 31) / 32 * 32;       // (whole rows, few idle threads)
    lay(threads);
    const int64_t mine = (p->positions + r.rows - 1) / r.rows * r.blocks;
    const size_t data = ((size_t)mine * kinds * r.threads * e * v + 15) / 16 * 16;
    const size_t more = ((size_t)r.rows * 2 * c + 4 * p->groups + (backward ? 2 * c : r.rows)) * 4;
    if (mine < (1 << 20) && data <= kHeldBytes && data + more <= 200 * 1024) {
        r.held = true;
        r.smem = data + more;
        const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(2048 / r.threads, 16), 220 * 1024 / (r.smem + 1024)));
        r.ctas = std::max<int64_t>(1, std::min<int64_t>(p->samples, per_sm * sm_count()));
        r.splits = 1;
        return r;
    }
    lay(vectors > 256 && vectors <= 512 ? (vectors + 31) / 32 * 32 : 256);
    const int64_t target = (int64_t)sm_count() * 8;
    const int64_t most = std::max<int64_t>(1, p->positions / (8 * r.rows));
    r.splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, (target + p->samples - 1) / std::max<int64_t>(1, p->samples)));
    r.split_positions = (p->positions + r.splits - 1) / r.splits;
    r.splits = (int)((p->positions + r.split_positions - 1) / r.split_positions);
    r.ctas = p->samples * r.splits;
    r.smem = ((size_t)r.rows * 2 * c + (backward ? 2 * p->groups : r.rows)) * 4;
    return r;
}

struct Vec {
    int n, elem;
    explicit Vec(const dcn_gnorm* p) : n(16 / elem_bytes(p->dtype)), elem(elem_bytes(p->dtype)) {
        while (n > 1 && p->channels % n != 0) n /= 2;
    }
    void by(const void* v) {
        while (v != nullptr && n > 1 && !aligned(v, n * elem)) n /= 2;
    }
};

GnormArgs gnorm_args(const dcn_gnorm* p, const Plan& r) {
    GnormArgs a = {};
    a.samples = p->samples, a.positions = p->positions, a.split_positions = r.split_positions, a.splits = r.splits;
    a.channels = (int)p->channels, a.groups = (int)p->groups, a.per_group = a.channels / a.groups, a.vectors = a.channels / r.v;
    a.act = p->act, a.wide_weights = p->weight_dtype == DCN_SEQ_F32;
    a.eps = p->eps;
    a.inv = (float)(1.0 / ((double)p->positions * a.per_group));
    return a;
}

template <typename K>
int launch_gnorm(K kernel, int64_t ctas, const Plan& r, size_t smem, const GnormArgs& a, cudaStream_t st) {
    // (one amount per kernel, so that calls of several host threads do not take it from one another)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) return DCN_ERR_CUDA;
    return launch_dependent(kernel, dim3((unsigned)ctas), dim3(r.threads), smem, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int V>
int forward_as(const GnormArgs& a, const Plan& r, cudaStream_t st) {
    if (r.held) return launch_gnorm(gnorm_held_kernel<T, V>, r.ctas, r, r.smem, a, st);
    const int rc = launch_gnorm(gnorm_sums_kernel<T, V>, r.ctas, r, r.smem, a, st);
    return rc != DCN_OK ? rc : launch_gnorm(gnorm_apply_kernel<T, V>, r.ctas, r, 2 * a.groups * 4, a, st);
}

template <typename T, int V>
int backward_as(const GnormArgs& a, const Plan& r, void* dw, void* db, cudaStream_t st) {
    int rc;
    if (r.held) {
        rc = launch_gnorm(gnorm_held_backward_kernel<T, V>, r.ctas, r, r.smem, a, st);
    } else {
        rc = launch_gnorm(gnorm_sums_backward_kernel<T, V>, r.ctas, r, r.smem, a, st);
        if (rc == DCN_OK && (a.dx != nullptr || a.dresidual != nullptr)) {
            const dim3 grid((unsigned)a.samples, (unsigned)std::min(8, (a.groups + 7) / 8));
            if (launch_dependent(gnorm_join_kernel<T>, grid, dim3(256), 0, st, a) != cudaSuccess) return DCN_ERR_CUDA;
            rc = launch_gnorm(gnorm_apply_backward_kernel<T, V>, r.ctas, r, 4 * a.groups * 4, a, st);
        }
    }
    if (rc != DCN_OK || (dw == nullptr && db == nullptr)) return rc;
    return launch_dependent(gnorm_weights_kernel<T>, dim3((a.channels + 31) / 32), dim3(32, 32), 0, st, (const float*)a.partial,
                            r.held ? r.ctas : a.samples * a.splits, a.channels, dw, db, a.wide_weights) != cudaSuccess
               ? DCN_ERR_CUDA
               : DCN_OK;
}

template <typename F>
int by_type(int dtype, int v, F&& f) {
    if (dtype == DCN_SEQ_F32)
        return v == 4   ? f((float*)nullptr, std::integral_constant<int, 4>())
               : v == 2 ? f((float*)nullptr, std::integral_constant<int, 2>())
                        : f((float*)nullptr, std::integral_constant<int, 1>());
    auto half = [&](auto* t) {
        return v == 8   ? f(t, std::integral_constant<int, 8>())
               : v == 4 ? f(t, std::integral_constant<int, 4>())
               : v == 2 ? f(t, std::integral_constant<int, 2>())
                        : f(t, std::integral_constant<int, 1>());
    };
    return dtype == DCN_SEQ_BF16 ? half((__nv_bfloat16*)nullptr) : half((__half*)nullptr);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
// (whatever vectors a call's pointers allow)
size_t gnorm_bytes(const dcn_gnorm* p, bool backward) {
    size_t most = 0;
    if (p->samples == 0 || p->positions == 0) return 0;
    for (int v = Vec(p).n; v >= 1; v /= 2)
        for (int residual = 0; residual < (backward ? 2 : 1); ++residual) {
            const Plan r = plan_of(p, v, backward, residual != 0);
            size_t n = 0;
            if (backward) n = up256((size_t)r.ctas * 2 * p->channels * 4) + (r.held ? 0 : up256((size_t)p->samples * p->groups * 8));
            else if (!r.held) n = up256((size_t)r.ctas * 2 * p->groups * 4);
            most = std::max(most, n);
        }
    return most;
}

bool gnorm_aligned(const dcn_gnorm* p, std::initializer_list<const void*> elems, std::initializer_list<const void*> weights) {
    for (const void* v : elems)
        if (!aligned(v, elem_bytes(p->dtype))) return false;
    for (const void* v : weights)
        if (!aligned(v, elem_bytes(p->weight_dtype))) return false;
    return true;
}

}  // namespace
}  // namespace seq
}  // namespace dcn

using namespace dcn::seq;

extern "C" size_t dcn_gnorm_workspace_bytes(const dcn_gnorm* p, int32_t backward) {
    return check_gnorm(p) != DCN_OK ? 0 : gnorm_bytes(p, backward != 0);
}

extern "C" int dcn_gnorm_forward(const dcn_gnorm* p, const void* x, const void* weight, const void* bias, const void* residual, void* y,
                                 float* stats, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_gnorm(p);
    if (bad != DCN_OK) return bad;
    if (p->samples == 0 || p->positions == 0) return DCN_OK;
    if (x == nullptr || y == nullptr) return DCN_ERR_NULL;
    if (!gnorm_aligned(p, {x, residual, y}, {weight, bias}) || !aligned(stats, 4)) return DCN_ERR_ALIGN;
    const size_t need = gnorm_bytes(p, false);
    if (need > 0 && (workspace == nullptr || !aligned(workspace, 4) || workspace_bytes < need)) return DCN_ERR_WORKSPACE;
    Vec vec(p);
    vec.by(x), vec.by(residual), vec.by(y);
    const Plan r = plan_of(p, vec.n, false, false);
    if (r.ctas >= 1ll << 31) return DCN_ERR_LIMIT;
    GnormArgs a = gnorm_args(p, r);
    a.x = x, a.weight = weight, a.bias = bias, a.residual = residual, a.y = y, a.stats = stats;
    a.partial = static_cast<float*>(workspace);
    return by_type(p->dtype, vec.n, [&](auto* t, auto v) {
        return forward_as<std::remove_pointer_t<decltype(t)>, decltype(v)::value>(a, r, (cudaStream_t)stream);
    });
}

extern "C" int dcn_gnorm_backward(const dcn_gnorm* p, const void* x, const void* weight, const void* bias, const void* residual,
                                  const float* stats, const void* dy, void* dx, void* dweight, void* dbias, void* dresidual,
                                  void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_gnorm(p);
    if (bad != DCN_OK) return bad;
    const cudaStream_t st = (cudaStream_t)stream;
    if (!gnorm_aligned(p, {x, residual, dy, dx, dresidual}, {weight, bias, dweight, dbias}) || !aligned(stats, 4)) return DCN_ERR_ALIGN;
    if (p->samples == 0 || p->positions == 0) {
        for (void* v : {dweight, dbias})
            if (v != nullptr && cudaMemsetAsync(v, 0, (size_t)p->channels * elem_bytes(p->weight_dtype), st) != cudaSuccess)
                return DCN_ERR_CUDA;
        return DCN_OK;
    }
    if (x == nullptr || dy == nullptr || stats == nullptr) return DCN_ERR_NULL;
    const size_t need = gnorm_bytes(p, true);
    if (workspace == nullptr || !aligned(workspace, 4) || workspace_bytes < need) return DCN_ERR_WORKSPACE;
    Vec vec(p);
    vec.by(x), vec.by(residual), vec.by(dy), vec.by(dx), vec.by(dresidual);
    const Plan r = plan_of(p, vec.n, true, residual != nullptr);
    if (r.ctas >= 1ll << 31) return DCN_ERR_LIMIT;
    GnormArgs a = gnorm_args(p, r);
    a.x = x, a.weight = weight, a.bias = bias, a.residual = residual, a.dy = dy, a.stats = const_cast<float*>(stats);
    a.dx = dx, a.dresidual = dresidual;
    a.partial = static_cast<float*>(workspace);
    a.sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + up256((size_t)r.ctas * 2 * p->channels * 4));
    return by_type(p->dtype, vec.n, [&](auto* t, auto v) {
        return backward_as<std::remove_pointer_t<decltype(t)>, decltype(v)::value>(a, r, dweight, dbias, st);
    });
}
