// Group norm with an activation over channels-last features, with means over the positions and the channels of a sample's group:
//     h = (x - mean) r,  r = (mean((x - mean)^2) + eps)^-1/2;   z = h w + b + residual;   y = act(z)
// and the gradient, with dz = dy act'(z):
//     dw = sum dz h,  db = sum dz,  dresidual = dz;   dx = r (dz w - mean(dz w) - h mean(dz w h))
//
// A thread has a vector of channels (16 bytes where the rows allow it) and walks positions, so that the loads of a warp lie next to one
// another and its sums are those of fixed channels.  Variances are sums of squares about the thread's first element, joined over threads
// as n_i (mean_i - mean)^2 + M_i: no difference of large numbers, however far the mean is from zero.
//
// Three splits.  Single positions: some lanes of a warp have a group, a vector each.  Samples that fit a CTA's shared memory are read once
// (`held`): CTAs walk over samples.  Larger ones take two passes, the second of which finds in L2 what the first has left there; it runs from
// the end backwards.  Both passes have the next eight vectors of a thread on their way to its own places in shared memory (`Ring`), and
// arithmetic in packed pairs, since loads in registers and single instructions bounded them (8x50176x64 bf16 with gradients: 103 us before,
// 86 after, 78 with the weights' sums spread out; 1816 with a first version).
//
// Kernels' times: 8x50176x64 by 32 bf16, 51 MB a tensor: 15.7 + 15.1 us forward (floor 16.0), 24.0 + 25.9 backward (23.9): DRAM and issue
// slots, either at some 60 %.  6x1183x256 by 32 float32: 4.8 + 6.1 + 6.3 + 7.0 us, latency of few loads a thread.  Single positions,
// 18498x128 by 32 float32: 6.9 and 8.7 us (2.9 and 4.4) and 5.4 for the weights' sums; 30000x512 by 8 bf16 with SiLU 22.5 (9.5).
#include <algorithm>

#include "seq_common.cuh"

namespace dcn {
namespace seq {
namespace {

constexpr int64_t kMostChannels = 8192;
constexpr int kThreads = 256;                    // of a CTA of the two passes, at most
constexpr int kHeldBytes = 96 * 1024;            // of a sample's tensors, so that two CTAs share an SM
constexpr int kMostShared = 227 * 1024;          // what a CTA may ask for

struct GnormArgs {
    const void *x, *weight, *bias, *residual, *dy;
    void *y, *dx, *dresidual;
    float *stats;                                // [samples][groups][2]
    float *partial;                              // [samples][splits][groups][2]
    float *channel_sums;                         // backward [CTAs][channels][2]
    void *dweight, *dbias;
    int64_t samples, positions, split_positions;
    int channels, groups, per_group, vectors, act, wide_weights, splits;
    int tiny;                                    // a group has one or two elements
    int lanes;                                   // of a group, where samples are single positions (a power of two)
    int beside;                                  // channels that a block of weight_gradients has
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

// The weights of V channels, all on their way at once
template <typename T, int V>
__device__ __forceinline__ void weights_at(const void* w, int c0, int wide, float none, float (&out)[V]) {
    if (w == nullptr) {
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = none;
    } else if (wide) {
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = gload(static_cast<const float*>(w) + c0 + e);
    } else {
        Pack<T, 1> p[V];
#pragma unroll
        for (int e = 0; e < V; ++e) p[e].get(static_cast<const T*>(w) + c0 + e);
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = p[e].at(0);
    }
}

// The elements of a vector in pairs, as the packed instructions take them (one alone beside a zero)
template <int V>
struct Pairs {
    static constexpr int kN = (V + 1) / 2;
    Lanes v[kN];
    template <typename T>
    __device__ __forceinline__ void from(const Pack<T, V>& p) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const float f[2] = {p.at(2 * i), 2 * i + 1 < V ? p.at(2 * i + 1 < V ? 2 * i + 1 : 0) : 0.0f};
            v[i] = lanes(f);
        }
    }
    template <typename T>
    __device__ __forceinline__ Pack<T, V> pack() const {
        float f[V];
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = v[e / 2].at(e % 2);
        Pack<T, V> p;
        p.set(f);
        return p;
    }
    __device__ __forceinline__ void fill(float f) {
#pragma unroll
        for (int i = 0; i < kN; ++i) v[i] = all_lanes(f);
    }
    __device__ __forceinline__ float at(int e) const { return v[e / 2].at(e % 2); }
    // each element of two vectors
    template <typename F>
    __device__ __forceinline__ void map(F&& f) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const float r[2] = {f(v[i].at(0), 2 * i), 2 * i + 1 < V ? f(v[i].at(1), 2 * i + 1) : 0.0f};
            v[i] = lanes(r);
        }
    }
};

// y = act(z)
template <int V>
__device__ __forceinline__ void activate(Pairs<V>& z, int act) {
    if (act == DCN_ACT_RELU) {
        z.map([](float v, int) {
            float r;
            asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
            return r;
        });
    } else if (act == DCN_ACT_SILU) {
        z.map([](float v, int) {
            float s, rest;
            logistic(v, s, rest);
            return v * s;
        });
    }
}
// dy act'(z)
template <int V>
__device__ __forceinline__ Pairs<V> activate_gradient(Pairs<V> z, const Pairs<V>& dy, int act) {
    if (act == DCN_ACT_RELU) {
        z.map([&](float v, int e) { return v <= 0.0f ? 0.0f : dy.at(e); });
    } else if (act == DCN_ACT_SILU) {
        z.map([&](float v, int e) {
            float s, rest;
            logistic(v, s, rest);
            return dy.at(e) * (s * fmaf(v, rest, 1.0f));
        });
    } else {
        z = dy;
    }
    return z;
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

// Sums over the rows of threads of entries [row][channel][2] in shared memory: the channels' to entries [channel][2] (and `out`, added
// to what is there where `add`), and the groups' of them times w to `sums` [group][2] (may be null).  In a fixed order.
template <typename W>
__device__ __forceinline__ void join_channels(const GnormArgs& a, int rows, float2* entries, float* out, bool add, float* sums, W&& weight) {
    const int n = blockDim.x, c = a.channels, parts = max(1, min(n / c, rows));
    __syncthreads();
    for (int c0 = 0; c0 < c; c0 += n) {
        const int ch = parts > 1 ? threadIdx.x % c : c0 + threadIdx.x, part = parts > 1 ? threadIdx.x / c : 0;
        const bool in = ch < c && part < parts;
        float2 s = {0.0f, 0.0f};
        if (in)
            for (int r = part; r < rows; r += parts) s.x += entries[r * c + ch].x, s.y += entries[r * c + ch].y;
        if (parts > 1) {
            __syncthreads();
            if (in) entries[part * c + ch] = s;
            __syncthreads();
            if (part == 0)
                for (int k = 1; k < parts; ++k) s.x += entries[k * c + ch].x, s.y += entries[k * c + ch].y;
        }
        if (in && part == 0) {
            entries[ch] = s;
            if (out != nullptr) {
                float2 o = add ? *reinterpret_cast<float2*>(out + 2 * ch) : make_float2(0.0f, 0.0f);
                o.x += s.x, o.y += s.y;
                *reinterpret_cast<float2*>(out + 2 * ch) = o;
            }
        }
    }
    if (sums == nullptr) return;
    __syncthreads();
    const bool few = a.per_group > 16 && a.groups < n;           // a warp has a group, or a thread
    const int step = few ? 32 : 1, lane = few ? threadIdx.x & 31 : 0;
    for (int g = threadIdx.x / step; g < a.groups; g += n / step) {
        float2 s = {0.0f, 0.0f};
        for (int i = lane; i < a.per_group; i += step) {
            const int ch = g * a.per_group + i;
            const float w = weight(ch);
            s.x = fmaf(entries[ch].x, w, s.x), s.y = fmaf(entries[ch].y, w, s.y);
        }
        if (few) s.x = warp_sum(s.x), s.y = warp_sum(s.y);
        if (lane == 0) *reinterpret_cast<float2*>(sums + 2 * g) = s;
    }
}

// Sums of one thread's column over its positions, from its first element on
template <int V>
struct Moments {
    Pairs<V> less, s, q;                         // less: the first element, negative
    int n = 0;
    template <typename T>
    __device__ __forceinline__ void add(const Pack<T, V>& p) {
        Pairs<V> x;
        x.from(p);
        if (n == 0) {
#pragma unroll
            for (int i = 0; i < Pairs<V>::kN; ++i) less.v[i] = x.v[i] * all_lanes(-1.0f);
            s.fill(0.0f), q.fill(0.0f);
        }
        ++n;
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) {
            const Lanes d = x.v[i] + less.v[i];
            s.v[i] = s.v[i] + d, q.v[i] = fma(d, d, q.v[i]);
        }
    }
    __device__ __forceinline__ void put(float* mean, float* sq) const {
        const float by = n > 0 ? 1.0f / (float)n : 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float m = n > 0 ? s.at(e) * by : 0.0f;
            mean[e] = n > 0 ? m - less.at(e) : 0.0f;
            sq[e] = n > 0 ? fmaxf(fmaf(-s.at(e), m, q.at(e)), 0.0f) : 0.0f;
        }
    }
};

// The groups of a thread's channels, one behind the other
struct GroupOf {
    int g, left, per;
    __device__ __forceinline__ GroupOf(const GnormArgs& a, int c0) : g(c0 / a.per_group), left((c0 / a.per_group + 1) * a.per_group - c0), per(a.per_group) {}
    __device__ __forceinline__ int next() {
        const int now = g;
        if (--left == 0) ++g, left = per;
        return now;
    }
};

// The threads' moments as entries of join_channels: counts times means, and squares, about one number of each group, which adds up
// (the mean of the group's first channel in the first row of threads)
template <int V>
__device__ __forceinline__ void put_first(const GnormArgs& a, const Moments<V>& m, int c0, float* about) {
    float mean[V], sq[V];
    m.put(mean, sq);
    GroupOf group(a, c0);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const bool first = group.left == a.per_group;
        const int g = group.next();
        if (first) about[g] = mean[e];
    }
}
template <int V>
__device__ __forceinline__ void put_entries(const GnormArgs& a, const Moments<V>& m, int c0, const float* about, float2* entries) {
    float mean[V], sq[V];
    m.put(mean, sq);
    GroupOf group(a, c0);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float d = mean[e] - about[group.next()], n = (float)m.n;
        entries[e] = make_float2(n * d, fmaf(n * d, d, sq[e]));
    }
}
// Another such number: the middle one of a channel's first, middle and last element, so that one that is far off does no harm
template <typename T>
__device__ __forceinline__ float typical(const GnormArgs& a, const T* x, int64_t positions) {
    Pack<T, 1> p, q, r;
    p.get(x), q.get(x + positions / 2 * a.channels), r.get(x + (positions - 1) * a.channels);
    return fmaxf(fminf(p.at(0), q.at(0)), fminf(fmaxf(p.at(0), q.at(0)), r.at(0)));
}
// The one or two elements of a tiny group
template <typename T>
__device__ __forceinline__ float2 two_of(const GnormArgs& a, const void* from, int64_t base, int g) {
    const T* const x = static_cast<const T*>(from) + base + g * a.per_group;
    Pack<T, 1> p, q;
    p.get(x), q.zero();
    if (a.inv < 1.0f) q.get(x + (a.per_group == 2 ? 1 : a.channels));
    return make_float2(p.at(0), q.at(0));
}
// Mean and 1 / sqrt(var + eps) of a tiny group, in the definition's own order of steps
template <typename T>
__device__ __forceinline__ float2 tiny_stats(const GnormArgs& a, int64_t base, int g) {
    const float2 v = two_of<T>(a, a.x, base, g);
    const float mean = __fmul_rn(__fadd_rn(v.x, v.y), a.inv), p = __fsub_rn(v.x, mean), q = a.inv < 1.0f ? __fsub_rn(v.y, mean) : 0.0f;
    return make_float2(mean, rsqrtf(__fadd_rn(__fmul_rn(__fadd_rn(__fmul_rn(p, p), __fmul_rn(q, q)), a.inv), a.eps)));
}
// A group's mean and 1 / sqrt(var + eps) from such sums
__device__ __forceinline__ float2 finish(const GnormArgs& a, float about, float2 s) {
    const float d = s.x * a.inv;
    return make_float2(about + d, rsqrtf(fmaf(fmaxf(fmaf(-s.x, d, s.y), 0.0f), a.inv, a.eps)));
}

// What a thread needs of its channels: z = (x - mean) (r w) + b
template <typename T, int V>
struct Channels {
    Pairs<V> less, rw, b;                        // less: the mean, negative
    __device__ __forceinline__ void get(const GnormArgs& a, int c0, const float* stats) {
        GroupOf group(a, c0);
        float m[V], r[V], w[V];
        weights_at<T, V>(a.weight, c0, a.wide_weights, 1.0f, r);
        weights_at<T, V>(a.bias, c0, a.wide_weights, 0.0f, w);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = group.next();
            m[e] = -stats[2 * g];
            r[e] *= stats[2 * g + 1];
        }
        less.map([&](float, int e) { return m[e]; });
        rw.map([&](float, int e) { return r[e]; });
        b.map([&](float, int e) { return w[e]; });
    }
    __device__ __forceinline__ Pairs<V> z(const Pairs<V>& x, const Pack<T, V>& res, bool residual) const {
        Pairs<V> out, more;
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) out.v[i] = fma(x.v[i] + less.v[i], rw.v[i], b.v[i]);
        if (residual) {
            more.from(res);
#pragma unroll
            for (int i = 0; i < Pairs<V>::kN; ++i) out.v[i] = out.v[i] + more.v[i];
        }
        return out;
    }
};

// A thread's vectors of the next positions, on their way to its own places in shared memory while it works: no barrier, no registers.
constexpr int kDepth = 8;
// (the most that any call asks for: three tensors' rings of 16 bytes a thread beside a channel's sums and two numbers of each group, or beside
// four numbers of each group and two of each thread)
static_assert(3 * kDepth * kThreads * 16 + (8 + 2 * 4) * kMostChannels + 8 <= kMostShared && 3 * kDepth * kThreads * 16 + 4 * 4 * kMostChannels + 8 * kThreads <= kMostShared,
              "a group a channel, and as many channels as there may be");
template <typename T, int V>
struct Ring {
    static constexpr int kBytes = sizeof(T) * V, kKind = kDepth * kThreads * kBytes;         // kKind: of a tensor
    char* at;
    __device__ __forceinline__ Ring(char* smem) : at(smem + threadIdx.x * kBytes) {}
    __device__ __forceinline__ void issue(int slot, int kind, const T* from) const {
        char* const to = at + kind * kKind + slot * (kThreads * kBytes);
        if constexpr (kBytes >= 4) {
            copy_async_all<kBytes>(to, from);
        } else {
            Pack<T, V> p;
            p.get(from);
            *reinterpret_cast<Raw<kBytes>*>(to) = p.raw;
        }
    }
    __device__ __forceinline__ void get(Pack<T, V>& p, int slot, int kind) const {
        const char* const from = at + kind * kKind + slot * (kThreads * kBytes);
        if constexpr (kBytes >= 4) load_shared(p.raw, from);
        else p.raw = *reinterpret_cast<const Raw<kBytes>*>(from);
    }
};
// n positions: issue(slot) asks for the next one's vectors, use(slot, ahead) has the oldest one's and calls ahead() when it has read them
template <typename I>
__device__ __forceinline__ void stream_begin(int n, I&& issue) {
#pragma unroll
    for (int j = 0; j < kDepth - 1; ++j) {
        if (j < n) issue(j);
        copies_issued();
    }
}
template <typename I, typename U>
__device__ __forceinline__ void stream(int n, I&& issue, U&& use) {
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        copies_arrived<kDepth - 2>();
        use(i % kDepth, [&] {
            if (i + kDepth - 1 < n) issue((i + kDepth - 1) % kDepth);
            copies_issued();
        });
    }
    copies_arrived<0>();
}

// ---- samples that a CTA holds ---------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_held_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    const int mine = (int)((a.positions + grid.rows - 1) / grid.rows) * grid.blocks;     // vectors of a thread
    Raw<sizeof(T) * V>* const held = reinterpret_cast<Raw<sizeof(T) * V>*>(smem);
    float2* const entries = reinterpret_cast<float2*>(smem + ((size_t)mine * blockDim.x * sizeof(T) * V + 15) / 16 * 16);
    float* const stats = reinterpret_cast<float*>(entries + grid.rows * a.channels);
    float* const about = stats + 2 * a.groups;
    pdl_wait();
    for (int64_t sample = blockIdx.x; sample < a.samples; sample += gridDim.x) {
        const int64_t base = sample * a.positions * a.channels;
        auto load = [&](int b, int& k, Moments<V>& m) {
            const int col = grid.col + b * blockDim.x;
            const T* const x = static_cast<const T*>(a.x) + base + col * V;
            int i = 0;
            for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++i) {
                if constexpr (sizeof(T) * V >= 4) copy_async_all<sizeof(T) * V>(&held[(size_t)(k + i) * blockDim.x + threadIdx.x], x + p * a.channels);
                else seq::load(held[(size_t)(k + i) * blockDim.x + threadIdx.x], x + p * a.channels);
            }
            copies_issued();
            copies_arrived<0>();
            for (int j = 0; j < i; ++j, ++k) {
                Pack<T, V> v;
                v.raw = held[(size_t)k * blockDim.x + threadIdx.x];
                m.add(v);
            }
        };
        int k = 0;
        Moments<V> m;
        auto in = [&](int b) { return grid.row >= 0 && grid.col + b * (int)blockDim.x < a.vectors; };
        auto own = [&](int b) { return entries + grid.row * a.channels + (grid.col + b * blockDim.x) * V; };
        if (grid.blocks == 1) {
            if (in(0)) load(0, k, m);
            if (grid.row == 0) put_first(a, m, grid.col * V, about);
            __syncthreads();
            if (in(0)) put_entries(a, m, grid.col * V, about, own(0));
        } else {
            for (int g = threadIdx.x; g < a.groups; g += blockDim.x)
                about[g] = typical(a, static_cast<const T*>(a.x) + base + g * a.per_group, a.positions);
            __syncthreads();
            for (int b = 0; b < grid.blocks; ++b) {
                if (!in(b)) continue;
                Moments<V> mb;
                load(b, k, mb);
                put_entries(a, mb, (grid.col + b * blockDim.x) * V, about, own(b));
            }
        }
        join_channels(a, grid.rows, entries, nullptr, false, stats, [](int) { return 1.0f; });
        __syncthreads();
        for (int g = threadIdx.x; g < a.groups; g += blockDim.x) {
            const float2 f = a.tiny ? tiny_stats<T>(a, base, g) : finish(a, about[g], make_float2(stats[2 * g], stats[2 * g + 1]));
            stats[2 * g] = f.x, stats[2 * g + 1] = f.y;
        }
        __syncthreads();
        if (a.stats != nullptr)
            for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) a.stats[sample * 2 * a.groups + i] = stats[i];
        k = 0;
        for (int b = 0; b < grid.blocks; ++b) {
            const int col = grid.col + b * blockDim.x;
            if (grid.row < 0 || col >= a.vectors) continue;
            Channels<T, V> ch;
            ch.get(a, col * V, stats);
            for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                const int64_t at = base + p * a.channels + col * V;
                Pack<T, V> x, res;
                x.raw = held[(size_t)k * blockDim.x + threadIdx.x];
                if (a.residual != nullptr) res.get(static_cast<const T*>(a.residual) + at);
                Pairs<V> v;
                v.from(x);
                v = ch.z(v, res, a.residual != nullptr);
                activate(v, a.act);
                v.template pack<T>().put(static_cast<T*>(a.y) + at);
            }
        }
        __syncthreads();
    }
}

// Sums over a sample's splits of f(split, first number, second, first number of split 0) by group, finished by g(group, sums, that
// number).  Threads share out (group, split); `room` holds two floats of each thread.
template <typename F, typename G>
__device__ __forceinline__ void gather_splits(const GnormArgs& a, int64_t sample, float* room, F&& f, G&& finish) {
    const float* const partial = a.partial + sample * a.splits * 2 * a.groups;
    const int n = blockDim.x, per = n / a.groups;               // threads of a group (0: each thread has several groups)
    for (int g0 = 0; g0 < a.groups; g0 += n) {
        const int g = per > 0 ? threadIdx.x % a.groups : g0 + threadIdx.x, part = per > 0 ? threadIdx.x / a.groups : 0;
        const bool in = per > 0 ? part < per : g < a.groups;
        float x = 0.0f, y = 0.0f, m0 = 0.0f;
        if (in) {
            m0 = gload(partial + 2 * g);
#pragma unroll 4
            for (int i = part; i < a.splits; i += max(per, 1)) {
                Pack<float, 2> p;
                p.get(partial + ((int64_t)i * a.groups + g) * 2);
                float xi, yi;
                f(i, p.at(0), p.at(1), m0, xi, yi);
                x += xi, y += yi;
            }
        }
        room[2 * threadIdx.x] = x, room[2 * threadIdx.x + 1] = y;
        __syncthreads();
        if (in && part == 0) {
            for (int k = 1; k < per; ++k) x += room[2 * (threadIdx.x + k * a.groups)], y += room[2 * (threadIdx.x + k * a.groups) + 1];
            finish(g, x, y, m0);
        }
        __syncthreads();
    }
}

// ---- two passes -----------------------------------------------------------------------------------------------------------
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) gnorm_sums_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    const Ring<T, V> ring(smem);
    // (in the ring's place, once nothing more comes into it)
    float2* const entries = reinterpret_cast<float2*>(smem + (grid.blocks == 1 ? 0 : ring.kKind));
    float* const about = reinterpret_cast<float*>(smem + (grid.blocks == 1 ? max((int)ring.kKind, grid.rows * 8 * a.channels) : ring.kKind + 8 * a.channels));
    float* const sums = about + a.groups + (a.groups & 1);
    pdl_wait();
    const int64_t sample = blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    const T* const x = static_cast<const T*>(a.x) + (sample * a.positions + begin) * a.channels;
    for (int g = threadIdx.x; g < a.groups; g += blockDim.x) about[g] = typical(a, x + g * a.per_group, end - begin);
    const int n = grid.row < 0 ? 0 : (int)((end - begin - grid.row + grid.rows - 1) / grid.rows);
    const int64_t step = (int64_t)grid.rows * a.channels;
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x, mine = col < a.vectors ? n : 0;
        Moments<V> m;
        const T* next = x + grid.row * a.channels + col * V;
        auto issue = [&](int slot) {
            ring.issue(slot, 0, next);
            next += step;
        };
        stream_begin(mine, issue);
        stream(mine, issue, [&](int slot, auto&& ahead) {
            Pack<T, V> v;
            ring.get(v, slot, 0);
            ahead();
            m.add(v);
        });
        if (grid.blocks == 1 || b == 0) __syncthreads();
        if (grid.row >= 0 && col < a.vectors) put_entries(a, m, col * V, about, entries + grid.row * a.channels + col * V);
    }
    join_channels(a, grid.rows, entries, nullptr, false, sums, [](int) { return 1.0f; });
    __syncthreads();
    // of a split: its mean, and its squares about that
    float* const out = a.partial + (int64_t)blockIdx.x * 2 * a.groups;
    const float by = 1.0f / ((float)(end - begin) * (float)a.per_group);
    for (int g = threadIdx.x; g < a.groups; g += blockDim.x) {
        const float d = sums[2 * g] * by;
        out[2 * g] = about[g] + d, out[2 * g + 1] = fmaxf(fmaf(-sums[2 * g], d, sums[2 * g + 1]), 0.0f);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 3) gnorm_apply_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const int kinds = a.residual != nullptr ? 2 : 1;
    const Ring<T, V> ring(smem);
    float* const stats = reinterpret_cast<float*>(smem + kinds * ring.kKind);
    const Grid grid(a.vectors);
    const int64_t block = gridDim.x - 1 - blockIdx.x, sample = block / a.splits;
    const int split = (int)(block % a.splits);
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    const int n = grid.row < 0 ? 0 : (int)((end - begin - grid.row + grid.rows - 1) / grid.rows);
    const int64_t first = (sample * a.positions + begin + grid.row) * a.channels, step = (int64_t)grid.rows * a.channels;
    const T *x, *res;
    auto issue = [&](int slot) {
        ring.issue(slot, 0, x);
        x += step;
        if (kinds == 2) ring.issue(slot, 1, res), res += step;
    };
    auto start = [&](int b) {
        const int col = grid.col + b * blockDim.x;
        x = static_cast<const T*>(a.x) + first + col * V, res = static_cast<const T*>(a.residual) + first + col * V;
        stream_begin(col < a.vectors ? n : 0, issue);
    };
    pdl_wait();
    start(0);
    // the splits' statistics, about the first one's mean: their means differ by little
    gather_splits(a, sample, stats + 2 * a.groups, [&](int i, float m, float q, float m0, float& sx, float& sy) {
        const int64_t from = i * a.split_positions;
        const float c = (float)((min(from + a.split_positions, a.positions) - from) * a.per_group), d = m - m0;
        sx = c * d, sy = fmaf(c * d, d, q);
    }, [&](int g, float sx, float sy, float m0) {
        const float2 f = a.tiny ? tiny_stats<T>(a, sample * a.positions * a.channels, g) : finish(a, m0, make_float2(sx, sy));
        stats[2 * g] = f.x, stats[2 * g + 1] = f.y;
    });
    if (a.stats != nullptr && split == 0)
        for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) a.stats[sample * 2 * a.groups + i] = stats[i];
    for (int b = 0; b < grid.blocks; ++b) {
        if (b > 0) start(b);
        const int col = grid.col + b * blockDim.x;
        if (grid.row < 0 || col >= a.vectors) continue;
        Channels<T, V> ch;
        ch.get(a, col * V, stats);
        T* y = static_cast<T*>(a.y) + first + col * V;
        stream(n, issue, [&](int slot, auto&& ahead) {
            Pack<T, V> v, r;
            ring.get(v, slot, 0);
            if (kinds == 2) ring.get(r, slot, 1);
            ahead();
            Pairs<V> z;
            z.from(v);
            z = ch.z(z, r, kinds == 2);
            activate(z, a.act);
            z.template pack<T>().put(y);
            y += step;
        });
    }
}

// ---- gradients ------------------------------------------------------------------------------------------------------------
// With d = x - mean: sums of dz and of dz d (h is d r);   dx = dz (r w) - (s1 + d s2), s1 = r mean(dz w), s2 = r^2 mean(dz w h)
template <typename T, int V>
struct Loads {
    Pack<T, V> x, dy, res;
    __device__ __forceinline__ void get(const GnormArgs& a, const Ring<T, V>& ring, int slot) {
        ring.get(x, slot, 0), ring.get(dy, slot, 1);
        if (a.residual != nullptr) ring.get(res, slot, 2);
    }
    __device__ __forceinline__ void get(const GnormArgs& a, int64_t at) {
        x.get(static_cast<const T*>(a.x) + at);
        dy.get(static_cast<const T*>(a.dy) + at);
        if (a.residual != nullptr) res.get(static_cast<const T*>(a.residual) + at);
    }
    // dz, and x - mean
    __device__ __forceinline__ Pairs<V> gradient(const GnormArgs& a, const Channels<T, V>& ch, Pairs<V>& d) const {
        Pairs<V> g, z;
        d.from(x), g.from(dy);
        if (a.act != DCN_ACT_NONE) z = ch.z(d, res, a.residual != nullptr);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) d.v[i] = d.v[i] + ch.less.v[i];
        return activate_gradient(z, g, a.act);
    }
};

// The next position's vectors of x, dy and the residual
template <typename T, int V>
struct Sources {
    const T *x, *dy, *res;
    int64_t step;
    __device__ __forceinline__ Sources(const GnormArgs& a, int64_t at, int64_t step_)
        : x(static_cast<const T*>(a.x) + at), dy(static_cast<const T*>(a.dy) + at),
          res(a.residual != nullptr ? static_cast<const T*>(a.residual) + at : nullptr), step(step_) {}
    __device__ __forceinline__ void issue(const Ring<T, V>& ring, int slot) {
        ring.issue(slot, 0, x), ring.issue(slot, 1, dy);
        x += step, dy += step;
        if (res != nullptr) ring.issue(slot, 2, res), res += step;
    }
};

template <typename T, int V>
struct Sums {
    Pairs<V> s, q;
    __device__ __forceinline__ Sums() { s.fill(0.0f), q.fill(0.0f); }
    __device__ __forceinline__ void add(const GnormArgs& a, const Channels<T, V>& ch, const Loads<T, V>& v) {
        Pairs<V> d;
        const Pairs<V> dz = v.gradient(a, ch, d);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) s.v[i] = s.v[i] + dz.v[i], q.v[i] = fma(dz.v[i], d.v[i], q.v[i]);
    }
    // to [channel][2] as sums of dz and dz h
    __device__ __forceinline__ void put(const GnormArgs& a, int c0, const float* stats, float2* out) const {
        GroupOf group(a, c0);
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = make_float2(s.at(e), q.at(e) * stats[2 * group.next() + 1]);
    }
};

// kTiny: where groups may have one or two elements (a.tiny says whether they do)
template <typename T, int V, bool kTiny>
struct Gradient {
    Channels<T, V> ch;
    Pairs<V> s1, s2;                             // negative
    float rr[kTiny ? V : 1], w[kTiny ? V : 1];   // (of tiny ones, whose s1 and s2 are the means themselves)
    __device__ __forceinline__ void get(const GnormArgs& a, int c0, const float* stats, const float* sums) {
        ch.get(a, c0, stats);
        GroupOf group(a, c0);
        float p[V], q[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int g = group.next();
            const float r = stats[2 * g + 1];
            p[e] = -r * (sums[2 * g] * a.inv), q[e] = -r * r * (sums[2 * g + 1] * a.inv);
            if constexpr (kTiny)
                if (a.tiny) p[e] = sums[2 * g], q[e] = sums[2 * g + 1], rr[e] = r;
        }
        if constexpr (kTiny)
            if (a.tiny) weights_at<T, V>(a.weight, c0, a.wide_weights, 1.0f, w);

        s1.map([&](float, int e) { return p[e]; });
        s2.map([&](float, int e) { return q[e]; });
    }
    __device__ __forceinline__ void put(const GnormArgs& a, const Loads<T, V>& v, int64_t at) const {
        Pairs<V> d, dx;
        const Pairs<V> dz = v.gradient(a, ch, d);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) dx.v[i] = fma(dz.v[i], ch.rw.v[i], fma(d.v[i], s2.v[i], s1.v[i]));
        // Of two elements, the three terms cancel down to eps / (var + eps) of them, of one to nothing: every factor as it stands in the sums
        if constexpr (kTiny)
            if (a.tiny) dx.map([&](float, int e) {
                const float dh = __fmul_rn(dz.at(e), w[e]), h = __fmul_rn(d.at(e), rr[e]);
                return __fmul_rn(rr[e], __fsub_rn(__fsub_rn(dh, s1.at(e)), __fmul_rn(h, s2.at(e))));
            });
        if (a.dx != nullptr) dx.template pack<T>().put(static_cast<T*>(a.dx) + at);
        if (a.dresidual != nullptr) dz.template pack<T>().put(static_cast<T*>(a.dresidual) + at);
    }
};

// mean(dz w) and mean(dz w h) of a tiny group
template <typename T>
__device__ __forceinline__ void tiny_sums(const GnormArgs& a, int64_t base, int g, const float* stats, float* sums) {
    const float2 x = two_of<T>(a, a.x, base, g), dy = two_of<T>(a, a.dy, base, g);
    const float2 res = a.residual != nullptr ? two_of<T>(a, a.residual, base, g) : make_float2(0.0f, 0.0f);
    float dh[2] = {}, h[2] = {};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if (e == 1 && a.inv == 1.0f) break;
        const int c = g * a.per_group + (a.per_group == 2 ? e : 0);
        const float w = weight_at<T>(a.weight, c, a.wide_weights, 1.0f), d = (e == 0 ? x.x : x.y) - stats[2 * g];
        Pairs<1> z, y;
        const float zy[4] = {fmaf(d, stats[2 * g + 1] * w, weight_at<T>(a.bias, c, a.wide_weights, 0.0f)) + (e == 0 ? res.x : res.y), 0.0f,
                             e == 0 ? dy.x : dy.y, 0.0f};
        const float zs[2] = {zy[0], zy[1]}, ys[2] = {zy[2], zy[3]};
        z.v[0] = lanes(zs), y.v[0] = lanes(ys);
        dh[e] = __fmul_rn(activate_gradient(z, y, a.act).at(0), w), h[e] = __fmul_rn(d, stats[2 * g + 1]);
    }
    sums[2 * g] = __fmul_rn(__fadd_rn(dh[0], dh[1]), a.inv);
    sums[2 * g + 1] = __fmul_rn(__fadd_rn(__fmul_rn(dh[0], h[0]), __fmul_rn(dh[1], h[1])), a.inv);
}

template <typename T, int V>
__global__ void __launch_bounds__(512) gnorm_held_backward_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    const int mine = (int)((a.positions + grid.rows - 1) / grid.rows) * grid.blocks;
    const int kinds = a.residual != nullptr ? 3 : 2;
    Raw<sizeof(T) * V>* const held = reinterpret_cast<Raw<sizeof(T) * V>*>(smem);
    float2* const entries = reinterpret_cast<float2*>(smem + ((size_t)mine * kinds * blockDim.x * sizeof(T) * V + 15) / 16 * 16);
    float* const stats = reinterpret_cast<float*>(entries + grid.rows * a.channels);
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
            Channels<T, V> ch;
            ch.get(a, col * V, stats);
            Sums<T, V> sum;
            for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                Loads<T, V> v;
                v.get(a, base + p * a.channels + col * V);
                sum.add(a, ch, v);
                held[(size_t)(kinds * k) * blockDim.x + threadIdx.x] = v.x.raw;
                held[(size_t)(kinds * k + 1) * blockDim.x + threadIdx.x] = v.dy.raw;
                if (kinds == 3) held[(size_t)(kinds * k + 2) * blockDim.x + threadIdx.x] = v.res.raw;
            }
            sum.put(a, col * V, stats, entries + grid.row * a.channels + col * V);
        }
        join_channels(a, grid.rows, entries, total, true, sums, [&](int c) { return weight_at<T>(a.weight, c, a.wide_weights, 1.0f); });
        __syncthreads();
        if (a.tiny) {
            for (int g = threadIdx.x; g < a.groups; g += blockDim.x) tiny_sums<T>(a, base, g, stats, sums);
            __syncthreads();
        }
        k = 0;
        if (a.dx != nullptr || a.dresidual != nullptr)
            for (int b = 0; b < grid.blocks; ++b) {
                const int col = grid.col + b * blockDim.x;
                if (grid.row < 0 || col >= a.vectors) continue;
                Gradient<T, V, true> gr;
                gr.get(a, col * V, stats, sums);
                for (int64_t p = grid.row; p < a.positions; p += grid.rows, ++k) {
                    Loads<T, V> v;
                    v.x.raw = held[(size_t)(kinds * k) * blockDim.x + threadIdx.x];
                    v.dy.raw = held[(size_t)(kinds * k + 1) * blockDim.x + threadIdx.x];
                    if (kinds == 3) v.res.raw = held[(size_t)(kinds * k + 2) * blockDim.x + threadIdx.x];
                    gr.put(a, v, base + p * a.channels + col * V);
                }
            }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * a.channels; i += blockDim.x) a.channel_sums[(int64_t)blockIdx.x * 2 * a.channels + i] = total[i];
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 2) gnorm_sums_backward_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Grid grid(a.vectors);
    const Ring<T, V> ring(smem);
    const int room = (a.residual != nullptr ? 3 : 2) * ring.kKind;
    float2* const entries = reinterpret_cast<float2*>(smem + (grid.blocks == 1 ? 0 : room));       // (as in the forward pass)
    float* const stats = reinterpret_cast<float*>(smem + (grid.blocks == 1 ? max(room, grid.rows * 8 * a.channels) : room + 8 * a.channels));
    pdl_wait();
    const int64_t sample = blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    const int n = grid.row < 0 ? 0 : (int)((end - begin - grid.row + grid.rows - 1) / grid.rows);
    const int64_t first = (sample * a.positions + begin + grid.row) * a.channels;
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x, mine = col < a.vectors ? n : 0;
        Sources<T, V> from(a, first + col * V, (int64_t)grid.rows * a.channels);
        auto issue = [&](int slot) { from.issue(ring, slot); };
        stream_begin(mine, issue);
        if (b == 0) {
            for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) stats[i] = gload(a.stats + sample * 2 * a.groups + i);
            __syncthreads();
        }
        Sums<T, V> sum;
        if (mine > 0) {
            Channels<T, V> ch;
            ch.get(a, col * V, stats);
            stream(mine, issue, [&](int slot, auto&& ahead) {
                Loads<T, V> v;
                v.get(a, ring, slot);
                ahead();
                sum.add(a, ch, v);
            });
        }
        if (grid.blocks == 1) __syncthreads();
        if (grid.row >= 0 && col < a.vectors) sum.put(a, col * V, stats, entries + grid.row * a.channels + col * V);
    }
    join_channels(a, grid.rows, entries, a.channel_sums + (int64_t)blockIdx.x * 2 * a.channels, false,
                  a.partial + (int64_t)blockIdx.x * 2 * a.groups, [&](int c) { return weight_at<T>(a.weight, c, a.wide_weights, 1.0f); });
}

// ---- single positions -----------------------------------------------------------------------------------------------------
// Samples of one position (the heads' outputs of an attention, feature vectors) whose groups are up to 32 vectors: a few lanes of a warp
// have a group, a vector each, and walk over samples, so that weights and their gradients' sums stay in registers; sums of a group are
// shuffles.  No barrier, one read: bound by DRAM, and by the arithmetic of the activation.
struct Place {
    int lane, group, row, rows, blocks;          // blocks: of a sample's groups; rows: samples of a CTA
    int64_t first, step;                         // samples
    bool in;
    __device__ __forceinline__ explicit Place(const GnormArgs& a) {
        const int most = kThreads / a.lanes, slot = threadIdx.x / a.lanes, beside = min(a.groups, most);
        lane = threadIdx.x % a.lanes;
        rows = most / beside, blocks = (a.groups + most - 1) / most;
        row = slot / beside, group = blockIdx.x % blocks * most + slot % beside;
        first = (int64_t)(blockIdx.x / blocks) * rows, step = (int64_t)(gridDim.x / blocks) * rows;
        in = row < rows && group < a.groups;
    }
};
__device__ __forceinline__ float over_lanes(float v, int lanes) {
    for (int o = lanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int V>
__device__ __forceinline__ float over_pairs(const Pairs<V>& p) {
    Lanes s = p.v[0];
#pragma unroll
    for (int i = 1; i < Pairs<V>::kN; ++i) s = s + p.v[i];
    return s.at(0) + s.at(1);
}
// d less its group's mean
template <int V>
__device__ __forceinline__ float centre(Pairs<V>& d, bool in, const GnormArgs& a) {
    if (V == 1) d.map([](float f, int e) { return e == 0 ? f : 0.0f; });
    if (!in) d.fill(0.0f);
    const float mean = over_lanes(over_pairs(d), a.lanes) * a.inv;
    const Lanes less = all_lanes(-mean);
#pragma unroll
    for (int i = 0; i < Pairs<V>::kN; ++i) d.v[i] = d.v[i] + less;
    if (V == 1) d.map([](float f, int e) { return e == 0 ? f : 0.0f; });
    if (!in) d.fill(0.0f);
    return mean;
}
template <int V>
__device__ __forceinline__ Pairs<V> add_residual(Pairs<V> z, const Pairs<V>& res) {
#pragma unroll
    for (int i = 0; i < Pairs<V>::kN; ++i) z.v[i] = z.v[i] + res.v[i];
    return z;
}
template <typename T, int V>
__device__ __forceinline__ void weights_of(const GnormArgs& a, int c, bool in, Pairs<V>& w, Pairs<V>& b) {
    float f[V] = {}, g[V] = {};
    if (in) weights_at<T, V>(a.weight, c, a.wide_weights, 1.0f, f), weights_at<T, V>(a.bias, c, a.wide_weights, 0.0f, g);
    w.map([&](float, int e) { return f[e]; });
    b.map([&](float, int e) { return g[e]; });
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) gnorm_rows_kernel(const GnormArgs a) {
    pdl_wait();
    const Place place(a);
    const bool in = place.in && place.lane * V < a.per_group, residual = a.residual != nullptr;
    const int c = place.group * a.per_group + place.lane * V;
    Pairs<V> w, b;
    weights_of<T, V>(a, c, in, w, b);
    Pack<T, V> x, res, next, next_res;
    next.zero(), next_res.zero();
    auto fetch = [&](int64_t sample) {
        if (!in || sample >= a.samples) return;
        next.get(static_cast<const T*>(a.x) + sample * a.channels + c);
        if (residual) next_res.get(static_cast<const T*>(a.residual) + sample * a.channels + c);
    };
    fetch(place.first + place.row);
    for (int64_t start = place.first; start < a.samples; start += place.step) {
        const int64_t sample = start + place.row;
        const bool here = in && sample < a.samples;
        x = next, res = next_res;
        fetch(sample + place.step);
        Pairs<V> d, z, more;
        d.from(x);
        // about the group's first element, so that a mean far from zero costs nothing
        const float about = __shfl_sync(0xffffffffu, d.at(0), 0, a.lanes);
        const Lanes less = all_lanes(-about);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) d.v[i] = d.v[i] + less;
        const float mean = about + centre(d, in, a);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) z.v[i] = d.v[i] * d.v[i];
        const float r = rsqrtf(fmaf(over_lanes(over_pairs(z), a.lanes), a.inv, a.eps));
        if (!here) continue;
        if (a.stats != nullptr && place.lane == 0) {
            float* const to = a.stats + (sample * a.groups + place.group) * 2;
            to[0] = mean, to[1] = r;
        }
        const Lanes by = all_lanes(r);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) z.v[i] = fma(d.v[i], w.v[i] * by, b.v[i]);
        if (residual) more.from(res), z = add_residual(z, more);
        activate(z, a.act);
        z.template pack<T>().put(static_cast<T*>(a.y) + sample * a.channels + c);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) gnorm_rows_backward_kernel(const GnormArgs a) {
    __shared__ float2 room[kThreads * V];
    pdl_wait();
    const Place place(a);
    const bool in = place.in && place.lane * V < a.per_group, residual = a.residual != nullptr;
    const int c = place.group * a.per_group + place.lane * V;
    Pairs<V> w, b, s, q;
    weights_of<T, V>(a, c, in, w, b);
    s.fill(0.0f), q.fill(0.0f);
    Loads<T, V> v, next;
    next.x.zero(), next.dy.zero(), next.res.zero();
    float mean = 0.0f, r = 0.0f, next_mean = 0.0f, next_r = 0.0f;
    auto fetch = [&](int64_t sample) {
        if (!in || sample >= a.samples) return;
        next.get(a, sample * a.channels + c);
        const float* const from = a.stats + (sample * a.groups + place.group) * 2;
        next_mean = gload(from), next_r = gload(from + 1);
    };
    fetch(place.first + place.row);
    for (int64_t start = place.first; start < a.samples; start += place.step) {
        const int64_t sample = start + place.row;
        const bool here = in && sample < a.samples;
        v = next, mean = next_mean, r = next_r;
        fetch(sample + place.step);
        const Lanes by = all_lanes(r), less = all_lanes(-mean);
        Pairs<V> d, z, dz, more, t, u;
        d.from(v.x), dz.from(v.dy);
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) d.v[i] = d.v[i] + less;
        centre(d, in, a);                        // (the mean has been rounded: in a group of nearly equal elements that would be seen)
        if (a.act != DCN_ACT_NONE) {
#pragma unroll
            for (int i = 0; i < Pairs<V>::kN; ++i) z.v[i] = fma(d.v[i], w.v[i] * by, b.v[i]);
            if (residual) more.from(v.res), z = add_residual(z, more);
        }
        dz = activate_gradient(z, dz, a.act);
        if (!here) dz.fill(0.0f), d.fill(0.0f);
        if (V == 1) dz.map([](float f, int e) { return e == 0 ? f : 0.0f; });
#pragma unroll
        for (int i = 0; i < Pairs<V>::kN; ++i) {
            d.v[i] = d.v[i] * by;                // h
            t.v[i] = dz.v[i] * w.v[i], u.v[i] = t.v[i] * d.v[i];
            s.v[i] = s.v[i] + dz.v[i], q.v[i] = fma(dz.v[i], d.v[i], q.v[i]);
        }
        const Lanes s1 = all_lanes(-over_lanes(over_pairs(t), a.lanes) * a.inv), s2 = all_lanes(-over_lanes(over_pairs(u), a.lanes) * a.inv);
        if (!here) continue;
        if (a.dresidual != nullptr) dz.template pack<T>().put(static_cast<T*>(a.dresidual) + sample * a.channels + c);
        if (a.dx != nullptr) {
#pragma unroll
            for (int i = 0; i < Pairs<V>::kN; ++i) t.v[i] = by * (t.v[i] + fma(d.v[i], s2, s1));
            t.template pack<T>().put(static_cast<T*>(a.dx) + sample * a.channels + c);
        }
    }
    if (a.dweight == nullptr && a.dbias == nullptr) return;
    // the CTA's rows in order
#pragma unroll
    for (int e = 0; e < V; ++e) room[threadIdx.x * V + e] = make_float2(s.at(e), q.at(e));
    __syncthreads();
    if (place.row != 0 || !in) return;
    float2* const to = reinterpret_cast<float2*>(a.channel_sums) + (int64_t)(blockIdx.x / place.blocks) * a.channels + c;
    const int beside = min(a.groups, kThreads / a.lanes) * a.lanes;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        float2 sum = make_float2(0.0f, 0.0f);
        for (int k = 0; k < place.rows; ++k) {
            const float2 f = room[(threadIdx.x + k * beside) * V + e];
            sum.x += f.x, sum.y += f.y;
        }
        to[e] = sum;
    }
}

// dw and db of a.beside channels (a power of two up to 32): sums of n partial ones [n][channels][2], in a fixed order
template <typename T>
__device__ __forceinline__ void weight_gradients(const GnormArgs& a, int block, int64_t n, float* room) {
    const int rows = blockDim.x / a.beside, col = threadIdx.x % a.beside, row = threadIdx.x / a.beside, c = block * a.beside + col;
    Lanes sum = all_lanes(0.0f);
    if (c < a.channels) {
#pragma unroll 8
        for (int64_t i = row; i < n; i += rows) {
            Pack<float, 2> p;
            p.get(a.channel_sums + (i * a.channels + c) * 2);
            const float f[2] = {p.at(0), p.at(1)};
            sum = sum + lanes(f);
        }
    }
    float s = sum.at(0), q = sum.at(1);
    for (int o = a.beside; o < 32; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o), q += __shfl_xor_sync(0xffffffffu, q, o);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (lane < a.beside) room[2 * (warp * a.beside + lane)] = s, room[2 * (warp * a.beside + lane) + 1] = q;
    __syncthreads();
    if (row != 0 || c >= a.channels) return;
    s = q = 0.0f;
    for (int k = 0; k < (int)blockDim.x / 32; ++k) s += room[2 * (k * a.beside + col)], q += room[2 * (k * a.beside + col) + 1];
    auto put = [&](void* p, float v) {
        if (p == nullptr) return;
        if (a.wide_weights) static_cast<float*>(p)[c] = v;
        else static_cast<T*>(p)[c] = from_float<T>(v);
    };
    put(a.dweight, q), put(a.dbias, s);
}

// kTiny: groups of one or two elements, of so many channels that no CTA holds a sample
template <typename T, int V, bool kTiny>
__global__ void __launch_bounds__(kThreads, 2) gnorm_apply_backward_kernel(const GnormArgs a) {
    extern __shared__ __align__(16) char smem[];
    const Ring<T, V> ring(smem);
    float* const stats = reinterpret_cast<float*>(smem + (a.residual != nullptr ? 3 : 2) * ring.kKind);
    float* const sums = stats + 2 * a.groups;
    const Grid grid(a.vectors);
    const int first = a.dweight != nullptr || a.dbias != nullptr ? (a.channels + a.beside - 1) / a.beside : 0;      // blocks for these
    pdl_wait();
    if ((int)blockIdx.x < first) {
        weight_gradients<T>(a, blockIdx.x, a.samples * a.splits, stats);
        return;
    }
    const int64_t block = gridDim.x - 1 - blockIdx.x, sample = block / a.splits;
    const int split = (int)(block % a.splits);
    const int64_t begin = split * a.split_positions, end = min(begin + a.split_positions, a.positions);
    const int n = grid.row < 0 ? 0 : (int)((end - begin - grid.row + grid.rows - 1) / grid.rows);
    const int64_t at = (sample * a.positions + begin + grid.row) * a.channels, step = (int64_t)grid.rows * a.channels;
    Sources<T, V> from(a, at + grid.col * V, step);
    auto issue = [&](int slot) { from.issue(ring, slot); };
    stream_begin(grid.col < a.vectors ? n : 0, issue);
    for (int i = threadIdx.x; i < 2 * a.groups; i += blockDim.x) stats[i] = gload(a.stats + sample * 2 * a.groups + i);
    gather_splits(a, sample, sums + 2 * a.groups, [&](int, float p, float q, float, float& x, float& y) { x = p, y = q; },
                  [&](int g, float x, float y, float) {
                      sums[2 * g] = x, sums[2 * g + 1] = y;
                      if constexpr (kTiny) tiny_sums<T>(a, sample * a.positions * a.channels, g, stats, sums);
                  });
    for (int b = 0; b < grid.blocks; ++b) {
        const int col = grid.col + b * blockDim.x;
        if (b > 0) {
            from = Sources<T, V>(a, at + col * V, step);
            stream_begin(col < a.vectors ? n : 0, issue);
        }
        if (grid.row < 0 || col >= a.vectors) continue;
        Gradient<T, V, kTiny> gr;
        gr.get(a, col * V, stats, sums);
        int64_t to = at + col * V;
        stream(n, issue, [&](int slot, auto&& ahead) {
            Loads<T, V> v;
            v.get(a, ring, slot);
            ahead();
            gr.put(a, v, to);
            to += step;
        });
    }
}

template <typename T>
__global__ void __launch_bounds__(512) gnorm_weights_kernel(const GnormArgs a, int64_t n) {
    extern __shared__ __align__(16) char smem[];
    pdl_wait();
    weight_gradients<T>(a, blockIdx.x, n, reinterpret_cast<float*>(smem));
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
    int v;                                       // elements of a vector
    int threads, rows, blocks, splits;
    int64_t split_positions, ctas;
    bool held, single;                           // single: samples of one position, some lanes to a group
    int lanes;
    size_t smem, ring;                           // ring: of one tensor
};

Plan plan_of(const dcn_gnorm* p, int v, bool backward, bool residual) {
    Plan r = {};
    const int e = elem_bytes(p->dtype), c = (int)p->channels;
    r.v = v;
    const int vectors = c / v;
    const int64_t all = (int64_t)vectors * p->positions;
    const int kinds = backward ? (residual ? 3 : 2) : 1, per = c / (int)p->groups;
    if (p->positions == 1 && per > 2) {
        while (r.v > 1 && per % r.v != 0) r.v /= 2;
        if (per / r.v <= 32) {
            r.single = true, r.threads = kThreads, r.splits = 1;
            for (r.lanes = 1; r.lanes * r.v < per; r.lanes *= 2) {}
            const int most = kThreads / r.lanes, blocks = ((int)p->groups + most - 1) / most, rows = most / std::min((int)p->groups, most);
            // (backward, a CTA's sums for the weights are read once more: half as many)
            const int64_t fit = std::max<int64_t>(1, (int64_t)sm_count() * (backward ? 4 : 8) / blocks);
            r.ctas = std::min(fit, (p->samples + rows - 1) / rows) * blocks, r.blocks = blocks;
            return r;
        }
        r.v = v;
    }
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
    const size_t held_sums = ((size_t)r.rows * 2 * c + 4 * p->groups + (backward ? 2 * c : 0)) * 4;
    if (mine < (1 << 20) && data <= kHeldBytes && data + held_sums <= 200 * 1024) {
        r.held = true;
        r.smem = data + held_sums;
        const int64_t per_sm = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(2048 / r.threads, 16), 220 * 1024 / (r.smem + 1024)));
        r.ctas = std::max<int64_t>(1, std::min<int64_t>(p->samples, per_sm * sm_count()));
        r.splits = 1;
        return r;
    }
    // One wave of CTAs, each with eight positions a thread or more, and so much of x that the splits' statistics, which each CTA of
    // the second pass reads, are an eighth of it: splits * groups * 8 bytes <= positions / splits * channels * e / 8
    const int blocks = (vectors + kThreads - 1) / kThreads, width = (vectors + blocks - 1) / blocks;
    lay((kThreads / width * width + 31) / 32 * 32);
    const int64_t target = (int64_t)sm_count() * ((backward ? 2 : 3) * kThreads / r.threads);
    int64_t most = std::max<int64_t>(1, p->positions / (8 * r.rows));
    while (most > 1 && most * most > p->positions * c * e / (64 * p->groups)) most = most * 7 / 8;
    r.splits = (int)std::max<int64_t>(1, std::min<int64_t>(most, target / std::max<int64_t>(1, p->samples)));
    r.split_positions = (p->positions + r.splits - 1) / r.splits;
    r.splits = (int)((p->positions + r.split_positions - 1) / r.split_positions);
    r.ctas = p->samples * r.splits;
    r.ring = (size_t)kDepth * kThreads * e * v;
    const size_t sums = (size_t)r.rows * 2 * c * 4, more = (size_t)(backward ? 2 : 4) * p->groups * 4 + 8;
    if (backward) r.smem = r.blocks == 1 ? std::max(kinds * r.ring, sums) + more : kinds * r.ring + sums + more;
    else r.smem = (r.blocks == 1 ? std::max(r.ring, sums) : r.ring + sums) + more;
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
    a.tiny = p->positions * a.per_group <= 2;
    a.lanes = r.lanes;
    // Few channels: more threads to each.  (8x50176x64: the second pass 34 us with two blocks of 32 before it, 26 with eight of 8; but
    // 6x1183x256: 6.8 with eight of 32, 9.3 with 32 of 8.  Alone, 592 sums of 128 channels: 11.6 us with 32, 5.4 with 8.)
    a.beside = 8;
    while (a.beside < 32 && a.channels > (r.held || r.single ? 64 : 8) * a.beside) a.beside *= 2;
    return a;
}

template <typename K>
int launch_gnorm(K kernel, int64_t ctas, const Plan& r, size_t smem, const GnormArgs& a, cudaStream_t st) {
    // (one amount per kernel, so that calls of several host threads do not take it from one another)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared) != cudaSuccess) return DCN_ERR_CUDA;
    return launch_dependent(kernel, dim3((unsigned)ctas), dim3(r.threads), smem, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int V>
int forward_as(const GnormArgs& a, const Plan& r, cudaStream_t st) {
    if (r.single)
        return launch_dependent(gnorm_rows_kernel<T, V>, dim3((unsigned)r.ctas), dim3(kThreads), 0, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
    if (r.held) return launch_gnorm(gnorm_held_kernel<T, V>, r.ctas, r, r.smem, a, st);
    const int rc = launch_gnorm(gnorm_sums_kernel<T, V>, r.ctas, r, r.smem, a, st);
    return rc != DCN_OK ? rc : launch_gnorm(gnorm_apply_kernel<T, V>, r.ctas, r, (a.residual != nullptr ? 2 : 1) * r.ring + (2 * a.groups + 2 * r.threads) * 4, a, st);
}

template <typename T, int V>
int backward_as(const GnormArgs& a, const Plan& r, cudaStream_t st) {
    const bool weights = a.dweight != nullptr || a.dbias != nullptr, data = a.dx != nullptr || a.dresidual != nullptr;
    const int blocks = weights ? (a.channels + a.beside - 1) / a.beside : 0;
    const size_t room = (a.residual != nullptr ? 3 : 2) * r.ring + 2 * r.threads * 4;
    const bool once = r.held || r.single;
    int rc;
    if (r.single) rc = launch_dependent(gnorm_rows_backward_kernel<T, V>, dim3((unsigned)r.ctas), dim3(kThreads), 0, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
    else rc = r.held ? launch_gnorm(gnorm_held_backward_kernel<T, V>, r.ctas, r, r.smem, a, st)
                     : launch_gnorm(gnorm_sums_backward_kernel<T, V>, r.ctas, r, r.smem, a, st);
    if (rc != DCN_OK || (!weights && once)) return rc;
    if (!once && data)
        return launch_gnorm(a.tiny ? gnorm_apply_backward_kernel<T, V, true> : gnorm_apply_backward_kernel<T, V, false>, blocks + r.ctas, r,
                            4 * a.groups * 4 + room, a, st);
    if (!weights) return DCN_OK;
    return launch_dependent(gnorm_weights_kernel<T>, dim3(blocks), dim3(512), 2 * 512 * 4, st, a, r.single ? r.ctas / r.blocks : r.held ? r.ctas : a.samples * a.splits) !=
                   cudaSuccess
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
            if (!r.held && !r.single) n = up256((size_t)r.ctas * 2 * p->groups * 4);
            if (backward) n += up256((size_t)r.ctas * 2 * p->channels * 4);
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
    if (need > 0 && (workspace == nullptr || !aligned(workspace, 8) || workspace_bytes < need)) return DCN_ERR_WORKSPACE;
    Vec vec(p);
    vec.by(x), vec.by(residual), vec.by(y);
    const Plan r = plan_of(p, vec.n, false, false);
    if (r.ctas >= 1ll << 31) return DCN_ERR_LIMIT;
    GnormArgs a = gnorm_args(p, r);
    a.x = x, a.weight = weight, a.bias = bias, a.residual = residual, a.y = y, a.stats = stats;
    a.partial = static_cast<float*>(workspace);
    return by_type(p->dtype, r.v, [&](auto* t, auto v) {
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
    if (workspace == nullptr || !aligned(workspace, 8) || workspace_bytes < need) return DCN_ERR_WORKSPACE;
    Vec vec(p);
    vec.by(x), vec.by(residual), vec.by(dy), vec.by(dx), vec.by(dresidual);
    const Plan r = plan_of(p, vec.n, true, residual != nullptr);
    if (r.ctas >= 1ll << 31) return DCN_ERR_LIMIT;
    GnormArgs a = gnorm_args(p, r);
    a.x = x, a.weight = weight, a.bias = bias, a.residual = residual, a.dy = dy, a.stats = const_cast<float*>(stats);
    a.dx = dx, a.dresidual = dresidual, a.dweight = dweight, a.dbias = dbias;
    a.channel_sums = static_cast<float*>(workspace);
    a.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + up256((size_t)r.ctas * 2 * p->channels * 4));
    return by_type(p->dtype, r.v, [&](auto* t, auto v) {
        return backward_as<std::remove_pointer_t<decltype(t)>, decltype(v)::value>(a, r, st);
    });
}
