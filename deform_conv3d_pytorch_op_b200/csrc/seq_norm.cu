// The norm behind a block, its gate, the scaled residual and the norm before the next block, as one pass over the rows:
//     yn = block r,  r = (mean(block^2) + eps)^-1/2;   stream = x + c s(gate) yn,  c = scale post
//     sn = stream q, q = (mean(stream^2) + eps)^-1/2;  normed = sn pre
// and the gradient, with dsn = dnormed pre and means over the channels:
//     ds = dstream + q (dsn - sn mean(dsn sn)) = dx;   dyn = ds c s(gate);   dblock = r (dyn - yn mean(dyn yn))
//     dgate = dyn yn (1 - s(gate));   Z = sum over rows of ds s(gate) yn:  dscale = Z post, dpost = Z scale;   dpre = sum dnormed sn
//
// A row lives in the registers of a row of threads, 32 bytes of each tensor a thread, so that every tensor is read or written
// once.  Rows of up to 32 threads (512 channels of 16 bits, 256 of float32) share a warp, and their sums are shuffles alone; above,
// a row is that of 64 to 512 (float32: 1024) threads of a CTA, which meet at a barrier of their own.  CTAs walk the rows; a
// thread's elements of the next row are on their way to its own places in shared memory meanwhile (cp.async, 16, 8 or 4 bytes at a
// time, as rows start on them).  Weights are in shared memory too, once a CTA (registers for them would cost a third of the
// threads), and the arithmetic goes in pairs through the packed float32 instructions.  The CTAs of the backward pass keep Z and
// dpre in registers and leave one partial sum each; a second kernel adds those in a fixed order.
//
// The bound is DRAM, and the arithmetic, which leaves a third of the issue slots, stands close behind.  Measured, forward and
// backward with the sums of the weights' gradients, against a copy of the same bytes at 6.5 TB/s:
//     32768 x 2048 bf16    117 us (5.7 TB/s, 88 %)   209 us (5.1 TB/s, 79 %)
//     32768 x 2044 bf16    143 us                    261 us      rows on 8 bytes: twice the loads and stores
//     32768 x 2046 bf16    192 us                    347 us      on 4 bytes: four times as many
//     32768 x 2047 bf16    248 us                    574 us      pairs that lie across the tensor's 4 bytes (392 and 887 us
//                                                                when elements were loaded and stored one by one)
//     16384 x 2046 float32 125 us                    205 us      on 8 bytes (by 4, at 2047: 174 and 286 us)
//     10080 x 2112 bf16     84 us (33 of a copy)     141 us (52)  132 of a row's 256 threads have elements, all issue
//     21289 x 2145 bf16    346 us (70)               780 us (112) the same, and odd rows
//     4096 x 8192 float32  140 us (4.8 TB/s, 74 %)   334 us (3.2 TB/s, 49 %)     above 4096 channels rows are too long to be held
//                                                                twice, nothing is ahead, and the backward pass spills registers
//     65536 x 64 bf16       10 us (4.0 TB/s)          22 us (3.1 TB/s)           in L2; eight rows to a warp
#include <algorithm>

#include "seq_common.cuh"

namespace dcn {
namespace seq {
namespace {

constexpr int64_t kMostChannels = 8192;

struct NormArgs {
    const void *x, *block, *gate, *scale, *post, *pre, *dstream, *dnormed;
    void *stream, *normed, *dx, *dblock, *dgate;
    float *stats, *partial;
    int64_t rows, x_row, block_row, gate_row, dstream_row, dnormed_row;
    int channels, threads, wide_weights;         // threads: of a row
    float eps, inv;
};

// How a row of elements T lies over threads, V at a time: the vectors j, j + threads, ... of thread j.  16-bit rows that start in
// the middle of 4 bytes (V 1) lie in pairs as well (kSkew): they move 4 bytes at a time, as these lie in the tensor, and a thread
// has its pair from two neighbouring ones.  Neighbours are those of a segment, the threads that a row and a warp share: its pairs
// are next to one another, whichever vectors they are, and its last thread fetches the 4 bytes behind them too.
template <typename T, int V>
struct Layout {
    static constexpr bool kSkew = V * sizeof(T) == 2;
    static constexpr int kV = kSkew ? 2 : V, kPer = 32 / (int)sizeof(T), kVectors = kPer / kV, kPairs = kPer / 2;
    static __device__ __forceinline__ int element(int j, int threads, int e) {
        if constexpr (kSkew) {
            const int s = segment(threads);
            return (j / s * s * kVectors + e / kV * s + j % s) * kV + e % kV;
        }
        return (j + e / kV * threads) * kV + e % kV;
    }
    static __host__ __device__ __forceinline__ int segment(int threads) { return threads < 32 ? threads : 32; }
    static __device__ __forceinline__ int at_segment(int threads) { return (int)threadIdx.x % segment(threads); }
};

// A thread's elements of a row
template <typename T, int V>
struct Slice {
    static constexpr int kV = Layout<T, V>::kV;
    Pack<T, kV> v[Layout<T, V>::kVectors];
    __device__ __forceinline__ float at(int e) const { return v[e / kV].at(e % kV); }
    __device__ __forceinline__ Lanes pair(int i) const {
        const float f[2] = {at(2 * i), at(2 * i + 1)};
        return lanes(f);
    }
};

template <typename T, int V>
__device__ __forceinline__ void put(void* base, int64_t offset, const Lanes (&f)[Layout<T, V>::kPairs], int j, int threads,
                                    int channels) {
    using L = Layout<T, V>;
    if (base == nullptr) return;
    T* out = static_cast<T*>(base) + offset;
    const bool skew = L::kSkew && reinterpret_cast<uintptr_t>(out) % 4 != 0;
    uint32_t words[L::kSkew ? L::kVectors : 1];
#pragma unroll
    for (int i = 0; i < L::kVectors; ++i) {
        const int c = L::element(j, threads, i * L::kV);
        float part[L::kV];
#pragma unroll
        for (int k = 0; k < L::kV; ++k) part[k] = f[(i * L::kV + k) / 2].at((i * L::kV + k) % 2);
        Pack<T, L::kV> mine;
        mine.set(part);
        if constexpr (L::kSkew) {
            words[i] = mine.raw.u[0];
        } else {
            if (c < channels) mine.put(out + c);
        }
    }
    if constexpr (L::kSkew) {
        // (every lane takes part in the shuffles, whatever its row's skew: a warp's rows may differ in it)
        const int s = L::segment(threads), l = L::at_segment(threads), next_lane = (int)threadIdx.x % 32 - l + (l + 1) % s;
        uint32_t nexts[L::kVectors];
#pragma unroll
        for (int i = 0; i < L::kVectors; ++i)
            nexts[i] = __shfl_sync(0xffffffffu, l == 0 && i + 1 < L::kVectors ? words[i + 1] : words[i], next_lane);
        if (skew) {                              // 4 bytes are a pair's second element and the next pair's first
#pragma unroll
            for (int i = 0; i < L::kVectors; ++i) {
                const int c = L::element(j, threads, i * L::kV);
                const bool both = c + 2 < channels && (i + 1 < L::kVectors || l + 1 < s);
                if (i == 0 && l == 0 && c < channels) store(out + c, Raw<2>{(uint16_t)words[i]});
                if (both) store(out + c + 1, Raw<4>{{__funnelshift_r(words[i], nexts[i], 16)}});
                if (!both && c + 1 < channels) store(out + c + 1, Raw<2>{(uint16_t)(words[i] >> 16)});
            }
        } else {
#pragma unroll
            for (int i = 0; i < L::kVectors; ++i) {
                const int c = L::element(j, threads, i * L::kV);
                if (c + 1 < channels) store(out + c, Raw<4>{{words[i]}});
                if (c + 1 == channels) store(out + c, Raw<2>{(uint16_t)words[i]});
            }
        }
    }
}

// A thread's elements of one row after the other, of kTensors tensors
template <typename T, int V, int kTensors, bool kStaged>
struct Rows {
    using L = Layout<T, V>;
    const T* base[kTensors];                     // nullptr: zeros
    int64_t stride[kTensors];
    int64_t rows, step;                          // rows in all, and from one of mine to the next
    int j, threads, channels;                    // my place in the row
    unsigned char* room;                         // mine of the first vector
    int width;                                   // bytes from one vector of a thread to its next: of the CTA's threads
    int stage = 0;
    int64_t now = 0;
    bool first = true, live = true;              // live: the row is there (rows of a warp end together)
    Slice<T, V> here[kStaged ? 1 : kTensors];    // the row's, where it is not in shared memory
    static constexpr int kMove = L::kV * (int)sizeof(T);
    static constexpr int kBytes = kStaged ? 2 * kTensors * L::kVectors * kMove : 0;    // of a thread: two rows
    static constexpr int kExtra = kStaged && L::kSkew ? 2 * kTensors * kMove : 0;      // of a segment: what its last thread fetches
    // where thread n of a CTA's has its first vector, in rows of `threads`; and `width` for n threads
    static __device__ __forceinline__ int offset_of(int n, int threads) {
        const int s = L::segment(threads);
        return (L::kSkew ? n / s * (s * L::kVectors + 1) + n % s : n) * kMove;
    }
    static __device__ __forceinline__ int width_of(int n, int threads) {
        return (L::kSkew ? n * L::kVectors + n / L::segment(threads) : n) * kMove;
    }
    __device__ __forceinline__ unsigned char* place(int s, int t, int i) const {
        if constexpr (L::kSkew) return room + (s * kTensors + t) * width + i * L::segment(threads) * kMove;
        return room + ((s * kTensors + t) * L::kVectors + i) * width;
    }
    __device__ __forceinline__ bool skewed(int t, int64_t row) const {
        return L::kSkew &&
               (((unsigned)(reinterpret_cast<uintptr_t>(base[t]) / 2) + (unsigned)row * (unsigned)stride[t]) & 1) != 0;
    }
    __device__ __forceinline__ void fetch(int s, int64_t row) {
        if (row < rows) {
            const bool whole = channels == threads * L::kPer;
#pragma unroll
            for (int t = 0; t < kTensors; ++t) {
                if (base[t] == nullptr) continue;
                const T* from = base[t] + row * stride[t] + L::element(j, threads, 0);
                if constexpr (L::kSkew) {        // zeros from the row's end on; nothing is read that lies before the tensor
                    const int skew = skewed(t, row), apart = L::kV * L::segment(threads);
                    from -= skew;
                    int left = channels - L::element(j, threads, 0) + skew;
                    if (from < base[t]) {
                        Pack<T, 1> one;
                        one.get(base[t]);
                        *reinterpret_cast<Raw<2>*>(place(s, t, 0) + 2) = one.raw;
                    } else if (left >= 0) {
                        copy_async_some<4>(place(s, t, 0), from, min(2 * left, 4));
                    }
#pragma unroll
                    for (int i = 1; i < L::kVectors; ++i) {
                        from += apart, left -= apart;
                        if (left >= 0) copy_async_some<4>(place(s, t, i), from, min(2 * left, 4));
                    }
                    if (L::at_segment(threads) + 1 == L::segment(threads) && left >= 2)
                        copy_async_some<4>(place(s, t, L::kVectors - 1) + 4, from + 2, min(2 * left - 4, 4));
                    continue;
                }
#pragma unroll
                for (int i = 0; i < L::kVectors; ++i, from += threads * V) {
                    if (whole) copy_async_all<kMove>(place(s, t, i), from);
                    else if (L::element(j, threads, i * V) < channels) copy_async<kMove>(place(s, t, i), from, true);
                    else copy_async<kMove>(place(s, t, i), base[t], false);
                }
            }
        }
        copies_issued();
    }
    // the row that next() goes to first
    __device__ __forceinline__ void begin(int64_t row) {
        if constexpr (kStaged && L::kSkew) {     // (what lies far behind the rows' ends is not fetched)
            for (int t = 0; t < 2 * kTensors; ++t)
                for (int i = 0; i < L::kVectors; ++i) {
                    *reinterpret_cast<uint32_t*>(place(0, t, i)) = 0;
                    if (i + 1 == L::kVectors && L::at_segment(threads) + 1 == L::segment(threads))
                        *reinterpret_cast<uint32_t*>(place(0, t, i) + 4) = 0;
                }
            __syncwarp();
        }
        if constexpr (kStaged) fetch(0, row);
    }
    // to row `row`, the next one since the last call or begin()
    __device__ __forceinline__ void next(int64_t row) {
        live = row < rows;
        now = row;
        if constexpr (kStaged) {
            stage = first ? 0 : stage ^ 1;
            first = false;
            if (L::kSkew) __syncwarp();          // (neighbours have read what is fetched over)
            fetch(stage ^ 1, row + step);
            copies_arrived<1>();
            if (L::kSkew) __syncwarp();
        } else {
#pragma unroll
            for (int t = 0; t < kTensors; ++t)
#pragma unroll
                for (int i = 0; i < L::kVectors; ++i) {
                    const int c = L::element(j, threads, i * L::kV);
                    here[t].v[i].zero();
                    if (!live || base[t] == nullptr || c >= channels) continue;
                    const T* from = base[t] + row * stride[t] + c;
                    if constexpr (L::kSkew) {
                        Raw<2> lo, hi{0};
                        load(lo, from);
                        if (c + 1 < channels) load(hi, from + 1);
                        here[t].v[i].raw.u[0] = lo.u | (uint32_t)hi.u << 16;
                    } else {
                        here[t].v[i].get(from);
                    }
                }
        }
    }
    // the row's elements of a tensor, until the next next(): from shared memory when they are asked for, so that registers hold
    // no more than what is in use
    __device__ __forceinline__ Slice<T, V> get(int t) const {
        if constexpr (!kStaged) {
            return here[t];
        } else {
            Slice<T, V> s;
#pragma unroll
            for (int i = 0; i < L::kVectors; ++i) {
                if (base[t] == nullptr || !live) {
                    s.v[i].zero();
                    continue;
                }
                load_shared(s.v[i].raw, place(stage, t, i));
                if constexpr (L::kSkew) {
                    Raw<4> next;
                    load_shared(next, place(stage, t, i) + 4);
                    s.v[i].raw.u[0] = __funnelshift_r(s.v[i].raw.u[0], next.u[0], skewed(t, now) ? 16 : 0);
                }
            }
            return s;
        }
    }
};

// A weight as float32: of its own type, or of the activations'
template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int c, int wide) {
    if (w == nullptr) return 1.0f;
    Pack<T, 1> v;
    if (wide) return gload(static_cast<const float*>(w) + c);
    v.get(static_cast<const T*>(w) + c);
    return v.at(0);
}

// A thread's elements of a weight, all on their way before the first is used; ones where there is no weight
template <typename W, typename T, int V>
__device__ __forceinline__ void load_weight(Pack<W, 1> (&f)[Layout<T, V>::kPer], const void* w, int j, int threads, int channels) {
#pragma unroll
    for (int e = 0; e < Layout<T, V>::kPer; ++e) {
        const int c = Layout<T, V>::element(j, threads, e);
        const float one[1] = {1.0f};
        f[e].set(one);
        if (w != nullptr && c < channels) f[e].get(static_cast<const W*>(w) + c);
    }
}

// scale post and pre of a row's threads, in shared memory: those of a thread four at a time
template <typename T, int V>
struct Weights {
    using L = Layout<T, V>;
    static constexpr int kBytes = 2 * L::kPer * 4;          // of a thread
    float4* at;
    int width;
    template <typename W>
    __device__ __forceinline__ void put_as(const NormArgs& p, int j, int threads) {
        Pack<W, 1> scale[L::kPer], post[L::kPer], pre[L::kPer];
        load_weight<W, T, V>(scale, p.scale, j, threads, p.channels);
        load_weight<W, T, V>(post, p.post, j, threads, p.channels);
        load_weight<W, T, V>(pre, p.pre, j, threads, p.channels);
#pragma unroll
        for (int i = 0; i < L::kPer; i += 4) {
            at[i / 4 * width] = make_float4(scale[i].at(0) * post[i].at(0), scale[i + 1].at(0) * post[i + 1].at(0),
                                            scale[i + 2].at(0) * post[i + 2].at(0), scale[i + 3].at(0) * post[i + 3].at(0));
            at[(L::kPer + i) / 4 * width] = make_float4(pre[i].at(0), pre[i + 1].at(0), pre[i + 2].at(0), pre[i + 3].at(0));
        }
    }
    __device__ __forceinline__ void put(const NormArgs& p, int j, int threads) {
        if (p.wide_weights) put_as<float>(p, j, threads);
        else put_as<T>(p, j, threads);
    }
    __device__ __forceinline__ void get(int which, Lanes (&f)[L::kPairs]) const {
#pragma unroll
        for (int i = 0; i < L::kPer / 4; ++i) {
            const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&at[(which * (L::kPer / 4) + i) * width]);
            f[2 * i].v = v.x;
            f[2 * i + 1].v = v.y;
        }
    }
};

// The rows of threads of a CTA: within warps (kWarp: up to 32 each), or of 64 and more.  The rows of a warp are walked together.
template <bool kWarp>
struct Team {
    int threads, j, group, groups;
    __device__ __forceinline__ explicit Team(int threads_) : threads(threads_) {
        j = threadIdx.x % threads;
        group = threadIdx.x / threads;
        groups = blockDim.x / threads;
    }
    // the first row that a thread of the warp walks: the loop goes on as long as it is there
    __device__ __forceinline__ int64_t warp_row(int64_t row) const {
        return kWarp ? row - (threadIdx.x % 32) / threads : row;
    }
};

// Sums over the threads of a row.  They use two areas in turn, so that one barrier a sum is enough: an area is written again
// behind the barrier of the sum in between.
template <bool kWarp>
struct RowSum {
    float (&room)[2][32];
    const Team<kWarp>& me;
    int side;
    __device__ __forceinline__ float operator()(Lanes pair) {
        float v = pair.at(0) + pair.at(1);
        if constexpr (kWarp) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                if (o < me.threads) v += __shfl_xor_sync(0xffffffffu, v, o);
        } else {
            v = warp_sum(v);
            const int warps = me.threads / 32;
            float* at = room[side] + me.group * warps;
            side ^= 1;
            if (me.j % 32 == 0) at[me.j / 32] = v;
            asm volatile("bar.sync %0, %1;" ::"r"(me.group + 1), "r"(me.threads) : "memory");
            v = 0.0f;
            for (int w = 0; w < warps; w += 2) v += at[w] + at[w + 1];
        }
        return v;
    }
};

template <typename T, int V>
__device__ __forceinline__ void gates_of(const Slice<T, V>& g, bool has, Lanes (&on)[Layout<T, V>::kPairs]) {
#pragma unroll
    for (int i = 0; i < Layout<T, V>::kPairs; ++i) {
        float s[2] = {1.0f, 1.0f}, rest;
        if (has) {
            logistic(g.at(2 * i), s[0], rest);
            logistic(g.at(2 * i + 1), s[1], rest);
        }
        on[i] = lanes(s);
    }
}

template <typename T, int V, bool kWarp, int kMost, bool kStaged>
__global__ void __launch_bounds__(kMost, kMost == 256 ? 3 : kMost == 384 ? 2 : 1) norm_forward_kernel(const NormArgs p) {
    using L = Layout<T, V>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float room[2][32];
    const Team<kWarp> me(p.threads);
    RowSum<kWarp> row_sum{room, me, 0};
    pdl_wait();
    Weights<T, V> weights{reinterpret_cast<float4*>(dynamic) + me.j, me.threads};
    const int64_t first = (int64_t)blockIdx.x * me.groups + me.group, step = (int64_t)gridDim.x * me.groups;
    using R = Rows<T, V, 3, kStaged>;
    R rows{{static_cast<const T*>(p.x), static_cast<const T*>(p.block), static_cast<const T*>(p.gate)},
           {p.x_row, p.block_row, p.gate_row},
           p.rows, step, me.j, me.threads, p.channels,
           dynamic + me.threads * Weights<T, V>::kBytes + R::offset_of(threadIdx.x, me.threads),
           R::width_of(blockDim.x, me.threads)};
    rows.begin(first);
    if (me.group == 0) weights.put(p, me.j, me.threads);
    __syncthreads();
    for (int64_t row = first; me.warp_row(row) < p.rows; row += step) {
        rows.next(row);
        const Slice<T, V> x = rows.get(0);
        Lanes s[L::kPairs], w[L::kPairs], sum = all_lanes(0.0f);
        float r = 0.0f;
        if (p.block != nullptr) {
            const Slice<T, V> y = rows.get(1);
            gates_of<T, V>(rows.get(2), p.gate != nullptr, s);
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) sum = fma(y.pair(i), y.pair(i), sum);
            r = rsqrtf(row_sum(sum) * p.inv + p.eps);
            weights.get(0, w);
            sum = all_lanes(0.0f);
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) {
                s[i] = fma(w[i] * s[i], y.pair(i) * all_lanes(r), x.pair(i));
                sum = fma(s[i], s[i], sum);
            }
            put<T, V>(p.stream, row * p.channels, s, me.j, me.threads, rows.live ? p.channels : 0);
        } else {
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) {
                s[i] = x.pair(i);
                sum = fma(s[i], s[i], sum);
            }
        }
        const float q = rsqrtf(row_sum(sum) * p.inv + p.eps);
        weights.get(1, w);
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) s[i] = s[i] * all_lanes(q) * w[i];
        put<T, V>(p.normed, row * p.channels, s, me.j, me.threads, rows.live ? p.channels : 0);
        if (p.stats != nullptr && me.j == 0 && rows.live) {
            p.stats[2 * row] = r;
            p.stats[2 * row + 1] = q;
        }
    }
    if constexpr (kStaged) copies_arrived<0>();
}

template <typename T, int V, bool kWarp, int kMost, bool kStaged>
__global__ void __launch_bounds__(kMost, kMost == 256 ? 2 : 1) norm_backward_kernel(const NormArgs p) {
    using L = Layout<T, V>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float room[2][32];
    const Team<kWarp> me(p.threads);
    RowSum<kWarp> row_sum{room, me, 0};
    pdl_wait();
    Weights<T, V> weights{reinterpret_cast<float4*>(dynamic) + me.j, me.threads};
    const int64_t first = (int64_t)blockIdx.x * me.groups + me.group, step = (int64_t)gridDim.x * me.groups;
    using R = Rows<T, V, 5, kStaged>;
    R rows{{static_cast<const T*>(p.x), static_cast<const T*>(p.block), static_cast<const T*>(p.gate),
            static_cast<const T*>(p.dstream), static_cast<const T*>(p.dnormed)},
           {p.x_row, p.block_row, p.gate_row, p.dstream_row, p.dnormed_row},
           p.rows, step, me.j, me.threads, p.channels,
           dynamic + me.threads * Weights<T, V>::kBytes + R::offset_of(threadIdx.x, me.threads),
           R::width_of(blockDim.x, me.threads)};
    rows.begin(first);
    if (me.group == 0) weights.put(p, me.j, me.threads);
    __syncthreads();
    Lanes z[L::kPairs], dpre[L::kPairs];
#pragma unroll
    for (int i = 0; i < L::kPairs; ++i) z[i] = dpre[i] = all_lanes(0.0f);
    float next_r = 0.0f, next_q = 0.0f;
    auto fetch_stats = [&](int64_t row) {
        if (row >= p.rows) return;
        next_r = gload(p.stats + 2 * row);
        next_q = gload(p.stats + 2 * row + 1);
    };
    fetch_stats(first);
    for (int64_t row = first; me.warp_row(row) < p.rows; row += step) {
        const float r = next_r, q = next_q;
        fetch_stats(row + step);
        rows.next(row);
        const Slice<T, V> y = rows.get(1);
        const Lanes rr = all_lanes(r), qq = all_lanes(q);
        Lanes on[L::kPairs], sn[L::kPairs], d[L::kPairs], w[L::kPairs], sum = all_lanes(0.0f);
        gates_of<T, V>(rows.get(2), p.gate != nullptr, on);
        const Slice<T, V> x = rows.get(0);
        if (p.block != nullptr) {
            weights.get(0, w);
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) sn[i] = fma(w[i] * on[i], y.pair(i) * rr, x.pair(i)) * qq;
        } else {
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) sn[i] = x.pair(i) * qq;
        }
        const Slice<T, V> dn = rows.get(4);
        weights.get(1, w);
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) {
            dpre[i] = fma(dn.pair(i), sn[i], dpre[i]);
            d[i] = dn.pair(i) * w[i];
            sum = fma(d[i], sn[i], sum);
        }
        const Lanes m = all_lanes(-row_sum(sum) * p.inv);
        const Slice<T, V> ds = rows.get(3);
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) d[i] = fma(qq, fma(sn[i], m, d[i]), ds.pair(i));
        put<T, V>(p.dx, row * p.channels, d, me.j, me.threads, rows.live ? p.channels : 0);
        if (p.block == nullptr) continue;
        weights.get(0, w);
        sum = all_lanes(0.0f);
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) {
            const Lanes yn = y.pair(i) * rr, u = d[i] * on[i];
            z[i] = fma(u, yn, z[i]);
            sn[i] = u * w[i];                    // the gradient of yn from here on
            sum = fma(sn[i], yn, sum);
        }
        const Lanes n = all_lanes(-row_sum(sum) * p.inv);
#pragma unroll
        for (int i = 0; i < L::kPairs; ++i) d[i] = rr * fma(y.pair(i) * rr, n, sn[i]);
        put<T, V>(p.dblock, row * p.channels, d, me.j, me.threads, rows.live ? p.channels : 0);
        if (p.dgate != nullptr) {
            const Slice<T, V> g = rows.get(2);
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) {
                float off[2], s;
                logistic(g.at(2 * i), s, off[0]);
                logistic(g.at(2 * i + 1), s, off[1]);
                d[i] = sn[i] * (y.pair(i) * rr) * lanes(off);
            }
            put<T, V>(p.dgate, row * p.channels, d, me.j, me.threads, rows.live ? p.channels : 0);
        }
    }
    if constexpr (kStaged) copies_arrived<0>();
    if (p.partial == nullptr) return;
    // the rows of threads add theirs up: those of a warp as a tree, the others in order (over the weights)
    int rows_left = me.groups, mine = me.group;
    if constexpr (kWarp) {
#pragma unroll
        for (int o = 16; o >= 4; o >>= 1) {
            if (o < me.threads) break;
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) z[i] = z[i] + shuffle_xor(z[i], o), dpre[i] = dpre[i] + shuffle_xor(dpre[i], o);
        }
        rows_left = blockDim.x / 32, mine = threadIdx.x % 32 < me.threads ? threadIdx.x / 32 : -1;
    }
    Lanes* all = reinterpret_cast<Lanes*>(dynamic) + me.j;
    for (int k = 0; k < rows_left; ++k) {
        __syncthreads();
        if (k == mine)
#pragma unroll
            for (int i = 0; i < L::kPairs; ++i) {
                if (k > 0) z[i] = all[2 * i * me.threads] + z[i], dpre[i] = all[(2 * i + 1) * me.threads] + dpre[i];
                all[2 * i * me.threads] = z[i], all[(2 * i + 1) * me.threads] = dpre[i];
            }
    }
    if (mine != rows_left - 1) return;
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.channels;
#pragma unroll
    for (int e = 0; e < L::kPer; ++e) {
        const int at = L::element(me.j, me.threads, e);
        if (at < p.channels) {
            out[at] = z[e / 2].at(e % 2);
            out[p.channels + at] = dpre[e / 2].at(e % 2);
        }
    }
}

// Column sums of the partial sums [n][2][channels]: 32 columns a CTA, 32 threads a column.
template <typename T>
__global__ void __launch_bounds__(1024) norm_weights_kernel(const float* partial, int n, int channels, const void* scale,
                                                            const void* post, void* dscale, void* dpost, void* dpre, int wide) {
    __shared__ float room[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x, which = blockIdx.y;
    pdl_wait();
    float sum = 0.0f;
    if (c < channels)
        for (int i = threadIdx.y; i < n; i += 32) sum += gload(partial + ((int64_t)i * 2 + which) * channels + c);
    room[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    sum = warp_sum(room[threadIdx.x][threadIdx.y]);
    const int at = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x != 0 || at >= channels) return;
    auto put_weight = [&](void* out, float v) {
        if (out == nullptr) return;
        if (wide) static_cast<float*>(out)[at] = v;
        else static_cast<T*>(out)[at] = from_float<T>(v);
    };
    if (which == 0) {
        put_weight(dscale, sum * weight_at<T>(post, at, wide));
        put_weight(dpost, sum * weight_at<T>(scale, at, wide));
    } else {
        put_weight(dpre, sum);
    }
}

// Threads of a row: a power of two up to 256, which share a CTA of 256, then a multiple of 64, so that few are idle and an SM holds
// two rows up to 384 (16384x4480 bf16, forward and backward: 169 and 354 us; 280 and 453 us with 512 threads a row)
int threads_of(int64_t channels, int elem) {
    const int64_t wanted = (channels * elem + 31) / 32;
    if (wanted > 256) return (int)((wanted + 63) / 64 * 64);
    int t = 4;
    while (t < wanted) t *= 2;
    return t;
}

// Threads of a CTA: 256, in rows of t, or one row of more
int cta_of(int t) { return t > 256 ? t : 256; }

// CTAs: as many as the SMs hold at once (so many threads by registers, and `smem` a CTA), and no more than there are rows for: one
// more would start when others end, and walk its rows alone (16384x4096 bf16, forward: 137 us, 156 us with a third CTA an SM).
constexpr int kForwardThreads = 768, kBackwardThreads = 512;

unsigned grid_of(int64_t rows, int64_t channels, int elem, int threads_an_sm, size_t smem = 0) {
    const int t = threads_of(channels, elem), cta = cta_of(t);
    const int64_t units = (rows + cta / t - 1) / (cta / t);
    const int held = std::max(1, std::min(threads_an_sm / cta, (int)(228 * 1024 / (smem + 1024))));
    const int64_t most = (int64_t)sm_count() * held;
    return (unsigned)(units < most ? units : most);
}

// `most`: the shared memory of the kernel's largest CTA.  It is what is asked for at every launch, so that calls of several host
// threads do not take it from one another.
template <typename K>
int launch(K kernel, unsigned grid, int cta, size_t smem, int most, const NormArgs& a, cudaStream_t st) {
    if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
        return DCN_ERR_CUDA;
    return launch_dependent(kernel, dim3(grid), dim3(cta), smem, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int V, bool kWarp, int kMost>
int run_as(const NormArgs& a, bool backward, cudaStream_t st) {
    // two rows of every tensor in shared memory where an SM has room for as many threads
    constexpr int kSM = 226 * 1024, kWeights = kMost * Weights<T, V>::kBytes, kSegments = kMost / (kWarp ? 4 : 32);
    using F = Rows<T, V, 3, true>;
    using B = Rows<T, V, 5, true>;
    constexpr int kForward = kMost * F::kBytes + kSegments * F::kExtra, kBackward = kMost * B::kBytes + kSegments * B::kExtra;
    constexpr bool f = kForward + kWeights <= kSM, b = kBackward + kWeights <= kSM;
    const int cta = cta_of(a.threads), segments = cta / (a.threads < 32 ? a.threads : 32);
    const size_t weights = (size_t)a.threads * Weights<T, V>::kBytes;
    if (backward)
        return launch(norm_backward_kernel<T, V, kWarp, kMost, b>, grid_of(a.rows, a.channels, sizeof(T), kBackwardThreads), cta,
                      weights + (b ? cta * B::kBytes + segments * B::kExtra : 0), kWeights + (b ? kBackward : 0), a, st);
    const size_t smem = weights + (f ? cta * F::kBytes + segments * F::kExtra : 0);
    return launch(norm_forward_kernel<T, V, kWarp, kMost, f>, grid_of(a.rows, a.channels, sizeof(T), kForwardThreads, smem), cta,
                  smem, kWeights + (f ? kForward : 0), a, st);
}

template <typename T, int V>
int run(NormArgs a, bool backward, cudaStream_t st) {
    a.threads = threads_of(a.channels, sizeof(T));
    if (a.threads <= 32) return run_as<T, V, true, 256>(a, backward, st);
    if (a.threads <= 256) return run_as<T, V, false, 256>(a, backward, st);
    if (a.threads <= 384) return run_as<T, V, false, 384>(a, backward, st);
    if constexpr (sizeof(T) == 4)
        if (a.threads > 512) return run_as<T, V, false, 1024>(a, backward, st);
    return run_as<T, V, false, 512>(a, backward, st);
}

template <typename T>
int run_weights(const NormArgs& a, int elem, void* dscale, void* dpost, void* dpre, cudaStream_t st) {
    const dim3 grid((a.channels + 31) / 32, 2), block(32, 32);
    const int n = (int)grid_of(a.rows, a.channels, elem, kBackwardThreads);
    return launch_dependent(norm_weights_kernel<T>, grid, block, 0, st, a.partial, n, a.channels, a.scale, a.post, dscale, dpost,
                            dpre, a.wide_weights) != cudaSuccess
               ? DCN_ERR_CUDA
               : DCN_OK;
}

int check_norm(const dcn_norm* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype) || (p->weight_dtype != DCN_SEQ_F32 && p->weight_dtype != p->dtype)) return DCN_ERR_UNSUPPORTED;
    if (p->rows < 0 || p->channels < 1) return DCN_ERR_SHAPE;
    if (p->rows >= 1ll << 31 || p->channels > kMostChannels) return DCN_ERR_LIMIT;
    return DCN_OK;
}

NormArgs args_of(const dcn_norm* p) {
    NormArgs a = {};
    a.rows = p->rows;
    a.channels = (int)p->channels;
    a.x_row = p->x_row, a.block_row = p->block_row, a.gate_row = p->gate_row;
    a.dstream_row = p->dstream_row, a.dnormed_row = p->dnormed_row;
    a.wide_weights = p->weight_dtype == DCN_SEQ_F32;
    a.eps = p->eps;
    a.inv = 1.0f / (float)p->channels;
    return a;
}

// Elements of a vector: 16 bytes, 8 or 4 where every row of every tensor starts on as many, one element otherwise (of which 16-bit
// ones move two at a time all the same).
struct Vector {
    int n, elem;
    explicit Vector(const dcn_norm* p) : n(16 / elem_bytes(p->dtype)), elem(elem_bytes(p->dtype)) {}
    void by(const void* v, int64_t row) {
        while (v != nullptr && n > 1 && (!aligned(v, n * elem) || row % n != 0)) n /= 2;
    }
};

template <typename T>
int run_16(int n, const NormArgs& a, bool backward, cudaStream_t st) {
    return n == 8   ? run<T, 8>(a, backward, st)
           : n == 4 ? run<T, 4>(a, backward, st)
           : n == 2 ? run<T, 2>(a, backward, st)
                    : run<T, 1>(a, backward, st);
}

int run_any(int dtype, int n, const NormArgs& a, bool backward, cudaStream_t st) {
    if (dtype == DCN_SEQ_F32)
        return n == 4   ? run<float, 4>(a, backward, st)
               : n == 2 ? run<float, 2>(a, backward, st)
                        : run<float, 1>(a, backward, st);
    if (dtype == DCN_SEQ_BF16) return run_16<__nv_bfloat16>(n, a, backward, st);
    return run_16<__half>(n, a, backward, st);
}

}  // namespace
}  // namespace seq
}  // namespace dcn

using namespace dcn::seq;

extern "C" int dcn_norm_forward(const dcn_norm* p, const void* x, const void* block, const void* gate, const void* scale,
                                const void* post, const void* pre, void* stream_out, void* normed, float* stats, void* stream) {
    const int bad = check_norm(p);
    if (bad != DCN_OK) return bad;
    if (p->rows == 0) return DCN_OK;
    if (x == nullptr || normed == nullptr || (block != nullptr) != (stream_out != nullptr)) return DCN_ERR_NULL;
    const int e = elem_bytes(p->dtype), we = elem_bytes(p->weight_dtype);
    for (const void* v : {x, block, gate, (const void*)stream_out, (const void*)normed})
        if (!aligned(v, e)) return DCN_ERR_ALIGN;
    for (const void* v : {scale, post, pre})
        if (!aligned(v, we)) return DCN_ERR_ALIGN;
    if (!aligned(stats, 4)) return DCN_ERR_ALIGN;
    NormArgs a = args_of(p);
    a.x = x, a.block = block, a.gate = block != nullptr ? gate : nullptr, a.scale = scale, a.post = post, a.pre = pre;
    a.stream = stream_out, a.normed = normed, a.stats = stats;
    Vector vec(p);
    vec.by(x, p->x_row), vec.by(block, p->block_row), vec.by(a.gate, p->gate_row);
    vec.by(stream_out, p->channels), vec.by(normed, p->channels);          // (so the channels are whole vectors too)
    const cudaStream_t st = (cudaStream_t)stream;
    return run_any(p->dtype, vec.n, a, false, st);
}

extern "C" size_t dcn_norm_workspace_bytes(const dcn_norm* p) {
    if (check_norm(p) != DCN_OK) return 0;
    return (size_t)grid_of(p->rows, p->channels, elem_bytes(p->dtype), kBackwardThreads) * 2 * p->channels * sizeof(float);
}

extern "C" int dcn_norm_backward(const dcn_norm* p, const void* x, const void* block, const void* gate, const void* scale,
                                 const void* post, const void* pre, const float* stats, const void* dstream,
                                 const void* dnormed, void* dx, void* dblock, void* dgate, void* dscale, void* dpost, void* dpre,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_norm(p);
    if (bad != DCN_OK) return bad;
    const bool weights = dscale != nullptr || dpost != nullptr || dpre != nullptr;
    const cudaStream_t st = (cudaStream_t)stream;
    const int e = elem_bytes(p->dtype), we = elem_bytes(p->weight_dtype);
    for (const void* v : {scale, post, pre, (const void*)dscale, (const void*)dpost, (const void*)dpre})
        if (!aligned(v, we)) return DCN_ERR_ALIGN;
    if (p->rows == 0) {
        for (void* v : {dscale, dpost, dpre})
            if (v != nullptr && cudaMemsetAsync(v, 0, (size_t)p->channels * we, st) != cudaSuccess) return DCN_ERR_CUDA;
        return DCN_OK;
    }
    if (x == nullptr || stats == nullptr || (block == nullptr && (dblock != nullptr || dgate != nullptr)) ||
        (gate == nullptr && dgate != nullptr))
        return DCN_ERR_NULL;
    for (const void* v : {x, block, gate, dstream, dnormed, (const void*)dx, (const void*)dblock, (const void*)dgate})
        if (!aligned(v, e)) return DCN_ERR_ALIGN;
    if (!aligned(stats, 4)) return DCN_ERR_ALIGN;
    if (weights && (workspace == nullptr || !aligned(workspace, 4) || workspace_bytes < dcn_norm_workspace_bytes(p)))
        return DCN_ERR_WORKSPACE;
    NormArgs a = args_of(p);
    a.x = x, a.block = block, a.gate = block != nullptr ? gate : nullptr, a.scale = scale, a.post = post, a.pre = pre;
    a.stats = const_cast<float*>(stats), a.dstream = dstream, a.dnormed = dnormed;
    a.dx = dx, a.dblock = dblock, a.dgate = dgate;
    a.partial = weights ? static_cast<float*>(workspace) : nullptr;
    Vector vec(p);
    vec.by(x, p->x_row), vec.by(block, p->block_row), vec.by(a.gate, p->gate_row);
    vec.by(dstream, p->dstream_row), vec.by(dnormed, p->dnormed_row);
    vec.by(x, p->channels);                      // (channels are whole vectors)
    vec.by(dx, p->channels), vec.by(dblock, p->channels), vec.by(dgate, p->channels);
    const int rc = run_any(p->dtype, vec.n, a, true, st);
    if (rc != DCN_OK || !weights) return rc;
    if (p->dtype == DCN_SEQ_F32) return run_weights<float>(a, e, dscale, dpost, dpre, st);
    if (p->dtype == DCN_SEQ_BF16) return run_weights<__nv_bfloat16>(a, e, dscale, dpost, dpre, st);
    return run_weights<__half>(a, e, dscale, dpost, dpre, st);
}
