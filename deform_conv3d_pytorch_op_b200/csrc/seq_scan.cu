// Gated linear recurrence over time, per channel:
//     a_t = s(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t          (s the logistic function)
// and its gradient.  With p_t the gradient that step t passes to the state before it,
//     p_t = a_t p_{t+1} + a_t dy_t   (p behind the last step: dlast),   D_t = dy_t + p_{t+1}
//     dx_t = D_t (1 - a_t),   dgate_t = D_t (h_{t-1} - x_t) a_t (1 - a_t),   dstate = p_0.
//
// A gate near one is the common case, and 1 - a is what matters of it: a state that lasts 10^4 steps would lose all of its
// digits to the rounding of a.  So a step is known by q = min(a, 1 - a) and which of the two it is, as one signed float s (-q for
// a = 1 - q, q for a = q), and every product with a is a sum with the product with q: a u = fma(s, u, s < 0 ? u : 0).
//
// Both directions are scans of affine maps h -> A h + B, whose composition is (A2 A1, A2 B1 + B2), A kept in the same form.  A thread holds kSteps steps of W
// channels in registers: it composes its steps, the warps of a CTA (one behind the other in time) compose theirs through shared
// memory and the CTAs of a cluster theirs through distributed shared memory; then every thread walks its steps once more from
// the state that reaches it.  So x and gate are read once and y is written once, whatever the length: the bound is DRAM.  A
// cluster walks the time axis in waves of (its CTAs) x 64 steps and carries the state from wave to wave in registers.
// The forward pass leaves the state before every 64th step; the backward pass recomputes the states in between from it, in
// float32, and reads no y: 4 bytes in 64 steps instead of an activation per step, and no rounded state in a gradient.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace cg = cooperative_groups;

namespace dcn {
namespace seq {
namespace {

constexpr int kSteps = 8;                        // of a thread
constexpr int kWarps = 8;                        // of a CTA, at most
constexpr int kChunk = kSteps * kWarps;          // steps between checkpoints
constexpr int kCluster = 8;                      // CTAs of a cluster, at most

struct ScanArgs {
    const void *x, *gate, *dy;
    const float *state, *dlast;
    const int64_t* lengths;
    void *y, *dx, *dgate;
    float *last, *dstate, *checkpoints;
    int64_t steps, channels, chunks;
    int64_t x_batch, x_step, gate_batch, gate_step, dy_batch, dy_step;
    int tiles;                                   // of 32 W channels
};

__device__ __forceinline__ bool near_one(float s) { return __float_as_int(s) < 0; }

// s of a gate; -0, a step that keeps the state as it is, outside the sequence
__device__ __forceinline__ float step_of(float gate, bool in) {
    const float t = __expf(-fabsf(gate)), q = t * __fdividef(1.0f, 1.0f + t);
    const uint32_t s = __float_as_uint(q) | (~__float_as_uint(gate) & 0x80000000u);
    return in ? __uint_as_float(s) : -0.0f;
}
// a u, and a h + (1 - a) x
__device__ __forceinline__ float times(float s, float u) { return fmaf(s, u, near_one(s) ? u : 0.0f); }
__device__ __forceinline__ float advance(float s, float h, float x) { return fmaf(s, h - x, near_one(s) ? h : x); }

// The product of gates, as A and as 1 - A: each is a sum or product of positive terms, so neither loses digits
struct Product {
    float a = 1.0f, rest = 0.0f;
    __device__ __forceinline__ void by(float s) {
        rest = fmaf(-s, a, near_one(s) ? rest : 1.0f);
        a = times(s, a);
    }
    __device__ __forceinline__ float signed_form() const { return rest < 0.5f ? -rest : a; }
};

// Where a thread works
template <int W>
struct Place {
    int lane, warp, warps, rank, ranks;
    int64_t b, c;
    bool live;
    __device__ __forceinline__ explicit Place(const ScanArgs& p) {
        const cg::cluster_group cluster = cg::this_cluster();
        lane = threadIdx.x;
        warp = threadIdx.y;
        warps = blockDim.y;
        rank = (int)cluster.block_rank();
        ranks = (int)cluster.num_blocks();
        const unsigned unit = blockIdx.x / ranks;
        b = unit / p.tiles;
        c = (int64_t)(unit % p.tiles) * 32 * W + lane * W;
        live = c < p.channels;
    }
};

__device__ __forceinline__ int64_t length_of(const ScanArgs& p, int64_t b) {
    if (p.lengths == nullptr) return p.steps;
    const int64_t n = gload_i64(p.lengths + b);
    return n < 0 ? 0 : n > p.steps ? p.steps : n;
}

template <int W>
__device__ __forceinline__ void load_state(float (&h)[W], const float* s, int64_t at, bool live) {
#pragma unroll
    for (int i = 0; i < W; ++i) h[i] = s != nullptr && live ? gload(s + at + i) : 0.0f;
}

// kSteps packs from step t0 on; zeros where there is none
template <typename T, int W>
__device__ __forceinline__ void load_steps(Pack<T, W> (&v)[kSteps], const T* base, int64_t t0, int64_t stride, int64_t len,
                                           bool live) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        v[k].zero();
        if (live && t0 + k < len) v[k].get(base + (t0 + k) * stride);
    }
}

// Zeros from step `from` on, shared out over the warps of the cluster
template <typename T, int W>
__device__ __forceinline__ void zero_rest(const Place<W>& me, T* out, int64_t from, int64_t steps, int64_t channels) {
    Pack<T, W> z;
    z.zero();
    if (me.live)
        for (int64_t t = from + me.rank * me.warps + me.warp; t < steps; t += me.ranks * me.warps) z.put(out + t * channels);
}

template <typename T, int W>
__global__ void __launch_bounds__(32 * kWarps, 3) scan_forward_kernel(const ScanArgs p) {
    // maps (A, B) of the warps and of the cluster's CTAs; two of each, so that a wave's are read while the next one's are written
    __shared__ float2 part[2][kWarps][W][32];
    __shared__ float2 whole[2][kCluster][W][32];
    const Place<W> me(p);
    pdl_wait();
    const int64_t len = length_of(p, me.b);
    const T* x = static_cast<const T*>(p.x) + me.b * p.x_batch + me.c;
    const T* gate = static_cast<const T*>(p.gate) + me.b * p.gate_batch + me.c;
    T* y = static_cast<T*>(p.y) + me.b * p.steps * p.channels + me.c;
    float carry[W];
    load_state<W>(carry, p.state, me.b * p.channels + me.c, me.live);

    const int chunk = me.warps * kSteps, wave = me.ranks * chunk;
    int64_t t0 = (int64_t)me.rank * chunk + me.warp * kSteps;      // my first step of this wave
    Pack<T, W> rx[kSteps], rg[kSteps];
    load_steps(rx, x, t0, p.x_step, len, me.live);
    load_steps(rg, gate, t0, p.gate_step, len, me.live);
    if (me.ranks > 1) cg::this_cluster().sync();                   // every CTA runs before another writes to its memory
    int side = 0;
    int64_t begin = 0;
    for (; begin < len; begin += wave, t0 += wave, side ^= 1) {
        float s[kSteps][W], v[kSteps][W], B[W];
        Product A[W];
#pragma unroll
        for (int i = 0; i < W; ++i) B[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                s[k][i] = step_of(rg[k].at(i), t0 + k < len);
                v[k][i] = rx[k].at(i);
                A[i].by(s[k][i]);
                B[i] = advance(s[k][i], B[i], v[k][i]);
            }
        load_steps(rx, x, t0 + wave, p.x_step, len, me.live);      // the next wave's, in flight during what follows
        load_steps(rg, gate, t0 + wave, p.gate_step, len, me.live);
#pragma unroll
        for (int i = 0; i < W; ++i) part[side][me.warp][i][me.lane] = make_float2(A[i].signed_form(), B[i]);
        __syncthreads();
        float h[W];
        if (me.ranks > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (me.warp == 0) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    Product a;
                    float sum = 0.0f;
                    for (int w = 0; w < me.warps; ++w) {
                        const float2 n = part[side][w][i][me.lane];
                        a.by(n.x);
                        sum = times(n.x, sum) + n.y;
                    }
                    const float2 m = make_float2(a.signed_form(), sum);
                    for (int r = 0; r < me.ranks; ++r) *cluster.map_shared_rank(&whole[side][me.rank][i][me.lane], r) = m;
                }
            }
            cluster.sync();
#pragma unroll
            for (int i = 0; i < W; ++i) h[i] = carry[i];
            for (int r = 0; r < me.ranks; ++r)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float2 m = whole[side][r][i][me.lane];
                    if (r == me.rank) h[i] = carry[i];
                    carry[i] = times(m.x, carry[i]) + m.y;
                }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) h[i] = carry[i];
        }
        if (p.checkpoints != nullptr && me.warp == 0 && me.live && t0 < len) {
            float* at = p.checkpoints + (me.b * p.chunks + t0 / kChunk) * p.channels + me.c;
#pragma unroll
            for (int i = 0; i < W; ++i) at[i] = h[i];
        }
        // from the state before the CTA's steps to the one before mine; a cluster of one also finds the state behind them here
        const int upto = me.ranks > 1 ? me.warp : me.warps;
        float mine[W];
#pragma unroll
        for (int i = 0; i < W; ++i) mine[i] = h[i];
        for (int w = 0; w < upto; ++w)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float2 m = part[side][w][i][me.lane];
                if (w == me.warp) mine[i] = h[i];
                h[i] = times(m.x, h[i]) + m.y;
            }
        if (me.ranks > 1) {
#pragma unroll
            for (int i = 0; i < W; ++i) mine[i] = h[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) carry[i] = h[i];
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const int64_t t = t0 + k;
            float out[W];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                mine[i] = advance(s[k][i], mine[i], v[k][i]);
                out[i] = t < len ? mine[i] : 0.0f;
            }
            Pack<T, W> to;
            to.set(out);
            if (me.live && t < p.steps) to.put(y + t * p.channels);
        }
    }
    zero_rest(me, y, begin, p.steps, p.channels);
    if (me.rank == 0 && me.warp == 0 && me.live) {
#pragma unroll
        for (int i = 0; i < W; ++i) p.last[me.b * p.channels + me.c + i] = carry[i];
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(32 * kWarps, 2) scan_backward_kernel(const ScanArgs p) {
    // of a warp: the product A of its gates (signed), the B of its forward map and the P of its backward map p -> A p + P
    __shared__ float part[2][kWarps][3][W][32];
    __shared__ float2 whole[2][kCluster][W][32];                   // (A, P) of the cluster's CTAs
    const Place<W> me(p);
    pdl_wait();
    const int64_t len = length_of(p, me.b);
    const T* x = static_cast<const T*>(p.x) + me.b * p.x_batch + me.c;
    const T* gate = static_cast<const T*>(p.gate) + me.b * p.gate_batch + me.c;
    const T* dy = static_cast<const T*>(p.dy) + me.b * p.dy_batch + me.c;
    T* dx = static_cast<T*>(p.dx) + me.b * p.steps * p.channels + me.c;
    T* dgate = static_cast<T*>(p.dgate) + me.b * p.steps * p.channels + me.c;
    float carry[W];
    load_state<W>(carry, p.dlast, me.b * p.channels + me.c, me.live);
    const bool has_dy = p.dy != nullptr && me.live;

    const int chunk = me.warps * kSteps, wave = me.ranks * chunk;
    const int64_t end = (len + wave - 1) / wave * wave;
    int64_t t0 = end - wave + (int64_t)me.rank * chunk + me.warp * kSteps;
    Pack<T, W> rx[kSteps], rg[kSteps], rd[kSteps];
    if (end > 0) {
        load_steps(rx, x, t0, p.x_step, len, me.live);
        load_steps(rg, gate, t0, p.gate_step, len, me.live);
        load_steps(rd, dy, t0, p.dy_step, len, has_dy);
    }
    if (me.ranks > 1) cg::this_cluster().sync();                   // every CTA runs before another writes to its memory
    int side = 0;
    for (int64_t begin = end - wave; begin >= 0; begin -= wave, t0 -= wave, side ^= 1) {
        float before[W];                                           // the state before the CTA's steps
        load_state<W>(before, p.checkpoints, (me.b * p.chunks + (t0 - me.warp * kSteps) / kChunk) * p.channels + me.c,
                      me.live && t0 - me.warp * kSteps < len);
        float s[kSteps][W], d[kSteps][W], h[kSteps][W];
        Pack<T, W> cx[kSteps];
        float B[W], P[W];
        Product A[W];
#pragma unroll
        for (int i = 0; i < W; ++i) B[i] = 0.0f, P[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            cx[k] = rx[k];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                s[k][i] = step_of(rg[k].at(i), t0 + k < len);
                d[k][i] = rd[k].at(i);
                A[i].by(s[k][i]);
                B[i] = advance(s[k][i], B[i], cx[k].at(i));
            }
        }
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k)
#pragma unroll
            for (int i = 0; i < W; ++i) P[i] = times(s[k][i], d[k][i] + P[i]);
        if (begin > 0) {
            load_steps(rx, x, t0 - wave, p.x_step, len, me.live);
            load_steps(rg, gate, t0 - wave, p.gate_step, len, me.live);
            load_steps(rd, dy, t0 - wave, p.dy_step, len, has_dy);
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            part[side][me.warp][0][i][me.lane] = A[i].signed_form();
            part[side][me.warp][1][i][me.lane] = B[i];
            part[side][me.warp][2][i][me.lane] = P[i];
        }
        __syncthreads();
        float g[W];                                                // the gradient that reaches the CTA's last step
#pragma unroll
        for (int i = 0; i < W; ++i) g[i] = carry[i];
        if (me.ranks > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (me.warp == 0) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    Product a;
                    float sum = 0.0f;
                    for (int w = me.warps - 1; w >= 0; --w) {
                        const float n = part[side][w][0][i][me.lane];
                        a.by(n);
                        sum = times(n, sum) + part[side][w][2][i][me.lane];
                    }
                    const float2 m = make_float2(a.signed_form(), sum);
                    for (int r = 0; r < me.ranks; ++r) *cluster.map_shared_rank(&whole[side][me.rank][i][me.lane], r) = m;
                }
            }
            cluster.sync();
            for (int r = me.ranks - 1; r >= 0; --r)
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float2 m = whole[side][r][i][me.lane];
                    if (r == me.rank) g[i] = carry[i];
                    carry[i] = times(m.x, carry[i]) + m.y;
                }
        }
        for (int w = 0; w < me.warp; ++w)
#pragma unroll
            for (int i = 0; i < W; ++i) before[i] = times(part[side][w][0][i][me.lane], before[i]) + part[side][w][1][i][me.lane];
        const int down = me.ranks > 1 ? me.warp + 1 : 0;
        float mine[W];
#pragma unroll
        for (int i = 0; i < W; ++i) mine[i] = g[i];
        for (int w = me.warps - 1; w >= down; --w)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (w == me.warp) mine[i] = g[i];
                g[i] = times(part[side][w][0][i][me.lane], g[i]) + part[side][w][2][i][me.lane];
            }
        if (me.ranks > 1) {
#pragma unroll
            for (int i = 0; i < W; ++i) mine[i] = g[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) carry[i] = g[i];
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i) {
                h[k][i] = before[i];
                before[i] = advance(s[k][i], before[i], cx[k].at(i));
            }
#pragma unroll
        for (int k = kSteps - 1; k >= 0; --k) {
            const int64_t t = t0 + k;
            float ox[W], og[W];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const float D = d[k][i] + mine[i], q = fabsf(s[k][i]);
                ox[i] = D * (near_one(s[k][i]) ? q : 1.0f - q);
                og[i] = D * (h[k][i] - cx[k].at(i)) * fmaf(-q, q, q);
                mine[i] = times(s[k][i], D);
                if (t >= len) ox[i] = og[i] = 0.0f;
            }
            Pack<T, W> vx, vg;
            vx.set(ox);
            vg.set(og);
            if (me.live && t < p.steps) {
                vx.put(dx + t * p.channels);
                vg.put(dgate + t * p.channels);
            }
        }
    }
    zero_rest(me, dx, end, p.steps, p.channels);
    zero_rest(me, dgate, end, p.steps, p.channels);
    if (p.dstate != nullptr && me.rank == 0 && me.warp == 0 && me.live) {
#pragma unroll
        for (int i = 0; i < W; ++i) p.dstate[me.b * p.channels + me.c + i] = carry[i];
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(128) scan_step_kernel(int64_t rows, int64_t channels, const T* x, int64_t x_row, const T* gate,
                                                        int64_t gate_row, float* state, int64_t pool, const int64_t* slots, T* y) {
    pdl_wait();
    const int64_t c = ((int64_t)blockIdx.x * 128 + threadIdx.x) * W;
    if (c >= channels) return;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        Pack<T, W> vx, vg, vy;
        vx.get(x + r * x_row + c);
        vg.get(gate + r * gate_row + c);
        const int64_t slot = slots != nullptr ? gload_i64(slots + r) : r;
        float out[W];
        if (slot >= 0 && slot < pool) {
            Pack<float, W> h;
            h.get(state + slot * channels + c);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                out[i] = advance(step_of(vg.at(i), true), h.at(i), vx.at(i));
            }
            h.set(out);
            h.put(state + slot * channels + c);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) out[i] = 0.0f;
        }
        vy.set(out);
        vy.put(y + r * channels + c);
    }
}

struct Launch {
    int warps, ranks;
    unsigned grid;
};

// CTAs along time: as many warps as the steps fill, and a cluster as long as the GPU has room for more CTAs.
Launch launch_of(int64_t units, int64_t steps) {
    Launch l;
    l.warps = (int)(steps >= kChunk ? kWarps : steps > kSteps ? (steps + kSteps - 1) / kSteps : 1);
    l.ranks = 1;
    while (l.ranks < kCluster && (int64_t)l.ranks * kChunk < steps && units * l.ranks < 2 * sm_count()) l.ranks *= 2;
    l.grid = (unsigned)(units * l.ranks);
    return l;
}

template <typename K>
int launch_scan(K kernel, const ScanArgs& a, int64_t batch, cudaStream_t st) {
    const Launch l = launch_of(batch * a.tiles, a.steps);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(l.grid);
    cfg.blockDim = dim3(32, l.warps);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = l.ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e != cudaSuccess || cudaGetLastError() != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

int check_scan(const dcn_scan* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype)) return DCN_ERR_UNSUPPORTED;
    if (p->batch < 0 || p->steps < 0 || p->channels < 0) return DCN_ERR_SHAPE;
    constexpr int64_t most = 1ll << 31;
    if (p->batch >= most || p->steps >= most || p->channels >= most) return DCN_ERR_LIMIT;
    if (p->batch * ((p->channels + 31) / 32) >= 1ll << 27) return DCN_ERR_LIMIT;       // CTAs of a grid, eight to a cluster
    return DCN_OK;
}

bool even(const void* p, int64_t batch, int64_t step) { return aligned(p, 4) && batch % 2 == 0 && step % 2 == 0; }

ScanArgs args_of(const dcn_scan* p, int w) {
    ScanArgs a = {};
    a.steps = p->steps;
    a.channels = p->channels;
    a.chunks = (p->steps + kChunk - 1) / kChunk;
    a.x_batch = p->x_batch, a.x_step = p->x_step;
    a.gate_batch = p->gate_batch, a.gate_step = p->gate_step;
    a.dy_batch = p->dy_batch, a.dy_step = p->dy_step;
    a.tiles = (int)((p->channels + 32 * w - 1) / (32 * w));
    return a;
}

}  // namespace
}  // namespace seq
}  // namespace dcn

using namespace dcn::seq;

extern "C" size_t dcn_scan_checkpoint_bytes(const dcn_scan* p) {
    if (check_scan(p) != DCN_OK) return 0;
    return (size_t)p->batch * ((p->steps + kChunk - 1) / kChunk) * p->channels * sizeof(float);
}

extern "C" int dcn_scan_forward(const dcn_scan* p, const void* x, const void* gate, const float* state, const int64_t* lengths,
                                void* y, float* last, float* checkpoints, void* stream) {
    const int bad = check_scan(p);
    if (bad != DCN_OK) return bad;
    if (p->batch == 0 || p->channels == 0) return DCN_OK;
    if (last == nullptr || (p->steps > 0 && (x == nullptr || gate == nullptr || y == nullptr))) return DCN_ERR_NULL;
    const int e = elem_bytes(p->dtype);
    if (!aligned(x, e) || !aligned(gate, e) || !aligned(y, e) || !aligned(state, 4) || !aligned(last, 4) ||
        !aligned(lengths, 8) || !aligned(checkpoints, 4))
        return DCN_ERR_ALIGN;
    // two channels a thread where pairs of 16-bit elements can be read as one word: lines of 128 bytes a warp
    const bool two = e == 2 && p->channels % 2 == 0 && even(x, p->x_batch, p->x_step) &&
                     even(gate, p->gate_batch, p->gate_step) && aligned(y, 4);
    ScanArgs a = args_of(p, two ? 2 : 1);
    a.x = x, a.gate = gate, a.state = state, a.lengths = lengths, a.y = y, a.last = last, a.checkpoints = checkpoints;
    const cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == DCN_SEQ_F32) return launch_scan(scan_forward_kernel<float, 1>, a, p->batch, st);
    if (p->dtype == DCN_SEQ_BF16)
        return two ? launch_scan(scan_forward_kernel<__nv_bfloat16, 2>, a, p->batch, st)
                   : launch_scan(scan_forward_kernel<__nv_bfloat16, 1>, a, p->batch, st);
    return two ? launch_scan(scan_forward_kernel<__half, 2>, a, p->batch, st)
               : launch_scan(scan_forward_kernel<__half, 1>, a, p->batch, st);
}

extern "C" int dcn_scan_backward(const dcn_scan* p, const void* x, const void* gate, const int64_t* lengths,
                                 const float* checkpoints, const void* dy, const float* dlast, void* dx, void* dgate,
                                 float* dstate, void* stream) {
    const int bad = check_scan(p);
    if (bad != DCN_OK) return bad;
    if (p->batch == 0 || p->channels == 0) return DCN_OK;
    if (p->steps > 0 && (x == nullptr || gate == nullptr || checkpoints == nullptr || dx == nullptr || dgate == nullptr))
        return DCN_ERR_NULL;
    const int e = elem_bytes(p->dtype);
    if (!aligned(x, e) || !aligned(gate, e) || !aligned(dy, e) || !aligned(dx, e) || !aligned(dgate, e) ||
        !aligned(dlast, 4) || !aligned(dstate, 4) || !aligned(lengths, 8) || !aligned(checkpoints, 4))
        return DCN_ERR_ALIGN;
    const bool two = e == 2 && p->channels % 2 == 0 && even(x, p->x_batch, p->x_step) &&
                     even(gate, p->gate_batch, p->gate_step) && (dy == nullptr || even(dy, p->dy_batch, p->dy_step)) &&
                     aligned(dx, 4) && aligned(dgate, 4);
    ScanArgs a = args_of(p, two ? 2 : 1);
    a.x = x, a.gate = gate, a.dy = dy, a.dlast = dlast, a.lengths = lengths, a.dx = dx, a.dgate = dgate, a.dstate = dstate;
    a.checkpoints = const_cast<float*>(checkpoints);
    const cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == DCN_SEQ_F32) return launch_scan(scan_backward_kernel<float, 1>, a, p->batch, st);
    if (p->dtype == DCN_SEQ_BF16)
        return two ? launch_scan(scan_backward_kernel<__nv_bfloat16, 2>, a, p->batch, st)
                   : launch_scan(scan_backward_kernel<__nv_bfloat16, 1>, a, p->batch, st);
    return two ? launch_scan(scan_backward_kernel<__half, 2>, a, p->batch, st)
               : launch_scan(scan_backward_kernel<__half, 1>, a, p->batch, st);
}

namespace {

template <typename T>
int launch_step(int64_t rows, int64_t channels, const void* x, int64_t x_row, const void* gate, int64_t gate_row, float* state,
                int64_t pool, const int64_t* slots, void* y, cudaStream_t st) {
    // four channels a thread where all rows allow it, one otherwise
    const size_t v = 4 * sizeof(T);
    const bool four = channels % 4 == 0 && x_row % 4 == 0 && gate_row % 4 == 0 && aligned(x, v) && aligned(gate, v) &&
                      aligned(y, v) && aligned(state, 16);
    const int w = four ? 4 : 1;
    const dim3 grid((unsigned)((channels + 128 * w - 1) / (128 * w)), (unsigned)(rows < 65535 ? rows : 65535));
    const auto kernel = four ? scan_step_kernel<T, 4> : scan_step_kernel<T, 1>;
    const cudaError_t e = dcn::launch_dependent(kernel, grid, dim3(128), 0, st, rows, channels, static_cast<const T*>(x), x_row,
                                                static_cast<const T*>(gate), gate_row, state, pool, slots, static_cast<T*>(y));
    return e != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

}  // namespace

extern "C" int dcn_scan_step(int32_t dtype, int64_t rows, int64_t channels, const void* x, int64_t x_row, const void* gate,
                             int64_t gate_row, float* state, int64_t pool, const int64_t* slots, void* y, void* stream) {
    if (!known_type(dtype)) return DCN_ERR_UNSUPPORTED;
    if (rows < 0 || channels < 0 || pool < 0 || (slots == nullptr && pool < rows)) return DCN_ERR_SHAPE;
    if (channels >= 1ll << 31) return DCN_ERR_LIMIT;
    if (rows == 0 || channels == 0) return DCN_OK;
    if (x == nullptr || gate == nullptr || y == nullptr || (state == nullptr && pool > 0)) return DCN_ERR_NULL;
    const int e = elem_bytes(dtype);
    if (!aligned(x, e) || !aligned(gate, e) || !aligned(y, e) || !aligned(state, 4) || !aligned(slots, 8)) return DCN_ERR_ALIGN;
    const cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DCN_SEQ_F32) return launch_step<float>(rows, channels, x, x_row, gate, gate_row, state, pool, slots, y, st);
    if (dtype == DCN_SEQ_BF16)
        return launch_step<__nv_bfloat16>(rows, channels, x, x_row, gate, gate_row, state, pool, slots, y, st);
    return launch_step<__half>(rows, channels, x, x_row, gate, gate_row, state, pool, slots, y, st);
}
