// The norm behind a block, its gate, the scaled residual and the norm before the next block, as one pass over the rows:
//     yn = block r,  r = (mean(block^2) + eps)^-1/2;   stream = x + c s(gate) yn,  c = scale post
//     sn = stream q, q = (mean(stream^2) + eps)^-1/2;  normed = sn pre
// and the gradient, with dsn = dnormed pre and means over the channels:
//     ds = dstream + q (dsn - sn mean(dsn sn)) = dx;   dyn = ds c s(gate);   dblock = r (dyn - yn mean(dyn yn))
//     dgate = dyn yn (1 - s(gate));   Z = sum over rows of ds s(gate) yn:  dscale = Z post, dpost = Z scale;   dpre = sum dnormed sn
//
// A row lives in the registers of a row of threads, eight elements each, so that every tensor is read or written once: the
// bound is DRAM.  Up to 256 channels a warp has a row for itself and sums by shuffles alone; above, a CTA has one row at a time.
// The CTAs of the backward pass walk the rows with Z and dpre in registers and leave one partial sum each; a second kernel
// adds those in a fixed order.
#include "seq_common.cuh"

namespace dcn {
namespace seq {
namespace {

constexpr int kPer = 8;                          // elements of a thread
constexpr int kMostChannels = 1024 * kPer;

struct NormArgs {
    const void *x, *block, *gate, *scale, *post, *pre, *dstream, *dnormed;
    void *stream, *normed, *dx, *dblock, *dgate;
    float *stats, *partial;
    int64_t rows, x_row, block_row, gate_row, dstream_row, dnormed_row;
    int channels, wide_weights;
    float eps, inv;
};

// kPer elements of a row, V at a time: the vectors j, j + threads, ...
template <typename T, int V>
struct Slice {
    Pack<T, V> v[kPer / V];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kPer / V; ++i) v[i].zero();
    }
    __device__ __forceinline__ float at(int e) const { return v[e / V].at(e % V); }
};

template <int V>
__device__ __forceinline__ int element(int j, int threads, int i) { return (j + i * threads) * V; }

template <typename T, int V>
__device__ __forceinline__ void get(Slice<T, V>& s, const void* base, int64_t offset, int j, int threads, int channels) {
#pragma unroll
    for (int i = 0; i < kPer / V; ++i) {
        const int c = element<V>(j, threads, i);
        s.v[i].zero();
        if (base != nullptr && c < channels) s.v[i].get(static_cast<const T*>(base) + offset + c);
    }
}

template <typename T, int V>
__device__ __forceinline__ void put(void* base, int64_t offset, const float (&f)[kPer], int j, int threads, int channels) {
    if (base == nullptr) return;
#pragma unroll
    for (int i = 0; i < kPer / V; ++i) {
        const int c = element<V>(j, threads, i);
        float part[V];
#pragma unroll
        for (int k = 0; k < V; ++k) part[k] = f[i * V + k];
        Pack<T, V> out;
        out.set(part);
        if (c < channels) out.put(static_cast<T*>(base) + offset + c);
    }
}

// A weight as float32: of its own type, or of the activations'
template <typename T>
__device__ __forceinline__ float weight(const void* w, int c, int wide) {
    if (w == nullptr) return 1.0f;
    Pack<T, 1> v;
    if (wide) return gload(static_cast<const float*>(w) + c);
    v.get(static_cast<const T*>(w) + c);
    return v.at(0);
}

template <typename T, int V>
__device__ __forceinline__ void get_weights(float (&c)[kPer], float (&pre)[kPer], const NormArgs& p, int j, int threads) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int at = element<V>(j, threads, e / V) + e % V;
        c[e] = pre[e] = 0.0f;
        if (at < p.channels) {
            c[e] = weight<T>(p.scale, at, p.wide_weights) * weight<T>(p.post, at, p.wide_weights);
            pre[e] = weight<T>(p.pre, at, p.wide_weights);
        }
    }
}

// Sums over the threads of a row.  They use two areas in turn, so that one barrier a sum is enough: an area is written again
// behind the barrier of the sum in between.
template <bool kWarp>
struct RowSum {
    float (&room)[2][32];
    int j, threads, side;
    __device__ __forceinline__ float operator()(float v) {
        v = warp_sum(v);
        if constexpr (!kWarp) {
            float* at = room[side];
            side ^= 1;
            if (j % 32 == 0) at[j / 32] = v;
            __syncthreads();
            v = warp_sum(j % 32 < threads / 32 ? at[j % 32] : 0.0f);
        }
        return v;
    }
};

template <typename T, int V, bool kWarp, int kMost>
__global__ void __launch_bounds__(kMost) norm_forward_kernel(const NormArgs p) {
    __shared__ float room[2][32];
    const int threads = kWarp ? 32 : blockDim.x, j = kWarp ? threadIdx.x % 32 : threadIdx.x;
    const int groups = kWarp ? blockDim.x / 32 : 1, group = kWarp ? threadIdx.x / 32 : 0;
    RowSum<kWarp> row_sum{room, j, threads, 0};
    pdl_wait();
    float c[kPer], pre[kPer];
    get_weights<T, V>(c, pre, p, j, threads);
    for (int64_t row = (int64_t)blockIdx.x * groups + group; row < p.rows; row += (int64_t)gridDim.x * groups) {
        Slice<T, V> x, y, g;
        get(x, p.x, row * p.x_row, j, threads, p.channels);
        get(y, p.block, row * p.block_row, j, threads, p.channels);
        get(g, p.gate, row * p.gate_row, j, threads, p.channels);
        float s[kPer], sum = 0.0f, r = 0.0f;
        if (p.block != nullptr) {
#pragma unroll
            for (int e = 0; e < kPer; ++e) sum = fmaf(y.at(e), y.at(e), sum);
            r = rsqrtf(row_sum(sum) * p.inv + p.eps);
        }
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            float on = 1.0f, off;
            if (p.gate != nullptr) logistic(g.at(e), on, off);
            s[e] = x.at(e);
            if (p.block != nullptr) s[e] = fmaf(c[e] * on, y.at(e) * r, s[e]);
            sum = fmaf(s[e], s[e], sum);
        }
        const float q = rsqrtf(row_sum(sum) * p.inv + p.eps);
        put<T, V>(p.stream, row * p.channels, s, j, threads, p.channels);
#pragma unroll
        for (int e = 0; e < kPer; ++e) s[e] = s[e] * q * pre[e];
        put<T, V>(p.normed, row * p.channels, s, j, threads, p.channels);
        if (p.stats != nullptr && j == 0) {
            p.stats[2 * row] = r;
            p.stats[2 * row + 1] = q;
        }
    }
}

template <typename T, int V, bool kWarp, int kMost>
__global__ void __launch_bounds__(kMost, kMost == 256 ? 2 : 1) norm_backward_kernel(const NormArgs p) {
    __shared__ float room[2][32];
    const int threads = kWarp ? 32 : blockDim.x, j = kWarp ? threadIdx.x % 32 : threadIdx.x;
    const int groups = kWarp ? blockDim.x / 32 : 1, group = kWarp ? threadIdx.x / 32 : 0;
    RowSum<kWarp> row_sum{room, j, threads, 0};
    pdl_wait();
    float c[kPer], pre[kPer], z[kPer], w[kPer];
    get_weights<T, V>(c, pre, p, j, threads);
#pragma unroll
    for (int e = 0; e < kPer; ++e) z[e] = w[e] = 0.0f;
    for (int64_t row = (int64_t)blockIdx.x * groups + group; row < p.rows; row += (int64_t)gridDim.x * groups) {
        Slice<T, V> x, y, g, ds, dn;
        get(x, p.x, row * p.x_row, j, threads, p.channels);
        get(y, p.block, row * p.block_row, j, threads, p.channels);
        get(g, p.gate, row * p.gate_row, j, threads, p.channels);
        get(ds, p.dstream, row * p.dstream_row, j, threads, p.channels);
        get(dn, p.dnormed, row * p.dnormed_row, j, threads, p.channels);
        const float r = p.block != nullptr ? gload(p.stats + 2 * row) : 0.0f, q = gload(p.stats + 2 * row + 1);
        float on[kPer], sn[kPer], d[kPer], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            float off;
            on[e] = 1.0f;
            if (p.gate != nullptr) logistic(g.at(e), on[e], off);
            sn[e] = (p.block != nullptr ? fmaf(c[e] * on[e], y.at(e) * r, x.at(e)) : x.at(e)) * q;
            w[e] = fmaf(dn.at(e), sn[e], w[e]);
            sum = fmaf(dn.at(e) * pre[e], sn[e], sum);
        }
        const float m = row_sum(sum) * p.inv;
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            d[e] = fmaf(q, fmaf(-sn[e], m, dn.at(e) * pre[e]), ds.at(e));
            const float yn = y.at(e) * r;
            z[e] = fmaf(d[e] * on[e], yn, z[e]);
            sum = fmaf(d[e] * c[e] * on[e], yn, sum);
        }
        put<T, V>(p.dx, row * p.channels, d, j, threads, p.channels);
        if (p.dblock != nullptr || p.dgate != nullptr) {
            const float n = row_sum(sum) * p.inv;
            float out[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) out[e] = r * fmaf(-y.at(e) * r, n, d[e] * c[e] * on[e]);
            put<T, V>(p.dblock, row * p.channels, out, j, threads, p.channels);
            if (p.dgate != nullptr) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    float s, off;
                    logistic(g.at(e), s, off);
                    out[e] = d[e] * c[e] * on[e] * (y.at(e) * r) * off;
                }
                put<T, V>(p.dgate, row * p.channels, out, j, threads, p.channels);
            }
        }
    }
    if (p.partial == nullptr) return;
    if constexpr (kWarp) {                       // the warps of a CTA add theirs up, in order
        __shared__ float all[2][32 * kPer];
        for (int k = 0; k < groups; ++k) {
            if (k == group) {
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int at = element<V>(j, threads, e / V) + e % V;
                    all[0][at] = z[e] = k == 0 ? z[e] : all[0][at] + z[e];
                    all[1][at] = w[e] = k == 0 ? w[e] : all[1][at] + w[e];
                }
            }
            __syncthreads();
        }
        if (group != groups - 1) return;
    }
    float* out = p.partial + (int64_t)blockIdx.x * 2 * p.channels;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const int at = element<V>(j, threads, e / V) + e % V;
        if (at < p.channels) {
            out[at] = z[e];
            out[p.channels + at] = w[e];
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
        put_weight(dscale, sum * weight<T>(post, at, wide));
        put_weight(dpost, sum * weight<T>(scale, at, wide));
    } else {
        put_weight(dpre, sum);
    }
}

int threads_of(int64_t channels) {
    int t = 32;
    while ((int64_t)t * kPer < channels) t *= 2;
    return t;
}

constexpr int kWarpGroups = 4;                   // rows of a CTA whose warps have one each

// CTAs: enough threads on every SM to have its share of memory traffic in flight, and no more than there are rows
unsigned grid_of(int64_t rows, int64_t channels, int threads_an_sm) {
    const int t = threads_of(channels), cta = t == 32 ? 32 * kWarpGroups : t;
    const int64_t units = t == 32 ? (rows + kWarpGroups - 1) / kWarpGroups : rows;
    const int64_t most = (int64_t)sm_count() * (threads_an_sm > cta ? threads_an_sm / cta : 1);
    return (unsigned)(units < most ? units : most);
}

constexpr int kForwardThreads = 1024, kBackwardThreads = 768;

template <typename T, int V>
int run_forward(const NormArgs& a, cudaStream_t st) {
    const int t = threads_of(a.channels);
    const dim3 grid(grid_of(a.rows, a.channels, kForwardThreads)), block(t == 32 ? 32 * kWarpGroups : t);
    const auto kernel = t == 32    ? norm_forward_kernel<T, V, true, 256>
                        : t <= 256 ? norm_forward_kernel<T, V, false, 256>
                                   : norm_forward_kernel<T, V, false, 1024>;
    return launch_dependent(kernel, grid, block, 0, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int V>
int run_backward(const NormArgs& a, cudaStream_t st) {
    const int t = threads_of(a.channels);
    const dim3 grid(grid_of(a.rows, a.channels, kBackwardThreads)), block(t == 32 ? 32 * kWarpGroups : t);
    const auto kernel = t == 32    ? norm_backward_kernel<T, V, true, 256>
                        : t <= 256 ? norm_backward_kernel<T, V, false, 256>
                                   : norm_backward_kernel<T, V, false, 1024>;
    return launch_dependent(kernel, grid, block, 0, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T>
int run_weights(const NormArgs& a, void* dscale, void* dpost, void* dpre, cudaStream_t st) {
    const dim3 grid((a.channels + 31) / 32, 2), block(32, 32);
    const int n = (int)grid_of(a.rows, a.channels, kBackwardThreads);
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

// 16-byte vectors where every row of `v` starts on one
bool wide(const void* v, int64_t row, int per) { return v == nullptr || (aligned(v, 16) && row % per == 0); }

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
    const int e = elem_bytes(p->dtype), we = elem_bytes(p->weight_dtype), per = 16 / e;
    for (const void* v : {x, block, gate, (const void*)stream_out, (const void*)normed})
        if (!aligned(v, e)) return DCN_ERR_ALIGN;
    for (const void* v : {scale, post, pre})
        if (!aligned(v, we)) return DCN_ERR_ALIGN;
    if (!aligned(stats, 4)) return DCN_ERR_ALIGN;
    NormArgs a = args_of(p);
    a.x = x, a.block = block, a.gate = block != nullptr ? gate : nullptr, a.scale = scale, a.post = post, a.pre = pre;
    a.stream = stream_out, a.normed = normed, a.stats = stats;
    const bool vec = p->channels % per == 0 && wide(x, p->x_row, per) && wide(block, p->block_row, per) &&
                     wide(a.gate, p->gate_row, per) && wide(stream_out, 0, per) && wide(normed, 0, per);
    const cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == DCN_SEQ_F32) return vec ? run_forward<float, 4>(a, st) : run_forward<float, 1>(a, st);
    if (p->dtype == DCN_SEQ_BF16) return vec ? run_forward<__nv_bfloat16, 8>(a, st) : run_forward<__nv_bfloat16, 1>(a, st);
    return vec ? run_forward<__half, 8>(a, st) : run_forward<__half, 1>(a, st);
}

extern "C" size_t dcn_norm_workspace_bytes(const dcn_norm* p) {
    if (check_norm(p) != DCN_OK) return 0;
    return (size_t)grid_of(p->rows, p->channels, kBackwardThreads) * 2 * p->channels * sizeof(float);
}

extern "C" int dcn_norm_backward(const dcn_norm* p, const void* x, const void* block, const void* gate, const void* scale,
                                 const void* post, const void* pre, const float* stats, const void* dstream,
                                 const void* dnormed, void* dx, void* dblock, void* dgate, void* dscale, void* dpost, void* dpre,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_norm(p);
    if (bad != DCN_OK) return bad;
    const bool weights = dscale != nullptr || dpost != nullptr || dpre != nullptr;
    const cudaStream_t st = (cudaStream_t)stream;
    const int e = elem_bytes(p->dtype), we = elem_bytes(p->weight_dtype), per = 16 / e;
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
    const bool vec = p->channels % per == 0 && wide(x, p->x_row, per) && wide(block, p->block_row, per) &&
                     wide(a.gate, p->gate_row, per) && wide(dstream, p->dstream_row, per) &&
                     wide(dnormed, p->dnormed_row, per) && wide(dx, 0, per) && wide(dblock, 0, per) && wide(dgate, 0, per);
    int rc;
    if (p->dtype == DCN_SEQ_F32) rc = vec ? run_backward<float, 4>(a, st) : run_backward<float, 1>(a, st);
    else if (p->dtype == DCN_SEQ_BF16) rc = vec ? run_backward<__nv_bfloat16, 8>(a, st) : run_backward<__nv_bfloat16, 1>(a, st);
    else rc = vec ? run_backward<__half, 8>(a, st) : run_backward<__half, 1>(a, st);
    if (rc != DCN_OK || !weights) return rc;
    if (p->dtype == DCN_SEQ_F32) return run_weights<float>(a, dscale, dpost, dpre, st);
    if (p->dtype == DCN_SEQ_BF16) return run_weights<__nv_bfloat16>(a, dscale, dpost, dpre, st);
    return run_weights<__half>(a, dscale, dpost, dpre, st);
}
