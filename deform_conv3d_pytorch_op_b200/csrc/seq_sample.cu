// One token of each row of logits, drawn by a given random number after temperature, top-k, top-p and min-p.
//
// Weights are whole numbers of 41 bits, w = floor(2^40 exp((x - largest) / temperature)) with the exponential in float32, and so are all
// sums: no order of addition, no split of a row changes a token.  Elements of weight 0 can neither come nor count.
//
// A cluster of CTAs has a row.  Descending order is found without sorting: by 2048 bins of the exponent's argument (equal widths, which
// the bulk of a row's logits spreads over), and inside the one bin that a limit falls into by the digits of the logit's bits; equal
// logits count by their index.  "Kept" is, for top-k and for top-p alike, what has less than a limit before it.
#include <cooperative_groups.h>

#include <algorithm>

#include "seq_common.cuh"

namespace cg = cooperative_groups;

namespace dcn {
namespace seq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kMostCluster = 8;
constexpr float kUnit = 1099511627776.0f;        // 2^40
constexpr float kBinsPerArgument = 73.0f;        // 2048 / 28: exp(-28) < 2^-40
constexpr int64_t kMostVocab = 1 << 20;

struct SampleArgs {
    const void* logits;
    const float *uniforms, *temperatures, *top_ps, *min_ps;
    const int64_t* top_ks;
    int64_t* tokens;
    float* logprobs;
    int64_t row_stride, top_k;
    int vocab;
    float temperature, top_p, min_p;
};

// Order of a type's elements as that of unsigned numbers, of the bits that they differ in as float32; -0 is 0
template <typename T>
struct Key {
    static constexpr int kBits = std::is_same<T, float>::value ? 32 : std::is_same<T, __nv_bfloat16>::value ? 16 : 24;
    static __device__ __forceinline__ uint32_t of(float x) {
        const uint32_t b = __float_as_uint(x + 0.0f);
        return (b & 0x80000000u ? ~b : b | 0x80000000u) >> (32 - kBits);
    }
};

struct Cut {                                     // what is kept: the bins before `bin`, and of that one keys above `key`, or equal up to `index`
    int bin;
    uint32_t key;
    int index;
};

struct Shared {
    uint32_t count[kBins];                       // of this CTA's elements
    unsigned long long mass[kBins];
    uint32_t all_count[kBins];                   // of the row's
    unsigned long long all_mass[kBins];
    float largest[kMostCluster];
    int odd[kMostCluster];
    unsigned long long sum[kMostCluster], warp_sum[kWarps], scan_mass[kWarps];
    uint32_t scan_count[kWarps];
    float warp_max[kWarps];
    int warp_odd[kWarps];
    int found;
    unsigned long long found_mass;
    uint32_t found_count;
};

template <typename T>
struct Row {
    static constexpr int kV = 16 / (int)sizeof(T);
    const T* x;
    int vocab, skew;                             // elements that the row's first 16 bytes have before it
    int begin, end;                              // of this warp's vectors
    float largest, inverse;

    __device__ __forceinline__ float argument(float v) const { return __fmul_rn(__fsub_rn(v, largest), inverse); }
    static __device__ __forceinline__ float weight_of(float e) { return e * kUnit; }
    // f(value, index) for the warp's elements, and their vectors one behind the other over the lanes
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        const int lane = threadIdx.x & 31;
        for (int i = begin + lane; i < end; i += 32) {
            const int at = i * kV - skew;
            if (at >= 0 && at + kV <= vocab) {
                Pack<T, kV> p;
                load_kept(p.raw, x + at);
#pragma unroll
                for (int e = 0; e < kV; ++e) f(p.at(e), at + e);
            } else {
                for (int e = 0; e < kV; ++e)
                    if (at + e >= 0 && at + e < vocab) {
                        Pack<T, 1> p;
                        p.get(x + at + e);
                        f(p.at(0), at + e);
                    }
            }
        }
    }
};

__device__ __forceinline__ int bin_of(float argument) { return min((int)(-argument * kBinsPerArgument), kBins - 1); }

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The row's counts and masses from those of its CTAs, which clear their own ones behind it
__device__ __forceinline__ void merge(Shared& s, cg::cluster_group& cluster) {
    cluster.sync();
    const int n = cluster.num_blocks();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        uint32_t c = 0;
        unsigned long long m = 0;
        for (int r = 0; r < n; ++r) {
            const Shared* const o = cluster.map_shared_rank(&s, r);
            c += o->count[i], m += o->mass[i];
        }
        s.all_count[i] = c, s.all_mass[i] = m;
    }
    cluster.sync();
}

__device__ __forceinline__ void clear(Shared& s) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0, s.mass[i] = 0;
    __syncthreads();
}

// The last bin with elements that has less than the limit before it, and what is before it
template <typename Less>
__device__ __forceinline__ int last_below(Shared& s, uint32_t count0, unsigned long long mass0, Less&& below, uint32_t& count,
                                          unsigned long long& mass) {
    constexpr int kEach = kBins / kThreads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t c = 0;
    unsigned long long m = 0;
    for (int i = 0; i < kEach; ++i) c += s.all_count[threadIdx.x * kEach + i], m += s.all_mass[threadIdx.x * kEach + i];
    uint32_t ci = c;
    unsigned long long mi = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, ci, o);
        const unsigned long long b = __shfl_up_sync(0xffffffffu, mi, o);
        if (lane >= o) ci += a, mi += b;
    }
    if (lane == 31) s.scan_count[warp] = ci, s.scan_mass[warp] = mi;
    if (threadIdx.x == 0) s.found = -1;
    __syncthreads();
    ci += count0 - c, mi += mass0 - m;
    for (int w = 0; w < warp; ++w) ci += s.scan_count[w], mi += s.scan_mass[w];
    int mine = -1;
    uint32_t mine_count = 0;
    unsigned long long mine_mass = 0;
    for (int i = 0; i < kEach; ++i) {
        const int b = threadIdx.x * kEach + i;
        if (s.all_count[b] > 0 && below(ci, mi)) mine = b, mine_count = ci, mine_mass = mi;
        ci += s.all_count[b], mi += s.all_mass[b];
    }
    if (mine >= 0) atomicMax(&s.found, mine);
    __syncthreads();
    if (mine >= 0 && s.found == mine) s.found_count = mine_count, s.found_mass = mine_mass;
    __syncthreads();
    count = s.found_count, mass = s.found_mass;
    const int found = s.found;
    __syncthreads();
    return found;
}

// The cut behind the last element that has less than a limit before it: below(count before, mass before).  `mass`: of what is kept.
// all_count and all_mass hold the first level's bins, and hold them again afterwards.
template <typename T, typename Less>
__device__ Cut cut_at(const Row<T>& row, Shared& s, cg::cluster_group& cluster, Less&& below, unsigned long long& kept_mass) {
    uint32_t count;
    unsigned long long mass;
    Cut cut;
    cut.bin = last_below(s, 0, 0, below, count, mass);
    cut.key = 0, cut.index = 0x7fffffff;
    const uint32_t in_bin = s.all_count[cut.bin];
    if (in_bin == 1) {
        kept_mass = mass + s.all_mass[cut.bin];
        return cut;
    }
    uint32_t prefix = 0, ties = 0;
    unsigned long long tie_mass = 0;
    for (int bits = 8; bits <= Key<T>::kBits; bits += 8) {
        __syncthreads();
        clear(s);
        row.each([&](float v, int) {
            const float a = row.argument(v);
            const unsigned long long w = (unsigned long long)Row<T>::weight_of(expf(a));
            if (w == 0 || bin_of(a) != cut.bin) return;
            const uint32_t key = Key<T>::of(v) >> (Key<T>::kBits - bits);
            if (key >> 8 != prefix) return;
            const int d = 255 - (int)(key & 255);
            atomicAdd(&s.count[d], 1u);
            atomicAdd(&s.mass[d], w);
        });
        merge(s, cluster);
        const int d = last_below(s, count, mass, below, count, mass);
        prefix = prefix << 8 | (uint32_t)(255 - d);
        ties = s.all_count[d], tie_mass = s.all_mass[d];
        __syncthreads();
    }
    cut.key = prefix;
    // equal logits have equal weights: the first n of them by index
    const unsigned long long w = tie_mass / ties;
    uint32_t lo = 1, hi = ties;                  // (the first one has less than the limit before it)
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (below(count + mid - 1, mass + w * (mid - 1))) lo = mid;
        else hi = mid - 1;
    }
    kept_mass = mass + w * lo;
    if (lo < ties) {
        // the index of the lo-th: how many each warp has, and where in the row's order
        uint32_t mine = 0;
        row.each([&](float v, int) { mine += Key<T>::of(v) == cut.key; });
        mine = __reduce_add_sync(0xffffffffu, mine);
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        __syncthreads();
        if (lane == 0) s.scan_count[warp] = mine;
        if (threadIdx.x == 0) s.found = -1;
        cluster.sync();
        uint32_t before = 0;
        const int rank = cluster.block_rank();
        for (int r = 0; r <= rank; ++r) {
            const Shared* const o = cluster.map_shared_rank(&s, r);
            for (int i = 0; i < (r < rank ? kWarps : warp); ++i) before += o->scan_count[i];
        }
        if (before < lo && before + mine >= lo) {
            // this warp has it: 32 vectors at a time
            uint32_t left = lo - before;
            constexpr int kV = Row<T>::kV;
            for (int i = row.begin; i < row.end; i += 32) {
                uint32_t mask = 0;
                const int at = (i + lane) * kV - row.skew;
                if (i + lane < row.end)
                    for (int e = 0; e < kV; ++e)
                        if (at + e >= 0 && at + e < row.vocab) {
                            Pack<T, 1> p;
                            p.get(row.x + at + e);
                            mask |= (uint32_t)(Key<T>::of(p.at(0)) == cut.key) << e;
                        }
                const uint32_t n = __popc(mask);
                uint32_t up = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t a = __shfl_up_sync(0xffffffffu, up, o);
                    if (lane >= o) up += a;
                }
                const uint32_t total = __shfl_sync(0xffffffffu, up, 31);
                if (left <= total) {
                    if (up - n < left && up >= left) {
                        for (uint32_t k = up - n + 1; k < left; ++k) mask &= mask - 1;
                        s.found = at + __ffs(mask) - 1;
                    }
                    break;
                }
                left -= total;
            }
        }
        cluster.sync();
        int index = -1;
        for (int r = 0; r < (int)cluster.num_blocks(); ++r) index = max(index, cluster.map_shared_rank(&s, r)->found);
        cut.index = index;
        cluster.sync();
    }
    return cut;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = cluster.block_rank(), ctas = cluster.num_blocks(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x / ctas;
    pdl_wait();

    auto number = [&](const float* p, float v) { return p != nullptr ? gload(p + r) : v; };
    float temperature = number(a.temperatures, a.temperature), top_p = number(a.top_ps, a.top_p), min_p = number(a.min_ps, a.min_p);
    const float uniform = gload(a.uniforms + r);
    int64_t top_k = a.top_ks != nullptr ? gload_i64(a.top_ks + r) : a.top_k;
    const bool bad = temperature != temperature || top_p != top_p || min_p != min_p || uniform != uniform;
    if (temperature == 0.0f) top_k = 1, temperature = 1.0f;
    temperature = fminf(fmaxf(temperature, 1e-3f), 1e3f);
    min_p = fminf(min_p, 1.0f);

    Row<T> row;
    row.x = static_cast<const T*>(a.logits) + r * a.row_stride;
    row.vocab = a.vocab;
    row.skew = (int)((reinterpret_cast<uintptr_t>(row.x) & 15) / sizeof(T));
    const int vectors = (row.skew + a.vocab + Row<T>::kV - 1) / Row<T>::kV, slices = ctas * kWarps, each = (vectors + slices - 1) / slices;
    row.begin = min((rank * kWarps + warp) * each, vectors), row.end = min(row.begin + each, vectors);

    float largest = -CUDART_INF_F;
    bool odd = false;
    row.each([&](float v, int) { largest = fmaxf(largest, v), odd = odd || v != v; });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    odd = __any_sync(0xffffffffu, odd);
    if (lane == 0) s.warp_max[warp] = largest, s.warp_odd[warp] = odd;
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0, s.mass[i] = 0;
    __syncthreads();
    if (threadIdx.x < ctas) {
        Shared* const to = cluster.map_shared_rank(&s, threadIdx.x);
        bool any = false;
        for (int w = 0; w < kWarps; ++w) largest = fmaxf(w == 0 ? s.warp_max[0] : largest, s.warp_max[w]), any = any || s.warp_odd[w];
        to->largest[rank] = largest, to->odd[rank] = any;
    }
    cluster.sync();
    odd = bad;
    largest = -CUDART_INF_F;
    for (int i = 0; i < ctas; ++i) largest = fmaxf(largest, s.largest[i]), odd = odd || s.odd[i];
    if (odd || isinf(largest)) {
        if (rank == 0 && threadIdx.x == 0) a.tokens[r] = -1, a.logprobs[r] = CUDART_NAN_F;
        return;                                  // (no CTA of the cluster reads another one's memory from here on)
    }
    row.largest = largest, row.inverse = 1.0f / temperature;

    const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0f;
    Cut cut = {kBins, 0, 0};
    if (by_count || by_mass) {
        row.each([&](float v, int) {
            const float x = row.argument(v);
            const unsigned long long w = (unsigned long long)Row<T>::weight_of(expf(x));
            if (w == 0) return;
            const int b = bin_of(x);
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], w);
        });
        merge(s, cluster);
        unsigned long long kept = 0;
        if (by_count) {
            cut = cut_at(row, s, cluster, [&](uint32_t count, unsigned long long) { return (int64_t)count < top_k; }, kept);
            if (by_mass) {                       // the bins again
                __syncthreads();
                clear(s);
                row.each([&](float v, int) {
                    const float x = row.argument(v);
                    const unsigned long long w = (unsigned long long)Row<T>::weight_of(expf(x));
                    if (w == 0) return;
                    const int b = bin_of(x);
                    atomicAdd(&s.count[b], 1u);
                    atomicAdd(&s.mass[b], w);
                });
                merge(s, cluster);
            }
        } else {
            for (int i = threadIdx.x; i < kBins; i += kThreads) kept += s.all_mass[i];
            kept = warp_sum64(kept);
            if (lane == 0) s.scan_mass[warp] = kept;
            __syncthreads();
            kept = 0;
            for (int w = 0; w < kWarps; ++w) kept += s.scan_mass[w];
            __syncthreads();
        }
        if (by_mass) {
            const double enough = fmax((double)top_p * (double)kept, 1e-300);
            cut = cut_at(row, s, cluster, [&](uint32_t, unsigned long long mass) { return (double)mass < enough; }, kept);
        }
    }

    // what is kept, and the token that the random number falls on
    auto weight = [&](float v, int index) -> unsigned long long {
        const float x = row.argument(v), e = expf(x);
        const unsigned long long w = (unsigned long long)Row<T>::weight_of(e);
        if (e < min_p) return 0;
        if (cut.bin < kBins && w != 0) {
            const int b = bin_of(x);
            if (b > cut.bin) return 0;
            if (b == cut.bin) {
                const uint32_t key = Key<T>::of(v);
                if (key < cut.key || (key == cut.key && index > cut.index)) return 0;
            }
        }
        return w;
    };
    unsigned long long mine = 0;
    row.each([&](float v, int index) { mine += weight(v, index); });
    mine = warp_sum64(mine);
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = mine;
    cluster.sync();
    unsigned long long total = 0, before = 0;
    for (int c = 0; c < ctas; ++c) {
        const Shared* const o = cluster.map_shared_rank(&s, c);
        for (int w = 0; w < kWarps; ++w) {
            if (c == rank && w == warp) before = total;
            total += o->warp_sum[w];
        }
    }
    cluster.sync();                              // (nothing of another CTA is read from here on)
    const double wanted = floor((double)fminf(fmaxf(uniform, 0.0f), 1.0f) * (double)total);
    const unsigned long long target = min((unsigned long long)wanted, total - 1);
    if (target < before || target >= before + mine) return;
    unsigned long long left = target - before;
    constexpr int kV = Row<T>::kV;
    for (int i = row.begin; i < row.end; i += 32) {
        const int at = (i + lane) * kV - row.skew;
        unsigned long long w[kV], sum = 0;
        for (int e = 0; e < kV; ++e) {
            w[e] = 0;
            if (i + lane < row.end && at + e >= 0 && at + e < a.vocab) {
                Pack<T, 1> p;
                p.get(row.x + at + e);
                w[e] = weight(p.at(0), at + e);
            }
            sum += w[e];
        }
        unsigned long long up = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long b = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += b;
        }
        const unsigned long long all = __shfl_sync(0xffffffffu, up, 31);
        if (left < all) {
            if (left >= up - sum && left < up) {
                left -= up - sum;
                for (int e = 0; e < kV; ++e) {
                    if (left < w[e]) {
                        a.tokens[r] = at + e;
                        a.logprobs[r] = (float)(log((double)w[e]) - log((double)total));
                        break;
                    }
                    left -= w[e];
                }
            }
            return;
        }
        left -= all;
    }
}

int check_sample(const dcn_sample* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype)) return DCN_ERR_UNSUPPORTED;
    if (p->rows < 0 || p->vocab < 1) return DCN_ERR_SHAPE;
    if (p->temperatures == nullptr && !(p->temperature == 0.0f || (p->temperature >= 1e-3f && p->temperature <= 1e3f))) return DCN_ERR_SHAPE;
    if (p->top_ps == nullptr && !(p->top_p >= 0.0f && p->top_p <= 1.0f)) return DCN_ERR_SHAPE;
    if (p->min_ps == nullptr && !(p->min_p >= 0.0f && p->min_p <= 1.0f)) return DCN_ERR_SHAPE;
    if (p->rows >= 1ll << 27 || p->vocab > kMostVocab) return DCN_ERR_LIMIT;
    return DCN_OK;
}

template <typename T>
int run_sample(const SampleArgs& a, int64_t rows, cudaStream_t st) {
    int cluster = 1;
    while (cluster < kMostCluster && rows * cluster * 2 <= 2 * dcn::sm_count() && a.vocab / (cluster * 2) >= 4096) cluster *= 2;
    constexpr size_t kBytes = sizeof(Shared);
    if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBytes) != cudaSuccess) return DCN_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = dcn::pdl_enabled() ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T>, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

}  // namespace
}  // namespace seq
}  // namespace dcn

using namespace dcn::seq;

extern "C" size_t dcn_sample_workspace_bytes(const dcn_sample*) { return 0; }

extern "C" int dcn_sample_tokens(const dcn_sample* p, const void* logits, const float* uniforms, int64_t* tokens, float* logprobs,
                                 void*, size_t, void* stream) {
    const int bad = check_sample(p);
    if (bad != DCN_OK) return bad;
    if (p->rows == 0) return DCN_OK;
    if (logits == nullptr || uniforms == nullptr || tokens == nullptr || logprobs == nullptr) return DCN_ERR_NULL;
    if (!aligned(logits, elem_bytes(p->dtype)) || !aligned(tokens, 8) || !aligned(p->top_ks, 8)) return DCN_ERR_ALIGN;
    for (const float* v : {uniforms, (const float*)logprobs, p->temperatures, p->top_ps, p->min_ps})
        if (!aligned(v, 4)) return DCN_ERR_ALIGN;
    const SampleArgs a = {logits, uniforms, p->temperatures, p->top_ps, p->min_ps, p->top_ks, tokens, logprobs, p->row_stride, p->top_k,
                          (int)p->vocab, p->temperature, p->top_p, p->min_p};
    const cudaStream_t st = (cudaStream_t)stream;
    return p->dtype == DCN_SEQ_F32    ? run_sample<float>(a, p->rows, st)
           : p->dtype == DCN_SEQ_BF16 ? run_sample<__nv_bfloat16>(a, p->rows, st)
                                      : run_sample<__half>(a, p->rows, st);
}
