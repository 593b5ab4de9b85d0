// One token of each row of logits, drawn by a given random number after temperature, top-k, top-p and min-p.
//
// Weights are whole numbers of 41 bits, w = floor(2^40 exp((x - largest) / temperature)) with the exponential in float32, and so are all
// sums: no order of addition, no split of a row changes a token.  Elements of weight 0 can neither come nor count.
//
// A cluster of CTAs has a row and reads it (from L2, but for the first time) a few times:
//   the largest logit;   how many logits lie in each of 2048 bins of equal widths of the exponential's argument, or (no count, no mass asked
//   for) each warp's sum;   the elements of the bins that a limit can lie in, which one CTA sorts.
// Where all that can be kept is in that list, its CTA draws the token from it.  Else a last pass sums what the cut keeps.  A list that
// would be too long (thousands of equal logits) is narrowed bin by bin by the digits of the logits' bits instead (cut_at).
// "Kept" is, for top-k and for top-p alike, what has less than a limit before it in falling order, equal logits by their index.
//
// Latency bounds it: a cluster's phases stand one behind the other, each with barriers, and reading takes a small part (64 x 131072 bf16, 50
// best and 0.9 of the mass: 55 to 89 us by the logits, floor 2.6; 37 x 50257 f16, 0.95: 55 to 72, floor 0.6; 16 x 400 float32: 5.9 from call to call).  Lists of
// the bins in question alone took the first from 187 to 89 us, limits found by bins rather than by sorting all that is kept before that.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "seq_common.cuh"

namespace cg = cooperative_groups;

namespace dcn {
namespace seq {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 2048, kMostCluster = 8, kList = 4096, kShort = 512, kFew = 64;
constexpr float kUnit = 1099511627776.0f;        // 2^40
constexpr float kBinsPerArgument = 73.0f;        // 2048 / 28: exp(-28) < 2^-40
constexpr int64_t kMostVocab = 1 << 20;
static_assert(kMostVocab <= (int64_t)kBins * kShort && kShort <= kThreads, "a bucket of indices has a thread for each");

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
    float warps_largest[kMostCluster * kWarps];  // of the row's warps
    float bound;
    unsigned long long warp_sum[kWarps], scan_mass[kWarps];
    uint32_t scan_count[kWarps];
    int found;
    unsigned long long found_mass;
    uint32_t found_count;
    unsigned long long shared_a[2][kMostCluster], shared_b[2][kMostCluster];     // of the CTAs (exchange)
    unsigned long long list[kList];              // candidates, of this CTA or (first CTA) of the row
    unsigned long long sorted[kShort], narrow[kShort];
    uint32_t listed, narrowed;
    uint32_t few_count[kFew], all_few_count[kFew];
    unsigned long long few_mass[kFew], all_few_mass[kFew];
    uint32_t high[kBins];                        // with the counts: sums of the high halves of weights above 2^-10
    Cut cut;
    unsigned long long kept;
    int failed;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
struct Row {
    static constexpr int kV = 16 / (int)sizeof(T);
    const T* x;
    int vocab, skew;                             // elements that the row's first 16 bytes have before it
    int begin, end;                              // of this warp's vectors
    float largest, inverse;

    __device__ __forceinline__ float argument(float v) const { return __fmul_rn(__fsub_rn(v, largest), inverse); }
    float floor;                                 // vectors without a logit that is as large can be left out

    // The warp's vector i; -inf for what does not belong to the row
    __device__ __forceinline__ Pack<T, kV> vector(int i) const {
        const int at = i * kV - skew;
        Pack<T, kV> p;
        if (at >= 0 && at + kV <= vocab) {
            load_kept(p.raw, x + at);
        } else {
            float f[kV];
#pragma unroll
            for (int e = 0; e < kV; ++e) {
                f[e] = -CUDART_INF_F;
                if (at + e >= 0 && at + e < vocab) {
                    Pack<T, 1> one;
                    one.get(x + at + e);
                    f[e] = one.at(0);
                }
            }
            p.set(f);
        }
        return p;
    }
    // (NaN where there is one)
    static __device__ __forceinline__ float largest_of(const Pack<T, kV>& p) {
        if constexpr (sizeof(T) == 4) {
            return max_nan(max_nan(p.at(0), p.at(1)), max_nan(p.at(2), p.at(3)));
        } else {
            const uint32_t m = max_pairs(max_pairs(p.raw.u[0], p.raw.u[1]), max_pairs(p.raw.u[2], p.raw.u[3]));
            return max_nan(half_of<T>(m, 0), half_of<T>(m, 1));
        }
    }
    static __device__ __forceinline__ uint32_t max_pairs(uint32_t a, uint32_t b) {
        uint32_t r;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    // f(vector, index of its first element) over the warp's vectors, which lie one behind the other over the lanes; the next one is on
    // its way
    template <typename F>
    __device__ __forceinline__ void vectors(F&& f) const {
        int i = begin + (threadIdx.x & 31);
        if (i >= end) return;
        Pack<T, kV> p = vector(i);
#pragma unroll 1
        for (; i < end; i += 32) {
            const Pack<T, kV> now = p;
            if (i + 32 < end) p = vector(i + 32);
            f(now, i * kV - skew);
        }
    }
    // f(value, index) for the elements of vectors that are not left out
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        vectors([&](const Pack<T, kV>& p, int at) {
            if (!(largest_of(p) >= floor)) return;
#pragma unroll
            for (int e = 0; e < kV; ++e) f(p.at(e), at + e);
        });
    }
    // leaves out what lies behind a bin, to be on the safe side of all roundings
    __device__ __forceinline__ void only_up_to(int last, float temperature) {
        floor = last >= kBins - 1 ? -CUDART_INF_F
                                  : largest - ((float)(last + 1) * (1.00001f / kBinsPerArgument) * temperature + 1e-5f * fabsf(largest) + 1e-30f);
    }
};

__device__ __forceinline__ int bin_of(float argument) { return min((int)(-argument * kBinsPerArgument), kBins - 1); }

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sums of weights in two halves of 20 bits, each exact in 32 bits over 4096 elements; a half is the floor that rounding towards zero
// beside 2^23 leaves
struct Halves {
    uint32_t high = 0, low = 0;
    __device__ __forceinline__ void add(float e) {
        const float a = e * 1048576.0f, h = __fadd_rz(a, 8388608.0f), r = a - (h - 8388608.0f), l = __fmaf_rz(r, 1048576.0f, 8388608.0f);
        high += __float_as_uint(h) - 0x4b000000u, low += __float_as_uint(l) - 0x4b000000u;
    }
    __device__ __forceinline__ unsigned long long sum() const { return ((unsigned long long)high << 20) + low; }
};
__device__ __forceinline__ unsigned long long weight_of(float e) {
    Halves h;
    h.add(e);
    return h.sum();
}

// Sums over the cluster of two numbers that each warp has one of.  Each CTA's own go to all (a load from another CTA's memory takes
// hundreds of cycles, a store none of the thread's).  Uses take turns between two places: a CTA writes for the next but one only behind
// the next one's barrier, when all have read.
struct Team {
    cg::cluster_group cluster;
    int rank, ctas, turn = 0;
    unsigned long long before_a;                 // the sums of the CTAs before this one
    __device__ __forceinline__ Team() : cluster(cg::this_cluster()), rank((int)cluster.block_rank()), ctas((int)cluster.num_blocks()) {}
    __device__ __forceinline__ void sync() {
        if (ctas > 1) cluster.sync();
        else __syncthreads();
    }
    __device__ __forceinline__ void exchange(Shared& s, unsigned long long& a, unsigned long long& b) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        __syncthreads();
        if (lane == 0) s.warp_sum[warp] = a, s.scan_mass[warp] = b;
        __syncthreads();
        if (warp == 0) {
            a = warp_sum64(lane < kWarps ? s.warp_sum[lane] : 0), b = warp_sum64(lane < kWarps ? s.scan_mass[lane] : 0);
            if (lane < ctas) {
                Shared* const to = cluster.map_shared_rank(&s, lane);
                to->shared_a[turn][rank] = a, to->shared_b[turn][rank] = b;
            }
        }
        sync();
        a = b = before_a = 0;
        for (int r = 0; r < ctas; ++r) {
            if (r < rank) before_a += s.shared_a[turn][r];
            a += s.shared_a[turn][r], b += s.shared_b[turn][r];
        }
        turn ^= 1;
    }
};

// A candidate as a number that falls with the logit, then with the index
__device__ __forceinline__ unsigned long long candidate(float v, int index) {
    return (unsigned long long)Key<float>::of(v) << 20 | (unsigned)(kMostVocab - 1 - index);
}
__device__ __forceinline__ int index_of(unsigned long long c) { return (int)(kMostVocab - 1) - (int)(c & (kMostVocab - 1)); }
__device__ __forceinline__ float logit_of(unsigned long long c) {
    const uint32_t k = (uint32_t)(c >> 20);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// The thread's number at its place among n different ones, the largest first (v is not to be `sorted`; up to kShort)
__device__ __forceinline__ void sort_short(const unsigned long long* v, int n, unsigned long long* sorted) {
    const unsigned long long mine = threadIdx.x < n ? v[threadIdx.x] : 0;
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += v[i] > mine;
    if (threadIdx.x < n) sorted[rank] = mine;
    __syncthreads();
}

// Sums in front of each thread's part of consecutive numbers, and of all
__device__ __forceinline__ unsigned long long scan64(Shared& s, unsigned long long mine, unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long b = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += b;
    }
    __syncthreads();
    if (lane == 31) s.scan_mass[warp] = up;
    __syncthreads();
    unsigned long long before = up - mine;
    total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s.scan_mass[w];
        total += s.scan_mass[w];
    }
    return before;
}

// This CTA's logits of at least `least` in bins first to last into its list (as many as it holds; all are counted).  kBefore: and how many
// lie in front of these bins, and their mass, for each thread's
template <bool kBefore, typename T>
__device__ __forceinline__ void collect(const Row<T>& row, Shared& s, int first, int last, float least, unsigned long long& count, unsigned long long& mass) {
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    const float from = (float)first, to = last == kBins - 1 ? kBins + 32.0f : (float)(last + 1);
    Halves before;
    uint32_t n = 0;
    row.each([&](float v, int index) {
        const float x = row.argument(v), t = -x * kBinsPerArgument;
        if (!(t < to) || v < least) return;
        if (kBefore && t < from) {
            before.add(expf(x));
            ++n;
            return;
        }
        const uint32_t at = atomicAdd(&s.listed, 1u);
        if (at < kList) s.list[at] = candidate(v, index);
    });
    __syncthreads();
    count = n, mass = before.sum();
}
template <typename T>
__device__ __forceinline__ void collect(const Row<T>& row, Shared& s, int last, float least) {
    unsigned long long count, mass;
    collect<false>(row, s, 0, last, least, count, mass);
}
// The CTAs' lists in the first one's; how many there are in all
__device__ __forceinline__ uint32_t join_lists(Shared& s, Team& team) {
    const uint32_t n = s.listed;
    unsigned long long count = threadIdx.x == 0 ? n : 0, none = 0;
    team.exchange(s, count, none);
    if (count > kShort) return (uint32_t)min(count, 0x7fffffffull);
    const uint32_t at = (uint32_t)team.before_a;
    if (team.rank > 0) {
        Shared* const first = team.cluster.map_shared_rank(&s, 0);
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) first->list[at + i] = s.list[i];
    }
    team.sync();
    return (uint32_t)count;
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

// The row's counts alone: each CTA adds up its share of the bins and tells all
__device__ __forceinline__ void merge_counts(Shared& s, Team& team) {
    team.sync();
    const int n = team.ctas, share = kBins / n;  // (n is a power of two)
    for (int i = team.rank * share + threadIdx.x; i < (team.rank + 1) * share; i += kThreads) {
        uint32_t c[kMostCluster], h[kMostCluster], sum = 0, high = 0;
#pragma unroll
        for (int r = 0; r < kMostCluster; ++r) {
            c[r] = h[r] = 0;
            if (r < n) c[r] = team.cluster.map_shared_rank(&s, r)->count[i], h[r] = team.cluster.map_shared_rank(&s, r)->high[i];
        }
#pragma unroll
        for (int r = 0; r < kMostCluster; ++r) sum += c[r], high += h[r];
        for (int r = 0; r < n; ++r) {
            Shared* const to = team.cluster.map_shared_rank(&s, r);
            to->all_count[i] = sum, to->all_mass[i] = (unsigned long long)high << 20;
        }
    }
    team.sync();
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
            const unsigned long long w = weight_of(expf(a));
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
    cut.key = prefix;                            // (made one of float32 at the end)
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
    if constexpr (Key<T>::kBits < 32)            // the bits that float32 has more, of a negative number's complement all ones
        cut.key = cut.key << (32 - Key<T>::kBits) | (cut.key >> (Key<T>::kBits - 1) ? 0u : (1u << (32 - Key<T>::kBits)) - 1u);
    return cut;
}

// A CTA's candidates, each thread with its own
struct Listed {
    static constexpr int kEach = kList / kThreads;
    unsigned long long weight[kEach];
    int bin[kEach];
    unsigned long long front_count = 0, front_mass = 0;          // what the thread has seen of bins before all of these
    template <typename T>
    __device__ __forceinline__ void get(const Row<T>& row, const Shared& s) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int i = threadIdx.x + j * kThreads;
            bin[j] = kBins, weight[j] = 0;
            if (i < s.listed) {
                const float x = row.argument(logit_of(s.list[i]));
                bin[j] = bin_of(x), weight[j] = weight_of(expf(x));
            }
        }
    }
    // over the cluster: how many lie in front of a bin, and their mass
    __device__ __forceinline__ void before(Shared& s, Team& team, int b, unsigned long long& count, unsigned long long& mass) const {
        count = front_count, mass = front_mass;
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (bin[j] < b) ++count, mass += weight[j];
        count = warp_sum64(count), mass = warp_sum64(mass);
        team.exchange(s, count, mass);
    }
};

// cut_at's from the CTAs' lists of all elements of bins up to `last`; `first`: a bin that is not behind the one the limit is in.  False where
// it is after all, where the limit lies behind the list, or too many elements share its bin.
template <typename T, typename Less>
__device__ bool cut_in(const Row<T>& row, Shared& s, Team& team, const Listed& mine, int first, int last, Less&& below, Cut& cut, unsigned long long& kept_mass) {
    unsigned long long count = 0, mass = 0, count_there = 0, mass_there = 0;
    int lo = first;                              // the last bin with elements that has less than the limit before it
    mine.before(s, team, first, count, mass);
    if (last - first < kFew) {
        // all bins' counts and masses at once
        if (threadIdx.x < kFew) s.few_count[threadIdx.x] = 0, s.few_mass[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < Listed::kEach; ++j)
            if (mine.bin[j] >= first && mine.bin[j] <= last) {
                atomicAdd(&s.few_count[mine.bin[j] - first], 1u);
                atomicAdd(&s.few_mass[mine.bin[j] - first], mine.weight[j]);
            }
        team.sync();
        if (threadIdx.x <= last - first) {
            uint32_t c[kMostCluster];
            unsigned long long m[kMostCluster];
#pragma unroll
            for (int r = 0; r < kMostCluster; ++r) {
                c[r] = 0, m[r] = 0;
                if (r < team.ctas) c[r] = team.cluster.map_shared_rank(&s, r)->few_count[threadIdx.x], m[r] = team.cluster.map_shared_rank(&s, r)->few_mass[threadIdx.x];
            }
#pragma unroll
            for (int r = 1; r < kMostCluster; ++r) c[0] += c[r], m[0] += m[r];
            s.all_few_count[threadIdx.x] = c[0], s.all_few_mass[threadIdx.x] = m[0];
        }
        team.sync();
        bool found = false;
        for (int b = first; b <= last; ++b) {
            const uint32_t c = s.all_few_count[b - first];
            if (c > 0 && below((uint32_t)count, mass)) found = true, lo = b, count_there = count, mass_there = mass;
            count += c, mass += s.all_few_mass[b - first];
        }
        if (!found || (last < kBins - 1 && below((uint32_t)count, mass))) return false;
    } else {
        count_there = count, mass_there = mass;
        if (!below((uint32_t)count, mass)) return false;
        mine.before(s, team, last + 1, count, mass);
        if (last < kBins - 1 && below((uint32_t)count, mass)) return false;
        int hi = last;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            mine.before(s, team, mid, count, mass);
            if (below((uint32_t)count, mass)) lo = mid, count_there = count, mass_there = mass;
            else hi = mid - 1;
        }
    }
    // its elements, to the first CTA
    Shared* const to = team.cluster.map_shared_rank(&s, 0);
    if (team.rank == 0 && threadIdx.x == 0) s.narrowed = 0;
    team.sync();
#pragma unroll
    for (int j = 0; j < Listed::kEach; ++j)
        if (mine.bin[j] == lo) {
            const uint32_t at = atomicAdd(&to->narrowed, 1u);
            if (at < kShort) to->narrow[at] = s.list[threadIdx.x + j * kThreads];
        }
    team.sync();
    if (team.rank == 0) {
        const int n = s.narrowed;
        if (threadIdx.x == 0) s.failed = n > kShort || n == 0, s.found = -1;
        __syncthreads();
        if (n <= kShort && n > 0) {
            sort_short(s.narrow, n, s.sorted);
            const bool in = threadIdx.x < n;
            const unsigned long long c = in ? s.sorted[threadIdx.x] : 0, w = in ? weight_of(expf(row.argument(logit_of(c)))) : 0;
            unsigned long long total, before = mass_there + scan64(s, w, total);
            const bool kept = in && below((uint32_t)count_there + threadIdx.x, before);
            if (kept) atomicMax(&s.found, (int)threadIdx.x);
            __syncthreads();
            if (kept && s.found == threadIdx.x) {
                s.cut = {kBins, (uint32_t)(c >> 20), index_of(c)};
                s.kept = before + w;
            }
        }
    }
    team.sync();
    const bool failed = to->failed != 0;
    cut = to->cut;
    kept_mass = to->kept;
    team.sync();
    return !failed;
}

// The bins' masses, about: the high halves' sums where those are most of it, else the exponentials in the middle of the bins
__device__ __forceinline__ void guess_masses(Shared& s) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        const float e = expf(((float)i + 0.5f) * (-1.0f / kBinsPerArgument));
        if (e < 0.0011f) s.all_mass[i] = (unsigned long long)((float)s.all_count[i] * (kUnit * e));
    }
    __syncthreads();
}
// The bin that a limit lies in; up_to: how many elements it and those before it have
template <typename Less>
__device__ __forceinline__ int place_of(Shared& s, Less&& below, uint32_t& up_to) {
    uint32_t count;
    unsigned long long mass;
    const int bin = last_below(s, 0, 0, below, count, mass);
    up_to = count + s.all_count[bin];
    return bin;
}

// Counts and masses of the first level's bins, for cut_at
template <typename T>
__device__ void histogram(const Row<T>& row, Shared& s, cg::cluster_group& cluster) {
    __syncthreads();
    clear(s);
    row.each([&](float v, int) {
        const float x = row.argument(v);
        const unsigned long long w = weight_of(expf(x));
        if (w == 0) return;
        const int b = bin_of(x);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], w);
    });
    merge(s, cluster);
}
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) char smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    Team team;
    cg::cluster_group& cluster = team.cluster;
    const int rank = team.rank, ctas = team.ctas, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = blockIdx.x / ctas;
    if (ctas > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");         // every CTA runs before another writes to its memory
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
    row.floor = -CUDART_INF_F;
    row.x = static_cast<const T*>(a.logits) + r * a.row_stride;
    row.vocab = a.vocab;
    row.skew = (int)((reinterpret_cast<uintptr_t>(row.x) & 15) / sizeof(T));
    const int vectors = (row.skew + a.vocab + Row<T>::kV - 1) / Row<T>::kV, slices = ctas * kWarps, each = (vectors + slices - 1) / slices;
    row.begin = min((rank * kWarps + warp) * each, vectors), row.end = min(row.begin + each, vectors);

    float largest = -CUDART_INF_F;               // (NaN where there is one)
    row.vectors([&](const Pack<T, Row<T>::kV>& p, int) { largest = max_nan(largest, Row<T>::largest_of(p)); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = s.high[i] = 0;
    if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (lane < ctas) cluster.map_shared_rank(&s, lane)->warps_largest[rank * kWarps + warp] = largest;
    team.sync();
    const int warps = ctas * kWarps;
    const float mine_of = threadIdx.x < warps ? s.warps_largest[threadIdx.x] : -CUDART_INF_F;
    for (int i = lane; i < warps; i += 32) largest = max_nan(largest, s.warps_largest[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) largest = max_nan(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    if (bad || largest != largest || isinf(largest)) {
        if (rank == 0 && threadIdx.x == 0) a.tokens[r] = -1, a.logprobs[r] = CUDART_NAN_F;
        return;                                  // (no CTA of the cluster reads another one's memory from here on)
    }
    row.largest = largest, row.inverse = 1.0f / temperature;

    const bool by_count = top_k > 0 && top_k < a.vocab, by_mass = top_p < 1.0f;
    const double u = (double)fminf(fmaxf(uniform, 0.0f), 1.0f);
    Cut cut = {-1, 0, 0};                        // bin -1: all; kBins: key and index alone; else the bins before it, and of it by key and index
    bool listed = false;                         // all that is kept is in the CTAs' lists
    Listed mine;
    if (by_count || by_mass) {
        const auto of_count = [&](uint32_t count, unsigned long long) { return (int64_t)count < top_k; };
        const auto of_share = [&](double enough) { return [=](uint32_t, unsigned long long mass) { return (double)mass < enough; }; };
        unsigned long long total = 0, none = 0;
        uint32_t all = kShort + 1;
        int last = kBins - 1, first = 0;
        if (a.vocab <= kShort) {                 // all of a small vocabulary
            collect(row, s, last, -CUDART_INF_F);
            all = join_lists(s, team);
        } else if (by_count && top_k <= warps) {
            // As many as are asked for are as large as the k-th largest of the warps' largest logits, and few more
            if (threadIdx.x < warps) {
                int above = 0;
                for (int i = 0; i < warps; ++i) {
                    const float o = s.warps_largest[i];
                    above += o > mine_of || (o == mine_of && i < threadIdx.x);
                }
                if (above == (int)top_k - 1) s.bound = mine_of;
            }
            __syncthreads();
            row.floor = s.bound;
            collect(row, s, last, s.bound);
            all = join_lists(s, team);
            row.floor = -CUDART_INF_F;
        }
        if (all > kShort) {
            // counts, and the sum where a share of it is asked for
            Halves sum;
            row.each([&](float v, int) {
                const float x = row.argument(v), t = -x * kBinsPerArgument;
                const int bin = min((int)t, kBins - 1);
                const bool in = t < kBins + 32.0f;
                if (in) atomicAdd(&s.count[bin], 1u);
                if (!by_count) {
                    const float e = expf(x);
                    sum.add(e);
                    if (e >= 0.0009765625f) atomicAdd(&s.high[bin], (uint32_t)(e * 1048576.0f));
                }
            });
            total = warp_sum64(sum.sum());
            if (!by_count) team.exchange(s, total, none);
            merge_counts(s, team);
            if (by_count) {
                first = last = place_of(s, of_count, all);
            } else {
                guess_masses(s);
                const double enough = fmax((double)top_p * (double)total, 1e-300);
                first = place_of(s, of_share(enough * 0.997), all);
                last = min(place_of(s, of_share(enough * 1.003), all) + 1, kBins - 1);
            }
            row.only_up_to(last, temperature);
            collect(row, s, last, -CUDART_INF_F);
            row.floor = -CUDART_INF_F;
            all = kShort + 1;
            if (by_count) all = join_lists(s, team);
        }
        const bool listing = all <= kShort;
        if (listing) {
            // all that can be kept, and what is like it: the first CTA draws from the list
            if (rank > 0) return;
            const int n = (int)all, limit = by_count ? (int)min((int64_t)n, top_k) : n, i = threadIdx.x;
            sort_short(s.list, n, s.sorted);
            const unsigned long long c = i < n ? s.sorted[i] : 0;
            const float e = i < limit ? expf(row.argument(logit_of(c))) : 0.0f;
            unsigned long long w = weight_of(e), counted, sums, own = 0;
            unsigned long long before = scan64(s, w, counted);
            if (by_count || a.vocab <= kShort) total = counted;
            const double enough = by_mass ? fmax((double)top_p * (double)total, 1e-300) : 2e300;
            if (w != 0 && (double)before < enough && (i == 0 || e >= min_p)) own = (unsigned long long)(kMostVocab - 1 - index_of(c)) << 41 | w;
            // by index: the kept ones are among the first
            if (i < kShort) s.list[i] = own;
            const int kept = __syncthreads_count(own != 0), reach = kept;
            if (threadIdx.x == 0) s.found = 0;
            __syncthreads();
            if (own != 0) atomicMax(&s.found, i + 1);
            __syncthreads();
            const int used = s.found;
            int place = 0;
#pragma unroll 8
            for (int k = 0; k < used; ++k) place += s.list[k] > own;
            __syncthreads();
            if (own != 0) s.sorted[place] = own;
            __syncthreads();
            own = i < reach ? s.sorted[i] : 0;
            w = own & ((1ull << 41) - 1);
            before = scan64(s, w, sums);
            const unsigned long long target = min((unsigned long long)floor(u * (double)sums), sums - 1);
            if (target >= before && target < before + w) {
                a.tokens[r] = (int64_t)(kMostVocab - 1) - (int64_t)(own >> 41);
                a.logprobs[r] = (float)(log((double)w) - log((double)sums));
            }
            return;
        }
        // More: the lists stay with their CTAs, each with what its warps have of the row.  Where they are too long, they are made anew, of
        // the bins alone that the limit can lie in, and the token is looked for in the row itself.
        const auto fits = [&] {
            unsigned long long longest = threadIdx.x == 0 && s.listed > kList ? 1 : 0;
            team.exchange(s, longest, none);
            return longest == 0;
        };
        unsigned long long kept = 0;
        bool narrow = false, usable = fits();
        if (!usable) {
            narrow = true;
            row.only_up_to(last, temperature);
            collect<true>(row, s, first, last, -CUDART_INF_F, mine.front_count, mine.front_mass);
            row.floor = -CUDART_INF_F;
            usable = fits();
        }
        mine.get(row, s);
        if (by_count) {
            usable = usable && cut_in(row, s, team, mine, first, last, of_count, cut, kept);
            if (!usable) {
                histogram(row, s, cluster);
                cut = cut_at(row, s, cluster, of_count, kept);
            }
            total = kept;
        }
        if (by_mass) {
            const auto below = of_share(fmax((double)top_p * (double)total, 1e-300));
            Cut other;
            // (the share of a count lies in front of its limit: a list of that one's bin alone does not have it)
            usable = usable && !(by_count && narrow) && cut_in(row, s, team, mine, by_count ? 0 : first, last, below, other, kept);
            if (!usable) {
                histogram(row, s, cluster);
                other = cut_at(row, s, cluster, below, kept);
            }
            cut = other;
        }
        listed = usable && !narrow;
        // nothing below the cut is looked at again
        if (cut.bin == kBins) row.floor = logit_of((unsigned long long)cut.key << 20);
        else row.only_up_to(cut.bin, temperature);
    }

    // what is kept, and the token that the random number falls on
    auto weight = [&](float v, int index) -> unsigned long long {
        // (most logits lie below the cut: their exponentials are not needed)
        const float x = row.argument(v);
        if (cut.bin >= 0) {
            const int b = cut.bin == kBins ? kBins : -x * kBinsPerArgument < (float)kBins ? bin_of(x) : kBins;
            if (b > cut.bin) return 0;
            if (b == cut.bin) {
                const uint32_t key = Key<float>::of(v);
                if (key < cut.key || (key == cut.key && index > cut.index)) return 0;
            }
        }
        const float e = expf(x);
        const unsigned long long w = e < min_p ? 0 : weight_of(e);
        return w;
    };
    unsigned long long of_warp = 0, none = 0;
    if (listed) {
        const unsigned long long least = (unsigned long long)cut.key << 20 | (unsigned)(kMostVocab - 1 - cut.index);
        int index[Listed::kEach];
#pragma unroll
        for (int j = 0; j < Listed::kEach; ++j) {
            const int i = threadIdx.x + j * kThreads;
            index[j] = 0x7fffffff;       // (not kept)
            if (i < s.listed) {
                const unsigned long long c = s.list[i];
                if (c >= least && expf(row.argument(logit_of(c))) >= min_p) index[j] = index_of(c), of_warp += mine.weight[j];
            }
        }
        unsigned long long total = warp_sum64(of_warp), own = total;
        team.exchange(s, total, none);           // (nothing of another CTA is read from here on)
        const unsigned long long target = min((unsigned long long)floor(u * (double)total), total - 1), before = team.before_a;
        own = s.shared_a[team.turn ^ 1][rank];
        if (target < before || target >= before + own) return;
        // The token among this CTA's: by buckets of indices, then inside of one
        const int base = max(rank * kWarps * each * Row<T>::kV - row.skew, 0), span = min(kWarps * each * Row<T>::kV, a.vocab - base);
        int shift = 0;                           // (up to 9: indices lie below 2^20, whatever a warp's whole vectors add up to)
        while ((span - 1) >> shift >= kBins) ++shift;
        clear(s);
#pragma unroll
        for (int j = 0; j < Listed::kEach; ++j)
            if (index[j] != 0x7fffffff && mine.weight[j] != 0) atomicAdd(&s.mass[(index[j] - base) >> shift], mine.weight[j]);
        if (threadIdx.x == 0) s.narrowed = 0;
        __syncthreads();
        constexpr int kPer = kBins / kThreads;
        unsigned long long sum = 0, all;
#pragma unroll
        for (int k = 0; k < kPer; ++k) sum += s.mass[threadIdx.x * kPer + k];
        unsigned long long up = before + scan64(s, sum, all);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const unsigned long long m = s.mass[threadIdx.x * kPer + k];
            if (target >= up && target < up + m) s.found = threadIdx.x * kPer + k, s.found_mass = up;
            up += m;
        }
        __syncthreads();
        const int bucket = s.found;
        up = s.found_mass;
#pragma unroll
        for (int j = 0; j < Listed::kEach; ++j)
            if (index[j] != 0x7fffffff && mine.weight[j] != 0 && (index[j] - base) >> shift == bucket) {
                const uint32_t at = atomicAdd(&s.narrowed, 1u);          // (a bucket has 2^20 / 2048 indices at most, which fit)
                if (at < kShort) s.narrow[at] = (unsigned long long)(index[j] - base) << 41 | mine.weight[j];
            }
        __syncthreads();
        constexpr unsigned long long kWeight = (1ull << 41) - 1;
        const int n = s.narrowed;
        if (threadIdx.x < n) {
            const unsigned long long c = s.narrow[threadIdx.x], w = c & kWeight;
            for (int k = 0; k < n; ++k) up += s.narrow[k] < c ? s.narrow[k] & kWeight : 0;
            if (target >= up && target < up + w) {
                a.tokens[r] = base + (int)(c >> 41);
                a.logprobs[r] = (float)(log((double)w) - log((double)total));
            }
        }
        return;
    }
    row.each([&](float v, int index) { of_warp += weight(v, index); });
    of_warp = warp_sum64(of_warp);
    unsigned long long total = of_warp;
    team.exchange(s, total, none);               // (nothing of another CTA is read from here on)
    unsigned long long before = team.before_a;
    for (int w = 0; w < warp; ++w) before += s.warp_sum[w];
    const double wanted = floor(u * (double)total);
    const unsigned long long target = min((unsigned long long)wanted, total - 1);
    if (target < before || target >= before + of_warp) return;
    unsigned long long left = target - before;
    constexpr int kV = Row<T>::kV;
#pragma unroll 1
    for (int i = row.begin; i < row.end; i += 32) {
        const int at = (i + lane) * kV - row.skew;
        Pack<T, kV> p;
        bool in = i + lane < row.end;
        if (in) p = row.vector(i + lane), in = Row<T>::largest_of(p) >= row.floor;
        unsigned long long w[kV], sum = 0;
#pragma unroll
        for (int e = 0; e < kV; ++e) w[e] = in ? weight(p.at(e), at + e) : 0, sum += w[e];
        unsigned long long up = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long b = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += b;
        }
        const unsigned long long all = __shfl_sync(0xffffffffu, up, 31);
        if (left < all) {
            left -= up - sum;                    // (of the lanes in front of it: none of its own any more)
            if (left < sum) {
#pragma unroll
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

// Clusters of this size that the current device has room for at once: asked once for each type, size and device
template <typename T>
int clusters_at_once(int size, const cudaLaunchConfig_t& cfg) {
    static std::atomic<int> known[64][4];        // (by device and log2 of the size; one more than the number, 0: not asked yet)
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
    std::atomic<int>& here = known[device][size == 8 ? 3 : size == 4 ? 2 : 1];
    int n = here.load(std::memory_order_relaxed);
    if (n == 0) {
        int found = 0;
        if (cudaOccupancyMaxActiveClusters(&found, sample_kernel<T>, &cfg) != cudaSuccess) {
            cudaGetLastError();                  // (it is no call's: a CTA to a row will do)
            return 0;
        }
        here.store(n = found + 1, std::memory_order_relaxed);
    }
    return n - 1;
}

template <typename T>
int run_sample(const SampleArgs& a, int64_t rows, cudaStream_t st) {
    constexpr size_t kBytes = sizeof(Shared);
    if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBytes) != cudaSuccess) return DCN_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    // As many CTAs to a row as leave room for all rows at once: 16-bit kernels fill an SM's registers with one CTA, float32's with two, and the
    // parts of the GPU hold whole clusters only (bf16, 50257 tokens, 50 best: 32 rows 12.6 us in clusters of four, 25.8 of eight; 16384 tokens,
    // 0.95 of the mass: 64 rows 26 us of two, 44 of four).  Where a CTA still has 12288 tokens, up to 7/4 as many CTAs as SMs: rows take
    // unequal times, and the last ones begin when the first end (131072 tokens, 0.95 of the mass: 48 rows 116 us of four, 140 of two; 16 rows
    // 55 us of eight, 84 of four; but of 50 best, 20 and 14).
    int cluster = 1;
    for (int size = 2; size <= kMostCluster && a.vocab / size >= 4096; size *= 2) {
        attr[0].val.clusterDim.x = size;
        cfg.gridDim = dim3((unsigned)(rows * size)), cfg.numAttrs = 1;
        if (rows > clusters_at_once<T>(size, cfg) && !(a.vocab / size >= 12288 && rows * size * 4 <= 7 * dcn::sm_count())) break;
        cluster = size;
    }
    cfg.gridDim = dim3((unsigned)(rows * cluster));
    attr[0].val.clusterDim.x = cluster;
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
