// Rows of logits: log-probabilities of given tokens, entropy and best alternatives; KL divergence from a teacher's best tokens;
// the gradients of both.
//
// Forward, one pass: every thread keeps the running maximum m of its logits, S = sum e and U = sum e d of
//     d = (z - m) / (temperature ln 2),  e = 2^d
// and rescales the sums where m grows; the threads of a row, and the CTAs of a cluster where rows are few, join theirs:
//     log p_j = ln 2 (d_j - log2 S),   entropy = ln 2 (log2 S - U / S).
// Backward, one pass over elements that are independent of one another given a row's (m, log2 S):
//     dz_j = p_j (c0 + c1 log2 p_j)  and a term more at the row's special tokens (the given one, the alternatives, the teacher's),
// which are written once the row's other elements are.  Both are bound by DRAM: a read of the logits, and a write of
// their gradient.  Rows start wherever they do: what lies before the first and behind the last whole 16-byte vector is taken
// element by element.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace cg = cooperative_groups;

namespace dcn {
namespace seq {
namespace {

constexpr int kThreads = 256;                    // of a CTA that has a row, or a part of one
constexpr int kWarpRows = 4;                     // rows of a CTA whose warps have one each
constexpr int kCluster = 8;
constexpr int kMostTop = DCN_SCORES_MOST_TOP, kMostK = DCN_DISTILL_MOST_K;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = 1e30f;                    // logits beyond it are shifted before they are scaled
constexpr float kNone = -__builtin_huge_valf();

enum Kind { kScores, kScoresTop, kDistill };

// The row's statistics for the backward pass
enum Stat { kM, kLogS, kEntropy, kRestM = 2, kRestLogS, kRestC, kMass, kNorm };

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// d = (v - m) k.  As one product and one sum, unless that could overflow where v - m does not (masks of a type's lowest value);
// the rounded m k is the same wherever a row's m is used, so it drops out of d - log2 S.
struct Shift {
    float m, k, mk;
    bool far;
    __device__ __forceinline__ Shift(float m_, float k_) : m(m_), k(k_) {
        mk = __fmul_rn(m, k);
        far = !(fabsf(m) < kFar);
    }
    __device__ __forceinline__ float operator()(float v) const {
        return far ? __fmul_rn(__fsub_rn(v, m), k) : __fmaf_rn(v, k, -mk);
    }
    // from sums at this m to sums at another
    __device__ __forceinline__ float to(const Shift& o) const {
        return max_nan(far || o.far ? __fmul_rn(__fsub_rn(m, o.m), k) : __fsub_rn(mk, o.mk), -kFar);
    }
};

struct Sums {
    float m, s, u;
    // the same sums at a maximum that is at least as large
    __device__ __forceinline__ void rescale(float to, float k) {
        if (m == kNone || m == to) {             // nothing summed yet, or nothing to do
            m = to;
            return;
        }
        const float d = Shift(m, k).to(Shift(to, k)), f = ex2(d);
        u = f * fmaf(s, d, u);
        s *= f;
        m = to;
    }
};

// A row, or a part of one: vectors [v0, v1), the elements before the first vector (head) and behind the last (from tail on)
template <typename T>
struct Row {
    static constexpr int kPer = 16 / sizeof(T);
    const T* p;
    int n, head, head_here, v0, v1, tail;
    __device__ __forceinline__ Row(const T* p_, int n_, int part, int parts) : p(p_), n(n_) {
        const int off = (int)(reinterpret_cast<uintptr_t>(p) % 16) / (int)sizeof(T);
        head = min(n, (kPer - off) % kPer);
        const int vectors = (n - head) / kPer;
        v0 = (int)((int64_t)vectors * part / parts);
        v1 = (int)((int64_t)vectors * (part + 1) / parts);
        tail = part == parts - 1 ? head + vectors * kPer : n;
        head_here = part == 0 ? head : 0;
    }
    __device__ __forceinline__ const T* vec(int v) const { return p + head + (int64_t)v * kPer; }
    // the part's elements: f(element, value), in any order
    template <typename F>
    __device__ __forceinline__ void each(int tid, int threads, F&& f) const {
        for (int e = tid; e < head_here; e += threads) f(e, one(e));
        for (int v = v0 + tid; v < v1; v += threads) {
            Pack<T, kPer> a;
            a.get(vec(v));
#pragma unroll
            for (int i = 0; i < kPer; ++i) f(head + v * kPer + i, a.at(i));
        }
        for (int e = tail + tid; e < n; e += threads) f(e, one(e));
    }
    __device__ __forceinline__ float one(int64_t e) const {
        Pack<T, 1> a;
        a.get(p + e);
        return a.at(0);
    }
};

// Marks of tokens in a part of a row: bit (element - head) + 8, so that a vector's bits lie within one byte
template <typename T>
__device__ __forceinline__ int mark_of(const Row<T>& row, int e) { return e - row.head - row.v0 * Row<T>::kPer + 8; }
template <typename T>
__device__ __forceinline__ bool in_part(const Row<T>& row, int e) {
    return e < row.head ? e < row.head_here : e >= row.tail || (e >= row.head + row.v0 * Row<T>::kPer && e < row.head + row.v1 * Row<T>::kPer);
}

template <bool kU>
__device__ __forceinline__ void add_one(Sums& a, float v, float k) {
    const float m = max_nan(a.m, v);
    if (m == kNone) return;
    a.rescale(m, k);
    float d = Shift(m, k)(v);
    if constexpr (kU) d = max_nan(d, -kFar);     // (0 times it is 0)
    const float e = ex2(d);
    a.s += e;
    if constexpr (kU) a.u = fmaf(e, d, a.u);
}

// The sums of a thread's elements.  kMarks: without the marked ones.
template <typename T, bool kU, bool kMarks>
__device__ __forceinline__ Sums sums_of(const Row<T>& row, int tid, int threads, float k, const uint8_t* marks) {
    constexpr int kPer = Row<T>::kPer, kBatch = 32 / kPer;
    Sums a{kNone, 0.0f, 0.0f};
    auto marked = [&](int e) {
        if constexpr (!kMarks) return false;
        const int b = mark_of(row, e);
        return (marks[b >> 3] >> (b & 7) & 1) != 0;
    };
    for (int e = tid; e < row.head_here; e += threads)
        if (!marked(e)) add_one<kU>(a, row.one(e), k);
    for (int v = row.v0 + tid; v < row.v1; v += kBatch * threads) {
        Pack<T, kPer> raw[kBatch];
        float f[kBatch * kPer];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (v + b * threads < row.v1) raw[b].get(row.vec(v + b * threads));
        float m = a.m;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const bool in = v + b * threads < row.v1;
            uint32_t bits = 0;
            if constexpr (kMarks) {
                const int at = 8 + (v + b * threads - row.v0) * kPer;
                if (in) bits = marks[at >> 3] >> (at & 7);
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                f[b * kPer + i] = in && !(kMarks && (bits >> i & 1)) ? raw[b].at(i) : kNone;
                m = max_nan(m, f[b * kPer + i]);
            }
        }
        if (m == kNone) continue;
        if (m != a.m) a.rescale(m, k);
        const Shift shift(m, k);
        if (shift.far) {
#pragma unroll
            for (int i = 0; i < kBatch * kPer; ++i) add_one<kU>(a, f[i], k);
        } else {
#pragma unroll
            for (int i = 0; i < kBatch * kPer; ++i) {
                float d = __fmaf_rn(f[i], k, -shift.mk);
                if constexpr (kU) d = max_nan(d, -kFar);
                const float e = ex2(d);
                a.s += e;
                if constexpr (kU) a.u = fmaf(e, d, a.u);
            }
        }
    }
    for (int e = row.tail + tid; e < row.n; e += threads)
        if (!marked(e)) add_one<kU>(a, row.one(e), k);
    return a;
}

// The threads of a row: a warp, or a CTA.
template <bool kWarp>
struct Team {
    float* room;                                 // 32 x 2 floats, of a CTA
    int tid, threads;
    __device__ __forceinline__ void sync() const {
        if constexpr (kWarp) __syncwarp();
        else __syncthreads();
    }
    template <typename F>
    __device__ __forceinline__ float fold(float v, float none, F&& f) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        if constexpr (!kWarp) {
            __syncthreads();
            if (tid % 32 == 0) room[tid / 32] = v;
            __syncthreads();
            v = tid % 32 < threads / 32 ? room[tid % 32] : none;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        }
        return v;
    }
    __device__ __forceinline__ float max(float v) const { return fold(v, kNone, [](float a, float b) { return max_nan(a, b); }); }
    __device__ __forceinline__ float sum(float v) const { return fold(v, 0.0f, [](float a, float b) { return a + b; }); }
    __device__ __forceinline__ Sums join(Sums a, float k, bool with_u) const {
        a.rescale(max(a.m), k);
        a.s = sum(a.s);
        if (with_u) a.u = sum(a.u);
        return a;
    }
};

// ---- the best alternatives ------------------------------------------------------------------------------------------------
// A key of 32 bits orders values as they are ranked (NaN first, then by size, -0 as 0); with the complement of the index
// behind it, equal values come by their index and no two keys are the same.  0 is less than every value's key.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    if (key == 0xffffffffu) return CUDART_NAN_F;
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

constexpr int kRoom = 1024;                      // entries of a list

struct TopRoom {
    unsigned long long above[kRoom], equal[kRoom];          // what is over the bound, and what is on it
    unsigned long long best[kCluster][kMostTop];            // the parts' results, in the first CTA of a cluster
    uint32_t maxima[kThreads];
    uint32_t bound;
    int n_above, n_equal, count[kThreads / 32];
};

// Entry i of a list goes to the place of its rank
__device__ __forceinline__ void place(const unsigned long long* list, int n, int tid, int top, unsigned long long* out) {
    for (int i = tid; i < n; i += kThreads) {
        const unsigned long long mine = list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list[j] > mine;
        if (rank < top && mine != 0) out[rank] = mine;
    }
}

__device__ __forceinline__ int block_count(TopRoom& r, int v, int tid) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (tid % 32 == 0) r.count[tid / 32] = v;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kThreads / 32; ++w) sum += r.count[w];
    return sum;
}

// The `top` largest keys of a CTA's part, in order, into out[0, top) (0 behind the last, where the part has fewer).
// Bound: the top-th largest of the threads' maxima `mine`, which at least `top` elements reach.  What is over it, rarely much more
// than `top`, is listed and ranked.  If fewer than `top` are over it, the bound is the value of the last places, which go to the
// lowest indices that have it.  If more are over it than the list holds (large values all in few threads' hands), the value
// of the last place is found by bisection.
template <typename T>
__device__ __forceinline__ void top_of(const Row<T>& row, float mine, int tid, int top, TopRoom& r, unsigned long long* out) {
    const bool any = row.v0 + tid < row.v1 || tid < row.head_here || row.tail + tid < row.n;
    r.maxima[tid] = any ? key_of(mine) : 0;
    if (tid < top) out[tid] = 0;
    if (tid == 0) r.n_above = r.n_equal = 0;
    __syncthreads();
    const uint32_t my_key = r.maxima[tid];
    int rank = 0;
    for (int j = 0; j < kThreads; ++j) rank += r.maxima[j] > my_key || (r.maxima[j] == my_key && j < tid);
    if (rank == top - 1) r.bound = my_key;
    __syncthreads();
    uint32_t bound = r.bound;
    for (int attempt = 0; attempt < 2; ++attempt) {
        const float least = bound == 0 ? kNone : value_of(bound);
        row.each(tid, kThreads, [&](int e, float v) {
            if (v < least) return;
            const uint32_t key = key_of(v);
            const unsigned long long entry = (unsigned long long)key << 32 | (uint32_t)~e;
            if (key > bound) {
                if (*(volatile int*)&r.n_above <= kRoom) {
                    const int at = atomicAdd(&r.n_above, 1);
                    if (at < kRoom) r.above[at] = entry;
                }
            } else if (key == bound && *(volatile int*)&r.n_equal <= kRoom) {
                const int at = atomicAdd(&r.n_equal, 1);
                if (at < kRoom) r.equal[at] = entry;
            }
        });
        __syncthreads();
        if (r.n_above <= kRoom) break;
        uint32_t hi = 0xffffffffu;               // the largest key that `top` elements reach: in [bound, hi]
        while (bound < hi) {
            const uint32_t mid = bound + (hi - bound) / 2 + 1;
            int n = 0;
            row.each(tid, kThreads, [&](int, float v) { n += key_of(v) >= mid; });
            if (block_count(r, n, tid) >= top) bound = mid;
            else hi = mid - 1;
        }
        __syncthreads();
        if (tid == 0) r.n_above = r.n_equal = 0;
        __syncthreads();
    }
    const int above = min(r.n_above, kRoom), equal = r.n_equal;
    place(r.above, above, tid, top, out);
    const int need = top - above;
    if (need > 0 && equal > 0) {
        if (equal <= kRoom) {
            place(r.equal, equal, tid, need, out + above);
        } else {                                 // dense: the first of them by index, a vector a thread at a time
            constexpr int kPer = Row<T>::kPer;
            int done = 0;
            auto take = [&](int e, float v, bool in, int& before) {
                if (in && key_of(v) == bound) {
                    if (before < need) out[above + before] = (unsigned long long)bound << 32 | (uint32_t)~e;
                    ++before;
                }
            };
            // threads in the order of their elements: places from a prefix sum of their counts
            auto places = [&](int mine_n) {
                int before = mine_n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int up = __shfl_up_sync(0xffffffffu, before, o);
                    if (tid % 32 >= o) before += up;
                }
                __syncthreads();
                if (tid % 32 == 31) r.count[tid / 32] = before;
                __syncthreads();
                int start = done, all = 0;
                for (int w = 0; w < kThreads / 32; ++w) {
                    if (w < tid / 32) start += r.count[w];
                    all += r.count[w];
                }
                done += all;
                return start + before - mine_n;
            };
            {
                const bool in = tid < row.head_here;
                const float v = in ? row.one(tid) : 0.0f;
                int at = places(in && key_of(v) == bound);
                take(tid, v, in, at);
            }
            for (int v0 = row.v0; v0 < row.v1 && done < need; v0 += kThreads) {
                const int v = v0 + tid;
                Pack<T, kPer> a;
                a.zero();
                if (v < row.v1) a.get(row.vec(v));
                int n = 0;
#pragma unroll
                for (int i = 0; i < kPer; ++i) n += v < row.v1 && key_of(a.at(i)) == bound;
                int at = places(n);
                if (n > 0)
#pragma unroll
                    for (int i = 0; i < kPer; ++i) take(row.head + v * kPer + i, a.at(i), true, at);
            }
            if (done < need) {
                const int e = row.tail + tid;
                const bool in = e < row.n;
                const float v = in ? row.one(e) : 0.0f;
                int at = places(in && key_of(v) == bound);
                take(e, v, in, at);
            }
        }
    }
    __syncthreads();
}

// ---- forward --------------------------------------------------------------------------------------------------------------
struct LogitsArgs {
    const void* logits;
    int64_t rows, stride;
    int vocab;
    float k, temperature;                        // k = log2 e / temperature
    float* stats;
    // scores
    const int64_t* tokens;
    int64_t ignore;
    int top;
    float *logprob, *entropy, *top_logprobs;
    int64_t* top_tokens;
    const float *dlogprob, *dentropy, *dtop;
    // distillation
    const void* teacher;
    const int64_t* teacher_tokens;
    int places, wide_teacher, tail;
    float* loss;
    const float* dloss;
    void* dlogits;
    int marks;                                   // bytes of a part's marks
};

template <typename T>
__device__ __forceinline__ float teacher_at(const LogitsArgs& p, int64_t at) {
    if (p.wide_teacher) return gload(static_cast<const float*>(p.teacher) + at);
    Pack<T, 1> v;
    v.get(static_cast<const T*>(p.teacher) + at);
    return v.at(0);
}

// log p of a value; -inf where the row has nothing.  Logits of the size of the type's range are not put in units of log 2.
__device__ __forceinline__ float log_p(float v, float m, float log_s, const LogitsArgs& p) {
    if (m == kNone) return kNone;
    const float plain = (v - m) / p.temperature;
    return fabsf(plain) > kFar ? plain - kLn2 * log_s : kLn2 * (Shift(m, p.k)(v) - log_s);
}

__device__ __forceinline__ float product_or_zero(float p, float v) { return p > 0.0f || p != p ? p * v : 0.0f; }

struct TeacherRoom {
    int token[kMostK];                           // -1: not used
    float log_q[kMostK], logit[kMostK];
};

// The teacher's places of a row: tokens and log q (normalised over them where there is no tail)
template <typename T, bool kWarp>
__device__ __forceinline__ float teacher_of(const LogitsArgs& p, int64_t row, const Team<kWarp>& team, TeacherRoom& r, int& used) {
    int n = 0;
    float m = kNone;
    for (int i = team.tid; i < p.places; i += team.threads) {
        const int64_t t = gload_i64(p.teacher_tokens + row * p.places + i);
        const bool in = t >= 0 && t < p.vocab;
        const float lq = in ? teacher_at<T>(p, row * p.places + i) : kNone;
        r.token[i] = in ? (int)t : -1;
        r.log_q[i] = lq;
        n += in;
        m = max_nan(m, lq);
    }
    used = (int)team.sum((float)n);
    float norm = 0.0f;
    if (!p.tail) {
        m = team.max(m);
        float s = 0.0f;
        for (int i = team.tid; i < p.places; i += team.threads) s += m == kNone ? 0.0f : expf(r.log_q[i] - m);
        norm = m == kNone ? 0.0f : m + logf(team.sum(s));
        if (m == kNone) used = 0;                // no probability anywhere: as if no place were used
        for (int i = team.tid; i < p.places; i += team.threads) r.log_q[i] -= norm;
    }
    team.sync();
    return norm;
}

template <typename T, bool kWarp>
__device__ __forceinline__ void distill_row(const LogitsArgs& p, int64_t row, const T* logits, const Team<kWarp>& team,
                                            TeacherRoom& r, Sums rest, float norm, int used) {
    // the student's sums over the teacher's tokens, each token once
    Sums best{kNone, 0.0f, 0.0f};
    float mass = 0.0f;
    for (int i = team.tid; i < p.places; i += team.threads) {
        const int t = r.token[i];
        if (t < 0) continue;
        mass += expf(r.log_q[i]);
        bool again = false;
        for (int j = 0; j < i; ++j) again |= r.token[j] == t;
        if (!again) add_one<false>(best, r.logit[i], p.k);
    }
    best = team.join(best, p.k, false);
    mass = team.sum(mass);
    const float m = max_nan(best.m, rest.m);
    Sums all = best, other = rest;
    if (m != kNone) {
        all.rescale(m, p.k);
        other.rescale(m, p.k);
    }
    const float log_s = log2f(all.s + other.s), rest_log_s = log2f(rest.s);
    float loss = 0.0f;
    for (int i = team.tid; i < p.places; i += team.threads) {
        if (r.token[i] < 0) continue;
        const float lq = r.log_q[i];
        loss += product_or_zero(expf(lq), lq - log_p(r.logit[i], m, log_s, p));
    }
    loss = team.sum(loss);
    if (team.tid != 0) return;
    float q_rest = 0.0f, c = 0.0f;
    if (p.tail && rest.m != kNone) q_rest = fmaxf(1.0f - mass, 0.0f);
    if (mass != mass) q_rest = mass;
    if (rest.m != kNone) {
        const float log_rest = kLn2 * (Shift(rest.m, p.k).to(Shift(m, p.k)) + rest_log_s - log_s);
        loss += product_or_zero(q_rest, logf(q_rest) - log_rest);
        c = fmaf(mass + q_rest, expf(log_rest), -q_rest);
    }
    if (used == 0) loss = c = mass = q_rest = 0.0f;
    p.loss[row] = loss * p.temperature * p.temperature;
    if (p.stats != nullptr) {
        float* s = p.stats + row * DCN_LOGITS_STATS;
        s[kM] = m, s[kLogS] = log_s, s[kRestM] = rest.m, s[kRestLogS] = rest_log_s;
        s[kRestC] = c, s[kMass] = mass + q_rest, s[kNorm] = norm;
    }
}

template <typename T, int kKind, bool kWarp>
__global__ void __launch_bounds__(kThreads) logits_forward_kernel(const LogitsArgs p) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float room[32];
    __shared__ Sums parts[kCluster];
    __shared__ TeacherRoom teachers[kKind == kDistill ? (kWarp ? kWarpRows : 1) : 1];
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = kWarp ? 0 : (int)cluster.block_rank(), ranks = kWarp ? 1 : (int)cluster.num_blocks();
    const int group = kWarp ? threadIdx.x / 32 : 0;
    const int64_t at = kWarp ? (int64_t)blockIdx.x * kWarpRows + group : blockIdx.x / ranks;
    const Team<kWarp> team{room, kWarp ? (int)threadIdx.x % 32 : (int)threadIdx.x, kWarp ? 32 : kThreads};
    if (ranks > 1) cluster.sync();               // every CTA runs before another writes to its memory
    if (at >= p.rows) return;                    // (a warp's row: a CTA's is always there)
    pdl_wait();
    const T* logits = static_cast<const T*>(p.logits) + at * p.stride;
    const Row<T> row(logits, p.vocab, rank, ranks);
    TopRoom& top = *reinterpret_cast<TopRoom*>(dynamic);
    TeacherRoom& teacher = teachers[kKind == kDistill ? group : 0];
    uint8_t* marks = dynamic + group * p.marks;
    float norm = 0.0f;
    int used = 0;
    if constexpr (kKind == kDistill) {
        for (int i = team.tid; i < p.marks / 4; i += team.threads) reinterpret_cast<uint32_t*>(marks)[i] = 0;
        norm = teacher_of<T, kWarp>(p, at, team, teacher, used);
        for (int i = team.tid; i < p.places; i += team.threads) {
            const int t = teacher.token[i];
            if (t < 0) continue;
            if (rank == 0) teacher.logit[i] = row.one(t);
            if (in_part(row, t)) {
                const int b = mark_of(row, t);
                atomicOr(reinterpret_cast<uint32_t*>(marks) + (b >> 5), 1u << (b & 31));
            }
        }
        team.sync();
    }
    const Sums mine = sums_of<T, kKind != kDistill, kKind == kDistill>(row, team.tid, team.threads, p.k, marks);
    Sums sums = team.join(mine, p.k, kKind != kDistill);
    if constexpr (kKind == kScoresTop) {
        if (ranks == 1) {
            top_of(row, mine.m, team.tid, p.top, top, top.best[0]);
        } else {
            top_of(row, mine.m, team.tid, p.top, top, top.best[rank]);
            if (rank > 0 && team.tid < p.top) *cluster.map_shared_rank(&top.best[rank][team.tid], 0) = top.best[rank][team.tid];
        }
    }
    if (ranks > 1) {
        if (team.tid == 0) *cluster.map_shared_rank(&parts[rank], 0) = sums;
        cluster.sync();
        if (rank > 0) return;
        float m = parts[0].m;
        for (int r = 1; r < ranks; ++r) m = max_nan(m, parts[r].m);
        sums = Sums{m, 0.0f, 0.0f};
        for (int r = 0; r < ranks; ++r) {
            Sums other = parts[r];
            other.rescale(m, p.k);
            sums.s += other.s;
            sums.u += other.u;
        }
    }
    if constexpr (kKind == kDistill) {
        distill_row<T, kWarp>(p, at, logits, team, teacher, sums, norm, used);
    } else {
        const float log_s = log2f(sums.s);
        const float entropy = sums.m == kNone ? 0.0f : kLn2 * (log_s - sums.u / sums.s);
        if (team.tid == 0) {
            if (p.logprob != nullptr) {
                const int64_t t = gload_i64(p.tokens + at);
                float v = CUDART_NAN_F;
                if (t == p.ignore) v = 0.0f;
                else if (t >= 0 && t < p.vocab) v = log_p(row.one(t), sums.m, log_s, p);
                p.logprob[at] = v;
            }
            if (p.entropy != nullptr) p.entropy[at] = entropy;
            if (p.stats != nullptr) {
                float* s = p.stats + at * DCN_LOGITS_STATS;
                s[kM] = sums.m, s[kLogS] = log_s, s[kEntropy] = entropy;
            }
        }
        if constexpr (kKind == kScoresTop) {
            unsigned long long* best = top.best[0];
            if (ranks > 1) {                     // the parts' best, ranked among one another
                for (int i = team.tid; i < ranks * p.top; i += kThreads) top.above[i] = top.best[i / p.top][i % p.top];
                __syncthreads();
                place(top.above, ranks * p.top, team.tid, p.top, top.equal);
                __syncthreads();
                best = top.equal;
            }
            for (int i = team.tid; i < p.top; i += kThreads) {
                const unsigned long long entry = best[i];
                p.top_tokens[at * p.top + i] = (int64_t)(uint32_t)~(uint32_t)entry;
                p.top_logprobs[at * p.top + i] = log_p(value_of((uint32_t)(entry >> 32)), sums.m, log_s, p);
            }
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------
// dz = 2^l (c0 + c1 l), l = log2 p: p from (m, log2 S)
struct Slope {
    Shift shift;
    float log_s, c0, c1;
    bool zero;
    __device__ __forceinline__ Slope(float m, float k, float log_s_, float c0_, float c1_)
        : shift(m, k), log_s(log_s_), c0(c0_), c1(c1_), zero(m == kNone) {}
    __device__ __forceinline__ float operator()(float v) const {
        if (zero) return 0.0f;
        const float l = max_nan(shift(v) - log_s, -kFar);
        return ex2(l) * fmaf(c1, l, c0);
    }
};

template <typename T, bool kDistilled>
__global__ void __launch_bounds__(kThreads) logits_backward_kernel(const LogitsArgs p, int parts) {
    constexpr int kPer = Row<T>::kPer;
    __shared__ int token[kMostTop + 1];
    __shared__ float weight[kMostTop + 1];
    __shared__ float room[32];
    const int tid = threadIdx.x, threads = blockDim.x;
    const int64_t at = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    pdl_wait();
    const Row<T> row(static_cast<const T*>(p.logits) + at * p.stride, p.vocab, part, parts);
    T* out = static_cast<T*>(p.dlogits) + at * p.vocab;
    const float* stat = p.stats + at * DCN_LOGITS_STATS;
    const float m = gload(stat + kM), log_s = gload(stat + kLogS);
    // the special tokens and what they get beside the slope
    const Team<false> team{room, tid, threads};
    int specials;
    Slope slope(m, p.k, log_s, 0.0f, 0.0f), special = slope;
    if constexpr (kDistilled) {
        specials = p.places;
        const float g = gload(p.dloss + at) * p.temperature;
        slope = Slope(gload(stat + kRestM), p.k, gload(stat + kRestLogS), g * gload(stat + kRestC), 0.0f);
        special.c0 = g * gload(stat + kMass);
        const float norm = gload(stat + kNorm);
        for (int i = tid; i < specials; i += threads) {
            const int64_t t = gload_i64(p.teacher_tokens + at * p.places + i);
            const bool in = t >= 0 && t < p.vocab;
            token[i] = in ? (int)t : -1;
            weight[i] = in ? -g * expf(teacher_at<T>(p, at * p.places + i) - norm) : 0.0f;
        }
    } else {
        specials = p.dtop != nullptr ? p.top + 1 : 1;
        const float scale = 1.0f / p.temperature;
        const float gh = p.dentropy != nullptr ? gload(p.dentropy + at) : 0.0f;
        float all = 0.0f;
        for (int i = tid; i < specials; i += threads) {
            float g = 0.0f;
            int64_t t = -1;
            if (i > 0) {
                t = gload_i64(p.top_tokens + at * p.top + i - 1);
                g = gload(p.dtop + at * p.top + i - 1);
            } else if (p.dlogprob != nullptr) {
                t = gload_i64(p.tokens + at);
                g = gload(p.dlogprob + at);
                if (t == p.ignore) t = -1;
            }
            const bool in = t >= 0 && t < p.vocab;
            token[i] = in ? (int)t : -1;
            weight[i] = in ? g * scale : 0.0f;
            all += weight[i];
        }
        if (specials > 1) {
            all = team.sum(all);
        } else {
            __syncthreads();
            all = weight[0];
        }
        slope.c0 = -fmaf(gh * scale, gload(stat + kEntropy), all);
        slope.c1 = -scale * kLn2 * gh;
        special = slope;
    }
    // vectors where the gradient's rows start as the logits' do, elements otherwise
    const bool same = reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(row.p) % 16;
    auto put = [&](int64_t e, float v) { out[e] = from_float<T>(v); };
    for (int e = tid; e < row.head_here; e += threads) put(e, slope(row.one(e)));
    constexpr int kBatch = 4;
    for (int v = row.v0 + tid; v < row.v1; v += kBatch * threads) {
        Pack<T, kPer> raw[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (v + b * threads < row.v1) raw[b].get(row.vec(v + b * threads));
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (v + b * threads >= row.v1) break;
            float f[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) f[i] = slope(raw[b].at(i));
            T* to = out + row.head + (int64_t)(v + b * threads) * kPer;
            if (same) {
                Pack<T, kPer> o;
                o.set(f);
                o.put(to);
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i) to[i] = from_float<T>(f[i]);
            }
        }
    }
    for (int e = row.tail + tid; e < row.n; e += threads) put(e, slope(row.one(e)));
    __syncthreads();                             // the part's special tokens are written over what stands there
    if (special.zero) return;
    for (int i = tid; i < specials; i += threads) {
        const int t = token[i];
        if (t < 0 || !in_part(row, t)) continue;
        float w = 0.0f;
        for (int j = 0; j < specials; ++j) w += token[j] == t ? weight[j] : 0.0f;
        put(t, special(row.one(t)) + w);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
constexpr int kWarpVocab = 2048;                 // rows up to this size: a warp each, where no alternatives are asked for

int parts_of(int64_t rows, int64_t vocab) {
    int parts = 1;
    while (parts < kCluster && rows * parts < 2 * sm_count() && vocab / parts > 4096) parts *= 2;
    return parts;
}

template <typename T, int kKind>
int run_forward(LogitsArgs a, cudaStream_t st) {
    const bool warp = kKind != kScoresTop && a.vocab <= kWarpVocab;
    const int parts = warp ? 1 : parts_of(a.rows, a.vocab);
    cudaLaunchConfig_t cfg = {};
    size_t smem = kKind == kScoresTop ? sizeof(TopRoom) : 0;
    if (kKind == kDistill) {
        const int per = 16 / (int)sizeof(T);
        a.marks = (int)(((a.vocab / per + parts - 1) / parts * per + 8 + 2 * per + 8 + 127) / 128 * 16);
        smem = (size_t)a.marks * (warp ? kWarpRows : 1);
    }
    cfg.gridDim = dim3((unsigned)(warp ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows * parts));
    cfg.blockDim = dim3(warp ? 32 * kWarpRows : kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = pdl_enabled() ? attr : attr + 1;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaError_t e = cudaSuccess;
    if constexpr (kKind == kScoresTop) {
        e = cudaLaunchKernelEx(&cfg, logits_forward_kernel<T, kKind, false>, a);
    } else if (warp) {
        e = cudaLaunchKernelEx(&cfg, logits_forward_kernel<T, kKind, true>, a);
    } else {
        if (smem > 40 * 1024) e = cudaFuncSetAttribute(logits_forward_kernel<T, kKind, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, logits_forward_kernel<T, kKind, false>, a);
    }
    return e != cudaSuccess || cudaGetLastError() != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, bool kDistilled>
int run_backward(const LogitsArgs& a, cudaStream_t st) {
    // parts of at most 16384 elements, of a CTA with a vector or more for each thread
    const int64_t parts = (a.vocab + 16383) / 16384;
    const int64_t vectors = a.vocab / parts * (int64_t)sizeof(T) / 16;
    const int threads = vectors >= 192 ? 256 : vectors >= 96 ? 128 : 64;
    if (a.rows * parts >= 1ll << 31) return DCN_ERR_LIMIT;
    return launch_dependent(logits_backward_kernel<T, kDistilled>, dim3((unsigned)(a.rows * parts)), dim3(threads), 0, st, a,
                            (int)parts) != cudaSuccess
               ? DCN_ERR_CUDA
               : DCN_OK;
}

int check_logits(const dcn_logits* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype)) return DCN_ERR_UNSUPPORTED;
    if (p->rows < 0 || p->vocab < 1 || !(p->temperature >= 1e-3f && p->temperature <= 1e3f)) return DCN_ERR_SHAPE;
    if (p->rows >= 1ll << 27 || p->vocab >= 1ll << 31) return DCN_ERR_LIMIT;
    return DCN_OK;
}

LogitsArgs args_of(const dcn_logits* p, const void* logits) {
    LogitsArgs a = {};
    a.logits = logits;
    a.rows = p->rows;
    a.stride = p->row_stride;
    a.vocab = (int)p->vocab;
    a.temperature = p->temperature;
    a.k = (float)(1.4426950408889634 / (double)p->temperature);
    return a;
}

template <int kKind>
int forward_of(int dtype, const LogitsArgs& a, cudaStream_t st) {
    if (dtype == DCN_SEQ_F32) return run_forward<float, kKind>(a, st);
    if (dtype == DCN_SEQ_BF16) return run_forward<__nv_bfloat16, kKind>(a, st);
    return run_forward<__half, kKind>(a, st);
}

template <bool kDistilled>
int backward_of(int dtype, const LogitsArgs& a, cudaStream_t st) {
    if (dtype == DCN_SEQ_F32) return run_backward<float, kDistilled>(a, st);
    if (dtype == DCN_SEQ_BF16) return run_backward<__nv_bfloat16, kDistilled>(a, st);
    return run_backward<__half, kDistilled>(a, st);
}

int check_distill(const dcn_logits* p, const void* logits, int32_t k, const void* teacher, int32_t teacher_dtype,
                  const int64_t* tokens, int32_t tail) {
    const int bad = check_logits(p);
    if (bad != DCN_OK) return bad;
    if (teacher_dtype != DCN_SEQ_F32 && teacher_dtype != p->dtype) return DCN_ERR_UNSUPPORTED;
    if (tail != 0 && tail != 1) return DCN_ERR_UNSUPPORTED;
    if (k < 1) return DCN_ERR_SHAPE;
    if (k > kMostK || p->vocab > DCN_DISTILL_MOST_VOCAB) return DCN_ERR_LIMIT;
    if (p->rows == 0) return DCN_OK;
    if (logits == nullptr || teacher == nullptr || tokens == nullptr) return DCN_ERR_NULL;
    if (!aligned(logits, elem_bytes(p->dtype)) || !aligned(teacher, elem_bytes(teacher_dtype)) || !aligned(tokens, 8))
        return DCN_ERR_ALIGN;
    return DCN_OK;
}

}  // namespace
}  // namespace seq
}  // namespace dcn

using namespace dcn::seq;

extern "C" int dcn_scores_forward(const dcn_logits* p, const void* logits, const int64_t* tokens, int64_t ignore_index,
                                  int32_t top, float* logprob, float* entropy, float* top_logprobs, int64_t* top_tokens,
                                  float* stats, void* stream) {
    const int bad = check_logits(p);
    if (bad != DCN_OK) return bad;
    if (top < 0 || top > p->vocab) return DCN_ERR_SHAPE;
    if (top > kMostTop) return DCN_ERR_LIMIT;
    if (p->rows == 0) return DCN_OK;
    if (logits == nullptr || (logprob != nullptr && tokens == nullptr) ||
        (top > 0 && (top_logprobs == nullptr || top_tokens == nullptr)))
        return DCN_ERR_NULL;
    if (!aligned(logits, elem_bytes(p->dtype)) || !aligned(tokens, 8) || !aligned(top_tokens, 8) || !aligned(logprob, 4) ||
        !aligned(entropy, 4) || !aligned(top_logprobs, 4) || !aligned(stats, 4))
        return DCN_ERR_ALIGN;
    LogitsArgs a = args_of(p, logits);
    a.tokens = tokens, a.ignore = ignore_index, a.top = top, a.logprob = logprob, a.entropy = entropy;
    a.top_logprobs = top_logprobs, a.top_tokens = top_tokens, a.stats = stats;
    const cudaStream_t st = (cudaStream_t)stream;
    return top > 0 ? forward_of<kScoresTop>(p->dtype, a, st) : forward_of<kScores>(p->dtype, a, st);
}

extern "C" int dcn_scores_backward(const dcn_logits* p, const void* logits, const int64_t* tokens, int64_t ignore_index,
                                   int32_t top, const int64_t* top_tokens, const float* stats, const float* dlogprob,
                                   const float* dentropy, const float* dtop, void* dlogits, void* stream) {
    const int bad = check_logits(p);
    if (bad != DCN_OK) return bad;
    if (top < 0 || top > p->vocab) return DCN_ERR_SHAPE;
    if (top > kMostTop) return DCN_ERR_LIMIT;
    if (p->rows == 0) return DCN_OK;
    if (logits == nullptr || stats == nullptr || dlogits == nullptr || (dlogprob != nullptr && tokens == nullptr) ||
        (top > 0 && dtop != nullptr && top_tokens == nullptr))
        return DCN_ERR_NULL;
    const int e = elem_bytes(p->dtype);
    if (!aligned(logits, e) || !aligned(dlogits, e) || !aligned(tokens, 8) || !aligned(top_tokens, 8) || !aligned(stats, 4) ||
        !aligned(dlogprob, 4) || !aligned(dentropy, 4) || !aligned(dtop, 4))
        return DCN_ERR_ALIGN;
    LogitsArgs a = args_of(p, logits);
    a.tokens = tokens, a.ignore = ignore_index, a.top = top, a.top_tokens = const_cast<int64_t*>(top_tokens);
    a.stats = const_cast<float*>(stats), a.dlogprob = dlogprob, a.dentropy = dentropy, a.dtop = top > 0 ? dtop : nullptr;
    a.dlogits = dlogits;
    return backward_of<false>(p->dtype, a, (cudaStream_t)stream);
}

extern "C" int dcn_distill_forward(const dcn_logits* p, const void* logits, int32_t k, const void* teacher_logprobs,
                                   int32_t teacher_dtype, const int64_t* teacher_tokens, int32_t tail, float* loss, float* stats,
                                   void* stream) {
    const int bad = check_distill(p, logits, k, teacher_logprobs, teacher_dtype, teacher_tokens, tail);
    if (bad != DCN_OK || p->rows == 0) return bad;
    if (loss == nullptr) return DCN_ERR_NULL;
    if (!aligned(loss, 4) || !aligned(stats, 4)) return DCN_ERR_ALIGN;
    LogitsArgs a = args_of(p, logits);
    a.teacher = teacher_logprobs, a.teacher_tokens = teacher_tokens, a.places = k, a.tail = tail;
    a.wide_teacher = teacher_dtype == DCN_SEQ_F32, a.loss = loss, a.stats = stats;
    return forward_of<kDistill>(p->dtype, a, (cudaStream_t)stream);
}

extern "C" int dcn_distill_backward(const dcn_logits* p, const void* logits, int32_t k, const void* teacher_logprobs,
                                    int32_t teacher_dtype, const int64_t* teacher_tokens, int32_t tail, const float* stats,
                                    const float* dloss, void* dlogits, void* stream) {
    const int bad = check_distill(p, logits, k, teacher_logprobs, teacher_dtype, teacher_tokens, tail);
    if (bad != DCN_OK || p->rows == 0) return bad;
    if (stats == nullptr || dloss == nullptr || dlogits == nullptr) return DCN_ERR_NULL;
    if (!aligned(stats, 4) || !aligned(dloss, 4) || !aligned(dlogits, elem_bytes(p->dtype))) return DCN_ERR_ALIGN;
    LogitsArgs a = args_of(p, logits);
    a.teacher = teacher_logprobs, a.teacher_tokens = teacher_tokens, a.places = k, a.tail = tail;
    a.wide_teacher = teacher_dtype == DCN_SEQ_F32, a.stats = const_cast<float*>(stats), a.dloss = dloss, a.dlogits = dlogits;
    return backward_of<true>(p->dtype, a, (cudaStream_t)stream);
}
