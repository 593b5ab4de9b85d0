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

#include <algorithm>

#include "seq_common.cuh"

namespace cg = cooperative_groups;

namespace dcn {
namespace seq {
namespace {

constexpr int kThreads = 256;                    // of a CTA that has a row, or a part of one
// of one that has a short row and up to 32 alternatives of it; up to 64: twice as many (4096x1000 bf16, 50 best 37 us, by 256 70 us)
constexpr int kFewThreads = 64;
constexpr int kWarpRows = 4;                     // rows of a CTA whose warps have one each
constexpr int kCluster = 8;
constexpr int kMostTop = DCN_SCORES_MOST_TOP, kMostK = DCN_DISTILL_MOST_K;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = 1e30f;                    // d is not below minus it: 0 times it is 0
constexpr float kGone = 1e4f;                    // 2^-kGone is 0, and what kGone is multiplied with stays finite
constexpr float kNear = 4194304.0f;              // 2^22: up to here a rounded m k is off by an eighth at most
constexpr float kNone = -__builtin_huge_valf();

enum Kind { kScores, kScoresTop, kDistill };

// The row's statistics for the backward pass
enum Stat { kM, kLogS, kEntropy, kRestM = 2, kRestLogS, kRestC, kMass, kNorm };

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// d = (v - m) k.  As one product and one sum, v k - c with c = m k, where m k is small: the rounded m k is the same wherever a row's
// m is used, so what it is off by drops out of d - log2 S.  Larger ones (masks of any finite value, and what is summed before
// anything else is seen) are off by more than 2^d has room for, or overflow where v - m does not: there the difference comes first,
// (v - b) k with b = m.
struct Shift {
    float k, b, c;
    bool far;
    __device__ __forceinline__ Shift(float m, float k_) : k(k_) {
        const float mk = __fmul_rn(m, k);
        far = !(fabsf(mk) < kNear);
        b = far ? m : 0.0f;
        c = far ? 0.0f : mk;
    }
    __device__ __forceinline__ float operator()(float v) const { return __fmaf_rn(__fsub_rn(v, b), k, -c); }
    // from sums at this m to sums at another, each as its d are formed
    __device__ __forceinline__ float to(const Shift& o) const {
        return max_nan(__fmaf_rn(__fsub_rn(b, o.b), k, __fsub_rn(c, o.c)), -kFar);
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

// A row, or a part of one: vectors [v0, v1), the elements before the first vector (head) and behind the last (from tail on).
// single: without vectors, all elements one by one.
template <typename T>
struct Row {
    static constexpr int kPer = 16 / sizeof(T);
    const T* p;
    int n, head, head_here, v0, v1, tail;
    __device__ __forceinline__ Row(const T* p_, int n_, int part, int parts, bool single = false) : p(p_), n(n_) {
        const int off = (int)(reinterpret_cast<uintptr_t>(p) % 16) / (int)sizeof(T);
        head = single ? n : min(n, (kPer - off) % kPer);
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
        for (int i = tid; i < n - tail; i += threads) f(tail + i, one(tail + i));     // (tail + tid may be past 31 bits)
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
    return e < row.head ? e < row.head_here
                        : e >= row.tail || (e >= row.head + row.v0 * Row<T>::kPer && e < row.head + row.v1 * Row<T>::kPer);
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

template <typename T>
__device__ __forceinline__ bool marked(const Row<T>& row, const uint8_t* marks, int e) {
    const int b = mark_of(row, e);
    return (marks[b >> 3] >> (b & 7) & 1) != 0;
}

// Elements one by one, those outside vectors.  Not inlined, so that the usual path stays short.
template <typename T, bool kU, bool kMarks>
__device__ __noinline__ Sums add_elements(Sums a, const Row<T>& row, int e0, int e1, int step, float k, const uint8_t* marks) {
    for (int e = e0; e < e1; e += step) {
        if constexpr (kMarks)
            if (marked(row, marks, e)) continue;
        add_one<kU>(a, row.one(e), k);
    }
    return a;
}

// Words of a vector as the type's own instructions take them
template <typename T>
struct Word {
    static constexpr int kPer = 4 / sizeof(T);
    static constexpr uint32_t kNothing = sizeof(T) == 4                            ? 0xff800000u
                                         : std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u
                                                                                 : 0xfc00fc00u;
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
        uint32_t r;
        if constexpr (sizeof(T) == 4) r = __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    static __device__ __forceinline__ float at(uint32_t w, int i) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else return half_of<T>(w, i);
    }
    // without the element
    static __device__ __forceinline__ uint32_t without(uint32_t w, int i) {
        if constexpr (sizeof(T) == 4) return kNothing;
        else return i == 0 ? (w & 0xffff0000u) | (kNothing & 0xffffu) : (w & 0xffffu) | (kNothing & 0xffff0000u);
    }
};

// Elements 2 i, 2 i + 1 of a vector's words
template <typename T>
__device__ __forceinline__ Lanes pair_of(const uint32_t* w, int i) {
    float f[2];
    if constexpr (sizeof(T) == 4) f[0] = __uint_as_float(w[2 * i]), f[1] = __uint_as_float(w[2 * i + 1]);
    else f[0] = half_of<T>(w[i], 0), f[1] = half_of<T>(w[i], 1);
    return lanes(f);
}

// The sums of a thread's elements.  kMarks: without the marked ones.  kAgain: the elements are read a second time.
template <typename T, bool kU, bool kMarks, bool kAgain, bool kSingle>
__device__ __forceinline__ Sums sums_of(const Row<T>& row, int tid, int threads, float k, const uint8_t* marks) {
    using W = Word<T>;
    constexpr int kPer = Row<T>::kPer, kBatch = 4, kWords = 4 * kBatch;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    Sums a{kNone, 0.0f, 0.0f};
    const int ends = row.head_here + (row.n - row.tail);          // elements outside vectors: at most one a thread, or all (kSingle)
    if (tid < ends) {
        const int e = tid < row.head_here ? tid : row.tail + tid - row.head_here;
        a = add_elements<T, kU, kMarks>(a, row, e, kSingle ? ends : e + 1, kSingle ? threads : 1, k, marks);
    }
    if constexpr (kSingle) return a;
    for (int v = row.v0 + tid; v < row.v1; v += kBatch * threads) {
        uint32_t w[kWords];
        const bool whole = v + (kBatch - 1) * threads < row.v1;
        auto fetch = [&](int b) {
            Raw<16> raw;
            if constexpr (kAgain) load_kept(raw, row.vec(v + b * threads));
            else load(raw, row.vec(v + b * threads));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * b + i] = raw.u[i];
        };
        if (whole) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) fetch(b);
        } else {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * b + i] = W::kNothing;
                if (v + b * threads < row.v1) fetch(b);
            }
        }
        if constexpr (kMarks) {
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int at = 8 + (v + b * threads - row.v0) * kPer;
                if (!whole && v + b * threads >= row.v1) break;
                const uint32_t bits = marks[at >> 3] >> (at & 7) & ((1u << kPer) - 1);
                if (bits == 0) continue;         // (nearly always)
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (bits >> i & 1) w[4 * b + i / W::kPer] = W::without(w[4 * b + i / W::kPer], i % W::kPer);
            }
        }
        uint32_t top = w[0];
#pragma unroll
        for (int i = 1; i < kWords; ++i) top = W::max(top, w[i]);
        float m = max_nan(a.m, W::at(top, 0));
        if constexpr (W::kPer == 2) m = max_nan(m, W::at(top, 1));
        if (m == kNone) continue;
        if (m != a.m) a.rescale(m, k);
        const Shift shift(m, k);
        auto add = [&](auto far) {
            const Lanes kk = all_lanes(k), shifted = all_lanes(far.value ? -shift.b : -shift.c);
            Lanes s = all_lanes(0.0f), u = s;
#pragma unroll
            for (int i = 0; i < kWords * W::kPer / 2; ++i) {
                // 0 times what is far below is 0, not NaN: logits of -inf are raised to where their d is finite
                if constexpr (kU && kBf16 && !far.value) w[i] = W::max(w[i], 0xf14af14au);            // -1e30
                Lanes d = far.value ? (pair_of<T>(w, i) + shifted) * kk : fma(pair_of<T>(w, i), kk, shifted);
                if constexpr (kU && (!kBf16 || far.value)) {
                    const float f[2] = {max_nan(d.at(0), -kFar), max_nan(d.at(1), -kFar)};
                    d = lanes(f);
                }
                const float e[2] = {ex2(d.at(0)), ex2(d.at(1))};
                s = s + lanes(e);
                if constexpr (kU) u = fma(lanes(e), d, u);
            }
            a.s += s.at(0) + s.at(1);
            if constexpr (kU) a.u += u.at(0) + u.at(1);
        };
        if (shift.far) add(std::true_type());
        else add(std::false_type());
    }
    return a;
}

// The threads of a row: a warp, or a CTA.  Its sums use two areas in turn, so that one barrier a sum is enough: an area is
// written again behind the barrier of the sum in between.
template <bool kWarp>
struct Team {
    float2 (&room)[2][32];
    int tid, threads, side = 0;
    __device__ __forceinline__ void sync() const {
        if constexpr (kWarp) __syncwarp();
        else __syncthreads();
    }
    template <typename F>
    __device__ __forceinline__ float2 fold(float2 v, float none, F&& f) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            v.x = f(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
            v.y = f(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
        }
        if constexpr (!kWarp) {
            float2* at = room[side];
            side ^= 1;
            if (tid % 32 == 0) at[tid / 32] = v;
            __syncthreads();
            v = make_float2(none, none);
#pragma unroll
            for (int w = 0; w < kThreads / 32; ++w)
                if (w < threads / 32) v = make_float2(f(v.x, at[w].x), f(v.y, at[w].y));
        }
        return v;
    }
    __device__ __forceinline__ float max(float v) {
        return fold(make_float2(v, v), kNone, [](float a, float b) { return max_nan(a, b); }).x;
    }
    __device__ __forceinline__ float2 sum2(float x, float y) {
        return fold(make_float2(x, y), 0.0f, [](float a, float b) { return a + b; });
    }
    __device__ __forceinline__ float sum(float v) { return sum2(v, 0.0f).x; }
    __device__ __forceinline__ Sums join(Sums a, float k) {
        a.rescale(max(a.m), k);
        const float2 v = sum2(a.s, a.u);
        a.s = v.x;
        a.u = v.y;
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

// What a CTA of kT threads needs for it
template <int kT>
struct TopRoom {
    static constexpr int kWarps = kT / 32, kRoom = 8 * kT, kParts = kT == kThreads ? kCluster : 1;
    unsigned long long list[kRoom];              // candidates
    unsigned long long best[kParts][kMostTop];   // the parts' results, where the list is too small; the row's in the end
    alignas(16) uint32_t keys[kT];               // the largest of the warps' lanes, of all CTAs of the cluster
    uint32_t bound;
    int n, counts[kParts], count[kWarps];
};

// Entry i of a list goes to the place of its rank
template <int kT>
__device__ __forceinline__ void place(const unsigned long long* list, int n, int tid, int top, unsigned long long* out) {
    for (int i = tid; i < n; i += kT) {
        const unsigned long long mine = list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list[j] > mine;
        if (rank < top && mine != 0) out[rank] = mine;
    }
}

template <int kT>
__device__ __forceinline__ int block_count(TopRoom<kT>& r, int v, int tid) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if (tid % 32 == 0) r.count[tid / 32] = v;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kT / 32; ++w) sum += r.count[w];
    return sum;
}

template <typename T>
__device__ __forceinline__ uint32_t vector_max(const Raw<16>& v) {
    using W = Word<T>;
    return W::max(W::max(v.u[0], v.u[1]), W::max(v.u[2], v.u[3]));
}

// Lists the elements that reach the bound in a room (another CTA's too), whose n counts them, listed or not.  Returns the number
// of the warp's.
template <bool kSingle, typename T, int kT>
__device__ __forceinline__ int list_candidates(const Row<T>& row, int tid, uint32_t bound, TopRoom<kT>& r) {
    using W = Word<T>;
    constexpr int kPer = Row<T>::kPer, kBatch = 4;
    const float least = bound == 0 ? kNone : value_of(bound);
    auto reaches = [&](float v) { return v >= least || v != v; };
    const int lane = tid % 32;
    int all = 0;
    // the lanes of a warp get their places from a prefix sum of their counts, and the warp its own from one addition
    auto list = [&](uint32_t mask, auto&& element_of) {
        if (!__any_sync(0xffffffffu, mask != 0)) return;
        const int n = __popc(mask);
        int at = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += up;
        }
        int base = 0;
        if (lane == 31) base = atomicAdd(&r.n, at);
        all += __shfl_sync(0xffffffffu, at, 31);
        at += __shfl_sync(0xffffffffu, base, 31) - n;
        for (; mask != 0 && at < TopRoom<kT>::kRoom; mask &= mask - 1, ++at) {
            const int e = element_of(__ffs(mask) - 1);
            r.list[at] = (unsigned long long)key_of(row.one(e)) << 32 | (uint32_t)~e;
        }
    };
    const int ends = row.head_here + (row.n - row.tail);
    for (int i = tid; i - tid < (kSingle ? ends : kT); i += kT) {
        const int e = i < row.head_here ? i : row.tail + i - row.head_here;
        list(i < ends && reaches(row.one(e)) ? 1u : 0u, [&](int) { return e; });
    }
    if constexpr (kSingle) return all;
    for (int first = row.v0 + tid - lane; first < row.v1; first += kBatch * kT) {       // (a warp's first vector)
        Raw<16> raw[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (first + lane + b * kT < row.v1) load_kept(raw[b], row.vec(first + lane + b * kT));
        uint32_t mask = 0;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (first + lane + b * kT >= row.v1) break;
            const uint32_t m = vector_max<T>(raw[b]);
            float top = W::at(m, 0);
            if constexpr (W::kPer == 2) top = max_nan(top, W::at(m, 1));
            if (reaches(top)) {                  // (rarely)
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (reaches(W::at(raw[b].u[i / W::kPer], i % W::kPer))) mask |= 1u << (b * kPer + i);
            }
        }
        list(mask, [&](int bit) { return row.head + (first + lane + bit / kPer * kT) * kPer + bit % kPer; });
    }
    return all;
}

template <typename T, int kT>
__device__ __noinline__ int count_from(const Row<T>& row, int tid, uint32_t bound, TopRoom<kT>& r) {
    int n = 0;
    row.each(tid, kT, [&](int, float v) { n += key_of(v) >= bound; });
    return block_count(r, n, tid);
}

// The largest key that `top` elements of the part reach, which is at least `bound`: by bisection
template <typename T, int kT>
__device__ __noinline__ uint32_t exact_bound(const Row<T>& row, int tid, int top, uint32_t bound, TopRoom<kT>& r) {
    uint32_t hi = 0xffffffffu;
    if (bound < hi && count_from(row, tid, bound + 1, r) < top) return bound;
    while (bound < hi) {
        const uint32_t mid = bound + (hi - bound) / 2 + 1;
        if (count_from(row, tid, mid, r) >= top) bound = mid;
        else hi = mid - 1;
    }
    return bound;
}

// Entries of the first `need` elements that are on the bound, by index: a vector a thread at a time
template <typename T, int kT>
__device__ __noinline__ void first_on_bound(const Row<T>& row, int tid, int need, uint32_t bound, TopRoom<kT>& r,
                                            unsigned long long* out) {
    constexpr int kPer = Row<T>::kPer;
    int done = 0;
    // a thread's place from a prefix sum of the counts, threads being in the order of their elements
    auto place_of = [&](int mine) {
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, before, o);
            if (tid % 32 >= o) before += up;
        }
        __syncthreads();
        if (tid % 32 == 31) r.count[tid / 32] = before;
        __syncthreads();
        int start = done, all = 0;
        for (int w = 0; w < kT / 32; ++w) {
            if (w < tid / 32) start += r.count[w];
            all += r.count[w];
        }
        done += all;
        return start + before - mine;
    };
    auto take = [&](int e0, int n) {             // n elements of mine from e0 on
        int count = 0;
        for (int i = 0; i < n; ++i) count += key_of(row.one(e0 + i)) == bound;
        int at = place_of(count);
        for (int i = 0; i < n && count > 0; ++i)
            if (key_of(row.one(e0 + i)) == bound) {
                if (at < need) out[at] = (unsigned long long)bound << 32 | (uint32_t)~(e0 + i);
                ++at;
            }
    };
    take(tid, tid < row.head_here ? 1 : 0);
    for (int v = row.v0; v < row.v1 && done < need; v += kT) take(row.head + (v + tid) * kPer, v + tid < row.v1 ? kPer : 0);
    if (done < need) take(row.tail + tid, tid < row.n - row.tail ? 1 : 0);
}

// The largest keys of a warp's lanes, `each` of them, into to[0, each) (0 behind the last element)
__device__ __forceinline__ void largest_of_warp(float mine, bool any, int each, uint32_t* to) {
    uint32_t key = any ? key_of(mine) : 0;
    for (int i = 0; i < each; ++i) {
        const uint32_t taken = __reduce_max_sync(0xffffffffu, key);
        const uint32_t who = __ballot_sync(0xffffffffu, key == taken);
        if (threadIdx.x % 32 == __ffs(who) - 1) {
            key = 0;
            to[i] = taken;
        }
    }
}

// The top-th largest of n published keys, each a lane's maximum: at least `top` elements of the row reach it
template <int kT>
__device__ __forceinline__ uint32_t bound_of(TopRoom<kT>& r, int n, int tid, int top) {
    if (tid == 0) r.bound = 0;
    if (tid >= n) r.keys[tid] = 0;               // (up to a whole number of vectors)
    __syncthreads();
    if (tid < n) {
        const uint32_t mine = r.keys[tid];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; j += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(&r.keys[j]);
            // equal keys by their place
            rank += (v.x > mine) + (v.y > mine) + (v.z > mine) + (v.w > mine);
            rank += (v.x == mine & j < tid) + (v.y == mine & j + 1 < tid) + (v.z == mine & j + 2 < tid) + (v.w == mine & j + 3 < tid);
        }
        if (rank == top - 1) r.bound = mine;
    }
    __syncthreads();
    return r.bound;
}

// Where the list cannot hold what reaches the bound (many equal values, or large ones all in few lanes' hands): the `top` largest
// of a CTA's part, in order, into out[0, top) (0 behind the last).  If they do not fit either, the value of the part's last place is
// found by bisection.  Fewer than `top` elements are larger and are listed; the places behind them go to the lowest indices that
// have the value.
template <typename T, int kT>
__device__ __noinline__ void top_of_part(const Row<T>& row, int tid, int top, uint32_t bound, int reach, TopRoom<kT>& r,
                                         unsigned long long* out) {
    __syncthreads();
    if (tid < top) out[tid] = 0;
    if (tid == 0) r.n = 0;
    int equal = 0;
    if (reach > TopRoom<kT>::kRoom) {
        bound = exact_bound(row, tid, top, bound, r);
        equal = 1;
    }
    __syncthreads();
    if (bound + equal >= bound) list_candidates<false>(row, tid, bound + equal, r);
    __syncthreads();
    const int n = r.n;
    if (equal) first_on_bound(row, tid, top - n, bound, r, out + n);
    place<kT>(r.list, n, tid, top, out);
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
    int top, top_each;                           // top_each: of the largest lanes of a warp, to find a bound from
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

// temperature times it, which float32 holds where log p is too low for it
__device__ __forceinline__ float scaled_log_p(float v, float m, float log_s, const LogitsArgs& p) {
    if (m == kNone) return kNone;
    const float apart = v - m;
    return fabsf(apart) > kFar ? fmaf(-kLn2 * p.temperature, log_s, apart) : kLn2 * p.temperature * (Shift(m, p.k)(v) - log_s);
}

__device__ __forceinline__ float product_or_zero(float p, float v) { return p > 0.0f || p != p ? p * v : 0.0f; }

struct TeacherRoom {
    int token[kMostK];                           // -1: not used
    float log_q[kMostK], logit[kMostK];
    int repeats;                                 // not 0: a token may be there twice
};

// The row's loss and statistics, by a warp, from the teacher's places and the student's sums over the other tokens
__device__ __forceinline__ void distill_row(const LogitsArgs& p, int64_t row, int lane, TeacherRoom& r, Sums rest) {
    const auto largest = [](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    };
    const auto total = [](float v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    float top = kNone, norm = 0.0f;
    bool used = false;
    for (int i = lane; i < p.places; i += 32) {
        used |= r.token[i] >= 0;
        top = max_nan(top, r.log_q[i]);
    }
    used = __any_sync(0xffffffffu, used);
    if (!p.tail) {                               // log q normalised over the places
        top = largest(top);
        float s = 0.0f;
        for (int i = lane; i < p.places; i += 32) s += top == kNone ? 0.0f : expf(r.log_q[i] - top);
        if (top != kNone) norm = top + logf(total(s));
        else used = false;                       // no probability anywhere: as if no place were used
        for (int i = lane; i < p.places; i += 32) r.log_q[i] -= norm;
    }
    // the student's sums over the teacher's tokens, each token once
    Sums best{kNone, 0.0f, 0.0f};
    float mass = 0.0f;
    for (int i = lane; i < p.places; i += 32) {
        const int t = r.token[i];
        if (t < 0) continue;
        mass += expf(r.log_q[i]);
        bool again = false;
        if (r.repeats != 0)
            for (int j = 0; j < i; ++j) again |= r.token[j] == t;
        if (!again) add_one<false>(best, r.logit[i], p.k);
    }
    best.rescale(largest(best.m), p.k);
    best.s = total(best.s);
    mass = total(mass);
    const float m = max_nan(best.m, rest.m);
    Sums all = best, other = rest;
    if (m != kNone) {
        all.rescale(m, p.k);
        other.rescale(m, p.k);
    }
    const float log_s = log2f(all.s + other.s), rest_log_s = log2f(rest.s);
    float loss = 0.0f;
    for (int i = lane; i < p.places; i += 32) {
        if (r.token[i] < 0) continue;
        const float lq = r.log_q[i];
        loss += product_or_zero(expf(lq), fmaf(p.temperature, lq, -scaled_log_p(r.logit[i], m, log_s, p)));
    }
    loss = total(loss);
    if (lane != 0) return;
    float q_rest = 0.0f, c = 0.0f;
    if (p.tail && rest.m != kNone) q_rest = fmaxf(1.0f - mass, 0.0f);
    if (mass != mass) q_rest = mass;
    if (rest.m != kNone) {
        const float apart = Shift(rest.m, p.k).to(Shift(m, p.k)), unit = kLn2 * p.temperature;
        float log_rest = unit * apart;           // times the temperature, as the others'
        if (!(apart > -0.5f * kFar)) log_rest = rest.m - m;                      // (rarely: where `to` is cut off)
        log_rest = fmaf(unit, rest_log_s - log_s, log_rest);
        loss += product_or_zero(q_rest, fmaf(p.temperature, logf(q_rest), -log_rest));
        c = fmaf(mass + q_rest, expf(kLn2 * (apart + (rest_log_s - log_s))), -q_rest);
    }
    if (!used) loss = c = mass = q_rest = 0.0f;
    p.loss[row] = loss * p.temperature;
    if (p.stats != nullptr) {
        float* s = p.stats + row * DCN_LOGITS_STATS;
        s[kM] = m, s[kLogS] = log_s, s[kRestM] = rest.m, s[kRestLogS] = rest_log_s;
        s[kRestC] = c, s[kMass] = mass + q_rest, s[kNorm] = norm;
    }
}

// 48 registers a thread where a fifth CTA of 256 threads is worth more (4096x8192 float32, 20 best: 56 us, 59 us with 58)
template <typename T, int kKind, int kT, bool kSingle>
constexpr int kHeld = kKind == kScoresTop && !kSingle && (std::is_same<T, __half>::value || (sizeof(T) == 4 && kT == kThreads))
                          ? 5 * kThreads / kT
                          : 0;

template <typename T, int kKind, bool kWarp, int kT, bool kSingle = false>
__global__ void __launch_bounds__(kT, (kHeld<T, kKind, kT, kSingle>)) logits_forward_kernel(const LogitsArgs p) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float2 room[2][32];
    __shared__ Sums parts[kCluster];
    __shared__ TeacherRoom teachers[kKind == kDistill ? (kWarp ? kWarpRows : 1) : 1];
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = kWarp ? 0 : (int)cluster.block_rank(), ranks = kWarp ? 1 : (int)cluster.num_blocks();
    const int group = kWarp ? threadIdx.x / 32 : 0;
    const int64_t at = kWarp ? (int64_t)blockIdx.x * kWarpRows + group : blockIdx.x / ranks;
    Team<kWarp> team{room, kWarp ? (int)threadIdx.x % 32 : (int)threadIdx.x, kWarp ? 32 : kT};
    // every CTA of a cluster runs before another writes to its memory
    if (ranks > 1) asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    auto arrived = [&] { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); };
    if (at >= p.rows) return;                    // (a warp's row: a CTA's is always there)
    pdl_wait();
    const T* logits = static_cast<const T*>(p.logits) + at * p.stride;
    const Row<T> row(logits, p.vocab, rank, ranks, kSingle);
    TopRoom<kT>& top = *reinterpret_cast<TopRoom<kT>*>(dynamic);
    constexpr int kWarps = kT / 32;
    TeacherRoom& teacher = teachers[kKind == kDistill ? group : 0];
    uint8_t* marks = dynamic + group * p.marks;
    float given = CUDART_NAN_F;
    int64_t token = p.ignore;
    if constexpr (kKind != kDistill) {           // (on its way while the row is read)
        if (team.tid == 0 && rank == 0 && p.logprob != nullptr) {
            token = gload_i64(p.tokens + at);
            if (token >= 0 && token < p.vocab) given = row.one(token);
        }
    }
    // The teacher's places, one or (in a warp's row) up to four a thread.  What the sums need of them are the marks; the student's
    // logits there are on their way while the row is read.
    constexpr int kPlaces = kKind != kDistill ? 1 : kWarp ? kMostK / 32 : 1;
    float at_place[kPlaces];
    if constexpr (kKind == kDistill && !kWarp) {  // (the row's beginning is on its way to L2 while the marks are made: 1 to 3 %)
        if (team.tid == 0 && row.v1 > row.v0)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(row.vec(row.v0)),
                         "r"(min(row.v1 - row.v0, 2048) * 16)
                         : "memory");
    }
    if constexpr (kKind == kDistill) {
        int64_t t[kPlaces];
        float lq[kPlaces];
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            const int i = team.tid + q * team.threads;
            t[q] = i < p.places ? gload_i64(p.teacher_tokens + at * p.places + i) : -1;
            lq[q] = i < p.places ? teacher_at<T>(p, at * p.places + i) : kNone;
        }
        for (int i = team.tid; i < p.marks / 16; i += team.threads) reinterpret_cast<uint4*>(marks)[i] = make_uint4(0, 0, 0, 0);
        if (team.tid == 0) teacher.repeats = ranks > 1;          // (no CTA of a cluster sees all places)
        team.sync();
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            const int i = team.tid + q * team.threads;
            const bool in = t[q] >= 0 && t[q] < p.vocab;
            at_place[q] = in && rank == 0 ? row.one(t[q]) : kNone;
            if (i < p.places) {
                teacher.token[i] = in ? (int)t[q] : -1;
                teacher.log_q[i] = in ? lq[q] : kNone;
            }
            if (in && in_part(row, (int)t[q])) {
                const int b = mark_of(row, (int)t[q]);
                const uint32_t bit = 1u << (b & 31);
                if (atomicOr(reinterpret_cast<uint32_t*>(marks) + (b >> 5), bit) & bit) teacher.repeats = 1;
            }
        }
        team.sync();
    }
    const Sums mine =
        sums_of<T, kKind != kDistill, kKind == kDistill, kKind == kScoresTop, kSingle>(row, team.tid, team.threads, p.k, marks);
    if constexpr (kKind == kDistill) {
#pragma unroll
        for (int q = 0; q < kPlaces; ++q) {
            const int i = team.tid + q * team.threads;
            if (i < p.places) teacher.logit[i] = at_place[q];
        }
        __syncwarp();                            // (a CTA's row: the barriers of the join)
    }
    Sums sums = team.join(mine, p.k);
    if constexpr (kKind == kScoresTop) {
        const int warp = team.tid / 32;
        const bool any = row.v0 + team.tid < row.v1 || team.tid < row.head_here + (row.n - row.tail);
        uint32_t* to = top.keys + (rank * kWarps + warp) * p.top_each;
        largest_of_warp(mine.m, any, p.top_each, to);
        if (team.tid == 0) top.n = 0;
        __syncwarp();
        if (ranks > 1) {
            const uint32_t key = team.tid % 32 < p.top_each ? to[team.tid % 32] : 0;
            arrived();
            for (int r = 0; r < ranks; ++r)
                if (team.tid % 32 < p.top_each) cluster.map_shared_rank(to, r)[team.tid % 32] = key;
        }
    }
    if (ranks > 1) {
        if constexpr (kKind != kScoresTop) arrived();
        if (team.tid < ranks) *cluster.map_shared_rank(&parts[rank], team.tid) = sums;
        cluster.sync();
        if constexpr (kKind != kScoresTop)
            if (rank > 0) return;
    }
    if constexpr (kKind == kScoresTop) {
        const uint32_t bound = bound_of<kT>(top, ranks * kWarps * p.top_each, team.tid, p.top);
        TopRoom<kT>& first = ranks > 1 ? *cluster.map_shared_rank(&top, 0) : top;
        const int listed = list_candidates<kSingle>(row, team.tid, bound, first);
        int n = 0;
        if (ranks > 1) {
            if (team.tid % 32 == 0) top.count[team.tid / 32] = listed;
            __syncthreads();
            if (team.tid < ranks) {
                for (int w = 0; w < kWarps; ++w) n += top.count[w];
                cluster.map_shared_rank(&top, team.tid)->counts[rank] = n;
            }
            cluster.sync();
            n = 0;
            for (int r = 0; r < ranks; ++r) n += top.counts[r];
        } else {
            __syncthreads();
            n = top.n;
        }
        if (n > TopRoom<kT>::kRoom) {            // (the same for all CTAs of the cluster)
            top_of_part(row, team.tid, p.top, bound, ranks > 1 ? top.counts[rank] : n, top, top.best[rank]);
            if (rank > 0)
                for (int i = team.tid; i < p.top; i += kT)
                    *cluster.map_shared_rank(&top.best[rank][i], 0) = top.best[rank][i];
            if (ranks > 1) cluster.sync();
            if (rank > 0) return;
            n = ranks * p.top;
            for (int i = team.tid; i < n; i += kT) top.list[i] = top.best[i / p.top][i % p.top];
            __syncthreads();
        }
        if (rank > 0) return;
        place<kT>(top.list, n, team.tid, p.top, top.best[0]);
        __syncthreads();
    }
    if (ranks > 1) {                             // the parts' sums, a lane each
        const int lane = team.tid % 32;
        Sums part{kNone, 0.0f, 0.0f};
        if (lane < ranks) part = parts[lane];
        float m = part.m;
#pragma unroll
        for (int o = kCluster / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        part.rescale(m, p.k);
#pragma unroll
        for (int o = kCluster / 2; o > 0; o >>= 1) {
            part.s += __shfl_xor_sync(0xffffffffu, part.s, o);
            part.u += __shfl_xor_sync(0xffffffffu, part.u, o);
        }
        sums.m = __shfl_sync(0xffffffffu, part.m, 0);
        sums.s = __shfl_sync(0xffffffffu, part.s, 0);
        sums.u = __shfl_sync(0xffffffffu, part.u, 0);
    }
    if constexpr (kKind == kDistill) {
        if (kWarp || team.tid < 32) distill_row(p, at, team.tid, teacher, sums);
    } else {
        const float log_s = log2f(sums.s);
        const float entropy = sums.m == kNone ? 0.0f : kLn2 * (log_s - sums.u / sums.s);
        if (team.tid == 0) {
            if (p.logprob != nullptr) {
                float v = CUDART_NAN_F;
                if (token == p.ignore) v = 0.0f;
                else if (token >= 0 && token < p.vocab) v = log_p(given, sums.m, log_s, p);
                p.logprob[at] = v;
            }
            if (p.entropy != nullptr) p.entropy[at] = entropy;
            if (p.stats != nullptr) {
                float* s = p.stats + at * DCN_LOGITS_STATS;
                s[kM] = sums.m, s[kLogS] = log_s, s[kEntropy] = entropy;
            }
        }
        if constexpr (kKind == kScoresTop) {
            for (int i = team.tid; i < p.top; i += kT) {
                const unsigned long long entry = top.best[0][i];
                p.top_tokens[at * p.top + i] = (int64_t)(uint32_t)~(uint32_t)entry;
                p.top_logprobs[at * p.top + i] = log_p(value_of((uint32_t)(entry >> 32)), sums.m, log_s, p);
            }
        }
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------
// dz = 2^l (c0 + c1 l), l = log2 p = (v - m) k - log2 S.  kLinear: c1 is 0.
template <bool kLinear>
struct Slope {
    float minus_m, k, minus_log_s, c0, c1;
    // (log_s of the sums as they were formed; here without what their m k is off by)
    __device__ __forceinline__ Slope(float m, float k_, float log_s, float c0_, float c1_)
        : minus_m(-m), k(k_), minus_log_s(-log_s), c0(c0_), c1(c1_) {
        const Shift shift(m, k);
        if (!shift.far) minus_log_s += __fmaf_rn(m, k, -shift.c);
    }
    __device__ __forceinline__ bool zero() const { return minus_m == -kNone; }
    __device__ __forceinline__ float operator()(float v) const {
        if (zero()) return 0.0f;
        const float l = max_nan(__fmaf_rn(__fadd_rn(v, minus_m), k, minus_log_s), -kGone);
        return ex2(l) * (kLinear ? c0 : fmaf(c1, l, c0));
    }
    // a vector's, where the row is not zero
    template <typename T>
    __device__ __forceinline__ void vector(const uint32_t* w, float (&f)[16 / sizeof(T)]) const {
        const Lanes kk = all_lanes(k), shifted = all_lanes(minus_m), ss = all_lanes(minus_log_s);
#pragma unroll
        for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
            Lanes l = fma(pair_of<T>(w, i) + shifted, kk, ss), c = all_lanes(c0);
            if constexpr (!kLinear) {
                const float far[2] = {max_nan(l.at(0), -kGone), max_nan(l.at(1), -kGone)};
                l = lanes(far);
                c = fma(all_lanes(c1), l, c);
            }
            const float e[2] = {ex2(l.at(0)), ex2(l.at(1))};
            c = lanes(e) * c;
            f[2 * i] = c.at(0);
            f[2 * i + 1] = c.at(1);
        }
    }
};

// kStream: the gradient's rows are whole 32-byte sectors, which then need not be kept in L2 (of others the rest comes from another
// warp, and sending them off early costs a second write)
template <typename T, bool kDistilled, bool kStream>
__global__ void __launch_bounds__(kThreads, 6) logits_backward_kernel(const LogitsArgs p, int parts) {
    constexpr int kPer = Row<T>::kPer;
    __shared__ int token[kMostTop + 1];
    __shared__ float weight[kMostTop + 1];
    __shared__ float2 room[2][32];
    const int tid = threadIdx.x, threads = blockDim.x;
    // the rows that were read last come first: in a loss, whose backward pass follows its forward pass, they are still in L2
    const int64_t at = p.rows - 1 - blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    pdl_wait();
    const Row<T> row(static_cast<const T*>(p.logits) + at * p.stride, p.vocab, part, parts);
    T* out = static_cast<T*>(p.dlogits) + at * p.vocab;
    const float* stat = p.stats + at * DCN_LOGITS_STATS;
    // what the row's elements get; the special tokens get a term more
    Slope<kDistilled> slope(gload(stat + (kDistilled ? kRestM : kM)), p.k, gload(stat + (kDistilled ? kRestLogS : kLogS)), 0.0f, 0.0f);
    int specials;
    if constexpr (kDistilled) {
        specials = p.places;
        slope.c0 = gload(p.dloss + at) * p.temperature * gload(stat + kRestC);
    } else {
        specials = p.dtop != nullptr ? p.top + 1 : 1;
        const float scale = 1.0f / p.temperature;
        const float gh = p.dentropy != nullptr ? gload(p.dentropy + at) : 0.0f;
        auto special_of = [&](int i) {
            int64_t t = -1;
            float v = 0.0f;
            if (i > 0) {
                t = gload_i64(p.top_tokens + at * p.top + i - 1);
                v = gload(p.dtop + at * p.top + i - 1);
            } else if (p.dlogprob != nullptr) {
                t = gload_i64(p.tokens + at);
                v = gload(p.dlogprob + at);
                if (t == p.ignore) t = -1;
            }
            const bool in = t >= 0 && t < p.vocab;
            token[i] = in ? (int)t : -1;
            return weight[i] = in ? v * scale : 0.0f;
        };
        float all = 0.0f;
        if (specials > 1) {
            for (int i = tid; i < specials; i += threads) all += special_of(i);
            Team<false> team{room, tid, threads};
            all = team.sum(all);
        } else {
            if (tid == 0) special_of(0);
            __syncthreads();
            all = weight[0];
        }
        slope.c0 = -fmaf(gh * scale, gload(stat + kEntropy), all);
        slope.c1 = -scale * kLn2 * gh;
    }
    auto put = [&](int64_t e, float v) { out[e] = from_float<T>(v); };
    const int ends = row.head_here + (row.n - row.tail);          // elements outside vectors: at most one a thread
    if (tid < ends) {
        const int e = tid < row.head_here ? tid : row.tail + tid - row.head_here;
        put(e, slope(row.one(e)));
    }
    // vectors where the gradient's rows start as the logits' do, elements otherwise and in rows that are zero
    constexpr int kBatch = 4;
    const bool alike = reinterpret_cast<uintptr_t>(out) % 16 == reinterpret_cast<uintptr_t>(row.p) % 16;
    const bool vectors = alike && !slope.zero();
    T* to = out + row.head;
    for (int v = row.v0 + tid; v < row.v1; v += kBatch * threads) {
        if (vectors && v + (kBatch - 1) * threads < row.v1) {
            Raw<16> raw[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) load(raw[b], row.vec(v + b * threads));
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                float f[kPer];
                slope.template vector<T>(raw[b].u, f);
                Pack<T, kPer> o;
                o.set(f);
                if constexpr (kStream) store_streaming(to + (int64_t)(v + b * threads) * kPer, o.raw);
                else o.put(to + (int64_t)(v + b * threads) * kPer);
            }
        } else {
#pragma unroll 1
            for (int u = v; u < min(v + kBatch * threads, row.v1); u += threads) {
                Raw<16> raw;
                load(raw, row.vec(u));
                float f[kPer];
                if (vectors) {
                    slope.template vector<T>(raw.u, f);
                    Pack<T, kPer> o;
                    o.set(f);
                    o.put(to + (int64_t)u * kPer);
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        put(row.head + (int64_t)u * kPer + i, slope(Word<T>::at(raw.u[i / Word<T>::kPer], i % Word<T>::kPer)));
                }
            }
        }
    }
    if constexpr (kDistilled) {                  // (read here: the registers were the row's)
        const float g = gload(p.dloss + at) * p.temperature, norm = gload(stat + kNorm);
        slope = Slope<true>(gload(stat + kM), p.k, gload(stat + kLogS), g * gload(stat + kMass), 0.0f);
        for (int i = tid; i < specials; i += threads) {
            const int64_t t = gload_i64(p.teacher_tokens + at * p.places + i);
            const bool in = t >= 0 && t < p.vocab;
            token[i] = in ? (int)t : -1;
            weight[i] = in ? -g * expf(teacher_at<T>(p, at * p.places + i) - norm) : 0.0f;
        }
    }
    __syncthreads();                             // the part's special tokens are written over what stands there
    if (slope.zero()) return;
    for (int i = tid; i < specials; i += threads) {
        const int t = token[i];
        if (t < 0 || !in_part(row, t)) continue;
        float w = 0.0f;
        for (int j = 0; j < specials; ++j) w += token[j] == t ? weight[j] : 0.0f;
        put(t, slope(row.one(t)) + w);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
constexpr int kWarpVocab = 2048;                 // rows up to this size: a warp each, or two where alternatives are asked for

constexpr int kBackwardPart = 32768;

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
    size_t smem = 0;
    int threads = kThreads;
    bool single = false;
    if (kKind == kScoresTop) {
        if (a.vocab <= kWarpVocab && a.top <= 64) threads = a.top <= 32 ? kFewThreads : 2 * kFewThreads;
        smem = threads == kThreads      ? sizeof(TopRoom<kThreads>)
               : threads == kFewThreads ? sizeof(TopRoom<kFewThreads>)
                                        : sizeof(TopRoom<2 * kFewThreads>);
        // of every warp whose lanes all have a vector its share, or one more where that is less than twice `top` in all (the more,
        // the less is listed that is not among the `top`); of all CTAs together not more than there are keys
        const int warps = threads / 32, vectors = a.vocab / (16 / (int)sizeof(T)) / parts;
        // Short rows of which many are asked for are read element by element: where not many more lanes than `top` have a vector,
        // the largest of the lanes bound little and most elements would be ranked.  Such rows are shorter than the list, so that
        // nothing but the usual path reads them.  (Element by element / in vectors, us, by 256 threads: 12332x320 bf16, 50 best 128 /
        // 558; 4096 rows of bf16, 1000 with 128 best 100 / 777, with 70 66 / 99; 2000 with 128 122 / 100; by 64 threads, 256 with
        // 20 31 / 26, with 28 the same, 128 with 32 27 / 40.)
        single = parts == 1 && 8 * std::min(vectors, 32 * warps) < (threads == kFewThreads ? 10 : 15) * a.top;
        const int lanes = single ? a.vocab : vectors;
        const int full = lanes / 32 < 1 ? 1 : lanes / 32 < warps ? lanes / 32 : warps;
        const int share = (a.top + parts * full - 1) / (parts * full), most = 32 / parts;
        a.top_each = parts * full * share < 2 * a.top ? share + 1 : share;
        if (a.top_each > most) a.top_each = most;
    }
    if (kKind == kDistill) {
        const int per = 16 / (int)sizeof(T);
        a.marks = (int)(((a.vocab / per + parts - 1) / parts * per + 8 + 2 * per + 8 + 127) / 128 * 16);
        smem = (size_t)a.marks * (warp ? kWarpRows : 1);
    }
    cfg.gridDim = dim3((unsigned)(warp ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows * parts));
    cfg.blockDim = dim3(warp ? 32 * kWarpRows : threads);
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
        const auto launch = [&](auto one_by_one) {
            constexpr bool kSingle = one_by_one.value;
            const auto kernel = threads == kThreads      ? logits_forward_kernel<T, kKind, false, kThreads, kSingle>
                                : threads == kFewThreads ? logits_forward_kernel<T, kKind, false, kFewThreads, kSingle>
                                                         : logits_forward_kernel<T, kKind, false, 2 * kFewThreads, kSingle>;
            return cudaLaunchKernelEx(&cfg, kernel, a);
        };
        e = single ? launch(std::true_type()) : launch(std::false_type());
    } else if (warp) {
        e = cudaLaunchKernelEx(&cfg, logits_forward_kernel<T, kKind, true, 32 * kWarpRows>, a);
    } else {
        const auto kernel = logits_forward_kernel<T, kKind, false, kThreads>;
        // (the same for every call, so that calls of several host threads do not take it from one another)
        constexpr int most = (DCN_DISTILL_MOST_VOCAB / 8 + 1024) / 16 * 16;
        if (smem > 40 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, a);
    }
    return e != cudaSuccess || cudaGetLastError() != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, bool kDistilled>
int run_backward(const LogitsArgs& a, cudaStream_t st) {
    // parts of at most kBackwardPart elements, of a CTA with a vector or more for each thread
    const int64_t parts = (a.vocab + kBackwardPart - 1) / kBackwardPart;
    const int64_t vectors = a.vocab / parts * (int64_t)sizeof(T) / 16;
    const int threads = vectors >= 192 ? 256 : vectors >= 96 ? 128 : 64;
    if (a.rows * parts >= 1ll << 31) return DCN_ERR_LIMIT;
    const bool stream = a.vocab * sizeof(T) % 32 == 0 && aligned(a.dlogits, 32);
    const auto kernel = stream ? logits_backward_kernel<T, kDistilled, true> : logits_backward_kernel<T, kDistilled, false>;
    return launch_dependent(kernel, dim3((unsigned)(a.rows * parts)), dim3(threads), 0, st, a, (int)parts) != cudaSuccess
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
