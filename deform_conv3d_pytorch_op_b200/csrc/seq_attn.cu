// Decayed linear attention over time, for each head with its decay g:
//     S_t = g S_{t-1} + k_t v_t^T,    out_t = scale S_t^T q_t
// In chunks of 64 steps, with X the state before a chunk and i, j steps of it,
//     out_i = scale (sum_{j <= i} g^(i-j) (q_i . k_j) v_j  +  g^(i+1) X^T q_i),     X' = g^64 X + sum_j g^(63-j) k_j v_j^T
// One kernel runs through (a, b, c) = (q, k, v) in this way.  The gradients are the same sums over other operands:
//     dq: (dout, v, k) with the states S^T;   back in time, with R_t = g R_{t+1} + scale q_t dout_t^T the gradient of S_t,
//     dk: (v, dout, q) with R^T;   dv: (k, q, dout) with R;   R starts as dlast with one power of g less: g^i X and g^(64-j).
//
// Two kernels run it.  16-bit sequences of more than a chunk go to the tensor cores (seq_attn_tc.cuh), laid out anew first where their rows
// are not what a bulk copy takes (pack_kernel; results in join_kernel).  This file's own has float32, in which every operand is a sum of two
// of TF32, and short sequences of any type: a CTA walks one sequence's chunks for one head and 64 columns of c, the state in the accumulators
// of its warps.  Four groups of warps have 16 steps each; the warps of a group share columns, of the scores, of c and of the state, and meet
// twice a chunk: the scores take the place of a's rows, which nobody else reads.  The state meets a as a rounded copy in shared memory.  What
// bounds it is the latency of products and of the loads of their operands, so that warps count: 43x507x12x(80, 32) float32 674 us with one
// group member, 374 us with four; 8x3000x2x(128, 96) float32 with gradients 1967 and 1021.  That is some 20 TFLOP/s of float32 products.
//
// Where there are fewer heads than the GPU holds CTAs, the time axis is split: a first launch sums each part's k_t v_t^T, and a CTA of the
// second folds what lies before its own part.
#include <algorithm>
#include <cmath>

#include <cuda.h>

#include "dcn_tc_common.cuh"
#include "seq_common.cuh"

namespace dcn {
namespace seq {
namespace {

constexpr int kChunk = 64, kCols = 64, kMostWidth = 128, kMostParts = 32;

struct Strides {
    int64_t batch, step, head;
};

struct Operand {
    const void* p;
    Strides s;
    int share;                                   // heads that read the same one
    int width, bytes;                            // elements of a row; bytes that are copied at once
    int map;                                     // of the call's tensor maps
};

struct Job {
    Operand a, b, c;
    void* out;                                   // [batch, steps, heads, room], dense; float32 where wide
    const float* init;                           // [batch, heads, ...]: element (i, j) at i * init_i + j * init_j; NULL: zeros
    float* end;                                  // [batch, heads, a.width, c.width] dense, or NULL
    int room;                                    // elements of a row of out: c's width, or the next multiple of 8
    int init_i, init_j;
    int reverse, wide;
    float init_scale, end_scale;
    int pairs;                                   // out's rows start on two elements
    int sectors;                                 // ... and on 32 bytes, which all columns fill
};

struct AttnArgs {
    Job job[3];
    const float* log_decay;
    const int64_t* lengths;
    float* parts;                                // [unit less `whole`][part][part_floats]: sums [a.width][part_cols] of a unit's 64 columns
    int part_floats, part_cols;
    int64_t steps, part_steps;
    int64_t whole;                               // units (job, head, tile) whose time axis is not split
    int batch, heads, jobs, tiles, n_parts;      // tiles: of 64 columns, the most that a job has
    int tile_of[3];
    float scale;
};

// Which unit and which part of its time axis a CTA has.  kEnds: of those parts alone that another one follows
struct Place {
    int tile, which, unit, part;
    int64_t part_steps, split;                   // split: the unit among those that are split
    template <bool kEnds>
    static __device__ __forceinline__ Place of(const AttnArgs& a) {
        Place p;
        const int64_t at = (int64_t)blockIdx.x - (kEnds ? 0 : a.whole);
        const int parts = kEnds ? a.n_parts - 1 : a.n_parts;
        int64_t u = blockIdx.x;
        p.part = 0, p.part_steps = a.steps, p.split = 0;
        if (at >= 0) p.split = at / parts, u = a.whole + p.split, p.part = (int)(at % parts), p.part_steps = a.part_steps;
        p.tile = (int)(u % a.tiles);
        u /= a.tiles;
        p.which = (int)(u % a.jobs), p.unit = (int)(u / a.jobs);
        return p;
    }
    __device__ __forceinline__ float* sums(const AttnArgs& a, int s) const { return a.parts + (split * a.n_parts + s) * a.part_floats; }
};

__device__ __forceinline__ double log_decay_of(const float* log_decay, int h) {
    const float g = gload(log_decay + h);
    return g > 0.0f ? 0.0 : (double)g;
}
// g^n, rounded once (1 for no steps, whatever the decay)
__device__ __forceinline__ float power_of(double log_decay, int64_t n) {
    return n == 0 && log_decay == log_decay ? 1.0f : (float)exp((double)n * log_decay);
}
// The decay of a whole block as the factors of one block after another, each rounded so that their product stays the power that it stands
// for.  (One and the same rounding adds up: states of 40000 steps were off by 10^-5.)
struct Carried {
    double decay, inverse, off;
    __device__ __forceinline__ void begin(double log_decay, int steps) {
        decay = exp(steps * log_decay), inverse = decay > 1e-20 ? 1.0 / decay : 0.0, off = 0.0;          // (of less nothing is left after two)
    }
    __device__ __forceinline__ float next() {
        const float f = (float)(decay - decay * off);
        off += ((double)f - decay) * inverse;
        return f;
    }
};
// from a table of them in shared memory
__device__ __forceinline__ float power(uint32_t table, int n) {
    float f;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(table + 4 * n));
    return f;
}

// Float16 has 11 bits of what lies between 2^-14 and 2^16 alone, and the scores, states and weighted rows that it takes part in do not stay there
// (128 products of numbers above 22, gradients of a loss that is not scaled).  So what is rounded to it is brought near its upper end first, by
// a power of two that the largest of a row of scores, of a head's state or of a block's rows gives, and back in float32.  From 2^14 on,
// elements down to 2^-29 of that largest one keep their 11 bits.  (Bfloat16 has float32's range.)
template <typename T>
constexpr bool kNarrow = std::is_same<T, __half>::value;
// n, where 2^n brings a largest magnitude (0 and above, not NaN) into [2^14, 2^15), as far as 2^n and 2^-n are normal numbers; 0 for none and for
// infinity, beside which the others stay as they are
__device__ __forceinline__ int shift_of(float most) {
    return most > 0.0f && most < CUDART_INF_F ? min(max(14 + 127 - (int)(__float_as_uint(most) >> 23), -113), 100) : 0;
}
__device__ __forceinline__ float two_to(int n) { return __uint_as_float((uint32_t)(127 + n) << 23); }
// The larger magnitudes of pairs of float16 numbers, whose shift is up alone: they are in range.  (NaN is left out.)
__device__ __forceinline__ uint32_t larger_pairs(uint32_t most, uint32_t pair) {
    uint32_t m;
    asm("{\n .reg .b32 a;\n abs.f16x2 a, %2;\n max.f16x2 %0, %1, a;\n}" : "=r"(m) : "r"(most), "r"(pair));
    return m;
}
// (weight: the largest that they meet)
__device__ __forceinline__ int shift_up(uint32_t most, float weight) { return max(shift_of(half_of<__half>(most, 0) * weight), 0); }

#include "seq_attn_tc.cuh"

// ---- products: D[16 x 8] += A[16 x k] B[k x 8], k = 16 for 16-bit types and 8 for float32 -----------------------------------------
// Operands come from tiles in shared memory, rows of `a` columns.  16-bit tiles are swizzled by 16 bytes (the row's low three bits);
// float32 tiles have 8 columns more than they need, and the elements 2t and 2t + 1 of k stand for the instruction's t and t + 4.
template <typename T>
struct Tile {
    static constexpr int kK = 16;
    static constexpr int row_elems(int cols) { return cols; }
    // address of 16 bytes
    static __device__ __forceinline__ uint32_t at(uint32_t base, int row, int col, int cols) {
        return base + row * cols * 2 + (((col >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
    }
};
template <>
struct Tile<float> {
    static constexpr int kK = 8;
    static constexpr int row_elems(int cols) { return cols + 8; }
    static __device__ __forceinline__ uint32_t at(uint32_t base, int row, int col, int cols) {
        return base + (row * (cols + 8) + col) * 4;
    }
};

template <typename T>
struct FragA {
    uint32_t v[4];
};
template <typename T>
struct FragB {
    uint32_t v[2];
};
// float32: each element as the sum of two of TF32 (11 bits each), which leaves 2^-22 of it
template <>
struct FragA<float> {
    uint32_t v[4], low[4];
};
template <>
struct FragB<float> {
    uint32_t v[2], low[2];
};

__device__ __forceinline__ void split(float f, uint32_t& big, uint32_t& low) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(big) : "f"(f));
    const float rest = f - __uint_as_float(big);
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(low) : "f"(rest));
}

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const FragA<T>& a, const FragB<T>& b) {
    if constexpr (std::is_same<T, float>::value) {
        // (the tensor cores' own sums are cut off, not rounded: of eight products at a time, that is lost in them)
        float t[4] = {};
        mma8(t, a.low, b.v);
        mma8(t, a.v, b.low);
        mma8(t, a.v, b.v);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] += t[e];
    } else {
        mma16<T>(d, a.v, b.v);
    }
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float lds_float(uint32_t a) {
    float f;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(a) : "memory");
    return f;
}
__device__ __forceinline__ float2 lds_float2(uint32_t a) {
    float2 f;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f.x), "=f"(f.y) : "r"(a) : "memory");
    return f;
}

// A[m][k] = tile[m0 + m][k0 + k]
template <typename T>
__device__ __forceinline__ void load_a(FragA<T>& f, uint32_t base, int m0, int k0, int cols, int lane) {
    if constexpr (std::is_same<T, float>::value) {
        const int g = lane >> 2, t = lane & 3;
        const float2 x = lds_float2(Tile<T>::at(base, m0 + g, k0 + 2 * t, cols));
        const float2 y = lds_float2(Tile<T>::at(base, m0 + g + 8, k0 + 2 * t, cols));
        split(x.x, f.v[0], f.low[0]), split(y.x, f.v[1], f.low[1]), split(x.y, f.v[2], f.low[2]), split(y.y, f.v[3], f.low[3]);
    } else {
        ldsm4(f.v, Tile<T>::at(base, m0 + (lane & 15), k0 + (lane >> 4) * 8, cols));
    }
}
// two of B[k][n] = tile[n0 + n][k0 + k], for n0 and n0 + 8
template <typename T>
__device__ __forceinline__ void load_b(FragB<T> (&f)[2], uint32_t base, int n0, int k0, int cols, int lane) {
    if constexpr (std::is_same<T, float>::value) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 x = lds_float2(Tile<T>::at(base, n0 + 8 * i + g, k0 + 2 * t, cols));
            split(x.x, f[i].v[0], f[i].low[0]), split(x.y, f[i].v[1], f[i].low[1]);
        }
    } else {
        uint32_t r[4];
        ldsm4(r, Tile<T>::at(base, n0 + (lane >> 4) * 8 + (lane & 7), k0 + ((lane >> 3) & 1) * 8, cols));
        f[0].v[0] = r[0], f[0].v[1] = r[1], f[1].v[0] = r[2], f[1].v[1] = r[3];
    }
}
// two of B[k][n] = tile[k0 + k][n0 + n], for n0 and n0 + 8
template <typename T>
__device__ __forceinline__ void load_bt(FragB<T> (&f)[2], uint32_t base, int k0, int n0, int cols, int lane) {
    if constexpr (std::is_same<T, float>::value) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                split(lds_float(Tile<T>::at(base, k0 + 2 * t + e, n0 + 8 * i + g, cols)), f[i].v[e], f[i].low[e]);
    } else {
        uint32_t r[4];
        ldsm4t(r, Tile<T>::at(base, k0 + (lane & 15), n0 + (lane >> 4) * 8, cols));
        f[0].v[0] = r[0], f[0].v[1] = r[1], f[1].v[0] = r[2], f[1].v[1] = r[3];
    }
}
// The largest magnitudes of what load_at reads in rows m0 + g and m0 + g + 8 of A, as shift_up takes them: float16
__device__ __forceinline__ void largest_at(uint32_t (&most)[2], uint32_t base, int k0, int m0, int cols, int lane) {
    uint32_t r[4];
    ldsm4t(r, Tile<__half>::at(base, k0 + (lane >> 4) * 8 + (lane & 7), m0 + ((lane >> 3) & 1) * 8, cols));
#pragma unroll
    for (int i = 0; i < 4; ++i) most[i & 1] = larger_pairs(most[i & 1], r[i]);
}
// A[m][k] = tile[k0 + k][m0 + m] * weight of row k0 + k.  16-bit: rounded, what the rounding left (low), and what that one's left (last);
// float16: times `by` of rows g and g + 8
template <typename T>
__device__ __forceinline__ void load_at(FragA<T>& f, FragA<T>& low, FragA<T>& last, uint32_t base, int k0, int m0, int cols, int lane, uint32_t table,
                                        int last_power, int rows, const float (&by)[2]) {
    const int g = lane >> 2, t = lane & 3;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int j = k0 + 2 * t + e;
            const float w = j < rows ? power(table, max(last_power - j, 0)) : 0.0f;
            split(w * lds_float(Tile<T>::at(base, j, m0 + g, cols)), f.v[2 * e], f.low[2 * e]);
            split(w * lds_float(Tile<T>::at(base, j, m0 + g + 8, cols)), f.v[2 * e + 1], f.low[2 * e + 1]);
        }
    } else {
        uint32_t r[4];
        // matrices: (k 0-7, m 0-7), (k 0-7, m 8-15), (k 8-15, m 0-7), (k 8-15, m 8-15), each transposed
        ldsm4t(r, Tile<T>::at(base, k0 + (lane >> 4) * 8 + (lane & 7), m0 + ((lane >> 3) & 1) * 8, cols));
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = k0 + 2 * t + (e & 1) + (e >> 1) * 8;
            w[e] = j < rows ? power(table, max(last_power - j, 0)) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {            // 0: (g, k 2t), 1: (g + 8, k 2t), 2: (g, k 2t + 8), 3: (g + 8, k 2t + 8)
            float x = half_of<T>(r[i], 0) * w[(i >> 1) * 2], y = half_of<T>(r[i], 1) * w[(i >> 1) * 2 + 1];
            if constexpr (kNarrow<T>) x *= by[i & 1], y *= by[i & 1];
            f.v[i] = word_of<T>(x, y);
            const float p = x - half_of<T>(f.v[i], 0), q = y - half_of<T>(f.v[i], 1);
            low.v[i] = word_of<T>(p, q);
            last.v[i] = word_of<T>(p - half_of<T>(low.v[i], 0), q - half_of<T>(low.v[i], 1));
        }
    }
}
// The warps of a group meet
template <int kCount>
__device__ __forceinline__ void group_sync(int barrier) {
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(kCount) : "memory");
}
// two scores side by side, as load_a finds them
template <typename T>
__device__ __forceinline__ void put_pair(uint32_t at, float p, float q) {
    if constexpr (std::is_same<T, float>::value) asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(p), "f"(q) : "memory");
    else asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(word_of<T>(p, q)) : "memory");
}

// ---- tiles ----------------------------------------------------------------------------------------------------------------
// Rows first, first + 1, ... of a sequence (back in time from `length` where reverse) into a tile of kCols_ columns; zeros beyond the
// length and the operand's width.
template <typename T, int kCols_, int kT>
__device__ __forceinline__ void load_tile(uint32_t base, const Operand& o, const char* from, int64_t first, int64_t length, int col0,
                                          bool reverse) {
    constexpr int kElem = sizeof(T), kVec = 16 / kElem, kPerRow = kCols_ / kVec;
    const int width = o.width - col0;            // (may be above kCols_)
    for (int i = threadIdx.x; i < kChunk * kPerRow; i += kT) {
        const int row = i / kPerRow, col = (i % kPerRow) * kVec;
        const int64_t pos = first + row;
        const bool in = pos < length && col < width;
        const int64_t t = reverse ? length - 1 - pos : pos;
        const char* src = from + (in ? (t * o.s.step + col0 + col) * kElem : 0);
        const uint32_t dst = Tile<T>::at(base, row, col, kCols_);
        const int bytes = in ? min(16, (width - col) * kElem) : 0;
        if (o.bytes == 16) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
        } else if (o.bytes == 8) {
#pragma unroll
            for (int e = 0; e < 16; e += 8)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + e), "l"(bytes > e ? src + e : from),
                             "r"(max(0, min(8, bytes - e))) : "memory");
        } else if (o.bytes == 4) {
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + e), "l"(bytes > e ? src + e : from),
                             "r"(max(0, min(4, bytes - e))) : "memory");
        } else {
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                Raw<2> r;
                r.u = 0;
                if (bytes > e) load(r, src + e);
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + e), "h"(r.u) : "memory");
            }
        }
    }
}

template <typename T, int KA, bool kEnds>
struct Shape {
    static constexpr bool kFloat = sizeof(T) == 4;
    // Warps of a group.  (Float32, 128 columns: 1114 us with two, 1016 with four for 8x3000x2x(128, 96) with gradients; 64 columns: two 660,
    // one 838, four 747 for 16x1000x8x(64, 64).  16-bit, 64 columns: 341 with one, 374 with two for 7x11440x6x(54, 47), 128 columns:
    // 1219 with one, 979 with two, 1189 with four for 16x2614x12x(107, 71), both before such sequences went to the tensor cores.)
    static constexpr int kAcross = kEnds ? 2 : kFloat && KA == 128 ? 4 : kFloat || KA == 128 ? 2 : 1;
    static constexpr int kThreads = 128 * kAcross, kWarps = 4 * kAcross;
    static constexpr int kStages = kFloat && !kEnds && KA == 64 ? 1 : 2;
    static constexpr int kTileA = kChunk * Tile<T>::row_elems(KA) * (int)sizeof(T);
    static constexpr int kTileC = kChunk * Tile<T>::row_elems(kCols) * (int)sizeof(T);
    static constexpr int kState = kEnds ? 0 : KA * Tile<T>::row_elems(kCols) * (int)sizeof(T);
    static constexpr int kB = kEnds ? 0 : kTileA, kC = kB + kTileA, kStage = kC + kTileC;                // b's and c's places
    static constexpr int kTable = kStages * kStage + kState + (int)sizeof(Carried);          // g^n, 0 to 64, behind what gives the last one
    static constexpr int kLargest = kTable + (kChunk + 1) * 4 + kWarps * 4;                  // of rows of scores, float16
    static constexpr int kBytes = kLargest + (kNarrow<T> && !kEnds ? kAcross * kChunk * 4 : 0);
    static constexpr int kHeld = kEnds ? (kFloat && KA == 128 ? 2 : 3) : kFloat && KA == 128 ? 1 : kFloat || KA == 128 ? 2 : 3;           // CTAs that an SM has room for
};

// The maximum of a CTA's states, for the power of two of their float16 copy
template <int kWarps>
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* slots) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    v = slots[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v = max(v, slots[w]);
    return v;
}

// kEnds: the sums of each part's b_j c_j^T alone
template <typename T, int KA, bool kEnds>
__global__ void __launch_bounds__(Shape<T, KA, kEnds>::kThreads, Shape<T, KA, kEnds>::kHeld) attn_kernel(const AttnArgs args) {
    using S = Shape<T, KA, kEnds>;
    using L = Tile<T>;
    constexpr int kM = KA / 64;                  // 16-row tiles of the state that a warp has
    constexpr int kAcross = S::kAcross, kN = kCols / 8 / kAcross;       // 8-column tiles of c, in pairs
    constexpr int kSteps = kChunk / L::kK;
    extern __shared__ __align__(128) char smem[];
    const uint32_t tiles = shared_address(smem), copy = tiles + S::kStages * S::kStage;
    float* const powers = reinterpret_cast<float*>(smem + S::kTable);
    Carried& carried = reinterpret_cast<Carried*>(powers)[-1];
    uint32_t* const slots = reinterpret_cast<uint32_t*>(powers + kChunk + 1);
    float* const largest = reinterpret_cast<float*>(smem + S::kLargest);         // [side][row]
    const uint32_t table = shared_address(powers);
    const int warp = (threadIdx.x >> 5) & 3, side = threadIdx.x >> 7, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    auto col_of = [side](int n) { return ((n >> 1) * kAcross + side) * 16 + (n & 1) * 8; };              // where a warp's n-th tile lies

    const Place place = Place::of<kEnds>(args);
    const int tile = place.tile, which = place.which, unit = place.unit, h = unit % args.heads, b = unit / args.heads;
    const Job& job = args.job[which];
    if (tile >= args.tile_of[which]) return;
    const int col0 = tile * kCols, part = place.part;
    pdl_wait();

    const int64_t steps = args.steps;
    int64_t length = steps;
    if (args.lengths != nullptr) length = min(max(gload_i64(args.lengths + b), (int64_t)0), steps);
    const int64_t begin = (int64_t)part * place.part_steps, stop = min(begin + place.part_steps, steps);
    const int64_t finish = min(stop, length);    // of the steps there are
    const bool reverse = job.reverse != 0;
    const double log_decay = log_decay_of(args.log_decay, h);
    if (threadIdx.x < kChunk) powers[threadIdx.x] = power_of(log_decay, threadIdx.x);
    else if (threadIdx.x == kChunk) carried.begin(log_decay, kChunk), powers[kChunk] = carried.next();
    const int extra = reverse ? 0 : 1;           // powers of g on the state before a chunk, at its first step
    const int wa = job.a.width, wc = job.c.width;
    const bool exact = job.end != nullptr;       // the state is a result
    const int k_end = (wa + L::kK - 1) / L::kK * L::kK, c_end = wc - col0;        // of a's width, of c's columns
    const char* const from_a = static_cast<const char*>(job.a.p) + (b * job.a.s.batch + h / job.a.share * job.a.s.head) * (int64_t)sizeof(T);
    const char* const from_b = static_cast<const char*>(job.b.p) + (b * job.b.s.batch + h / job.b.share * job.b.s.head) * (int64_t)sizeof(T);
    const char* const from_c = static_cast<const char*>(job.c.p) + (b * job.c.s.batch + h / job.c.share * job.c.s.head) * (int64_t)sizeof(T);
    auto fetch = [&](int stage, int64_t first) {
        const uint32_t base = tiles + stage * S::kStage;
        if constexpr (!kEnds) load_tile<T, KA, S::kThreads>(base, job.a, from_a, first, length, 0, reverse);
        load_tile<T, KA, S::kThreads>(base + S::kB, job.b, from_b, first, length, 0, reverse);
        load_tile<T, kCols, S::kThreads>(base + S::kC, job.c, from_c, first, length, col0, reverse);
        copies_issued();
    };
    if (S::kStages == 2 && begin < finish) fetch(0, begin);

    // the state before this part
    float x[kM][kN][4];
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[m][n][e] = 0.0f;
                if constexpr (!kEnds) {
                    const int i = (m * 4 + warp) * 16 + g + (e >> 1) * 8, j = col0 + col_of(n) + 2 * t + (e & 1);
                    if (job.init != nullptr && i < wa && j < wc)
                        x[m][n][e] = job.init_scale * gload(job.init + (int64_t)unit * wa * wc + (int64_t)i * job.init_i + (int64_t)j * job.init_j);
                }
            }
    if constexpr (!kEnds) {
        const float whole = power_of(log_decay, place.part_steps);
        for (int s = 0; s < part; ++s) {
            const float* const sums = place.sums(args, s);
            // (a part that the sequence ends in is the last one that anything reads)
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = (m * 4 + warp) * 16 + g + (e >> 1) * 8, j = col0 + col_of(n) + 2 * t + (e & 1);
                        if (i < wa && j < wc && begin < length) x[m][n][e] = fmaf(x[m][n][e], whole, gload(sums + i * args.part_cols + j - col0));
                    }
        }
    }

    float by = 1.0f, back = 1.0f;                // float16: the copy is the state times `by`
    auto put_copy = [&]() {
        if constexpr (kNarrow<T>) {
            float most = 0.0f;
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(x[m][n][e]));
            const int shift = shift_of(__uint_as_float(cta_max<S::kWarps>(__float_as_uint(most), slots)));
            by = two_to(shift), back = two_to(-shift);
        }
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    put_pair<T>(L::at(copy, (m * 4 + warp) * 16 + g + half * 8, col_of(n) + 2 * t, kCols), x[m][n][2 * half] * by,
                                x[m][n][2 * half + 1] * by);
    };
    if constexpr (!kEnds) put_copy();

    int stage = 0;
    for (int64_t first = begin; first < finish; first += kChunk) {
        const int rows = (int)min((int64_t)kChunk, finish - first);
        if constexpr (S::kStages == 1) fetch(0, first);
        copies_arrived<0>();
        __syncthreads();                         // this chunk's tiles and the copy of the state are there
        if (S::kStages == 2 && first + kChunk < finish) fetch(stage ^ 1, first + kChunk);
        const uint32_t at = tiles + (S::kStages == 2 ? stage : 0) * S::kStage, bt = at + S::kB, ct = at + S::kC;
        if constexpr (!kEnds) {
            // which 16 steps a warp has goes round, so that the long rows of the triangle do not always meet the same scheduler
            const int m0 = ((warp + blockIdx.x + (int)(first / kChunk)) & 3) * 16;
            if (m0 < rows) {
                // a . X and a . b^T, each warp some pairs of columns of either
                float o[kN][4] = {}, s[kN][4] = {};
#pragma unroll 2
                for (int k = 0; k < k_end; k += L::kK) {
                    FragA<T> fa;
                    load_a<T>(fa, at, m0, k, KA, lane);
#pragma unroll
                    for (int n = 0; n < kN; n += 2) {
                        if (col_of(n) < c_end) {
                            FragB<T> fb[2];
                            load_bt<T>(fb, copy, k, col_of(n), kCols, lane);
                            mma<T>(o[n], fa, fb[0]);
                            mma<T>(o[n + 1], fa, fb[1]);
                        }
                        if (col_of(n) <= m0) {
                            FragB<T> fb[2];
                            load_b<T>(fb, bt, col_of(n), k, KA, lane);
                            mma<T>(s[n], fa, fb[0]);
                            mma<T>(s[n + 1], fa, fb[1]);
                        }
                    }
                }
                const float w0 = power(table, m0 + g + extra) * back, w1 = power(table, m0 + g + 8 + extra) * back;
#pragma unroll
                for (int n = 0; n < kN; ++n) o[n][0] *= w0, o[n][1] *= w0, o[n][2] *= w1, o[n][3] *= w1;
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = m0 + g + (e >> 1) * 8 - (col_of(n) + 2 * t + (e & 1));
                        s[n][e] = d >= 0 ? s[n][e] * power(table, max(d, 0)) : 0.0f;
                    }
                float score_by[2] = {1.0f, 1.0f}, score_back[2] = {1.0f, 1.0f};
                if constexpr (kNarrow<T>) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float most = 0.0f;
#pragma unroll
                        for (int n = 0; n < kN; ++n) most = fmaxf(fmaxf(most, fabsf(s[n][2 * half])), fabsf(s[n][2 * half + 1]));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1)), most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                        score_by[half] = most;
                        if (kAcross > 1 && t == 0) largest[side * kChunk + m0 + g + half * 8] = most;
                    }
                }
                // the scores take the place of these 16 steps of a, which these warps alone have read
                group_sync<32 * kAcross>(1 + warp);
                if constexpr (kNarrow<T>) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        for (int k = 0; kAcross > 1 && k < kAcross; ++k) score_by[half] = fmaxf(score_by[half], largest[k * kChunk + m0 + g + half * 8]);
                        const int shift = shift_of(score_by[half]);
                        score_by[half] = two_to(shift), score_back[half] = two_to(-shift);
                    }
                }
#pragma unroll
                for (int n = 0; n < kN; ++n)
                    if (col_of(n & ~1) <= m0) {
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            put_pair<T>(L::at(at, m0 + g + half * 8, col_of(n) + 2 * t, KA), s[n][2 * half] * score_by[half], s[n][2 * half + 1] * score_by[half]);
                    }
                group_sync<32 * kAcross>(1 + warp);
                // (float16: apart from the state's part, whose power of two is another)
                if constexpr (kNarrow<T>) {
#pragma unroll
                    for (int n = 0; n < kN; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
                }
                float (&product)[kN][4] = kNarrow<T> ? s : o;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if (k * L::kK > m0 + 15 || k * L::kK >= rows) continue;
                    FragA<T> fa;
                    load_a<T>(fa, at, m0, k * L::kK, KA, lane);
#pragma unroll
                    for (int n = 0; n < kN; n += 2) {
                        if (col_of(n) >= c_end) continue;
                        FragB<T> fb[2];
                        load_bt<T>(fb, ct, k * L::kK, col_of(n), kCols, lane);
                        mma<T>(product[n], fa, fb[0]);
                        mma<T>(product[n + 1], fa, fb[1]);
                    }
                }
                if constexpr (kNarrow<T>) {
#pragma unroll
                    for (int n = 0; n < kN; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][e] = fmaf(s[n][e], score_back[e >> 1], o[n][e]);
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int row = m0 + g + half * 8;
                    if (row >= rows) continue;
                    const int64_t pos = first + row, step = reverse ? length - 1 - pos : pos;
                    const int64_t to = (((int64_t)b * steps + step) * args.heads + h) * wc + col0;
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        const int c = col_of(n) + 2 * t;
                        const float p = o[n][2 * half] * args.scale, q = o[n][2 * half + 1] * args.scale;
                        const bool both = c + 1 < wc - col0, pairs = job.pairs != 0;
                        if (c >= wc - col0) continue;
                        if (std::is_same<T, float>::value || job.wide) {
                            float* const d = static_cast<float*>(job.out) + to + c;
                            if (both && pairs) *reinterpret_cast<float2*>(d) = make_float2(p, q);
                            else {
                                d[0] = p;
                                if (both) d[1] = q;
                            }
                        } else {
                            T* const d = static_cast<T*>(job.out) + to + c;
                            if constexpr (!std::is_same<T, float>::value) {
                                if (both && pairs) store(d, Raw<4>{{word_of<T>(p, q)}});
                                else {
                                    d[0] = from_float<T>(p);
                                    if (both) d[1] = from_float<T>(q);
                                }
                            }
                        }
                    }
                }
            }
        }
        // the state behind this chunk
        const float whole = power(table, rows);
        const int last_power = rows - extra;
        if constexpr (kNarrow<T>) {
            // (the sum of a chunk by itself: its power of two would take a large state out of float32)
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const int i0 = (m * 4 + warp) * 16;
                if (i0 >= wa) continue;
                uint32_t most[2] = {};
                for (int k = 0; k < rows; k += L::kK) largest_at(most, bt, k, i0, KA, lane);
                float row_by[2], row_back[2], sum[kN][4] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    most[half] = larger_pairs(most[half], __shfl_xor_sync(0xffffffffu, most[half], 1));
                    most[half] = larger_pairs(most[half], __shfl_xor_sync(0xffffffffu, most[half], 2));
                    const int shift = shift_up(max(most[half] & 0xffffu, most[half] >> 16), power(table, 1 - extra));
                    row_by[half] = two_to(shift), row_back[half] = two_to(-shift);
                }
#pragma unroll 1
                for (int k = 0; k < rows; k += L::kK) {
                    FragA<T> fa, low, lowest;
                    load_at<T>(fa, low, lowest, bt, k, i0, KA, lane, table, last_power, rows, row_by);
#pragma unroll
                    for (int n = 0; n < kN; n += 2) {
                        if (col_of(n) >= c_end) continue;
                        FragB<T> fb[2];
                        load_bt<T>(fb, ct, k, col_of(n), kCols, lane);
                        mma<T>(sum[n], fa, fb[0]);
                        mma<T>(sum[n + 1], fa, fb[1]);
                        mma<T>(sum[n], low, fb[0]);
                        mma<T>(sum[n + 1], low, fb[1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[m][n][e] = fmaf(x[m][n][e], whole, sum[n][e] * row_back[e >> 1]);
            }
        } else {
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[m][n][e] *= whole;
#pragma unroll 1
            for (int k = 0; k < rows; k += L::kK) {
                FragB<T> fb[kN / 2][2];
#pragma unroll
                for (int n = 0; n < kN; n += 2)
                    if (col_of(n) < c_end) load_bt<T>(fb[n / 2], ct, k, col_of(n), kCols, lane);
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    if ((m * 4 + warp) * 16 >= wa) continue;
                    FragA<T> fa, low, lowest;
                    load_at<T>(fa, low, lowest, bt, k, (m * 4 + warp) * 16, KA, lane, table, last_power, rows, {1.0f, 1.0f});
#pragma unroll
                    for (int n = 0; n < kN; n += 2) {
                        if (col_of(n) >= c_end) continue;
                        mma<T>(x[m][n], fa, fb[n / 2][0]);
                        mma<T>(x[m][n + 1], fa, fb[n / 2][1]);
                        if constexpr (!std::is_same<T, float>::value) {
                            mma<T>(x[m][n], low, fb[n / 2][0]);
                            mma<T>(x[m][n + 1], low, fb[n / 2][1]);
                            if (exact) {
                                mma<T>(x[m][n], lowest, fb[n / 2][0]);
                                mma<T>(x[m][n + 1], lowest, fb[n / 2][1]);
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();                         // every warp is done with the tiles and the copy
        if (threadIdx.x == 0) powers[kChunk] = carried.next();           // (read behind the next barrier)
        if constexpr (!kEnds) put_copy();
        stage ^= 1;
    }

    // (the first part ends a sequence of no steps)
    const bool ends_here = kEnds || (length > begin && length <= begin + place.part_steps) || (length == 0 && part == 0);
    float* const to = kEnds ? place.sums(args, part) - col0 : job.end != nullptr ? job.end + (int64_t)unit * wa * wc : nullptr;
    const int row = kEnds ? args.part_cols : wc;
    if (ends_here && to != nullptr) {
        const float by = kEnds ? 1.0f : job.end_scale;
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int n = 0; n < kN; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = (m * 4 + warp) * 16 + g + (e >> 1) * 8, j = col0 + col_of(n) + 2 * t + (e & 1);
                    if (i < wa && j < wc) to[(int64_t)i * row + j] = by * x[m][n][e];
                }
    }
    if constexpr (!kEnds) {
        // zeros behind the length
        const int64_t from = max(begin, length);
        const int n = min(kCols, wc - col0);
        const int64_t count = (stop - from) * n;
        for (int64_t i = threadIdx.x; i < count; i += S::kThreads) {
            const int64_t step = from + i / n, to_ = (((int64_t)b * steps + step) * args.heads + h) * wc + col0 + i % n;
            if (std::is_same<T, float>::value || job.wide) static_cast<float*>(job.out)[to_] = 0.0f;
            else static_cast<T*>(job.out)[to_] = from_float<T>(0.0f);
        }
    }
}

// Narrow loads that stay in L1: their neighbours find the rest of a sector there (without, each fetched it from L2 again, and joining
// 502 K rows of 71 took 131 us)
__device__ __forceinline__ uint32_t load_word(const void* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
template <typename T>
__device__ __forceinline__ float load_element(const T* p) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(load_word(p));
    } else {
        uint16_t v;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
        return to_float(*reinterpret_cast<const T*>(&v));
    }
}

// Rows that a bulk copy does not take (widths that 8 does not divide, odd strides, inputs that are broadcast) as rows that it takes: the
// width rounded up to 8, heads and steps dense.  A thread moves 16 bytes, read as aligned words of 4; what lies behind a row's end is
// not written, nor ever read.
struct PackArgs {
    struct One {
        const char* from;
        char* to;
        int64_t batch, step, head;               // bytes
        int width, vecs, heads;
    } of[4];
    const int64_t* lengths;
    int64_t rows, steps;                         // rows: batch * steps
    int span;                                    // 16 bytes that a CTA has at a time, about
};

__global__ void __launch_bounds__(256) pack_kernel(const PackArgs args) {
    const PackArgs::One o = args.of[blockIdx.y];
    pdl_wait();
    const int row_vecs = o.heads * o.vecs, block_rows = max(1, args.span / row_vecs);
    for (int64_t row0 = (int64_t)blockIdx.x * block_rows; row0 < args.rows; row0 += (int64_t)gridDim.x * block_rows) {
        const int64_t b0 = row0 / args.steps, t0 = row0 - b0 * args.steps;
        const int count = (int)min((int64_t)block_rows, args.rows - row0) * row_vecs;
#pragma unroll 4
        for (int i = threadIdx.x; i < count; i += 256) {
            const int row = i / row_vecs, in_row = i - row * row_vecs, h = in_row / o.vecs, v = in_row - h * o.vecs;
            const uint32_t from0 = (uint32_t)t0 + row, more = from0 / (uint32_t)args.steps;
            const int64_t b = b0 + more, t = from0 - more * (uint32_t)args.steps;
            const bool live = args.lengths == nullptr || t < gload_i64(args.lengths + b);
            const char* const from = o.from + b * o.batch + t * o.step + h * o.head + v * 16;
            const int bytes = live ? min(16, (o.width - v * 8) * 2) : 0, skew = (int)(reinterpret_cast<uintptr_t>(from) & 2);
            uint32_t w[5];
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                w[k] = bytes > 0 && 4 * k - skew < bytes ? load_word(from - skew + 4 * k) : 0;
            }
            Raw<16> out;
#pragma unroll
            for (int k = 0; k < 4; ++k) out.u[k] = __funnelshift_r(w[k], w[k + 1], skew * 8);
            if (live) store(o.to + ((row0 + row) * row_vecs + in_row) * 16, out);
        }
    }
}

// Gradients of keys and values that heads share, as sums over these (From: float); or results with rows of a multiple of 8 (From: T) as
// the dense ones that they are.  A thread writes 16 bytes, whichever rows they are of.
template <typename T, typename From>
__global__ void __launch_bounds__(256) join_kernel(const From* from, T* to, int64_t count, int share, int width, int room) {
    constexpr int kVec = 16 / (int)sizeof(T), kSpan = 256 * kVec;
    pdl_wait();
    const int64_t skew = (int64_t)(reinterpret_cast<uintptr_t>(to) % 16 / sizeof(T));
    for (int64_t start = (int64_t)blockIdx.x * kSpan - skew; start < count; start += (int64_t)gridDim.x * kSpan) {
        const int64_t row0 = max(start, (int64_t)0) / width;
        const int in = (int)(start - row0 * width) + (int)threadIdx.x * kVec;    // (may begin in front of the first row)
        const int64_t first = start + (int64_t)threadIdx.x * kVec;
        const int row = max(in, 0) / width;
        int col = in - row * width;
        const From* p = from + (row0 + row) * share * room;
        float sum[kVec] = {};
        int at[kVec];
        bool there[kVec], all = true, any = false;
#pragma unroll
        for (int e = 0, before = 0; e < kVec; ++e) {
            there[e] = first + e >= 0 && first + e < count;
            at[e] = there[e] ? before + col : 0;
            all = all && there[e], any = any || there[e];
            if (++col == width) col = 0, before += share * room;
        }
        for (int s = 0; s < (std::is_same<From, float>::value ? share : 1); ++s, p += room) {
            float f[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) f[e] = any ? load_element(p + at[e]) : 0.0f;
#pragma unroll
            for (int e = 0; e < kVec; ++e) sum[e] += f[e];
        }
        if (all) {
            Pack<T, kVec> out;
            out.set(sum);
            out.put(to + first);
        } else {
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                if (there[e]) to[first + e] = from_float<T>(sum[e]);
        }
    }
}

// ---- a single step --------------------------------------------------------------------------------------------------------
// A CTA advances a head's state of one sequence, kW columns of dv a thread, rows of dk over the rest; it is read and written once, which is
// what bounds it: 256 sequences of 16 heads of 128 x 128, 537 MB in 102 us, 0.82 of a copy's rate.
struct StepArgs {
    const void *q, *k, *v;
    Strides qs, ks, vs;
    const float* log_decay;
    float* state;
    const int64_t* slots;
    void* out;
    int64_t pool;
    int heads, share, dk, dv;
    float scale;
};

template <typename T, int kW, int kT>
__global__ void __launch_bounds__(kT) attn_step_kernel(const StepArgs a) {
    __shared__ float key[kMostWidth], query[kMostWidth], sums[kT * kW];
    pdl_wait();
    const int h = blockIdx.x % a.heads;
    const int64_t r = blockIdx.x / a.heads;
    const int64_t slot = a.slots != nullptr ? gload_i64(a.slots + r) : r;
    T* const out = static_cast<T*>(a.out) + (r * a.heads + h) * a.dv;
    if (slot < 0 || slot >= a.pool) {
        for (int j = threadIdx.x; j < a.dv; j += kT) out[j] = from_float<T>(0.0f);
        return;
    }
    const int groups = (a.dv + kW - 1) / kW, sets = kT / groups, set = threadIdx.x / groups, j = threadIdx.x % groups * kW;
    const T* const q = static_cast<const T*>(a.q) + r * a.qs.batch + h * a.qs.head;
    const T* const k = static_cast<const T*>(a.k) + r * a.ks.batch + h / a.share * a.ks.head;
    const T* const v = static_cast<const T*>(a.v) + r * a.vs.batch + h / a.share * a.vs.head;
    // (and what its rounding leaves, which would add up over a stream's steps.  Rounded down, so that this is above zero: infinity stays infinity)
    const double whole = exp(log_decay_of(a.log_decay, h));
    const float decay = __double2float_rd(whole), rest = fmaxf((float)(whole - (double)decay), decay * 1e-12f);
    for (int i = threadIdx.x; i < a.dk; i += kT) {
        Pack<T, 1> p;
        p.get(k + i), key[i] = p.at(0);
        p.get(q + i), query[i] = p.at(0) * a.scale;
    }
    float value[kW], sum[kW];
#pragma unroll
    for (int e = 0; e < kW; ++e) {
        Pack<T, 1> p;
        p.zero();
        if (set < sets && j + e < a.dv) p.get(v + j + e);
        value[e] = p.at(0), sum[e] = 0.0f;
    }
    __syncthreads();
    float* const state = a.state + (slot * a.heads + h) * (int64_t)a.dk * a.dv;
    if (set < sets) {
#pragma unroll 8
        for (int i = set; i < a.dk; i += sets) {
            Pack<float, kW> s;
            float f[kW];
            s.get(state + (int64_t)i * a.dv + j);
#pragma unroll
            for (int e = 0; e < kW; ++e) {
                f[e] = fmaf(s.at(e), decay, fmaf(s.at(e), rest, key[i] * value[e]));
                sum[e] = fmaf(f[e], query[i], sum[e]);
            }
            s.set(f);
            s.put(state + (int64_t)i * a.dv + j);
        }
#pragma unroll
        for (int e = 0; e < kW; ++e) sums[(set * groups + threadIdx.x % groups) * kW + e] = sum[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.dv; c += kT) {
        float s = 0.0f;
        for (int p = 0; p < sets; ++p) s += sums[p * groups * kW + c];
        out[c] = from_float<T>(s);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int check_attn(const dcn_attn* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype)) return DCN_ERR_UNSUPPORTED;
    if (p->batch < 0 || p->steps < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0 || p->dk < 1 || p->dv < 1)
        return DCN_ERR_SHAPE;
    if (!std::isfinite(p->scale) || p->scale == 0.0f || !std::isfinite(1.0f / p->scale)) return DCN_ERR_SHAPE;
    if (p->dk > kMostWidth || p->dv > kMostWidth || p->heads > 65535 || p->steps >= 1ll << 30) return DCN_ERR_LIMIT;
    if (p->batch >= (1ll << 27) / p->heads) return DCN_ERR_LIMIT;
    return DCN_OK;
}

int wide_of(const dcn_attn* p, bool backward) { return (int)(backward ? std::max(p->dk, p->dv) : p->dk) > 64 ? 128 : 64; }

// How the work is shared out.  Time goes in chunks of a CTA; a GPU holds `held` CTAs at once.  As many units (job, head, 64 columns)
// as fill it a whole number of times have their time axis to themselves; that of the others is split.  More parts fill the GPU, and cost
// a pass over b and c for their sums (half of a chunk's time) and the folding (a quarter of a chunk's for each part before), and each CTA
// what it costs to begin and to end.  (5x331x6x(40, 72) float32, 30 heads: three parts instead of one.  2x16384x16x128 bf16, where
// the backward pass has 192 units: 764 us with its gradients, 834 us when all units were whole.)
int held_of(bool wide_type, int width) {
    if (wide_type) return width == 128 ? Shape<float, 128, false>::kHeld : Shape<float, 64, false>::kHeld;
    return width == 128 ? Shape<__half, 128, false>::kHeld : Shape<__half, 64, false>::kHeld;
}
struct Split {
    int64_t whole;
    int parts;
};
Split split_of(const dcn_attn* p, bool backward, bool tensor, int jobs, int tiles) {
    const int64_t chunk = tensor ? tcgen::kSteps : kChunk;
    const int64_t units = p->batch * p->heads * tiles * jobs, chunks = (p->steps + chunk - 1) / chunk;
    const int64_t held = (int64_t)sm_count() * (tensor ? 1 : held_of(p->dtype == DCN_SEQ_F32, wide_of(p, backward)));
    const int64_t sums_held = (int64_t)sm_count() * (tensor ? 1 : wide_of(p, backward) == 128 ? Shape<float, 128, true>::kHeld : Shape<float, 64, true>::kHeld);
    const double fixed = tensor ? 2 : 0.7;
    if (!tensor && p->dtype != DCN_SEQ_F32) return {units, 1};           // (short ones)
    const int64_t full = units / held * held, rest = units - full;
    Split best = {units, 1};
    double least = (double)((rest + held - 1) / held) * (chunks + fixed);
    for (int n = 2; n <= kMostParts && n <= chunks; ++n) {
        const int64_t each = (chunks + n - 1) / n;
        if ((chunks + each - 1) / each != n) continue;
        const double waves = (double)((rest * n + held - 1) / held), sums = (double)((rest * (n - 1) + sums_held - 1) / sums_held);
        const double time = waves * (each + fixed + 0.25 * (n - 1)) + sums * (0.5 * each + fixed) + 0.5 * fixed;
        if (time < least * 0.97) least = time, best = {full, n};
    }
    return best;
}

unsigned ctas_of(const AttnArgs& a, bool ends) {
    const int64_t rest = (int64_t)a.batch * a.heads * a.jobs * a.tiles - a.whole;
    return (unsigned)(ends ? rest * (a.n_parts - 1) : a.whole + rest * a.n_parts);
}

template <typename T, int KA, bool kEnds>
int launch_attn(const AttnArgs& a, cudaStream_t st) {
    using S = Shape<T, KA, kEnds>;
    constexpr int kBytes = S::kBytes;
    if (cudaFuncSetAttribute(attn_kernel<T, KA, kEnds>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess)
        return DCN_ERR_CUDA;
    const dim3 grid(ctas_of(a, kEnds));
    return launch_dependent(attn_kernel<T, KA, kEnds>, grid, dim3(S::kThreads), kBytes, st, a) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int KA, bool kEnds>
int launch_attn_tc(const AttnArgs& a, const tcgen::Maps& maps, cudaStream_t st) {
    constexpr int kBytes = tcgen::Room<T, KA>::kBytes;
    const auto kernel = tcgen::attn_tc_kernel<T, KA, kEnds>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess) return DCN_ERR_CUDA;
    const dim3 grid(ctas_of(a, kEnds));
    return launch_dependent(kernel, grid, dim3(tcgen::kThreads), kBytes, st, a, maps) != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int KA>
int run_parts(const AttnArgs& a, const tcgen::Maps* maps, cudaStream_t st) {
    if constexpr (!std::is_same<T, float>::value)
        if (maps != nullptr) {
            const int rc = a.n_parts > 1 ? launch_attn_tc<T, KA, true>(a, *maps, st) : DCN_OK;
            return rc != DCN_OK ? rc : launch_attn_tc<T, KA, false>(a, *maps, st);
        }
    if constexpr (std::is_same<T, float>::value)
        if (a.n_parts > 1) {
            const int rc = launch_attn<T, KA, true>(a, st);
            if (rc != DCN_OK) return rc;
        }
    return launch_attn<T, KA, false>(a, st);
}

template <typename T>
int run_attn(const AttnArgs& a, int wide, const tcgen::Maps* maps, cudaStream_t st) {
    return wide == 128 ? run_parts<T, 128>(a, maps, st) : run_parts<T, 64>(a, maps, st);
}

// maps: those of the call's operands, or null where the tensor cores' kernel does not take them
int run_attn_any(const dcn_attn* p, const AttnArgs& a, bool backward, const tcgen::Maps* maps, cudaStream_t st) {
    const int wide = wide_of(p, backward);
    return p->dtype == DCN_SEQ_F32    ? run_attn<float>(a, wide, nullptr, st)
           : p->dtype == DCN_SEQ_BF16 ? run_attn<__nv_bfloat16>(a, wide, maps, st)
                                      : run_attn<__half>(a, wide, maps, st);
}

// Bytes that every row of an operand starts on, as cp.async takes them (2: element by element)
Operand operand(const dcn_attn* p, int map, const void* at, int64_t batch, int64_t step, int64_t head, int64_t width, int share) {
    const int e = elem_bytes(p->dtype);
    Operand o = {at, {p->batch > 1 ? batch : 0, p->steps > 1 ? step : 0, head}, share, (int)width, 16, map};
    while (o.bytes > 2 && (!aligned(at, o.bytes) || o.s.batch * e % o.bytes != 0 || o.s.step * e % o.bytes != 0 || head * e % o.bytes != 0))
        o.bytes /= 2;
    return o;
}

struct Operands {
    Operand q, k, v, d;
    Operand* begin() { return &q; }
    Operand* end() { return &d + 1; }
};
Operands operands(const dcn_attn* p, const void* q, const void* k, const void* v, const void* dout) {
    const int share = (int)(p->heads / p->kv_heads);
    return {operand(p, 0, q, p->q_batch, p->q_step, p->heads > 1 ? p->q_head : 0, p->dk, 1),
            operand(p, 1, k, p->k_batch, p->k_step, p->kv_heads > 1 ? p->k_head : 0, p->dk, share),
            operand(p, 2, v, p->v_batch, p->v_step, p->kv_heads > 1 ? p->v_head : 0, p->dv, share),
            operand(p, 3, dout, p->dout_batch, p->dout_step, p->heads > 1 ? p->dout_head : 0, p->dv, 1)};
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
int up8(int64_t width) { return (int)((width + 7) / 8 * 8); }

// What a call does with its operands and its workspace, by its sizes, type and strides alone
struct Plan {
    bool tensor;                                 // the tensor cores' kernel, if the pointers allow it
    bool pack[4];                                // operands that are laid out anew for it (q, k, v, dout)
    bool shared;                                 // gradients of k and v are sums over heads
    int room_k, room_v;                          // elements of a row of results dk and dv wide, as that kernel writes them
    size_t packed[4], dq, dk, dv, bytes;         // places in the workspace (parts are at its beginning): packed operands, results
};

int64_t parts_floats(const dcn_attn* p, bool backward, bool tensor);

Plan plan_of(const dcn_attn* p, bool backward) {
    Plan w = {};
    // Sequences of one chunk: a CTA of the other kernel begins and ends sooner, and two or three share an SM (1024 heads of 64 steps and
    // 128 x 128 bf16: 129 us, 178 us on the tensor cores; of 128 steps: 200 and 184)
    w.tensor = p->dtype != DCN_SEQ_F32 && p->steps > kChunk;
    w.shared = backward && p->heads != p->kv_heads;
    w.room_k = w.tensor ? up8(p->dk) : (int)p->dk, w.room_v = w.tensor ? up8(p->dv) : (int)p->dv;
    size_t at = rounded((size_t)parts_floats(p, backward, false) * 4);
    if (w.tensor) at = std::max(at, rounded((size_t)parts_floats(p, backward, true) * 4));
    auto place = [&](size_t n) {
        const size_t here = at;
        at += rounded(n);
        return here;
    };
    const size_t rows = (size_t)p->batch * p->steps;
    if (w.tensor) {
        const Operands all = operands(p, nullptr, nullptr, nullptr, nullptr);
        const Operand* const of[4] = {&all.q, &all.k, &all.v, &all.d};
        for (int i = 0; i < (backward ? 4 : 3); ++i) {
            const Operand& o = *of[i];
            const int64_t heads = p->heads / o.share, most = 1ll << 38;
            w.pack[i] = o.bytes != 16 || (p->batch > 1 && o.s.batch <= 0) || (p->steps > 1 && o.s.step <= 0) || (heads > 1 && o.s.head <= 0) ||
                        o.s.batch >= most || o.s.step >= most || o.s.head >= most;
            if (w.pack[i]) w.packed[i] = place(rows * heads * up8(o.width) * 2);
        }
    }
    // (results that are joined or that have rows of another length)
    if (backward && w.room_k != p->dk) w.dq = place(rows * p->heads * w.room_k * 2);
    if (backward && (w.shared || w.room_k != p->dk)) w.dk = place(rows * p->heads * w.room_k * (w.shared ? 4 : 2));
    if (w.shared || w.room_v != p->dv) w.dv = place(rows * p->heads * w.room_v * (w.shared ? 4 : 2));
    w.bytes = at;
    return w;
}

// Whether the pointers allow what is planned for the tensor cores
bool allowed(const Plan& w, const Operands& o, const dcn_attn* p, std::initializer_list<const void*> results_k, std::initializer_list<const void*> results_v,
             const void* state, const void* workspace) {
    if (!w.tensor || !aligned(state, 16) || !aligned(workspace, 16)) return false;
    const Operand* const of[4] = {&o.q, &o.k, &o.v, &o.d};
    for (int i = 0; i < 4; ++i)
        if (!w.pack[i] && !aligned(of[i]->p, 16)) return false;
    // (results with rows of another length, and those that heads share, go through the workspace)
    for (const void* r : results_k)
        if (w.room_k == p->dk && !aligned(r, 16)) return false;
    for (const void* r : results_v)
        if (w.room_v == p->dv && !aligned(r, 16)) return false;
    return true;
}

// The driver's function, found at run time: the library is not linked with the driver's
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return found;
}

// Lays out anew what the plan says, and makes the maps
bool prepare(const dcn_attn* p, const Plan& w, Operands& o, const int64_t* lengths, void* workspace, tcgen::Maps& maps, cudaStream_t st) {
    const EncodeTiled encode = encode_tiled();
    if (encode == nullptr) return false;
    // (the driver's function wants a context, which a thread that has launched nothing yet does not have: an engine's first backward pass)
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaSetDevice(device) != cudaSuccess) return false;
    PackArgs args = {};
    args.lengths = lengths, args.rows = p->batch * p->steps, args.steps = p->steps;
    int64_t most = 0;
    unsigned packs = 0;
    int i = 0;
    for (Operand& x : o) {
        if (w.pack[i++] && x.p != nullptr) {
            const int heads = (int)(p->heads / x.share), room = up8(x.width);
            char* const to = static_cast<char*>(workspace) + w.packed[i - 1];
            args.of[packs++] = {static_cast<const char*>(x.p), to, x.s.batch * 2, x.s.step * 2, x.s.head * 2, x.width, room / 8, heads};
            most = std::max(most, args.rows * heads * (room / 8));
            x.p = to, x.s = {p->steps * heads * room, (int64_t)heads * room, room}, x.bytes = 16;
        }
    }
    for (const Operand* x : {&o.q, &o.k, &o.v, &o.d}) {
        if (x->p == nullptr) continue;
        const cuuint64_t heads = (cuuint64_t)(p->heads / x->share), row = ((cuuint64_t)x->width * 2 + 15) / 16 * 16;
        const cuuint64_t dims[4] = {(cuuint64_t)x->width, heads, (cuuint64_t)p->steps, (cuuint64_t)p->batch};
        const cuuint64_t strides[3] = {heads > 1 ? (cuuint64_t)x->s.head * 2 : row, p->steps > 1 ? (cuuint64_t)x->s.step * 2 : row,
                                       p->batch > 1 ? (cuuint64_t)x->s.batch * 2 : row};
        const cuuint32_t box[4] = {64, 1, tcgen::kSteps, 1}, ones[4] = {1, 1, 1, 1};
        const CUtensorMapDataType type = p->dtype == DCN_SEQ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        if (encode(&maps.of[x->map], type, 4, const_cast<void*>(x->p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    }
    args.span = most > 1024 * 1024 ? 1024 : 256;
    const unsigned ctas = (unsigned)std::min<int64_t>(most / args.span + 1, 148 * 8);
    return packs == 0 || launch_dependent(pack_kernel, dim3(ctas, packs), dim3(256), 0, st, args) == cudaSuccess;
}

AttnArgs attn_args(const dcn_attn* p, const float* log_decay, const int64_t* lengths) {
    AttnArgs a = {};
    a.log_decay = log_decay, a.lengths = lengths;
    a.steps = p->steps;
    a.batch = (int)p->batch, a.heads = (int)p->heads;
    a.scale = p->scale;
    return a;
}

// Parts' sums are kept of the units that are split alone, of 64 columns each: the most that any job has.  (Of every unit, a batch of
// thousands of heads would need gigabytes for the few that do not fill the GPU.)
struct PartSize {
    int rows, cols;
};
PartSize part_of(const dcn_attn* p, bool backward, bool tensor) {
    const int row_k = (int)(tensor ? up8(p->dk) : p->dk), row_v = (int)(tensor ? up8(p->dv) : p->dv);
    return {(int)(backward ? std::max(p->dk, p->dv) : p->dk), std::min(kCols, backward ? std::max(row_k, row_v) : row_v)};
}

// (once the jobs are there)
void share_out(AttnArgs& a, const dcn_attn* p, bool backward, bool tensor, void* workspace) {
    const Split split = split_of(p, backward, tensor, a.jobs, a.tiles);
    const int64_t chunk = tensor ? tcgen::kSteps : kChunk, chunks = (p->steps + chunk - 1) / chunk;
    const PartSize size = part_of(p, backward, tensor);
    a.n_parts = split.parts, a.whole = split.whole;
    a.part_steps = std::max<int64_t>(1, (chunks + a.n_parts - 1) / a.n_parts) * chunk;
    a.parts = static_cast<float*>(workspace), a.part_cols = size.cols, a.part_floats = size.rows * size.cols;
}

void add(AttnArgs& a, const Job& j, int elem) {
    a.tile_of[a.jobs] = (j.c.width + kCols - 1) / kCols;
    a.tiles = std::max(a.tiles, a.tile_of[a.jobs]);
    a.job[a.jobs] = j;
    a.job[a.jobs].sectors = j.room % 16 == 0 && aligned(j.out, 32);
    a.job[a.jobs++].pairs = j.room % 2 == 0 && aligned(j.out, 2 * (j.wide ? 4 : elem));
}

// Floats that the parts' sums take, whichever gradients a call wants: their number, and the columns of the widest, decide the split
int64_t parts_floats(const dcn_attn* p, bool backward, bool tensor) {
    int64_t most = 0;
    for (int jobs = 1; jobs <= (backward ? 3 : 1); ++jobs)
        for (int tiles = 1; tiles <= 2; ++tiles) {
            const Split split = split_of(p, backward, tensor, jobs, tiles);
            if (split.parts > 1) most = std::max(most, (p->batch * p->heads * jobs * tiles - split.whole) * split.parts);
        }
    const PartSize size = part_of(p, backward, tensor);
    return most * size.rows * size.cols;
}

// Results in the workspace to where they belong
template <typename From>
int join(const dcn_attn* p, const void* from, void* to, int64_t heads, int share, int64_t width, int room, cudaStream_t st) {
    const int64_t count = p->batch * p->steps * heads * width, span = 256 * (16 / elem_bytes(p->dtype));
    const dim3 grid((unsigned)std::min<int64_t>(count / span + 2, 148 * 16));      // (one more where the first 16 bytes are not whole)
    auto go = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        using F = std::conditional_t<std::is_same<From, float>::value, float, T>;
        return launch_dependent(join_kernel<T, F>, grid, dim3(256), 0, st, static_cast<const F*>(from), static_cast<T*>(to), count, share, (int)width, room);
    };
    const cudaError_t e = p->dtype == DCN_SEQ_F32    ? go((float*)nullptr)
                          : p->dtype == DCN_SEQ_BF16 ? go((__nv_bfloat16*)nullptr)
                                                     : go((__half*)nullptr);
    return e == cudaSuccess ? DCN_OK : DCN_ERR_CUDA;
}

bool attn_aligned(const dcn_attn* p, std::initializer_list<const void*> elems, std::initializer_list<const void*> floats) {
    for (const void* v : elems)
        if (!aligned(v, elem_bytes(p->dtype))) return false;
    for (const void* v : floats)
        if (!aligned(v, 4)) return false;
    return true;
}

}  // namespace

int attn_check_status(cudaStream_t st) {
    unsigned int v = 0;
    if (cudaStreamSynchronize(st) != cudaSuccess || cudaMemcpyFromSymbol(&v, tc::g_tc_status, sizeof(v)) != cudaSuccess) return DCN_ERR_CUDA;
    if (v == 0) return DCN_OK;
    const unsigned int zero = 0;
    cudaMemcpyToSymbol(tc::g_tc_status, &zero, sizeof(zero));
    return DCN_ERR_TIMEOUT;
}

}  // namespace seq
}  // namespace dcn

using namespace dcn::seq;
using dcn::launch_dependent;

extern "C" size_t dcn_attn_workspace_bytes(const dcn_attn* p, int32_t backward) {
    if (check_attn(p) != DCN_OK || p->batch == 0) return 0;
    return plan_of(p, backward != 0).bytes;
}

extern "C" int dcn_attn_forward(const dcn_attn* p, const void* q, const void* k, const void* v, const float* log_decay,
                                const float* state, const int64_t* lengths, void* out, float* last, void* workspace,
                                size_t workspace_bytes, void* stream) {
    const int bad = check_attn(p);
    if (bad != DCN_OK) return bad;
    if (p->batch == 0) return DCN_OK;
    if (log_decay == nullptr || last == nullptr || (p->steps > 0 && (q == nullptr || k == nullptr || v == nullptr || out == nullptr)))
        return DCN_ERR_NULL;
    if (!attn_aligned(p, {q, k, v, out}, {log_decay, state, last}) || !aligned(lengths, 8)) return DCN_ERR_ALIGN;
    const Plan w = plan_of(p, false);
    if (w.bytes > 0 && (workspace == nullptr || !aligned(workspace, 4) || workspace_bytes < w.bytes)) return DCN_ERR_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    Operands o = operands(p, q, k, v, nullptr);
    tcgen::Maps maps = {};
    const bool tensor = allowed(w, o, p, {}, {out}, last, workspace);
    if (tensor && !prepare(p, w, o, lengths, workspace, maps, st)) return DCN_ERR_CUDA;
    const int room = tensor ? w.room_v : (int)p->dv;
    void* const to = room != p->dv ? static_cast<char*>(workspace) + w.dv : out;
    AttnArgs a = attn_args(p, log_decay, lengths);
    add(a, {o.q, o.k, o.v, to, state, last, room, (int)p->dv, 1, 0, 0, 1.0f, 1.0f}, elem_bytes(p->dtype));
    share_out(a, p, false, tensor, workspace);
    const int rc = run_attn_any(p, a, false, tensor ? &maps : nullptr, st);
    return rc != DCN_OK || to == out ? rc : join<void>(p, to, out, p->heads, 1, p->dv, room, st);
}

extern "C" int dcn_attn_backward(const dcn_attn* p, const void* q, const void* k, const void* v, const float* log_decay,
                                 const float* state, const int64_t* lengths, const void* dout, const float* dlast, void* dq, void* dk,
                                 void* dv, float* dstate, void* workspace, size_t workspace_bytes, void* stream) {
    const int bad = check_attn(p);
    if (bad != DCN_OK) return bad;
    if (p->batch == 0) return DCN_OK;
    if (log_decay == nullptr || (p->steps > 0 && (q == nullptr || k == nullptr || v == nullptr))) return DCN_ERR_NULL;
    if (!attn_aligned(p, {q, k, v, dout, dq, dk, dv}, {log_decay, state, dlast, dstate}) || !aligned(lengths, 8)) return DCN_ERR_ALIGN;
    const Plan w = plan_of(p, true);
    if (w.bytes > 0 && (workspace == nullptr || !aligned(workspace, 4) || workspace_bytes < w.bytes)) return DCN_ERR_WORKSPACE;
    const cudaStream_t st = (cudaStream_t)stream;
    if (p->steps > 0 && (dout == nullptr || (dstate != nullptr && dv == nullptr))) return DCN_ERR_NULL;
    if (dq == nullptr && dk == nullptr && dv == nullptr && dstate == nullptr) return DCN_OK;
    Operands o = operands(p, q, k, v, dout);
    tcgen::Maps maps = {};
    const bool tensor = w.shared ? allowed(w, o, p, {dq}, {}, dstate, workspace) : allowed(w, o, p, {dq, dk}, {dv}, dstate, workspace);
    if (tensor && !prepare(p, w, o, lengths, workspace, maps, st)) return DCN_ERR_CUDA;
    AttnArgs a = attn_args(p, log_decay, lengths);
    const int room_k = tensor ? w.room_k : (int)p->dk, room_v = tensor ? w.room_v : (int)p->dv;
    const bool other_k = room_k != p->dk, other_v = room_v != p->dv;             // rows of another length than the results'
    char* const at = static_cast<char*>(workspace);
    void* const to_q = other_k ? at + w.dq : dq;
    void* const to_k = w.shared || other_k ? at + w.dk : dk;
    void* const to_v = w.shared || other_v ? at + w.dv : dv;
    const int across = (int)p->dv, elem = elem_bytes(p->dtype), shared = w.shared;
    const float s = p->scale;
    if (dq != nullptr) add(a, {o.d, o.v, o.k, to_q, state, nullptr, room_k, 1, across, 0, 0, 1.0f, 1.0f}, elem);
    if (dk != nullptr) add(a, {o.v, o.d, o.q, to_k, dlast, nullptr, room_k, 1, across, 1, shared, 1.0f / s, 1.0f}, elem);
    if (dv != nullptr || dstate != nullptr) add(a, {o.k, o.q, o.d, to_v, dlast, dstate, room_v, across, 1, 1, shared, 1.0f / s, s}, elem);
    share_out(a, p, true, tensor, workspace);
    int rc = run_attn_any(p, a, true, tensor ? &maps : nullptr, st);
    if (rc != DCN_OK || p->steps == 0) return rc;
    const int share = (int)(p->heads / p->kv_heads);
    auto sum = [&](const void* from, void* to, int64_t width, int room) {
        return w.shared ? join<float>(p, from, to, p->kv_heads, share, width, room, st) : join<void>(p, from, to, p->heads, 1, width, room, st);
    };
    if (dq != nullptr && to_q != dq) rc = join<void>(p, to_q, dq, p->heads, 1, p->dk, room_k, st);
    if (rc == DCN_OK && dk != nullptr && to_k != dk) rc = sum(to_k, dk, p->dk, room_k);
    if (rc == DCN_OK && dv != nullptr && to_v != dv) rc = sum(to_v, dv, p->dv, room_v);
    return rc;
}

extern "C" int dcn_attn_step(const dcn_attn* p, const void* q, const void* k, const void* v, const float* log_decay,
                             float* pool_state, int64_t pool, const int64_t* slots, void* out, void* stream) {
    const int bad = check_attn(p);
    if (bad != DCN_OK) return bad;
    if (p->steps != 1 || pool < 0 || (slots == nullptr && pool < p->batch)) return DCN_ERR_SHAPE;
    if (p->batch == 0) return DCN_OK;
    if (q == nullptr || k == nullptr || v == nullptr || log_decay == nullptr || out == nullptr || (pool_state == nullptr && pool > 0))
        return DCN_ERR_NULL;
    if (!attn_aligned(p, {q, k, v, out}, {log_decay, pool_state}) || !aligned(slots, 8)) return DCN_ERR_ALIGN;
    StepArgs a = {q, k, v, {p->q_batch, 0, p->q_head}, {p->k_batch, 0, p->k_head}, {p->v_batch, 0, p->v_head}, log_decay, pool_state,
                  slots, out, pool, (int)p->heads, (int)(p->heads / p->kv_heads), (int)p->dk, (int)p->dv, p->scale};
    const dim3 grid((unsigned)(p->batch * p->heads));
    const cudaStream_t st = (cudaStream_t)stream;
    const bool wide = p->dv % 4 == 0 && aligned(pool_state, 16);
    auto go = [&](auto* type) {
        using T = std::remove_pointer_t<decltype(type)>;
        // More threads to a head where they have one column each (200x8x(107, 71) bf16: 45.8 us with 128, 30.8 with 512) or where there are too
        // few heads to fill the GPU (8x8x(128, 128): 8.6 and 4.5; 64x8x(128, 128), where there are enough: 10.3 and 11.1)
        const bool few = grid.x < 2u * (unsigned)dcn::sm_count();
        return !wide ? launch_dependent(attn_step_kernel<T, 1, 512>, grid, dim3(512), 0, st, a)
               : few ? launch_dependent(attn_step_kernel<T, 4, 512>, grid, dim3(512), 0, st, a)
                     : launch_dependent(attn_step_kernel<T, 4, 128>, grid, dim3(128), 0, st, a);
    };
    const cudaError_t e = p->dtype == DCN_SEQ_F32    ? go((float*)nullptr)
                          : p->dtype == DCN_SEQ_BF16 ? go((__nv_bfloat16*)nullptr)
                                                     : go((__half*)nullptr);
    return e == cudaSuccess ? DCN_OK : DCN_ERR_CUDA;
}
