// Decayed attention on the fifth-generation tensor cores, 16-bit types: see seq_attn.cu, which this file is a part of, for the
// mathematics.  Chunks are of 128 steps here:
//     scores = A B^T                  128 x 128                    (a's and b's rows as they lie)
//     P      = scores, weighted by g^(i-j) and cut above the diagonal, as 16-bit operand in tensor memory
//     O1     = A X,  O2 = P C         128 x 64                     out = scale (g^(i+1) O1 + O2)
//     U      = B^T C', C'_j = g^(127-j) c_j                        X'  = g^128 X + U
// C' is the sum of three bfloat16 (two float16) tiles, so that the products of the state are those of float32; X is in the registers of
// four warps in float32, and meets A as a rounded copy in shared memory.
//
// A CTA has one job's head (or a part of its time axis) and 64 columns of c: two such tiles of a chunk and a copy ahead fill shared
// memory.  Four warps load (cp.async, two chunks), four make P and the output, four make C' and the state, one thread issues the products.
// The loop that bounds the chain is C' -> U -> X -> O1; everything else runs beside it.
namespace tcgen {

constexpr int kSteps = 128, kDv = 64, kThreads = 13 * 32;
constexpr uint32_t kTmScores = 0, kTmO1 = 128, kTmO2 = 192, kTmU = 256, kTmP = 320;      // columns of tensor memory

template <typename T, int KA>
struct Room {
    static constexpr int kParts = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
    static constexpr int kHalf = kSteps * 128;                   // bytes of a tile of 64 columns
    static constexpr int kA = KA / 64 * kHalf, kStage = 2 * kA + kHalf;
    static constexpr int kWeighted = 2 * kStage, kState = kWeighted + kParts * kHalf, kControl = kState + KA * 128;
    static constexpr int kBytes = kControl + 2048 + 1024;        // (and what aligns it to 1024)
};

struct Control {
    uint64_t full[2], empty[2], scores_full, scores_empty, p_full, out_full, out_empty, c_full, u_full, x_full;
    uint32_t tmem;
    float up[2], most[4];
    float power[kSteps + 1];                     // g^n
    alignas(16) float back[32];                  // g^(31-n)
};

template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n, int a_mn_major, int b_mn_major) {
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// D (+)= A B with A in tensor memory
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
                 "l"(b_desc), "r"(id), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
        "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A tile's rows first, first + 1, ... of an operand, 64 columns to a half; zeros beyond the length and the width.  128 threads
template <int kCols_>
__device__ __forceinline__ void load_rows(uint32_t to, const Operand& o, const char* from, int64_t first, int64_t length, int col0, bool reverse,
                                          int tid) {
    constexpr int kChunks = kCols_ / 8, kRows = 128 / kChunks;   // of 16 bytes in a row; rows at a time (a multiple of 8)
    const int c = tid % kChunks, r0 = tid / kChunks, left = (o.width - col0 - c * 8) * 2, bytes = left <= 0 ? 0 : left >= 16 ? 16 : left;
    const int64_t t0 = reverse ? length - 1 - first - r0 : first + r0, step = (reverse ? -kRows : kRows) * o.s.step * 2;
    const char* src = from + (t0 * o.s.step + col0 + c * 8) * 2;
    uint32_t dst = to + (c >> 3) * (kSteps * 128) + tc::swz_offset(r0, c & 7);
    const int rows = (int)min((int64_t)kSteps, length - first) - r0;             // row r0 + p * kRows is there while p * kRows < rows
#pragma unroll
    for (int p = 0; p < kSteps / kRows; ++p) {
        const bool in = p * kRows < rows && bytes > 0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(in ? src : from), "r"(in ? bytes : 0) : "memory");
        src += step, dst += kRows * 128;
    }
}

// kEnds: the sums of each part's b_j c_j^T alone
template <typename T, int KA, bool kEnds>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const AttnArgs args) {
    using R = Room<T, KA>;
    extern __shared__ char raw[];
    char* const smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = tc::smem_u32(smem);
    Control& ctl = *reinterpret_cast<Control*>(smem + R::kControl);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    int u = blockIdx.x;
    const int tile = u % args.tiles;
    u /= args.tiles;
    const int which = u % args.jobs;
    const int unit = u / args.jobs, h = unit % args.heads, b = unit / args.heads;
    const Job& job = args.job[which];
    if (tile >= args.tile_of[which]) return;
    const int col0 = tile * kDv, part = blockIdx.y;

    if (warp == 12) {
        tc::tmem_alloc(&ctl.tmem, 512);
        tc::tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) tc::mbar_init(&ctl.full[s], 4), tc::mbar_init(&ctl.empty[s], 1 + 4);
        tc::mbar_init(&ctl.scores_full, 1), tc::mbar_init(&ctl.scores_empty, 4), tc::mbar_init(&ctl.p_full, 4);
        tc::mbar_init(&ctl.out_full, 1), tc::mbar_init(&ctl.out_empty, 4);
        tc::mbar_init(&ctl.c_full, 4), tc::mbar_init(&ctl.u_full, 1), tc::mbar_init(&ctl.x_full, 4);
        tc::fence_barrier_init();
    }
    pdl_wait();
    if (threadIdx.x <= kSteps) {
        float g;
        asm volatile("ld.global.f32 %0, [%1];" : "=f"(g) : "l"(args.log_decay + h));
        g = g > 0.0f ? 0.0f : g;
        const int n = threadIdx.x;
        const float w = n == 0 ? (g != g ? g : 1.0f) : (float)exp((double)n * (double)g);
        ctl.power[n] = w;
        if (n < 32) ctl.back[31 - n] = w;
    }
    const int64_t steps = args.steps;
    int64_t length = steps;
    if (args.lengths != nullptr) length = min(max(gload_i64(args.lengths + b), (int64_t)0), steps);
    const int64_t begin = (int64_t)part * args.part_steps, stop = min(begin + args.part_steps, steps);
    const int64_t finish = min(stop, length);
    const int chunks = finish > begin ? (int)((finish - begin + kSteps - 1) / kSteps) : 0;
    const bool reverse = job.reverse != 0;
    const int extra = reverse ? 0 : 1, wa = job.a.width, wc = job.c.width;
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = ctl.tmem;
    const int64_t parts_of = ((int64_t)which * args.batch * args.heads + unit) * args.n_parts;

    if (warp < 4) {
        // ---- loads
        const char* const from_a = static_cast<const char*>(job.a.p) + (b * job.a.s.batch + h / job.a.share * job.a.s.head) * 2;
        const char* const from_b = static_cast<const char*>(job.b.p) + (b * job.b.s.batch + h / job.b.share * job.b.s.head) * 2;
        const char* const from_c = static_cast<const char*>(job.c.p) + (b * job.c.s.batch + h / job.c.share * job.c.s.head) * 2;
        auto issue = [&](int n) {
            const uint32_t to = base + (n & 1) * R::kStage;
            const int64_t first = begin + (int64_t)n * kSteps;
            if constexpr (!kEnds) load_rows<KA>(to, job.a, from_a, first, length, 0, reverse, threadIdx.x);
            load_rows<KA>(to + R::kA, job.b, from_b, first, length, 0, reverse, threadIdx.x);
            load_rows<kDv>(to + 2 * R::kA, job.c, from_c, first, length, col0, reverse, threadIdx.x);
            copies_issued();
        };
        auto arrived = [&](int n) {
            tc::fence_proxy_async_smem();
            tc::mbar_arrive_warp(&ctl.full[n & 1]);
        };
        for (int n = 0; n < chunks; ++n) {
            if (n >= 2 && !tc::mbar_wait(&ctl.empty[n & 1], ((n >> 1) & 1) ^ 1)) break;
            issue(n);
            if (n == 0 && chunks > 1) continue;
            if (n == 1) {
                copies_arrived<1>();
                arrived(0);
            }
            copies_arrived<0>();
            arrived(n);
        }
    } else if (warp < 8) {
        // ---- scores to weights, and the output
        if constexpr (!kEnds) {
            const int w = warp & 3, i = w * 32 + lane;
            const uint32_t rows_at = tmem + ((uint32_t)(w * 32) << 16);
            bool ok = true;
            const float near = ctl.power[lane + 1];
            for (int n = 0; n < chunks; ++n) {
                ok = tc::mbar_wait(&ctl.scores_full, n & 1);
                if (!ok) break;
                __syncwarp();
                tc::tc_fence_after();
#pragma unroll 1
                for (int cb = 0; cb < 4; ++cb) {
                    uint32_t packed[16];
                    if (cb > w) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) packed[k] = 0;
                    } else {
                        uint32_t v[32];
                        tc::tmem_ld32(rows_at + kTmScores + cb * 32, v);
                        tc::tmem_ld_wait();
                        if (cb == w) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const int d = lane - 2 * k;      // steps back
                                const float x = d >= 0 ? __uint_as_float(v[2 * k]) * ctl.power[max(d, 0)] : 0.0f;
                                const float y = d >= 1 ? __uint_as_float(v[2 * k + 1]) * ctl.power[max(d - 1, 0)] : 0.0f;
                                packed[k] = word_of<T>(x, y);
                            }
                        } else {
                            const Lanes f = all_lanes(near * ctl.power[32 * (w - cb - 1)]);
#pragma unroll
                            for (int k = 0; k < 16; k += 2) {
                                const float4 c = *reinterpret_cast<const float4*>(&ctl.back[2 * k]);
                                const float c0[2] = {c.x, c.y}, c1[2] = {c.z, c.w};
                                const float x0[2] = {__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])};
                                const float x1[2] = {__uint_as_float(v[2 * k + 2]), __uint_as_float(v[2 * k + 3])};
                                const Lanes p = lanes(x0) * (f * lanes(c0)), q = lanes(x1) * (f * lanes(c1));
                                packed[k] = word_of<T>(p.at(0), p.at(1)), packed[k + 1] = word_of<T>(q.at(0), q.at(1));
                            }
                        }
                    }
                    tmem_st16(rows_at + kTmP + cb * 16, packed);
                }
                tmem_st_wait();
                tc::tc_fence_before();
                tc::mbar_arrive_warp(&ctl.scores_empty);
                tc::mbar_arrive_warp(&ctl.p_full);
                ok = tc::mbar_wait(&ctl.out_full, n & 1);
                if (!ok) break;
                __syncwarp();
                tc::tc_fence_after();
                const int64_t pos = begin + (int64_t)n * kSteps + i;
                const float w1 = ctl.power[i + extra] * ctl.up[n & 1];
                const Lanes f1 = all_lanes(w1 * args.scale), f2 = all_lanes(args.scale);
                const int64_t step = reverse ? length - 1 - pos : pos, at = (((int64_t)b * steps + step) * args.heads + h) * wc + col0;
#pragma unroll 1
                for (int cb = 0; cb < 2; ++cb) {
                    uint32_t p[32], q[32];
                    tc::tmem_ld32(rows_at + kTmO1 + cb * 32, p);
                    tc::tmem_ld32(rows_at + kTmO2 + cb * 32, q);
                    tc::tmem_ld_wait();
                    if (cb == 1) {
                        tc::tc_fence_before();
                        tc::mbar_arrive_warp(&ctl.out_empty);
                    }
                    if (pos < finish) {
                    float o[32];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        const float a[2] = {__uint_as_float(p[k]), __uint_as_float(p[k + 1])}, c[2] = {__uint_as_float(q[k]), __uint_as_float(q[k + 1])};
                        const Lanes r = fma(lanes(a), f1, lanes(c) * f2);
                        o[k] = r.at(0), o[k + 1] = r.at(1);
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {            // (widths are multiples of 8)
                        if (col0 + cb * 32 + k >= wc) continue;
                        if (job.wide) {
                            float4* const d = reinterpret_cast<float4*>(static_cast<float*>(job.out) + at + cb * 32 + k);
                            d[0] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]), d[1] = make_float4(o[k + 4], o[k + 5], o[k + 6], o[k + 7]);
                        } else {
                            store(static_cast<T*>(job.out) + at + cb * 32 + k,
                                  Raw<16>{{word_of<T>(o[k], o[k + 1]), word_of<T>(o[k + 2], o[k + 3]), word_of<T>(o[k + 4], o[k + 5]),
                                           word_of<T>(o[k + 6], o[k + 7])}});
                        }
                    }
                    }
                    __syncwarp();
                }
            }
            // zeros behind the length
            const int64_t from = max(begin, length);
            const int cols = min(kDv, wc - col0) / 8;
            for (int64_t k = threadIdx.x - 128; k < (stop - from) * cols; k += 128) {
                const int64_t at = (((int64_t)b * steps + from + k / cols) * args.heads + h) * wc + col0 + k % cols * 8;
                if (job.wide) {
                    float4* const d = reinterpret_cast<float4*>(static_cast<float*>(job.out) + at);
                    d[0] = d[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                } else {
                    store(static_cast<T*>(job.out) + at, Raw<16>{{0, 0, 0, 0}});
                }
            }
        }
    } else if (warp < 12) {
        // ---- the weighted c, and the state
        const int tid = threadIdx.x - 256, w = warp & 3, i = w * 32 + lane;
        const uint32_t rows_at = tmem + ((uint32_t)(w * 32) << 16) + kTmU;
        const bool mine = i < KA;                // (the products have 128 rows: behind a's 64 columns they find those of c)
        float x[kDv];
        {
            const float* const init = !kEnds && job.init != nullptr ? job.init + (int64_t)unit * wa * wc + (int64_t)i * job.init_i + (int64_t)col0 * job.init_j : nullptr;
#pragma unroll
            for (int k = 0; k < kDv; ++k) x[k] = init != nullptr && i < wa && col0 + k < wc ? job.init_scale * gload(init + (int64_t)k * job.init_j) : 0.0f;
        }
        if constexpr (!kEnds) {
            if (part > 0 && begin < length && i < wa) {
                float g;
                asm volatile("ld.global.f32 %0, [%1];" : "=f"(g) : "l"(args.log_decay + h));
                const float whole = (float)exp((double)args.part_steps * (double)(g > 0.0f ? 0.0f : g));
                for (int s = 0; s < part; ++s) {
                    const float* const sums = args.parts + (parts_of + s) * wa * wc + (int64_t)i * wc + col0;
#pragma unroll
                    for (int k = 0; k < kDv; k += 4)
                        if (col0 + k < wc) {
                            Pack<float, 4> p;
                            p.get(sums + k);
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[k + e] = fmaf(x[k + e], whole, p.at(e));
                        }
                }
            }
        }
        auto put_copy = [&](int n) {             // the state before chunk n
            float down = 1.0f;
            if constexpr (std::is_same<T, __half>::value) {
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < kDv; ++k) most = fmaxf(most, mine ? fabsf(x[k]) : 0.0f);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (lane == 0) ctl.most[w] = most;
                asm volatile("bar.sync 1, 128;" ::: "memory");
                most = fmaxf(fmaxf(ctl.most[0], ctl.most[1]), fmaxf(ctl.most[2], ctl.most[3]));
                asm volatile("bar.sync 1, 128;" ::: "memory");
                const int over = min(max((int)(__float_as_uint(most) >> 23) - 127 - 14, 0), 126);
                down = __uint_as_float((uint32_t)(127 - over) << 23);
                if (tid == 0) ctl.up[n & 1] = __uint_as_float((uint32_t)(127 + over) << 23);
            } else {
                if (tid == 0) ctl.up[n & 1] = 1.0f;
            }
            if (mine) {
                const uint32_t row = base + R::kState;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float* const v = x + 8 * c;
                    tc::st_shared_v4(row + tc::swz_offset(i, c), word_of<T>(v[0] * down, v[1] * down), word_of<T>(v[2] * down, v[3] * down),
                                     word_of<T>(v[4] * down, v[5] * down), word_of<T>(v[6] * down, v[7] * down));
                }
            }
            tc::fence_proxy_async_smem();
            tc::mbar_arrive_warp(&ctl.x_full);
        };
        const int c = tid & 7, r0 = tid >> 3;    // of the tile of c: 16 bytes of rows r0, r0 + 16, ...
        const uint32_t place = tc::swz_offset(r0, c);
        bool ok = true;
        for (int n = 0; n < chunks; ++n) {
            if constexpr (!kEnds) put_copy(n);
            ok = tc::mbar_wait(&ctl.full[n & 1], (n >> 1) & 1);
            if (!ok) break;
            const int rows = (int)min((int64_t)kSteps, finish - begin - (int64_t)n * kSteps), top = rows - extra;
            const uint32_t from = base + (n & 1) * R::kStage + 2 * R::kA + place, to = base + R::kWeighted + place;
#pragma unroll 2
            for (int p = 0; p < 8; ++p) {
                const int j = r0 + 16 * p;
                const float weight = j < rows ? ctl.power[top - j] : 0.0f;
                const Lanes f = all_lanes(weight);
                const uint4 v = tc::lds128(from + p * 2048);
                const uint32_t in[4] = {v.x, v.y, v.z, v.w};
                uint32_t out[R::kParts][4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float e[2] = {half_of<T>(in[k], 0), half_of<T>(in[k], 1)};
                    Lanes r = lanes(e) * f;
#pragma unroll
                    for (int q = 0; q < R::kParts; ++q) {
                        out[q][k] = word_of<T>(r.at(0), r.at(1));
                        if (q + 1 < R::kParts) {
                            const float t[2] = {half_of<T>(out[q][k], 0), half_of<T>(out[q][k], 1)};
                            r = r - lanes(t);
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < R::kParts; ++q)
                    tc::st_shared_v4(to + q * R::kHalf + p * 2048, out[q][0], out[q][1], out[q][2], out[q][3]);
            }
            tc::fence_proxy_async_smem();
            tc::tc_fence_before();               // (U of the chunk before has been read)
            tc::mbar_arrive_warp(&ctl.c_full);
            tc::mbar_arrive_warp(&ctl.empty[n & 1]);
            ok = tc::mbar_wait(&ctl.u_full, n & 1);
            if (!ok) break;
            __syncwarp();
            tc::tc_fence_after();
            const Lanes whole = all_lanes(ctl.power[rows]);
#pragma unroll
            for (int cb = 0; cb < 2; ++cb) {
                uint32_t v[32];
                tc::tmem_ld32(rows_at + cb * 32, v);
                tc::tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float a[2] = {x[cb * 32 + k], x[cb * 32 + k + 1]}, e[2] = {__uint_as_float(v[k]), __uint_as_float(v[k + 1])};
                    const Lanes r = fma(lanes(a), whole, lanes(e));
                    x[cb * 32 + k] = r.at(0), x[cb * 32 + k + 1] = r.at(1);
                }
            }
        }
        const bool ends_here = kEnds || (length > begin && length <= begin + args.part_steps) || (length == 0 && part == 0);
        float* const to = kEnds ? args.parts + (parts_of + part) * wa * wc : job.end != nullptr ? job.end + (int64_t)unit * wa * wc : nullptr;
        if (ok && ends_here && to != nullptr && mine && i < wa) {
            const float by = kEnds ? 1.0f : job.end_scale;
#pragma unroll
            for (int k = 0; k < kDv; k += 4)
                if (col0 + k < wc)
                    *reinterpret_cast<float4*>(to + (int64_t)i * wc + col0 + k) = make_float4(by * x[k], by * x[k + 1], by * x[k + 2], by * x[k + 3]);
        }
    } else if (lane == 0) {
        // ---- products
        bool ok = true;
        for (int n = 0; n < chunks && ok; ++n) {
            const int s = n & 1;
            const uint32_t a = base + s * R::kStage, bt = a + R::kA, ct = a + 2 * R::kA;
            ok = tc::mbar_wait(&ctl.full[s], (n >> 1) & 1);
            if (!ok) break;
            if constexpr (!kEnds) {
                ok = n == 0 || tc::mbar_wait(&ctl.scores_empty, (n - 1) & 1);
                if (!ok) break;
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < KA / 16; ++k) {
                    const uint32_t off = (k >> 2) * R::kHalf + (k & 3) * 32;
                    tc::umma_bf16(tmem + kTmScores, tc::make_desc(a + off, 16, 1024), tc::make_desc(bt + off, 16, 1024), idesc<T>(128, 128, 0, 0), k > 0);
                }
                tc::umma_commit(&ctl.scores_full);
                ok = tc::mbar_wait(&ctl.x_full, n & 1) && (n == 0 || tc::mbar_wait(&ctl.out_empty, (n - 1) & 1));
                if (!ok) break;
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < KA / 16; ++k) {
                    const uint32_t off = (k >> 2) * R::kHalf + (k & 3) * 32;
                    tc::umma_bf16(tmem + kTmO1, tc::make_desc(a + off, 16, 1024), tc::make_desc(base + R::kState + k * 2048, R::kHalf, 1024),
                                  idesc<T>(128, kDv, 0, 1), k > 0);
                }
            }
            ok = tc::mbar_wait(&ctl.c_full, n & 1);
            if (!ok) break;
            tc::tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < R::kParts; ++q)
#pragma unroll
                for (int k = 0; k < kSteps / 16; ++k)
                    tc::umma_bf16(tmem + kTmU, tc::make_desc(bt + k * 2048, R::kHalf, 1024),
                                  tc::make_desc(base + R::kWeighted + q * R::kHalf + k * 2048, R::kHalf, 1024), idesc<T>(128, kDv, 1, 1), q + k > 0);
            tc::umma_commit(&ctl.u_full);
            if constexpr (!kEnds) {
                ok = tc::mbar_wait(&ctl.p_full, n & 1);
                if (!ok) break;
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < kSteps / 16; ++k)
                    umma_ts(tmem + kTmO2, tmem + kTmP + k * 8, tc::make_desc(ct + k * 2048, R::kHalf, 1024), idesc<T>(128, kDv, 0, 1), k > 0);
                tc::umma_commit(&ctl.out_full);
            }
            tc::umma_commit(&ctl.empty[s]);
        }
        if (ok && chunks > 0) tc::mbar_wait(&ctl.empty[(chunks - 1) & 1], ((chunks - 1) >> 1) & 1);       // nothing is under way at the end
    }

    pdl_trigger();
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

}  // namespace tcgen
