// Decayed attention on the fifth-generation tensor cores, 16-bit types: see seq_attn.cu, which this file is a part of, for the
// mathematics.  Chunks are of 128 steps here:
//     scores = A B^T                  128 x 128                    (a's and b's rows as they lie)
//     P      = scores, weighted by g^(i-j) and cut above the diagonal, as 16-bit operand in tensor memory
//     O1     = A X,  O2 = P C         128 x 64                     out = scale (g^(i+1) O1 + O2)
//     U      = B^T C', C'_j = g^(127-j) c_j                        X'  = g^128 X + U
// C' is a sum of 16-bit tiles, so many that what the state is made of is exact to 2^-17 (two of bfloat16) where it only meets A, and to
// float32's own 2^-24 (three) where it is a result, in its last 1.5 decays; two of float16, brought up by a power of two that c's largest
// element gives, are exact to 2^-22, or 2^-40 of that element where this is more.  X is in the registers of four warps in float32, and meets A
// as a copy in shared memory that is rounded to the type, as P is: the products take both operands in one type, tensor memory (P) and shared
// memory (X) are full, and a second 16-bit part of either would double O1 or O2.  It makes a 16-bit result's error 1.4 times that of its own
// rounding (2.3e-3 and 1.7e-3 of bfloat16's norm).
//
// A CTA has one job's head (or a part of its time axis) and 64 columns of c: two chunks' tiles (three of up to 64 columns), C' and X fill
// shared memory.  One warp loads (TMA), three issue products (scores; O1 and O2; U), each as soon as its own operands are there, four
// make P, four the output, four C' (half a chunk ahead of its product), four keep the state: 20 warps.
//
// Rows of a tile are steps in the order of time.  Back in time, position i of a chunk is row 127 - i, and triangle and weights are mirrored.
//
// Float16 pays for its powers of two, of c's and X's largest elements in each chunk, with 920 us where 780 were without them, 310 and 268
// forward (2x16384x16x128): a tile of c comes when C' waits for it, and the state's copy is in the chain from chunk to chunk.  (C''s own warps look
// for c's largest: two other roles that did it a chunk ahead took 1100.  Leaving infinities out of the maxima cost 60.)
//
// 2x16384x16x128 bf16 with its gradients takes 750 us (850 over seconds of it; its bytes alone 168, its products, some 450 GFLOP, 270).  A chunk takes about 2.5 us:
// products some 1.2 us at the measured rate, the rest is the chain scores - P - O2 with its two ways through tensor memory, which one CTA an SM (shared
// memory) overlaps with the next chunk's scores only, and shared memory's bandwidth, of which operands, C' and X take about half.  What
// moved it most: code of the roles in short loops instead of unrolled (1356 to 1168 us: together they did not stay in the instruction
// caches), products issued by one lane of a converged warp with descriptors in uniform registers (957 to 886), tables read by shared
// addresses (886 to 834), and the split of a part of the units alone (834 to 764).
namespace tcgen {

constexpr int kSteps = 128, kDv = 64, kThreads = 20 * 32;
constexpr uint32_t kTmScores = 0, kTmU = 128, kTmP = 192, kTmO1 = 256, kTmO2 = 320, kTmTurn = 128;  // columns of tensor memory; O1 and O2 twice

template <typename T, int KA>
struct Room {
    static constexpr int kParts = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
    static constexpr int kHalf = kSteps * 128;                   // bytes of a tile of 64 columns
    static constexpr int kA = KA / 64 * kHalf, kStage = 2 * kA + kHalf, kStages = KA == 64 ? 3 : 2;
    static constexpr int kWeighted = kStages * kStage, kState = kWeighted + kParts * kHalf, kControl = kState + KA * 128;
    static constexpr int kBytes = kControl + 2048 + 1024;        // (and what aligns it to 1024)
};

struct Control {
    uint64_t full[3], full_c[3], empty[3], zeroed, scores_full, scores_empty, p_full, p_empty, out_full[2], out_empty[2], c_full[2], c_empty[2], u_full, u_empty,
        x_full, x_empty;
    Carried carried;
    uint32_t tmem;
    float whole[8];                              // g^128 of a chunk's turn, by the warp that loads, which is four ahead of the state at most
    float up[4];                                 // the state's copy, back to its size
    uint32_t most[2][4];
    uint32_t c_most[2][4];
    float c_back[2];                             // C', back to its size
    int8_t score_shift[4][kSteps];               // rows of P are times 2^this; kept until the output has left its chunk, which P is two ahead of at most
    float power[kSteps + 1];                     // g^n
    float diagonal[64];                          // [32 + row - column]: weights of 32 x 32 scores on the diagonal, 0 behind it
    alignas(16) float across[32];                // [column]: those of a row in front of such a block, from its last column but one on
};

// Bounded wait: gives up after tc::kWaitCycles, raises the status word and returns false
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
    const uint32_t at = tc::smem_u32(bar);
    const long long t0 = clock64();
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i) {
            uint32_t done;
            asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.b32 %0, 1, 0, p;\n}"
                         : "=r"(done) : "r"(at), "r"(parity) : "memory");
            if (done) return true;
        }
        if (clock64() - t0 > tc::kWaitCycles) {
            atomicOr(&tc::g_tc_status, 1u);
            return false;
        }
    }
}

// The larger magnitude
__device__ __forceinline__ float larger(float most, Lanes y) { return fmaxf(fmaxf(most, fabsf(y.at(0))), fabsf(y.at(1))); }

// From a table in shared memory that does not change any more, by its shared address (through a generic one the 32 loads of a block
// of scores took 600 cycles)
__device__ __forceinline__ float table(uint32_t at) {
    float f;
    asm("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(at));
    return f;
}

template <typename T>
__host__ __device__ constexpr uint32_t idesc(int m, int n, int a_mn_major, int b_mn_major) {
    const uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(m >> 4) << 24);
}

// Products and their commits are issued by one lane of a warp that runs as one, so that descriptors are in uniform registers
__device__ __forceinline__ uint32_t elected() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(yes));
    return yes;
}
// D (+)= A B of tiles in shared memory
__device__ __forceinline__ void umma(uint32_t yes, uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate), "r"(yes)
        : "memory");
}
// ... with A in tensor memory
__device__ __forceinline__ void umma_ts(uint32_t yes, uint32_t d, uint32_t a, uint64_t b_desc, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(b_desc), "r"(id), "r"(accumulate), "r"(yes)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t yes, uint64_t* bar) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(tc::smem_u32(bar)),
        "r"(yes)
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

// The operands as [batch][steps][heads][width], boxes of 64 elements of 128 steps
struct alignas(64) Maps {
    CUtensorMap of[4];
};

// 128 rows of 64 elements from `col`, row 0 at time t (zeros outside of the tensor, before time 0 too)
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap& map, int col, int head, int t, int batch, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to),
                 "l"(reinterpret_cast<uint64_t>(&map)), "r"(col), "r"(head), "r"(t), "r"(batch), "r"(tc::smem_u32(bar))
                 : "memory");
}

static_assert(sizeof(Control) <= 2048, "the control block's place in shared memory");

// kEnds: the sums of each part's b_j c_j^T alone
template <typename T, int KA, bool kEnds>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const AttnArgs args, const __grid_constant__ Maps maps) {
    using R = Room<T, KA>;
    extern __shared__ char raw[];
    char* const smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t base = tc::smem_u32(smem);
    Control& ctl = *reinterpret_cast<Control*>(smem + R::kControl);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const Place place = Place::of<kEnds>(args);
    const int tile = place.tile, which = place.which, unit = place.unit, h = unit % args.heads, b = unit / args.heads;
    const Job& job = args.job[which];
    if (tile >= args.tile_of[which]) return;
    const int col0 = tile * kDv, part = place.part;

    if (warp == 3) {
        tc::tmem_alloc(&ctl.tmem, 512);
        tc::tmem_relinquish();
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < R::kStages; ++s) tc::mbar_init(&ctl.full[s], 1), tc::mbar_init(&ctl.full_c[s], 1), tc::mbar_init(&ctl.empty[s], 1 + 4 + (kEnds ? 0 : 2));
        for (int s = 0; s < 2; ++s) tc::mbar_init(&ctl.c_full[s], 4), tc::mbar_init(&ctl.c_empty[s], 1), tc::mbar_init(&ctl.out_full[s], 1), tc::mbar_init(&ctl.out_empty[s], 4);
        tc::mbar_init(&ctl.zeroed, 4);
        tc::mbar_init(&ctl.scores_full, 1), tc::mbar_init(&ctl.scores_empty, 4), tc::mbar_init(&ctl.p_full, 4);
        tc::mbar_init(&ctl.p_empty, 1);
        tc::mbar_init(&ctl.u_full, 1), tc::mbar_init(&ctl.u_empty, 4), tc::mbar_init(&ctl.x_full, 4), tc::mbar_init(&ctl.x_empty, 1);
        tc::fence_barrier_init();
    }
    pdl_wait();
    float log_decay;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(log_decay) : "l"(args.log_decay + h));
    log_decay = log_decay > 0.0f ? 0.0f : log_decay;
    if (threadIdx.x <= kSteps) {
        const int n = threadIdx.x;
        const float w = n == 0 ? (log_decay != log_decay ? log_decay : 1.0f) : (float)exp((double)n * (double)log_decay);
        ctl.power[n] = w;
        if (n == kSteps) ctl.carried.begin(log_decay, kSteps), ctl.whole[0] = ctl.carried.next();
        if (n < 32) {
            ctl.across[job.reverse ? n : 31 - n] = w;
            ctl.diagonal[job.reverse ? 32 - n : 32 + n] = w;
            if (n > 0) ctl.diagonal[job.reverse ? 32 + n : 32 - n] = 0.0f;
        }
    }
    const int steps = (int)args.steps, part_steps = (int)place.part_steps;       // (below 2^30)
    int length = steps;
    if (args.lengths != nullptr) length = (int)min(max(gload_i64(args.lengths + b), (int64_t)0), (int64_t)steps);
    const int begin = part * part_steps, finish = min(min(begin + part_steps, steps), length);
    const int chunks = finish > begin ? (finish - begin + kSteps - 1) / kSteps : 0;
    const bool ends_here = kEnds || (length > begin && length <= begin + part_steps) || (length == 0 && part == 0);
    const bool reverse = job.reverse != 0;
    const int extra = reverse ? 0 : 1, wa = job.a.width, wc = job.c.width, room = job.room;
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = ctl.tmem, power = tc::smem_u32(ctl.power);
    // Tiles that C' is the sum of: all where the state is a result and the chunk so near its end that two would be seen in it (those
    // before it count e^-1.5 and less), else two
    const auto parts_of_chunk = [&](int n) {
        const float after = (float)(length - begin - (n + 1) * kSteps);
        return job.end != nullptr && after * -log_decay < 1.5f ? R::kParts : 2;
    };

    // Behind a sequence's end, but inside the tensor, rows hold what they may: b's and c's of the last chunk are made zeros
    const int ragged = !reverse && length < steps && chunks > 0 && length < begin + chunks * kSteps ? chunks - 1 : -1;

    if (warp == 0) {
        // ---- loads
        if (lane == 0) {
            int n = 0;
            tc::Ring ring;
            for (; n < chunks; ++n, ring.next(R::kStages)) {
                uint64_t* const bar = &ctl.full[ring.i];
                if (n >= R::kStages && !wait(&ctl.empty[ring.i], ring.ph ^ 1)) break;
                const uint32_t to = base + ring.i * R::kStage;
                const int first = begin + n * kSteps, t = reverse ? length - kSteps - first : first;
                tc::mbar_arrive_expect_tx(bar, kEnds ? R::kA : 2 * R::kA);
#pragma unroll
                for (int k = 0; k < KA / 64; ++k) {
                    load_box(to + R::kA + k * R::kHalf, maps.of[job.b.map], 64 * k, h / job.b.share, t, b, bar);
                    if constexpr (!kEnds) load_box(to + k * R::kHalf, maps.of[job.a.map], 64 * k, h / job.a.share, t, b, bar);
                }
                tc::mbar_arrive_expect_tx(&ctl.full_c[ring.i], R::kHalf);
                load_box(to + 2 * R::kA, maps.of[job.c.map], col0, h / job.c.share, t, b, &ctl.full_c[ring.i]);
                ctl.whole[(n + 1) & 7] = ctl.carried.next();     // (there with the next chunk's tiles)
            }
            for (int k = max(n - R::kStages, 0); k < n; ++k)     // (nothing is under way at the end)
                wait(&ctl.full[k % R::kStages], k / R::kStages & 1), wait(&ctl.full_c[k % R::kStages], k / R::kStages & 1);
        }
    } else if (warp >= 4 && warp < 8) {
        // ---- scores to weights
        if constexpr (!kEnds) {
            const int w = warp & 3;
            const uint32_t rows_at = tmem + ((uint32_t)(w * 32) << 16), diagonal = tc::smem_u32(ctl.diagonal + 32 + lane);
            const float near = table(power + 4 * (reverse ? 32 - lane : lane + 1));
            int shift = 0;                       // float16: of this row, as the chunk before left it
            for (int n = 0; n < chunks; ++n) {
                if (!wait(&ctl.scores_full, n & 1) || (n > 0 && !wait(&ctl.p_empty, (n - 1) & 1))) break;
                __syncwarp();
                tc::tc_fence_after();
                // (short code in loops: the roles' instructions together would not stay in the caches that feed the schedulers)
                // Float16: a row is right when its largest weight lies in [2^-8, 2^15), so that those down to 2^-6 of it have their 11 bits and
                // smaller ones are off by 2^-17 of it; if not, it is brought to 2^6 and the warp's rows are made once more.  Rows at a place in
                // their chunk differ little from chunk to chunk, so that this is rare.
                for (bool again = false;; again = true) {
                    const float by = kNarrow<T> ? two_to(shift) : 1.0f;
                    float most = 0.0f;
#pragma unroll 1
                    for (int cb = 0; cb < 4; ++cb) {
                        const int back = reverse ? cb - w : w - cb;      // blocks of 32 steps back
                        if (back < 0 && n > 0) continue;                 // (zeros already)
                        uint32_t v[32];
                        if (back >= 0) {
                            tc::tmem_ld32(rows_at + kTmScores + cb * 32, v);
                            tc::tmem_ld_wait();
                        }
                        if (back > 0) {
                            const Lanes f = all_lanes(near * table(power + 128 * (back - 1)) * by);
#pragma unroll
                            for (int k = 0; k < 16; k += 2) {
                                Raw<16> c;
                                load_shared(c, ctl.across + 2 * k);
                                const float c0[2] = {__uint_as_float(c.u[0]), __uint_as_float(c.u[1])}, c1[2] = {__uint_as_float(c.u[2]), __uint_as_float(c.u[3])};
                                const float x0[2] = {__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])};
                                const float x1[2] = {__uint_as_float(v[2 * k + 2]), __uint_as_float(v[2 * k + 3])};
                                const Lanes y0 = lanes(x0) * (f * lanes(c0)), y1 = lanes(x1) * (f * lanes(c1));
                                if constexpr (kNarrow<T>) most = larger(larger(most, y0), y1);
                                v[k] = word_of<T>(y0.at(0), y0.at(1)), v[k + 1] = word_of<T>(y1.at(0), y1.at(1));
                            }
                        } else if (back == 0) {
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                const float x[2] = {__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])}, c[2] = {table(diagonal - 8 * k), table(diagonal - 8 * k - 4)};
                                Lanes y = lanes(x) * lanes(c);
                                if constexpr (kNarrow<T>) y = y * all_lanes(by), most = larger(most, y);
                                v[k] = word_of<T>(y.at(0), y.at(1));
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < 16; ++k) v[k] = 0;
                        }
                        tmem_st16(rows_at + kTmP + cb * 16, *reinterpret_cast<uint32_t(*)[16]>(v));
                    }
                    if constexpr (!kNarrow<T>) break;
                    const bool fits = most == 0.0f || most == CUDART_INF_F || (most >= 0.00390625f && most < 32768.0f);
                    if (again || __all_sync(0xffffffffu, fits)) break;
                    tmem_st_wait();              // (before the same places are written again)
                    if (!fits) shift = min(max(shift + 6 + 127 - (int)(__float_as_uint(most) >> 23), -60), 60);
                }
                if constexpr (kNarrow<T>) ctl.score_shift[n & 3][w * 32 + lane] = (int8_t)shift;
                tmem_st_wait();
                tc::tc_fence_before();
                tc::mbar_arrive_warp(&ctl.scores_empty);
                tc::mbar_arrive_warp(&ctl.p_full);
            }
        }
    } else if (warp >= 8 && warp < 12) {
        // ---- the output
        if constexpr (!kEnds) {
            const bool wide = job.wide != 0;
            char* const out = static_cast<char*>(job.out);
            const int w = warp & 3, r = w * 32 + lane, i = reverse ? kSteps - 1 - r : r;     // the row, and its position
            const uint32_t rows_at = tmem + ((uint32_t)(w * 32) << 16);
            const float scale = args.scale, weight = table(power + 4 * (i + extra)) * scale;
            const int64_t row_bytes = (int64_t)args.heads * room * (wide ? 4 : 2);
            char* const first_row = out + (((int64_t)b * steps * args.heads + h) * room + col0) * (wide ? 4 : 2);
            for (int n = 0; n < chunks; ++n) {
                if (!wait(&ctl.out_full[n & 1], (n >> 1) & 1)) break;
                __syncwarp();
                tc::tc_fence_after();
                const float w1 = weight * ctl.up[n & 3], w2 = kNarrow<T> ? scale * two_to(-ctl.score_shift[n & 3][r]) : scale;
                const bool in = i < finish - begin - n * kSteps;
                const int t = reverse ? length - kSteps - begin - n * kSteps + r : begin + n * kSteps + r;
                char* to = first_row + t * row_bytes;
#pragma unroll 1
                for (int cb = 0; cb < 4; ++cb) {
                    uint32_t p[16], q[16];
                    tc::tmem_ld16(rows_at + kTmO1 + (n & 1) * kTmTurn + cb * 16, p);
                    tc::tmem_ld16(rows_at + kTmO2 + (n & 1) * kTmTurn + cb * 16, q);
                    tc::tmem_ld_wait();
                    if (cb == 3) {
                        tc::tc_fence_before();
                        tc::mbar_arrive_warp(&ctl.out_empty[n & 1]);
                    }
                    float o[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[k] = fmaf(__uint_as_float(p[k]), w1, __uint_as_float(q[k]) * w2);
                    if (in && col0 + cb * 16 < room) {           // (a multiple of 8)
                        const bool both = col0 + cb * 16 + 8 < room;
                        if (wide) {
#pragma unroll
                            for (int k = 0; k < 16; k += 4)
                                if (k < 8 || both) *reinterpret_cast<float4*>(to + k * 4) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                        } else {
                            uint32_t v[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] = word_of<T>(o[2 * k], o[2 * k + 1]);
                            if (job.sectors) {                   // whole sectors of 32 bytes
                                asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                                             "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                                             : "memory");
                            } else {
                                store(to, Raw<16>{{v[0], v[1], v[2], v[3]}});
                                if (both) store(to + 16, Raw<16>{{v[4], v[5], v[6], v[7]}});
                            }
                        }
                    }
                    to += wide ? 64 : 32;
                    __syncwarp();
                }
            }
            // zeros behind the length
            const int from = max(begin, length), cols = min(kDv, room - col0) / 8;
            for (int64_t k = threadIdx.x - 256; k < (int64_t)(min(begin + part_steps, steps) - from) * cols; k += 128) {
                const int64_t at = (((int64_t)b * steps + from + k / cols) * args.heads + h) * room + col0 + k % cols * 8;
                if (job.wide) {
                    float4* const d = reinterpret_cast<float4*>(static_cast<float*>(job.out) + at);
                    d[0] = d[1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                } else {
                    store(static_cast<T*>(job.out) + at, Raw<16>{{0, 0, 0, 0}});
                }
            }
        }
    } else if (warp >= 12 && warp < 16) {
        // ---- the weighted c, half a chunk at a time
        const int tid = threadIdx.x - 384, c = tid & 7, r0 = tid >> 3;           // 16 bytes of rows r0, r0 + 16, ...
        const uint32_t spot = tc::swz_offset(r0, c);
        bool ok = true;
        tc::Ring ring;
        // (a warp that gives up goes on to the others' barriers: these have no limit)
        for (int n = 0; n < chunks; ++n, ring.next(R::kStages)) {
            ok = ok && wait(&ctl.full_c[ring.i], ring.ph);
            const int rows = min(kSteps, finish - begin - n * kSteps), top = rows - extra, parts = parts_of_chunk(n);
            if (n == ragged) {
                ok = ok && wait(&ctl.full[ring.i], ring.ph);
                const uint32_t tile = base + ring.i * R::kStage + R::kA;        // b's halves, and c's behind them
                for (int k = tid; ok && k < (KA / 64 + 1) * (kSteps - rows) * 8; k += 128)
                    tc::st_shared_v4(tile + k / ((kSteps - rows) * 8) * R::kHalf + tc::swz_offset(rows + k / 8 % (kSteps - rows), k % 8), 0, 0, 0, 0);
                tc::fence_proxy_async_smem();
                if (ok) tc::mbar_arrive_warp(&ctl.zeroed);
                asm volatile("bar.sync 2, 128;" ::: "memory");
            }
            float by = 1.0f, back = 1.0f;
            if constexpr (kNarrow<T>) {
                // the tile's largest
                uint32_t m[4] = {};              // (chains of their own)
#pragma unroll
                for (int p = 0; p < 8; ++p) {
                    const uint4 v = tc::lds128(base + ring.i * R::kStage + 2 * R::kA + spot + p * 2048);
                    m[0] = larger_pairs(m[0], v.x), m[1] = larger_pairs(m[1], v.y), m[2] = larger_pairs(m[2], v.z), m[3] = larger_pairs(m[3], v.w);
                }
                uint32_t most = larger_pairs(larger_pairs(m[0], m[1]), larger_pairs(m[2], m[3]));
                most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
                if ((tid & 31) == 0) ctl.c_most[n & 1][warp & 3] = most;
                asm volatile("bar.sync 2, 128;" ::: "memory");
#pragma unroll
                for (int k = 0; k < 4; ++k) most = max(most, ctl.c_most[n & 1][k]);
                const int shift = shift_up(most, table(power + 4 * (1 - extra)));
                by = two_to(shift), back = two_to(-shift);
            }
            for (int half = 0; half < 2 && ok; ++half) {
                ok = n == 0 || wait(&ctl.c_empty[half], (n - 1) & 1);
                if (!ok) break;
                // (behind the wait: the state has taken the chunk before the last)
                if (kNarrow<T> && half == 0 && tid == 0) ctl.c_back[n & 1] = back;
                const uint32_t from = base + ring.i * R::kStage + 2 * R::kA + spot + half * 8192, to = base + R::kWeighted + spot + half * 8192;
#pragma unroll 1
                for (int p = 0; p < 4; ++p) {
                    const int row = r0 + 16 * p + 64 * half, j = reverse ? kSteps - 1 - row : row;
                    const Lanes f = all_lanes(j < rows ? table(power + 4 * max(top - j, 0)) * by : 0.0f);
                    const uint4 v = tc::lds128(from + p * 2048);
                    const uint32_t in[4] = {v.x, v.y, v.z, v.w};
                    uint32_t out[R::kParts][4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float e[2] = {half_of<T>(in[k], 0), half_of<T>(in[k], 1)};
                        Lanes r = lanes(e) * f;
#pragma unroll
                        for (int q = 0; q < R::kParts; ++q) {
                            if (q == 2 && parts <= 2) break;
                            out[q][k] = word_of<T>(r.at(0), r.at(1));
                            if (q + 1 < R::kParts) {
                                const float t[2] = {half_of<T>(out[q][k], 0), half_of<T>(out[q][k], 1)};
                                r = r - lanes(t);
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < R::kParts; ++q)
                        if (q < 2 || parts > 2) tc::st_shared_v4(to + q * R::kHalf + p * 2048, out[q][0], out[q][1], out[q][2], out[q][3]);
                }
                tc::fence_proxy_async_smem();
                tc::mbar_arrive_warp(&ctl.c_full[half]);
            }
            if (ok) tc::mbar_arrive_warp(&ctl.empty[ring.i]);
        }
    } else if (warp >= 16) {
        // ---- the state
        const int tid = threadIdx.x - 512, w = warp & 3, i = w * 32 + lane;
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
                const float whole = (float)exp((double)part_steps * (double)log_decay);
                for (int s = 0; s < part; ++s) {
                    const float* const sums = place.sums(args, s) + i * args.part_cols;
#pragma unroll
                    for (int k = 0; k < kDv; k += 4)
                        if (col0 + k < room) {           // (the parts' rows are multiples of 8, and reach as far as any job's)
                            Pack<float, 4> p;
                            p.get(sums + k);
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[k + e] = fmaf(x[k + e], whole, p.at(e));
                        }
                }
            }
        }
        bool ok = true;
        auto put_copy = [&](int n) {             // the state before chunk n (a warp that gives up goes on to the others' barriers)
            float by = 1.0f;
            if constexpr (kNarrow<T>) {
                float m[4] = {};                 // (chains of their own)
#pragma unroll
                for (int k = 0; k < kDv; k += 2) m[k / 2 & 3] = fmaxf(fmaxf(m[k / 2 & 3], fabsf(x[k])), fabsf(x[k + 1]));
                uint32_t most = __reduce_max_sync(0xffffffffu, mine ? __float_as_uint(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))) : 0);
                if (lane == 0) ctl.most[n & 1][w] = most;
                asm volatile("bar.sync 1, 128;" ::: "memory");
#pragma unroll
                for (int k = 0; k < 4; ++k) most = max(most, ctl.most[n & 1][k]);
                const int shift = shift_of(__uint_as_float(most));
                by = two_to(shift);
                if (tid == 0) ctl.up[n & 3] = two_to(-shift);
            } else {
                if (tid == 0) ctl.up[n & 3] = 1.0f;
            }
            if (!ok) return;
            if (mine) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float* const v = x + 8 * c;
                    tc::st_shared_v4(base + R::kState + tc::swz_offset(i, c), word_of<T>(v[0] * by, v[1] * by), word_of<T>(v[2] * by, v[3] * by),
                                     word_of<T>(v[4] * by, v[5] * by), word_of<T>(v[6] * by, v[7] * by));
                }
            }
            tc::fence_proxy_async_smem();
            tc::mbar_arrive_warp(&ctl.x_full);
        };
        if constexpr (!kEnds) put_copy(0);
        for (int n = 0; n < chunks; ++n) {
            const int rows = min(kSteps, finish - begin - n * kSteps);
            ok = ok && wait(&ctl.u_full, n & 1);
            if (ok) {
                __syncwarp();
                tc::tc_fence_after();
                const Lanes whole = all_lanes(rows == kSteps ? ctl.whole[n & 7] : table(power + 4 * rows));
                const Lanes back = all_lanes(kNarrow<T> ? ctl.c_back[n & 1] : 1.0f);
#pragma unroll
                for (int cb = 0; cb < 4; ++cb) {
                    uint32_t v[16];
                    tc::tmem_ld16(rows_at + cb * 16, v);
                    tc::tmem_ld_wait();
                    if (cb == 3) {
                        tc::tc_fence_before();
                        tc::mbar_arrive_warp(&ctl.u_empty);
                    }
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float a[2] = {x[cb * 16 + k], x[cb * 16 + k + 1]}, e[2] = {__uint_as_float(v[k]), __uint_as_float(v[k + 1])};
                        const Lanes r = fma(lanes(a), whole, kNarrow<T> ? lanes(e) * back : lanes(e));
                        x[cb * 16 + k] = r.at(0), x[cb * 16 + k + 1] = r.at(1);
                    }
                }
            }
            if constexpr (!kEnds) {
                if (n + 1 < chunks) {
                    ok = ok && wait(&ctl.x_empty, n & 1);       // A has met the copy before
                    __syncwarp();
                    put_copy(n + 1);
                }
            }
        }
        const int row = kEnds ? args.part_cols : wc, cols = kEnds ? room : wc;
        float* const to = (kEnds ? place.sums(args, part) : job.end != nullptr ? job.end + (int64_t)unit * wa * wc + col0 : nullptr) + (int64_t)i * row;
        if (ok && ends_here && (kEnds || job.end != nullptr) && mine && i < wa) {
            const float by = kEnds ? 1.0f : job.end_scale;
#pragma unroll
            for (int k = 0; k < kDv; ++k) x[k] *= by;
            if (row % 4 == 0) {
#pragma unroll
                for (int k = 0; k < kDv; k += 4)
                    if (col0 + k < cols) *reinterpret_cast<float4*>(to + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
            } else {
#pragma unroll
                for (int k = 0; k < kDv; ++k)
                    if (col0 + k < cols) to[k] = x[k];
            }
        }
    } else if (warp == 1) {
        // ---- scores
        if constexpr (!kEnds) {
            const uint32_t yes = elected();
            const uint64_t a_desc = tc::make_desc(base, 16, 1024), b_desc = tc::make_desc(base + R::kA, 16, 1024);
            tc::Ring ring;
            for (int n = 0; n < chunks; ++n, ring.next(R::kStages)) {
                const uint64_t stage = (uint64_t)(ring.i * R::kStage >> 4);
                if (!wait(&ctl.full[ring.i], ring.ph) || (n == ragged && !wait(&ctl.zeroed, 0)) || (n > 0 && !wait(&ctl.scores_empty, (n - 1) & 1))) break;
                __syncwarp();
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < KA / 16; ++k) {
                    const uint64_t off = stage + ((k >> 2) * R::kHalf + (k & 3) * 32 >> 4);
                    umma(yes, tmem + kTmScores, a_desc + off, b_desc + off, idesc<T>(128, 128, 0, 0), k > 0);
                }
                commit(yes, &ctl.scores_full);
                commit(yes, &ctl.empty[ring.i]);
            }
        }
    } else if (warp == 2) {
        // ---- O1 and O2
        if constexpr (!kEnds) {
            const uint32_t yes = elected();
            const uint64_t a_desc = tc::make_desc(base, 16, 1024), c_desc = tc::make_desc(base + 2 * R::kA, R::kHalf, 1024);
            const uint64_t x_desc = tc::make_desc(base + R::kState, R::kHalf, 1024);
            tc::Ring ring;
            for (int n = 0; n < chunks; ++n, ring.next(R::kStages)) {
                const uint64_t stage = (uint64_t)(ring.i * R::kStage >> 4);
                const uint32_t turn = tmem + (n & 1) * kTmTurn;
                if (!wait(&ctl.full[ring.i], ring.ph) || !wait(&ctl.x_full, n & 1) || (n >= 2 && !wait(&ctl.out_empty[n & 1], ((n >> 1) & 1) ^ 1))) break;
                __syncwarp();
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < KA / 16; ++k)
                    umma(yes, turn + kTmO1, a_desc + stage + ((k >> 2) * R::kHalf + (k & 3) * 32 >> 4), x_desc + (k * 2048 >> 4),
                         idesc<T>(128, kDv, 0, 1), k > 0);
                commit(yes, &ctl.x_empty);
                if (!wait(&ctl.full_c[ring.i], ring.ph) || (n == ragged && !wait(&ctl.zeroed, 0)) || !wait(&ctl.p_full, n & 1)) break;
                __syncwarp();
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < kSteps / 16; ++k)
                    umma_ts(yes, turn + kTmO2, tmem + kTmP + k * 8, c_desc + stage + (k * 2048 >> 4), idesc<T>(128, kDv, 0, 1), k > 0);
                commit(yes, &ctl.p_empty);
                commit(yes, &ctl.out_full[n & 1]);
                commit(yes, &ctl.empty[ring.i]);
            }
        }
    } else if (warp == 3) {
        // ---- U
        const uint32_t yes = elected();
        const uint64_t b_desc = tc::make_desc(base + R::kA, R::kHalf, 1024), w_desc = tc::make_desc(base + R::kWeighted, R::kHalf, 1024);
        bool ok = true;
        tc::Ring ring;
        for (int n = 0; n < chunks && ok; ++n, ring.next(R::kStages)) {
            const uint64_t stage = (uint64_t)(ring.i * R::kStage >> 4);
            ok = wait(&ctl.full[ring.i], ring.ph) && (n != ragged || wait(&ctl.zeroed, 0)) && (n == 0 || wait(&ctl.u_empty, (n - 1) & 1));
            for (int half = 0; half < 2 && ok; ++half) {
                ok = wait(&ctl.c_full[half], n & 1);
                if (!ok) break;
                __syncwarp();
                tc::tc_fence_after();
#pragma unroll 1
                for (int q = 0, parts = parts_of_chunk(n); q < parts; ++q)
#pragma unroll
                    for (int k = 0; k < kSteps / 32; ++k) {
                        const uint64_t rows = (uint64_t)(half * 4 + k) * (2048 >> 4);
                        umma(yes, tmem + kTmU, b_desc + stage + rows, w_desc + (uint64_t)q * (R::kHalf >> 4) + rows, idesc<T>(128, kDv, 1, 1),
                             half + q + k > 0);
                    }
                commit(yes, &ctl.c_empty[half]);
            }
            if (!ok) break;
            commit(yes, &ctl.u_full);
            commit(yes, &ctl.empty[ring.i]);
        }
    }
    // nothing is under way at the end: the last chunks' places have been given back by all who read them
    if (warp == 3)
        for (int k = max(chunks - R::kStages, 0); k < chunks; ++k) wait(&ctl.empty[k % R::kStages], k / R::kStages & 1);

    pdl_trigger();
    tc::tc_fence_before();
    __syncthreads();
    if (warp == 3) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, 512);
    }
}

}  // namespace tcgen
