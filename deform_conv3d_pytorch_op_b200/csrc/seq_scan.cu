// Gated linear recurrence over time, per channel:
//     a_t = s(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t,  y_t = h_t          (s the logistic function)
// and its gradient.  With p_t the gradient that step t passes to the state before it,
//     p_t = a_t p_{t+1} + a_t dy_t   (p behind the last step: dlast),   D_t = dy_t + p_{t+1}
//     dx_t = D_t (1 - a_t),   dgate_t = D_t (h_{t-1} - x_t) a_t (1 - a_t),   dstate = p_0.
//
// Both directions are scans of affine maps h -> A h + B, whose composition is (A2 A1, A2 B1 + B2).  A lane has a pair of
// channels, in the packed float32 instructions, and K steps of them: it composes its steps, the warps of a CTA (one behind the
// other in time) compose theirs through shared memory and the CTAs of a cluster theirs through distributed shared memory, a warp
// for all; the state that reaches a lane then gives all of its steps.  So x and gate are read once and y is written once, whatever
// the length.  A cluster walks the time axis in waves of (its CTAs) x 64 steps and carries the state from wave to wave in
// registers.  Every warp copies its own steps of the next waves to shared memory meanwhile (cp.async, two waves ahead; the gates
// of the backward pass one, which lets an SM hold four CTAs), and sends its results out from there: 16 bytes an instruction where
// addresses allow it, and no address arithmetic in the recurrence.
//
// What bounds it depends on how many sequences there are.  Measured, bf16, against a copy of the same bytes at 6.5 TB/s:
//     64 x 1024 x 2048 (2048 units, one CTA each)   forward 140 us (5.8 TB/s, 88 %)   backward 254 us (5.3 TB/s, 81 %): DRAM
//     2 x 16384 x 2048 (64 units in clusters)       forward 101 us (4.0 TB/s, 61 %)   backward 150 us (4.5 TB/s, 69 %)
// Few long sequences walk few clusters through many waves, and in each wave's exchange of maps its warps have nothing but copies
// under way: latency, with DRAM 43 % busy and 53 % of the issue slots taken in the forward pass.  Sequences of fewer than 64 steps
// are far from a copy (56 x 9 x 3776 fp16: 18 and 26 us, 2 and 3 at a copy's rate): a CTA takes the shared memory of 64 steps however
// many it has, and a last wave that is not whole is copied with its guards.  A tile of 64 channels that a width does not fill costs
// what a full one does (38 x 6862 x 257 fp16: 234 and 416 us, 62 and 103 at a copy's rate; the narrow rows' 4-byte copies are in it).
//
// A state that lasts 10^4 steps has gates within 10^-4 of one, and what matters of them is 1 - a: the rounding of a alone would
// cost it three digits.  So the product over a thread's steps is also formed as 1 - A = sum (1 - a_t) a_1 .. a_{t-1}, of which no
// term is a difference, and A is handed on as a float and the rest that its rounding left.
//
// The forward pass leaves the state before every 64th step; the backward pass recomputes the states in between from it, in
// float32, and reads no y: 4 bytes in 64 steps instead of an activation per step, and no rounded state in a gradient.
#include <cooperative_groups.h>

#include "seq_common.cuh"

namespace cg = cooperative_groups;

namespace dcn {
namespace seq {
namespace {

constexpr int kTile = 64;                        // channels of a CTA: two a lane
constexpr int kChunk = 64;                       // steps of a CTA in a wave, and between checkpoints
constexpr int kCluster = 8;                      // CTAs of a cluster, at most

struct ScanArgs {
    const void *x, *gate, *dy;
    const float *state, *dlast;
    const int64_t* lengths;
    void *y, *dx, *dgate;
    float *last, *dstate, *checkpoints;
    int64_t steps, channels, chunks;
    int64_t x_batch, x_step, gate_batch, gate_step, dy_batch, dy_step;
    int tiles;
};

// What is left of a product of gates that float32 does not hold: an infinite state times it is infinite, as the recurrence has it,
// and any other state times it is nothing beside what it was.
constexpr float kTrace = 9.2e-41f;               // 2^-133, the least that bfloat16 holds

// h -> A h + B, A = a + more to more digits than a float has, both above zero
struct Map {
    Lanes a, more, b;
    __device__ __forceinline__ Lanes operator()(Lanes h) const { return fma(a, h, fma(more, h, b)); }
};

// A product of gates, and one minus it.  (Not a product alone, so that it does not become zero: 64x1024x2048 bf16, forward, 1 %; a
// look at the states for infinite ones costs float32 and long sequences 2 to 3 %.)
struct Product {
    Lanes a = all_lanes(1.0f), rest = all_lanes(0.0f);
    __device__ __forceinline__ void by(Lanes gate, Lanes one_minus) {
        rest = fma(one_minus, a, rest);
        a = fma(gate, a, all_lanes(kTrace));
    }
    __device__ __forceinline__ void by(const Map& m) { by(m.a, all_lanes(1.0f) - m.a - m.more); }
    __device__ __forceinline__ Map map(Lanes b) const {
        float top[2], more[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float near = __fsub_rd(1.0f, rest.at(i));       // (what it lacks is not negative)
            const bool close = rest.at(i) < 0.5f;
            top[i] = close ? near : a.at(i);
            more[i] = close ? fmaxf((1.0f - near) - rest.at(i), kTrace) : kTrace;
        }
        return {lanes(top), lanes(more), b};
    }
};

__device__ __forceinline__ Map identity() { return {all_lanes(1.0f), all_lanes(kTrace), all_lanes(0.0f)}; }

// Maps of two channels in shared memory, a lane each.  `more` is below the last digit of a: eight digits of it are plenty, and
// what they save lets an SM hold another CTA.
struct MapRoom {
    static constexpr uint32_t kBytes = (2 * sizeof(Lanes) + 4) * 32;
    struct alignas(16) Pair {
        Lanes a, b;
    };
    Pair ab[32];
    uint32_t more[32];
    static __device__ __forceinline__ uint32_t packed(Lanes more) { return word_of<__nv_bfloat16>(more.at(0), more.at(1)); }
    __device__ __forceinline__ void put(int lane, const Map& m) { ab[lane] = {m.a, m.b}, more[lane] = packed(m.more); }
    __device__ __forceinline__ Map get(int lane, Lanes b) const {                  // with another b: its own is not read
        const uint32_t w = more[lane];
        const float f[2] = {half_of<__nv_bfloat16>(w, 0), half_of<__nv_bfloat16>(w, 1)};
        return {ab[lane].a, lanes(f), b};
    }
    __device__ __forceinline__ Map get(int lane) const { return get(lane, ab[lane].b); }
};

// Set where a wait for a map of another CTA gave up (which nothing but a fault of the GPU brings about)
__device__ unsigned int g_scan_status;
constexpr long long kWaitCycles = 1ll << 32;                     // some two seconds

// The exchange of maps in a cluster.  Each CTA sends its own to all (st.async, which counts its bytes on the barrier of the CTA it
// goes to): a cluster barrier instead holds every warp until its results of the wave before are in memory (2x16384x2048 bf16,
// forward: 120 us with it, 101 us without).  Two of everything: a CTA sends a wave's map when all maps of the wave before have
// arrived, so the one it writes over has been read.
struct Exchange {
    MapRoom maps[2][kCluster];
    alignas(8) uint64_t arrived[2];
    int gave_up;

    // by warp 0; the places of CTAs that are not there hold maps that change nothing
    __device__ __forceinline__ void begin(int lane, int ranks) {
        for (int r = ranks; r < kCluster; ++r) maps[0][r].put(lane, identity()), maps[1][r].put(lane, identity());
        if (lane == 0) {
            gave_up = 0;
            for (int s = 0; s < 2; ++s)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&arrived[s])) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    // by one thread a wave: so many maps will come
    __device__ __forceinline__ void expect(int side, int ranks) {
        asm volatile("{\n .reg .b64 s;\n mbarrier.arrive.expect_tx.shared::cta.b64 s, [%0], %1;\n}" ::"r"(
                         shared_address(&arrived[side])),
                     "r"(ranks * MapRoom::kBytes)
                     : "memory");
    }
    // my lane's part of the map of the CTA `rank`, to the CTA `to`
    __device__ __forceinline__ void send(int side, int rank, int to, int lane, const Map& m) {
        uint32_t there;                          // this object, in that CTA
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(shared_address(this)), "r"(to));
        const uint32_t here = shared_address(this), bar = there + shared_address(&arrived[side]) - here;
        const uint32_t ab = there + shared_address(&maps[side][rank].ab[lane]) - here,
                       more = there + shared_address(&maps[side][rank].more[lane]) - here;
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(ab), "l"(m.a.v),
                     "l"(m.b.v), "r"(bar)
                     : "memory");
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(more),
                     "r"(MapRoom::packed(m.more)), "r"(bar)
                     : "memory");
    }
    __device__ __forceinline__ void send_all(int side, int rank, int ranks, int lane, const Map& m) {
        if (lane == 0) expect(side, ranks);
#pragma unroll
        for (int r = 0; r < kCluster; ++r)
            if (r < ranks) send(side, rank, r, lane, m);
    }
    // until all maps of the n-th wave are there.  Bounded: a wait that gives up raises the status word, and the kernel runs to its
    // end without waiting again.
    __device__ __forceinline__ void wait(int side, int n) {
        const uint32_t bar = shared_address(&arrived[side]), parity = n / 2 % 2;
        long long began = 0;
        for (;;) {
            uint32_t ok;
            asm volatile(
                "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
                " selp.b32 %0, 1, 0, p;\n}"
                : "=r"(ok)
                : "r"(bar), "r"(parity)
                : "memory");
            if (ok || *(volatile int*)&gave_up) return;
            const long long now = clock64();
            if (began == 0) began = now;
            if (now - began > kWaitCycles) {
                *(volatile int*)&gave_up = 1;
                atomicOr(&g_scan_status, 1u);
                return;
            }
        }
    }
};

// Where a thread works
struct Place {
    int lane, warp, warps, rank, ranks;
    int64_t b, c;                                // c: the CTA's first channel
    int width, mine;                             // channels of the CTA, and of them mine
    __device__ __forceinline__ explicit Place(const ScanArgs& p) {
        const cg::cluster_group cluster = cg::this_cluster();
        lane = threadIdx.x;
        warp = threadIdx.y;
        warps = blockDim.y;
        rank = (int)cluster.block_rank();
        ranks = (int)cluster.num_blocks();
        const unsigned unit = blockIdx.x / ranks;
        b = unit / p.tiles;
        c = (int64_t)(unit % p.tiles) * kTile;
        width = (int)(p.channels - c < kTile ? p.channels - c : kTile);
        mine = width - 2 * lane < 0 ? 0 : width - 2 * lane > 2 ? 2 : width - 2 * lane;
    }
    __device__ __forceinline__ Lanes load(const float* s, int64_t row, int64_t channels) const {
        float h[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) h[i] = s != nullptr && i < mine ? gload(s + row * channels + c + 2 * lane + i) : 0.0f;
        return lanes(h);
    }
    __device__ __forceinline__ void store(float* s, int64_t row, int64_t channels, Lanes h) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (i < mine) s[row * channels + c + 2 * lane + i] = h.at(i);
    }
};

__device__ __forceinline__ int64_t length_of(const ScanArgs& p, int64_t b) {
    if (p.lengths == nullptr) return p.steps;
    const int64_t n = gload_i64(p.lengths + b);
    return n < 0 ? 0 : n > p.steps ? p.steps : n;
}

// Where rows start on 4 bytes or in the middle of them (kBytes 2): 0 or 1 element, for the even and the odd ones behind step t0
template <typename T, int kBytes>
struct Skew {
    int even = 0, odd = 0;
    __device__ __forceinline__ Skew(const T* base, int64_t t0, int64_t stride) {
        if constexpr (kBytes == 2) {
            even = (int)(((unsigned)(reinterpret_cast<uintptr_t>(base) / 2) + (unsigned)t0 * (unsigned)stride) & 1);
            odd = (even + (int)stride) & 1;
        }
    }
    __device__ __forceinline__ int at(int t) const { return kBytes == 2 ? (t % 2 == 0 ? even : odd) : 0; }
};

// K steps of the CTA's channels in shared memory, a warp's own.  They come and go 16 bytes at a time, or 4 where that is what all
// rows start on.  16-bit rows that start in the middle of 4 bytes (kBytes 2) move 4 bytes at a time too: they arrive in shared memory
// with their skew, which align() takes out, and the elements at their ends that share 4 bytes with others leave on their own.
// Measured, bf16, forward and backward: 64x1024x2046 183 and 416 us, 64x1024x2047 248 and 500 us (378 and 682 us element by element),
// against 143 and 255 us at 2048 channels: four times the copies, in a kernel whose issue slots are two thirds taken.
template <typename T, int kBytes, int K>
struct Block {
    static constexpr int kMove = kBytes == 2 ? 4 : kBytes, kPer = kMove / (int)sizeof(T), kSlots = kTile / kPer;
    static constexpr int kRows = kSlots <= 32 ? 32 / kSlots : 1;  // rows of a move
    static constexpr int kMoves = K * kSlots / 32, kHalves = kSlots <= 32 ? 1 : kSlots / 32;       // kHalves: moves of a row
    T v[K][kTile + (kBytes == 2 ? 2 : 0)];
    static __device__ __forceinline__ int row(int lane, int j) { return kSlots <= 32 ? lane / kSlots + j * kRows : j / kHalves; }
    static __device__ __forceinline__ int slot(int lane, int j) { return kSlots <= 32 ? lane % kSlots : lane + 32 * (j % kHalves); }
    // from step t0 on; zeros behind the sequence's end.  left: channels to the tensor's end; what lies behind them is left as it is.
    __device__ __forceinline__ void fill(const T* tensor, const T* base, int64_t t0, int64_t stride, int64_t len, int left,
                                         int lane) {
        const Skew<T, kBytes> skew(base, t0, stride);
        const T* q = base + t0 * stride;
        const bool all = t0 + K <= len;
        if (kBytes == 2 && all && q - 1 >= tensor) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int bytes = min(2 * (left + skew.at(p) - 2 * lane), 4);
                const T* from = q + p * stride - skew.at(p) + 2 * lane;
                if (bytes > 0)
#pragma unroll
                    for (int i = 0; i < K / 2; ++i, from += 2 * stride) copy_async_some<4>(&v[2 * i + p][2 * lane], from, bytes);
            }
            if (lane < K && skew.at(lane) != 0 && left >= kTile)
                copy_async_some<4>(&v[lane][kTile], q + lane * stride - 1 + kTile, left > kTile ? 4 : 2);
            return;
        }
        if (kBytes != 2 && all) {
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                const T* from = q + row(lane, 0) * stride + slot(lane, h) * kPer;
                if (slot(lane, h) * kPer < left)
#pragma unroll
                    for (int j = h; j < kMoves; j += kHalves, from += kRows * stride)
                        copy_async_all<kMove>(&v[row(lane, j)][slot(lane, j) * kPer], from);
            }
            return;
        }
#pragma unroll 1
        for (int j = lane; j < K * (kSlots + (kBytes == 2)); j += 32) {
            const int r = kBytes == 2 ? j / (kSlots + 1) : j / kSlots, i = kBytes == 2 ? j % (kSlots + 1) : j % kSlots;
            const int sk = skew.at(r);
            const T* from = q + r * stride - sk + i * kPer;
            const int there = t0 + r < len ? left + sk - i * kPer : 0;
            if (kBytes != 2 || from >= tensor || there <= 0) {
                const T* any = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(tensor) / kMove * kMove);
                copy_async_some<kMove>(&v[r][i * kPer], there > 0 ? from : any,
                                       there <= 0 ? 0 : there >= kPer ? kMove : there * (int)sizeof(T));
            } else {                             // nothing is read that lies before the tensor
                Pack<T, 1> one;
                one.get(tensor);
                *reinterpret_cast<Raw<sizeof(T)>*>(&v[r][1]) = one.raw;
            }
        }
    }
    // Rows t0, ..., t0 + K - 1 of a tensor's `steps`, from word(row, move, skew) and one(row, channel)
    template <typename F, typename G>
    static __device__ __forceinline__ void send(T* base, int64_t t0, int64_t stride, int64_t steps, int width, int lane, F&& word,
                                                G&& one) {
        const Skew<T, kBytes> skew(base, t0, stride);
        T* q = base + t0 * stride;
        const bool all = t0 + K <= steps;
        if constexpr (kBytes == 2) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {        // (behind a skew, a lane's word has its second element and the next lane's first)
                const int sk = skew.at(p);
                T* to = q + p * stride + sk + 2 * lane;
                if (2 * lane + sk + 1 >= width) continue;
                if (all) {
#pragma unroll
                    for (int i = 0; i < K / 2; ++i, to += 2 * stride) store(to, word(2 * i + p, lane, sk));
                } else {
#pragma unroll 1
                    for (int r = p; r < K && t0 + r < steps; r += 2, to += 2 * stride) store(to, word(r, lane, sk));
                }
            }
            // the first element behind a skew, and the last where words end before it
            const int r = lane / 2, sk = skew.at(r);
            if (r < K && t0 + r < steps && (lane % 2 == 0 ? sk : (width + sk) % 2) != 0) {
                const int c = lane % 2 == 0 ? 0 : width - 1;
                store(q + r * stride + c, one(r, c));
            }
        } else {
#pragma unroll
            for (int h = 0; h < kHalves; ++h) {
                T* to = q + row(lane, 0) * stride + slot(lane, h) * kPer;
                if (slot(lane, h) * kPer >= width) continue;
                if (all) {
#pragma unroll
                    for (int j = h; j < kMoves; j += kHalves, to += kRows * stride) store(to, word(row(lane, j), slot(lane, j), 0));
                } else {
#pragma unroll 1
                    for (int j = h; j < kMoves; j += kHalves, to += kRows * stride)
                        if (t0 + row(lane, j) < steps) store(to, word(row(lane, j), slot(lane, j), 0));
                }
            }
        }
    }
    // to the steps before `steps`
    __device__ __forceinline__ void drain(T* base, int64_t t0, int64_t stride, int64_t steps, int width, int lane) const {
        send(base, t0, stride, steps, width, lane,
             [&](int r, int i, int skew) {
                 Raw<kMove> w = *reinterpret_cast<const Raw<kMove>*>(&v[r][i * kPer]);
                 if (kBytes == 2 && skew != 0) w.u[0] = __funnelshift_r(w.u[0], word(r, i + 1), 16);
                 return w;
             },
             [&](int r, int c) { return *reinterpret_cast<const Raw<sizeof(T)>*>(&v[r][c]); });
    }
    __device__ __forceinline__ uint32_t& word(int r, int i) { return reinterpret_cast<uint32_t*>(&v[r][0])[i]; }
    __device__ __forceinline__ const uint32_t& word(int r, int i) const { return reinterpret_cast<const uint32_t*>(&v[r][0])[i]; }
    // takes the rows' skew out, once they have arrived
    __device__ __forceinline__ void align(const T* base, int64_t t0, int64_t stride, int lane) {
        if constexpr (kBytes == 2) {
            const Skew<T, kBytes> skew(base, t0, stride);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                if (skew.at(p) == 0) continue;
                uint32_t w[K / 2];
#pragma unroll
                for (int i = 0; i < K / 2; ++i) w[i] = __funnelshift_r(word(2 * i + p, lane), word(2 * i + p, lane + 1), 16);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < K / 2; ++i) word(2 * i + p, lane) = w[i];
            }
            __syncwarp();
        }
    }
    __device__ __forceinline__ Pack<T, 2> get(int k, int lane) const {
        Pack<T, 2> p;
        p.raw = *reinterpret_cast<const Raw<2 * sizeof(T)>*>(&v[k][2 * lane]);
        return p;
    }
    __device__ __forceinline__ Lanes at(int k, int lane) const {
        const Pack<T, 2> p = get(k, lane);
        const float f[2] = {p.at(0), p.at(1)};
        return lanes(f);
    }
    __device__ __forceinline__ void put(int k, int lane, Lanes x) {
        const float f[2] = {x.at(0), x.at(1)};
        Pack<T, 2> p;
        p.set(f);
        *reinterpret_cast<Raw<2 * sizeof(T)>*>(&v[k][2 * lane]) = p.raw;
    }
};

// Gate and one minus it; one and zero, a step that keeps the state, behind a sequence's end
template <typename T>
__device__ __forceinline__ void gates_of(const Pack<T, 2>& g, bool in, Lanes& a, Lanes& keep) {
    float fa[2], fk[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        logistic(g.at(i), fa[i], fk[i]);
        if (!in) fa[i] = 1.0f, fk[i] = 0.0f;
    }
    a = lanes(fa);
    keep = lanes(fk);
}

// Zeros from step `from` on, shared out over the warps of the cluster
template <typename T, int kBytes>
__device__ __forceinline__ void zero_rest(const Place& me, T* out, int64_t from, int64_t steps, int64_t channels) {
    using B = Block<T, kBytes, 4>;
    constexpr int kRows = 4;                     // of a warp at a time
    const int64_t all = (int64_t)me.ranks * me.warps * kRows;
    for (int64_t t = from + (int64_t)(me.rank * me.warps + me.warp) * kRows; t < steps; t += all)
        B::send(out, t, channels, steps, me.width, me.lane, [](int, int, int) { return Raw<B::kMove>{}; },
                [](int, int) { return Raw<sizeof(T)>{}; });
}

template <typename T, int kBytes, int K>
struct ForwardRoom {
    static constexpr int kWarps = kChunk / K;
    Block<T, kBytes, K> x[2][kWarps], gate[2][kWarps];
    MapRoom part[kWarps];                     // of the warps
    Lanes start[kWarps][32];                  // the states before their steps
    Exchange cluster;
};

template <typename T, int kBytes, int K>
__global__ void __launch_bounds__(32 * (kChunk / K), 4) scan_forward_kernel(const ScanArgs p) {
    constexpr int kWarps = kChunk / K;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto& room = *reinterpret_cast<ForwardRoom<T, kBytes, K>*>(dynamic);
    const Place me(p);
    pdl_wait();
    const int64_t len = length_of(p, me.b);
    const T* x = static_cast<const T*>(p.x) + me.b * p.x_batch + me.c;
    const T* gate = static_cast<const T*>(p.gate) + me.b * p.gate_batch + me.c;
    T* y = static_cast<T*>(p.y) + me.b * p.steps * p.channels + me.c;
    Lanes carry = me.load(p.state, me.b, p.channels);

    const int chunk = me.warps * K, wave = me.ranks * chunk;
    int64_t t0 = (int64_t)me.rank * chunk + me.warp * K;           // my first step of this wave
    int64_t begin = 0;
    const int left = (int)(p.channels - me.c < 2 * kTile ? p.channels - me.c : 2 * kTile);
    auto fill = [&](auto& block, const void* tensor, const T* from, int64_t t, int64_t stride) {
        if (t - me.rank * chunk - me.warp * K < len)               // (a wave that does not come is not filled)
            block.fill(static_cast<const T*>(tensor), from, t, stride, len, left, me.lane);
        copies_issued();
    };
    if (me.warp == 0) {
        if (me.ranks > 1) room.cluster.begin(me.lane, me.ranks);
        for (int w = me.warps; w < kWarps; ++w) {                  // (warps that are not there change nothing)
            room.part[w].put(me.lane, identity());
        }
    }
    for (int s = 0; s < 2; ++s) {
        fill(room.gate[s][me.warp], p.gate, gate, t0 + s * wave, p.gate_step);
        fill(room.x[s][me.warp], p.x, x, t0 + s * wave, p.x_step);
    }
    if (me.ranks > 1) cg::this_cluster().sync();                   // every CTA runs before another writes to its memory
    for (int side = 0, n = 0; begin < len; begin += wave, t0 += wave, side ^= 1, ++n) {
        auto &bx = room.x[side][me.warp], &bg = room.gate[side][me.warp];
        copies_arrived<2>();
        __syncwarp();
        bg.align(gate, t0, p.gate_step, me.lane);
        bx.align(x, t0, p.x_step, me.lane);
        // after each of my steps: y = A h + B of the state h before the first
        Lanes A[K], B[K], sum = all_lanes(0.0f);
        Product product;
        const bool all = begin + wave <= len;
        auto compose = [&](auto whole) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                Lanes a, keep;
                gates_of<T>(bg.get(k, me.lane), whole.value || t0 + k < len, a, keep);
                product.by(a, keep);
                sum = fma(a, sum, keep * bx.at(k, me.lane));
                A[k] = product.a;
                B[k] = sum;
            }
        };
        if (all) compose(std::true_type());
        else compose(std::false_type());
        room.part[me.warp].put(me.lane, product.map(sum));
        __syncthreads();
        if (me.warp == 0) {
            Lanes h = carry;
            if (me.ranks > 1) {
                Product product_of;
                Lanes s = all_lanes(0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const Map m = room.part[w].get(me.lane);
                    product_of.by(m);
                    s = m(s);
                }
                room.cluster.send_all(side, me.rank, me.ranks, me.lane, product_of.map(s));
                room.cluster.wait(side, n);
#pragma unroll
                for (int r = 0; r < kCluster; ++r) {
                    if (r == me.rank) h = carry;
                    carry = room.cluster.maps[side][r].get(me.lane)(carry);
                }
            }
            if (p.checkpoints != nullptr && t0 < len) me.store(p.checkpoints, me.b * p.chunks + t0 / kChunk, p.channels, h);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                room.start[w][me.lane] = h;
                h = room.part[w].get(me.lane)(h);
            }
            if (me.ranks == 1) carry = h;
        }
        fill(bg, p.gate, gate, t0 + 2 * wave, p.gate_step);
        __syncthreads();
        const Lanes mine = room.start[me.warp][me.lane];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Lanes v = fma(A[k], mine, B[k]);
            if (!all && t0 + k >= len) v = all_lanes(0.0f);
            bx.put(k, me.lane, v);
        }
        __syncwarp();
        bx.drain(y, t0, p.channels, p.steps, me.width, me.lane);
        __syncwarp();
        fill(bx, p.x, x, t0 + 2 * wave, p.x_step);
    }
    copies_arrived<0>();
    if (me.ranks > 1) cg::this_cluster().sync();                   // (no CTA ends while another could still send to it)
    zero_rest<T, kBytes>(me, y, begin, p.steps, p.channels);
    if (me.rank == 0 && me.warp == 0) me.store(p.last, me.b, p.channels, carry);
}

template <typename T, int kBytes, int K>
struct BackwardRoom {
    static constexpr int kWarps = kChunk / K;
    Block<T, kBytes, K> x[2][kWarps], dy[2][kWarps], gate[kWarps];
    MapRoom part[kWarps];                        // of the warps; b gives way to the states before their steps
    // the b of the warps' backward maps p -> A p + b, which have the forward ones' A; then the gradients behind their steps
    Lanes back[kWarps][32];
    Exchange cluster;
};

template <typename T, int kBytes, int K>
__global__ void __launch_bounds__(32 * (kChunk / K), K == 16 ? 4 : 2) scan_backward_kernel(const ScanArgs p) {
    constexpr int kWarps = kChunk / K;
    extern __shared__ __align__(16) unsigned char dynamic[];
    auto& room = *reinterpret_cast<BackwardRoom<T, kBytes, K>*>(dynamic);
    const Place me(p);
    pdl_wait();
    const int64_t len = length_of(p, me.b);
    const T* x = static_cast<const T*>(p.x) + me.b * p.x_batch + me.c;
    const T* gate = static_cast<const T*>(p.gate) + me.b * p.gate_batch + me.c;
    const T* dy = static_cast<const T*>(p.dy) + me.b * p.dy_batch + me.c;
    T* dx = static_cast<T*>(p.dx) + me.b * p.steps * p.channels + me.c;
    T* dgate = static_cast<T*>(p.dgate) + me.b * p.steps * p.channels + me.c;
    Lanes carry = me.load(p.dlast, me.b, p.channels);

    const int chunk = me.warps * K, wave = me.ranks * chunk;
    const int64_t end = (len + wave - 1) / wave * wave;
    int64_t begin = end - wave;
    int64_t t0 = begin + (int64_t)me.rank * chunk + me.warp * K;
    const int left = (int)(p.channels - me.c < 2 * kTile ? p.channels - me.c : 2 * kTile);
    // (a wave that does not come is not filled)
    auto fill = [&](int side, int64_t t) {
        if (t >= 0) {
            room.x[side][me.warp].fill(static_cast<const T*>(p.x), x, t, p.x_step, len, left, me.lane);
            room.dy[side][me.warp].fill(static_cast<const T*>(p.dy), dy, t, p.dy_step, p.dy == nullptr ? t : len, left, me.lane);
        }
        copies_issued();
    };
    auto fill_gate = [&](int64_t t) {
        if (t >= 0) room.gate[me.warp].fill(static_cast<const T*>(p.gate), gate, t, p.gate_step, len, left, me.lane);
        copies_issued();
    };
    if (me.warp == 0) {
        if (me.ranks > 1) room.cluster.begin(me.lane, me.ranks);
        for (int w = me.warps; w < kWarps; ++w) {                  // (warps that are not there change nothing)
            room.part[w].put(me.lane, identity());
            room.back[w][me.lane] = all_lanes(0.0f);
        }
    }
    fill(0, t0);
    fill_gate(t0);
    fill(1, t0 - wave);
    if (me.ranks > 1) cg::this_cluster().sync();                   // every CTA runs before another writes to its memory
    for (int side = 0, n = 0; begin >= 0; begin -= wave, t0 -= wave, side ^= 1, ++n) {
        auto &bx = room.x[side][me.warp], &bg = room.gate[me.warp], &bd = room.dy[side][me.warp];
        copies_arrived<1>();
        __syncwarp();
        bg.align(gate, t0, p.gate_step, me.lane);
        bx.align(x, t0, p.x_step, me.lane);
        if (p.dy != nullptr) bd.align(dy, t0, p.dy_step, me.lane);
        Lanes a[K], keep[K], before[K], sum = all_lanes(0.0f), passed = sum;
        Product product;
        const bool all = begin + wave <= len;
        auto compose = [&](auto whole) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                gates_of<T>(bg.get(k, me.lane), whole.value || t0 + k < len, a[k], keep[k]);
                product.by(a[k], keep[k]);
                sum = fma(a[k], sum, keep[k] * bx.at(k, me.lane));
            }
        };
        if (all) compose(std::true_type());
        else compose(std::false_type());
#pragma unroll
        for (int k = K - 1; k >= 0; --k) passed = a[k] * (bd.at(k, me.lane) + passed);
        room.part[me.warp].put(me.lane, product.map(sum));
        room.back[me.warp][me.lane] = passed;
        __syncthreads();
        fill_gate(t0 - wave);
        if (me.warp == (me.warps > 1 ? 1 : 0)) {                   // the states, from the one before the CTA's steps
            const int64_t first = t0 - me.warp * K;
            Lanes h = me.load(first < len ? p.checkpoints : nullptr, me.b * p.chunks + first / kChunk, p.channels);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const Map m = room.part[w].get(me.lane);
                room.part[w].ab[me.lane].b = h;
                h = m(h);
            }
        }
        if (me.warp == 0) {                                        // the gradients, from the one that reaches the CTA's last step
            auto back_map = [&](int w) { return room.part[w].get(me.lane, room.back[w][me.lane]); };
            Lanes g = carry;
            if (me.ranks > 1) {
                Product product_of;
                Lanes s = all_lanes(0.0f);
#pragma unroll
                for (int w = kWarps - 1; w >= 0; --w) {
                    const Map m = back_map(w);
                    product_of.by(m);
                    s = m(s);
                }
                room.cluster.send_all(side, me.rank, me.ranks, me.lane, product_of.map(s));
                room.cluster.wait(side, n);
#pragma unroll
                for (int r = kCluster - 1; r >= 0; --r) {
                    if (r == me.rank) g = carry;
                    carry = room.cluster.maps[side][r].get(me.lane)(carry);
                }
            }
#pragma unroll
            for (int w = kWarps - 1; w >= 0; --w) {
                const Map m = back_map(w);
                room.back[w][me.lane] = g;
                g = m(g);
            }
            if (me.ranks == 1) carry = g;
        }
        __syncthreads();
        Lanes h = room.part[me.warp].ab[me.lane].b, mine = room.back[me.warp][me.lane];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            before[k] = h;
            h = fma(a[k], h, keep[k] * bx.at(k, me.lane));
        }
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
            const Lanes d = bd.at(k, me.lane) + mine;
            Lanes ox = d * keep[k], og = ox * a[k] * (before[k] - bx.at(k, me.lane));
            mine = a[k] * d;
            if (!all && t0 + k >= len) ox = og = all_lanes(0.0f);
            bx.put(k, me.lane, ox);
            bd.put(k, me.lane, og);
        }
        __syncwarp();
        bx.drain(dx, t0, p.channels, p.steps, me.width, me.lane);
        bd.drain(dgate, t0, p.channels, p.steps, me.width, me.lane);
        __syncwarp();
        fill(side, t0 - 2 * wave);
    }
    copies_arrived<0>();
    if (me.ranks > 1) cg::this_cluster().sync();                   // (no CTA ends while another could still send to it)
    zero_rest<T, kBytes>(me, dx, end, p.steps, p.channels);
    zero_rest<T, kBytes>(me, dgate, end, p.steps, p.channels);
    if (p.dstate != nullptr && me.rank == 0 && me.warp == 0) me.store(p.dstate, me.b, p.channels, carry);
}

// One step of each row's state, in place: W channels a thread, and as many threads as there are channels, for the fewest dependent
// loads: gate and x, the slot, the state.  A call of 16 x 512 float32 takes 1.8 us on the GPU, most of it launch and two trips to
// memory, and 4.9 us from call to call, which is the host's share.  Widths that four do not divide take one channel a thread: 1555 x
// 1286 bf16 12.3 us, 4.3 at a copy's rate.
template <typename T, int W>
__global__ void __launch_bounds__(128)
    scan_step_kernel(int64_t rows, int64_t channels, const T* x, int64_t x_row, const T* gate, int64_t gate_row, float* state,
                     int64_t pool, const int64_t* slots, T* y) {
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
                // a h + (1 - a) x as a step from the larger share: no product with a gate near one is rounded.  As it stands where
                // the two are further apart than float32 holds.
                float a, keep;
                logistic(vg.at(i), a, keep);
                const float from = a < keep ? vx.at(i) : h.at(i), to = a < keep ? h.at(i) : vx.at(i), way = to - from;
                out[i] = fabsf(way) < CUDART_INF_F ? fmaf(a < keep ? a : keep, way, from) : fmaf(a, h.at(i), keep * vx.at(i));
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

// CTAs of a kernel that an SM holds with its shared memory, asked for once per device (0: it cannot be launched)
template <typename Room, typename K>
int resident(K kernel, int threads) {
    constexpr int kMostDevices = 64;
    static std::atomic<int> of_device[kMostDevices];
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMostDevices) return 0;
    int n = of_device[dev];
    if (n == 0) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Room)) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, sizeof(Room)) != cudaSuccess)
            return 0;
        of_device[dev] = n;                      // racing first calls find the same number
    }
    return n;
}

// As many warps as the steps fill, and CTAs along time as long as the GPU holds all of them at once: a cluster walks the whole
// time axis, and one that had to wait for another would double the time.  (Any number of them, and not powers of two alone: where
// an SM held three CTAs, the backward pass of 2x16384x2048 bf16 took 156 us in clusters of six, 185 us in clusters of four.)
template <typename K>
int launch_scan(K kernel, int held, size_t smem, int per_thread, const ScanArgs& a, int64_t batch, cudaStream_t st) {
    if (held == 0) return DCN_ERR_CUDA;
    const int64_t units = batch * a.tiles;
    const int64_t filled = (a.steps + per_thread - 1) / per_thread;
    const int warps = (int)(a.steps >= kChunk ? kChunk / per_thread : filled > 1 ? filled : 1);
    int ranks = 1;
    while (ranks < kCluster && (int64_t)ranks * kChunk < a.steps && units * (ranks + 1) <= (int64_t)held * sm_count()) ++ranks;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * ranks));
    cfg.blockDim = dim3(32, warps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e != cudaSuccess || cudaGetLastError() != cudaSuccess ? DCN_ERR_CUDA : DCN_OK;
}

template <typename T, int kBytes, int K>
int forward_as(const ScanArgs& a, int64_t batch, cudaStream_t st) {
    using Room = ForwardRoom<T, kBytes, K>;
    const int held = resident<Room>(scan_forward_kernel<T, kBytes, K>, 32 * kChunk / K);
    return launch_scan(scan_forward_kernel<T, kBytes, K>, held, sizeof(Room), K, a, batch, st);
}

template <typename T, int kBytes, int K>
int backward_as(const ScanArgs& a, int64_t batch, cudaStream_t st) {
    using Room = BackwardRoom<T, kBytes, K>;
    const int held = resident<Room>(scan_backward_kernel<T, kBytes, K>, 32 * kChunk / K);
    return launch_scan(scan_backward_kernel<T, kBytes, K>, held, sizeof(Room), K, a, batch, st);
}

// Steps of a thread, 16 or 8: with 16 the joining of maps costs half as much of a step, with 8 a thread has registers to spare, and
// float32 data holds the SM's shared memory anyhow.  Measured (us, 16 / 8): forward, bf16, 64x1024x2048 141 / 165, 2x16384x2048
// 101 / 141; float32, 2x8192x2048 82 / 86.  Backward, bf16, 64x1024x2048 252 / 326, 2x16384x2048 151 / 187; float32,
// 2x8192x2048 132 / 127, 46x238x3008 113 / 102.
template <typename T, int kBytes>
int run_forward(const ScanArgs& a, int64_t batch, cudaStream_t st) {
    return forward_as<T, kBytes, 16>(a, batch, st);
}

template <typename T, int kBytes>
int run_backward(const ScanArgs& a, int64_t batch, cudaStream_t st) {
    return backward_as<T, kBytes, sizeof(T) == 2 ? 16 : 8>(a, batch, st);
}

int check_scan(const dcn_scan* p) {
    if (p == nullptr) return DCN_ERR_NULL;
    if (!known_type(p->dtype)) return DCN_ERR_UNSUPPORTED;
    if (p->batch < 0 || p->steps < 0 || p->channels < 0) return DCN_ERR_SHAPE;
    constexpr int64_t most = 1ll << 31;
    if (p->batch >= most || p->steps >= most || p->channels >= most) return DCN_ERR_LIMIT;
    // (CTAs of a grid, eight to a cluster)
    if (p->batch * ((p->channels + kTile - 1) / kTile) >= 1ll << 27) return DCN_ERR_LIMIT;
    return DCN_OK;
}

// Bytes that every row of every tensor starts on: 16, 8 (float32 alone: 2x8192x2046 90 + 206 us, and 103 + 226 us by 4; bf16,
// 64x1024x2044: 174 + 433 us, and 183 + 416 us by 4), 4 or an element's
struct Bytes {
    int n, e;
    void by(const void* p, int64_t batch, int64_t step) {
        while (n > e && (!aligned(p, n) || batch * e % n != 0 || step * e % n != 0)) n = n == 16 && e == 2 ? 4 : n > 4 ? n / 2 : e;
    }
};

template <typename T, typename F>
int with_bytes(int n, F&& run) {
    constexpr bool kWide = sizeof(T) == 4;
    if (n == 16) return run(std::integral_constant<int, 16>());
    if (n == (kWide ? 8 : 4)) return run(std::integral_constant<int, kWide ? 8 : 4>());
    return run(std::integral_constant<int, kWide ? 4 : 2>());
}

ScanArgs args_of(const dcn_scan* p) {
    ScanArgs a = {};
    a.steps = p->steps;
    a.channels = p->channels;
    a.chunks = (p->steps + kChunk - 1) / kChunk;
    a.x_batch = p->x_batch, a.x_step = p->x_step;
    a.gate_batch = p->gate_batch, a.gate_step = p->gate_step;
    a.dy_batch = p->dy_batch, a.dy_step = p->dy_step;
    a.tiles = (int)((p->channels + kTile - 1) / kTile);
    return a;
}

}  // namespace

int scan_check_status(cudaStream_t st) {
    unsigned int v = 0;
    if (cudaStreamSynchronize(st) != cudaSuccess || cudaMemcpyFromSymbol(&v, g_scan_status, sizeof(v)) != cudaSuccess)
        return DCN_ERR_CUDA;
    if (v == 0) return DCN_OK;
    const unsigned int zero = 0;
    cudaMemcpyToSymbol(g_scan_status, &zero, sizeof(zero));
    return DCN_ERR_TIMEOUT;
}

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
    Bytes rows{16, e};
    rows.by(x, p->x_batch, p->x_step);
    rows.by(gate, p->gate_batch, p->gate_step);
    rows.by(y, p->channels, p->channels);
    ScanArgs a = args_of(p);
    a.x = x, a.gate = gate, a.state = state, a.lengths = lengths, a.y = y, a.last = last, a.checkpoints = checkpoints;
    const cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == DCN_SEQ_F32) return with_bytes<float>(rows.n, [&](auto n) { return run_forward<float, n.value>(a, p->batch, st); });
    if (p->dtype == DCN_SEQ_BF16)
        return with_bytes<__nv_bfloat16>(rows.n, [&](auto n) { return run_forward<__nv_bfloat16, n.value>(a, p->batch, st); });
    return with_bytes<__half>(rows.n, [&](auto n) { return run_forward<__half, n.value>(a, p->batch, st); });
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
    Bytes rows{16, e};
    rows.by(x, p->x_batch, p->x_step);
    rows.by(gate, p->gate_batch, p->gate_step);
    if (dy != nullptr) rows.by(dy, p->dy_batch, p->dy_step);
    rows.by(dx, p->channels, p->channels);
    rows.by(dgate, p->channels, p->channels);
    ScanArgs a = args_of(p);
    a.x = x, a.gate = gate, a.dy = dy, a.dlast = dlast, a.lengths = lengths, a.dx = dx, a.dgate = dgate, a.dstate = dstate;
    a.checkpoints = const_cast<float*>(checkpoints);
    const cudaStream_t st = (cudaStream_t)stream;
    if (p->dtype == DCN_SEQ_F32) return with_bytes<float>(rows.n, [&](auto n) { return run_backward<float, n.value>(a, p->batch, st); });
    if (p->dtype == DCN_SEQ_BF16)
        return with_bytes<__nv_bfloat16>(rows.n, [&](auto n) { return run_backward<__nv_bfloat16, n.value>(a, p->batch, st); });
    return with_bytes<__half>(rows.n, [&](auto n) { return run_backward<__half, n.value>(a, p->batch, st); });
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
