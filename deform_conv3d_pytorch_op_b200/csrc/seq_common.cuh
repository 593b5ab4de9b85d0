// What the kernels of the sequence operators (seq_*.cu) share: element types, loads and stores of several elements, reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <type_traits>

#include "../../include/dcn_seq.h"
#include "dcn_internal.h"

namespace dcn {
namespace seq {

// N bytes as one load or store moves them
template <int N>
struct alignas(N) Raw {
    uint32_t u[N / 4];
};
template <>
struct alignas(2) Raw<2> {
    uint16_t u;
};

// Loads that stay behind pdl_wait() (see gload in dcn_common.cuh).  The data is read once: it is not kept in L1.
__device__ __forceinline__ void load(Raw<2>& r, const void* p) {
    asm volatile("ld.global.L1::no_allocate.u16 %0, [%1];" : "=h"(r.u) : "l"(p));
}
__device__ __forceinline__ void load(Raw<4>& r, const void* p) {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r.u[0]) : "l"(p));
}
__device__ __forceinline__ void load(Raw<8>& r, const void* p) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.u[0]), "=r"(r.u[1]) : "l"(p));
}
__device__ __forceinline__ void load(Raw<16>& r, const void* p) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]) : "l"(p));
}
// The same where the data is read again soon
__device__ __forceinline__ void load_kept(Raw<16>& r, const void* p) {
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]) : "l"(p));
}
// From shared memory, each time anew
__device__ __forceinline__ void load_shared(Raw<16>& r, const void* p) {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3]) : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void load_shared(Raw<8>& r, const void* p) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.u[0]), "=r"(r.u[1]) : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void load_shared(Raw<4>& r, const void* p) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r.u[0]) : "r"((uint32_t)__cvta_generic_to_shared(p)));
}
__device__ __forceinline__ void store(void* p, const Raw<2>& r) { *static_cast<uint16_t*>(p) = r.u; }
__device__ __forceinline__ void store(void* p, const Raw<4>& r) { *static_cast<uint32_t*>(p) = r.u[0]; }
__device__ __forceinline__ void store(void* p, const Raw<8>& r) { *static_cast<uint2*>(p) = make_uint2(r.u[0], r.u[1]); }
__device__ __forceinline__ void store(void* p, const Raw<16>& r) {
    *static_cast<uint4*>(p) = make_uint4(r.u[0], r.u[1], r.u[2], r.u[3]);
}

// A result that is not read again soon: it does not push out of L2 what is
__device__ __forceinline__ void store_streaming(void* p, const Raw<16>& r) {
    asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(r.u[0]), "r"(r.u[1]), "r"(r.u[2]), "r"(r.u[3])
                 : "memory");
}

__device__ __forceinline__ int64_t gload_i64(const int64_t* p) {
    long long r;
    asm volatile("ld.global.s64 %0, [%1];" : "=l"(r) : "l"(p));
    return r;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Pairs of 16-bit elements in a word: one instruction an element in, one a pair out
template <typename T>
__device__ __forceinline__ float half_of(uint32_t word, int i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        return __uint_as_float(i == 0 ? word << 16 : word & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word));
        return i == 0 ? f.x : f.y;
    }
}
template <typename T>
__device__ __forceinline__ uint32_t word_of(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// W elements of type T
template <typename T, int W>
struct Pack {
    Raw<sizeof(T) * W> raw;
    __device__ __forceinline__ void zero() { memset(&raw, 0, sizeof(raw)); }
    __device__ __forceinline__ void get(const void* p) { load(raw, p); }
    __device__ __forceinline__ void put(void* p) const { store(p, raw); }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(raw.u[i]);
        } else if constexpr (W == 1) {
            return to_float(*reinterpret_cast<const T*>(&raw.u));
        } else {
            return half_of<T>(raw.u[i / 2], i % 2);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[W]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < W; ++i) raw.u[i] = __float_as_uint(f[i]);
        } else if constexpr (W == 1) {
            const T v = from_float<T>(f[0]);
            raw.u = *reinterpret_cast<const uint16_t*>(&v);
        } else {
#pragma unroll
            for (int i = 0; i < W; i += 2) raw.u[i / 2] = word_of<T>(f[i], f[i + 1]);
        }
    }
};

__device__ __forceinline__ float ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// s(v) = 1 / (1 + exp(-v)) and 1 - s(v): neither is formed as a difference.  The larger one is right to 4 x 2^-24 of itself.  The
// smaller one is off by what the rounding of the exponent's argument makes of it, which grows with |v|: measured, 4 x 2^-24 up to 1, 10
// up to 8, 17 up to 16, 30 up to 32, 64 up to 87, and it is 0 beyond (an argument in two parts would cost three instructions an
// element in kernels that are bound by them).
__device__ __forceinline__ void logistic(float v, float& s, float& rest) {
    const float t = ex2(-1.4426950408889634f * fabsf(v));
    const float r = rcp(1.0f + t), q = t * r;
    s = v < 0.0f ? q : r;
    rest = v < 0.0f ? r : q;
}

// Two floats as the packed float32 instructions take them
struct Lanes {
    uint64_t v;
    __device__ __forceinline__ float at(int i) const { return __uint_as_float((uint32_t)(i == 0 ? v : v >> 32)); }
};
__device__ __forceinline__ Lanes lanes(const float (&f)[2]) {
    Lanes r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(f[0]), "f"(f[1]));
    return r;
}
__device__ __forceinline__ Lanes all_lanes(float f) {
    const float a[2] = {f, f};
    return lanes(a);
}
__device__ __forceinline__ Lanes fma(Lanes a, Lanes b, Lanes c) {
    Lanes r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Lanes operator*(Lanes a, Lanes b) {
    Lanes r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Lanes operator+(Lanes a, Lanes b) {
    Lanes r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Lanes operator-(Lanes a, Lanes b) { return fma(b, all_lanes(-1.0f), a); }

__device__ __forceinline__ Lanes shuffle_xor(Lanes a, int o) {
    return {__shfl_xor_sync(0xffffffffu, (unsigned long long)a.v, o)};
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Copies to shared memory that run on while the thread goes on; nothing is read and zeros are written where `in` is false
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int kBytes>
__device__ __forceinline__ void copy_async(void* to, const void* from, bool in) {
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(to)), "l"(from), "r"(in ? 16 : 0)
                     : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(shared_address(to)), "l"(from), "n"(kBytes),
                     "r"(in ? kBytes : 0)
                     : "memory");
}
template <int kBytes>
__device__ __forceinline__ void copy_async_all(void* to, const void* from) {
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_address(to)), "l"(from) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(shared_address(to)), "l"(from), "n"(kBytes) : "memory");
}
// the first `bytes` of kBytes, zeros behind them
template <int kBytes>
__device__ __forceinline__ void copy_async_some(void* to, const void* from, int bytes) {
    if constexpr (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(shared_address(to)), "l"(from), "r"(bytes) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(shared_address(to)), "l"(from), "n"(kBytes), "r"(bytes)
                     : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all of the thread's groups but the `kLast` issued last
template <int kLast>
__device__ __forceinline__ void copies_arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(kLast) : "memory"); }

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int elem_bytes(int dtype) { return dtype == DCN_SEQ_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == DCN_SEQ_F32 || dtype == DCN_SEQ_BF16 || dtype == DCN_SEQ_F16; }

}  // namespace seq
}  // namespace dcn
