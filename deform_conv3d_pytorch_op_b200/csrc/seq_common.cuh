// What the kernels of the sequence operators (seq_*.cu) share: element types, loads and stores of several elements, reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "../../include/dcn_seq.h"
#include "dcn_internal.h"

namespace dcn {
namespace seq {

// N bytes as one load or store moves them
template <int N>
struct Raw {
    uint32_t u[N / 4];
};
template <>
struct Raw<2> {
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
__device__ __forceinline__ void store(void* p, const Raw<2>& r) { *static_cast<uint16_t*>(p) = r.u; }
__device__ __forceinline__ void store(void* p, const Raw<4>& r) { *static_cast<uint32_t*>(p) = r.u[0]; }
__device__ __forceinline__ void store(void* p, const Raw<8>& r) { *static_cast<uint2*>(p) = make_uint2(r.u[0], r.u[1]); }
__device__ __forceinline__ void store(void* p, const Raw<16>& r) {
    *static_cast<uint4*>(p) = make_uint4(r.u[0], r.u[1], r.u[2], r.u[3]);
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
            const uint16_t v = (uint16_t)(raw.u[i / 2] >> (i % 2 * 16));
            return to_float(*reinterpret_cast<const T*>(&v));
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
            for (int i = 0; i < W; i += 2) {
                const T a = from_float<T>(f[i]), b = from_float<T>(f[i + 1]);
                raw.u[i / 2] = (uint32_t) * reinterpret_cast<const uint16_t*>(&a) |
                               (uint32_t) * reinterpret_cast<const uint16_t*>(&b) << 16;
            }
        }
    }
};

// s(v) = 1 / (1 + exp(-v)) and 1 - s(v), both to a few units in the last place: neither is formed as a difference.
__device__ __forceinline__ void logistic(float v, float& s, float& rest) {
    const float t = __expf(-fabsf(v));
    const float r = __fdividef(1.0f, 1.0f + t), q = t * r;
    s = v >= 0.0f ? r : q;
    rest = v >= 0.0f ? q : r;
    if (v != v) s = rest = v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int elem_bytes(int dtype) { return dtype == DCN_SEQ_F32 ? 4 : 2; }
inline bool known_type(int dtype) { return dtype == DCN_SEQ_F32 || dtype == DCN_SEQ_BF16 || dtype == DCN_SEQ_F16; }

}  // namespace seq
}  // namespace dcn
