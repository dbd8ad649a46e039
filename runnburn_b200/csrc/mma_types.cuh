// 16-bit floating types as template arguments of the paged cache's kernels: conversions, and the warp-level product of each.
#pragma once
#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace rnb {

struct F16 {
    uint16_t bits;
};
struct Bf16 {
    uint16_t bits;
};

#ifdef __CUDACC__
// two f32 rounded to nearest, the first in the lower half
template <class T>
__device__ __forceinline__ uint32_t pk_pack(float x, float y) {
    uint32_t r;
    if constexpr (std::is_same<T, F16>::value) {
        const __half2 h = __floats2half2_rn(x, y);
        r = *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        r = *reinterpret_cast<const uint32_t *>(&h);
    }
    return r;
}
template <class T>
__device__ __forceinline__ float2 pk_unpack(uint32_t v) {
    if constexpr (std::is_same<T, F16>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ float pk_value(T v) {
    if constexpr (std::is_same<T, F16>::value) return f16_bits_to_f32(v.bits);
    else return __uint_as_float((uint32_t)v.bits << 16);
}
template <>
__device__ __forceinline__ float pk_value<float>(float v) { return v; }
template <class T>
__device__ __forceinline__ T pk_rounded(float v) {
    return {(uint16_t)(pk_pack<T>(v, 0.f) & 0xffffu)};
}
template <>
__device__ __forceinline__ float pk_rounded<float>(float v) { return v; }
// (x, y) rounded to T, and what the rounding left of them, rounded again
template <class T>
__device__ __forceinline__ void pk_split(float x, float y, uint32_t &hi, uint32_t &lo) {
    hi = pk_pack<T>(x, y);
    const float2 h = pk_unpack<T>(hi);
    lo = pk_pack<T>(x - h.x, y - h.y);
}
__device__ __forceinline__ void pk_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pk_ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// c += a b, m16n8k16
template <class T>
__device__ __forceinline__ void pk_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, F16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
#endif  // __CUDACC__

}  // namespace rnb
