// 16-bit floating types as template arguments of the paged cache's kernels: conversions, and the warp-level product of each.
#pragma once
#include <cuda_bf16.h>

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
#endif  // __CUDACC__

}  // namespace rnb
