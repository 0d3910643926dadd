// The 8-bit cache formats: int8 codes in [-127, 127] or fp8 e4m3 codes in [-448, 448], one fp32 scale per
// (page, KV head); code * scale is the value.  Both formats are exact in fp16, so the attention kernels multiply
// codes on the tensor cores and apply the scales in fp32.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "view_plan.h"

namespace gb200 {

enum : int { kElemF16 = 0, kElemInt8 = 1, kElemE4M3 = 2 };  // what a cache holds; 1 + cache_dtype for the 8-bit ones

template <int kElem>
__host__ __device__ constexpr float q8_max() { return kElem == kElemInt8 ? 127.f : 448.f; }

// Two neighbouring codes (the low 16 bits) as fp16.
__device__ __forceinline__ __half2 e4m3x2_to_half2(uint32_t w) {
    return __half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xFFFFu), __NV_E4M3));
}

// Four codes (byte i is element i) as fp32.
template <int kElem>
__device__ __forceinline__ float4 q8_decode4(uint32_t w) {
    if (kElem == kElemInt8)
        return make_float4((float)(int8_t)(w & 0xFF), (float)(int8_t)((w >> 8) & 0xFF), (float)(int8_t)((w >> 16) & 0xFF),
                           (float)(int8_t)(w >> 24));
    const float2 a = __half22float2(e4m3x2_to_half2(w)), b = __half22float2(e4m3x2_to_half2(w >> 16));
    return make_float4(a.x, a.y, b.x, b.y);
}

// Round to nearest even; |x| is at most the code range's end, up to a rounding error.
template <int kElem>
__device__ __forceinline__ uint32_t q8_encode4(float4 x) {
    if (kElem == kElemInt8) {
        // adding 1.5 * 2^23 leaves the rounded integer in the low bits of the sum
        auto one = [](float f) { return __float_as_uint(__fadd_rn(f, 12582912.f)); };
        return __byte_perm(__byte_perm(one(x.x), one(x.y), 0x0040), __byte_perm(one(x.z), one(x.w), 0x0040), 0x5410);
    }
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x.x, x.y), __NV_SATFINITE, __NV_E4M3) |
           ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x.z, x.w), __NV_SATFINITE, __NV_E4M3) << 16);
}

}  // namespace gb200
