// 8-bit numbers with a scale per block of 128: value = e4m3 * scale, the block's largest magnitude at 448.
#pragma once
#include "come_internal.cuh"

#include <cuda_fp8.h>

namespace come {

constexpr int kScaleBlock = 128;
constexpr float kE4m3Max = 448.0f;
// Block maxima below this take its scale, the smallest normal number: the scale and its reciprocal stay normal.
constexpr float kSmallestMax = 448.0f * 1.17549435e-38f;

// 448 / top for top in [kSmallestMax, inf]: the reciprocal of top / 256 leaves the range of normal numbers at neither end.
__device__ __forceinline__ float inverse_scale(float top) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(top * 0.00390625f));
    return r * 1.75f;
}

// Four numbers, already divided by their scale, as e4m3 (round to nearest even, saturating; NaN stays NaN).
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

}  // namespace come
