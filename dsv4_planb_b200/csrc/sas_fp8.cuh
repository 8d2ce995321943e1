// e4m3 codes, their scales and request lookup, shared by the kernels of the 8-bit cache.
#pragma once

#include <stdint.h>

#include "sas_common.cuh"

namespace sas_fp8 {

// Scales outside [2^-60, 2^60] (zero, negative, infinite or NaN ones among them) are no scales.
constexpr float kScaleMin = 8.673617379884035e-19f, kScaleMax = 1.152921504606846976e18f;
__device__ __forceinline__ bool scale_ok(float s) { return s >= kScaleMin && s <= kScaleMax; }

// Smallest power of two s with amax <= 448 s, clamped to the scales' range (amax finite, >= 0).
// amax = m 2^e with m in [1, 2); 448 = 1.75 2^8: k = e - 8 where m <= 1.75, else e - 7.
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    int k = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
    k = max(-60, min(60, k));  // zero and subnormal maxima: exponent field 0, below the range
    return __uint_as_float((uint32_t)(k + 127) << 23);
}

// Two floats to two codes (a in the low byte): nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    return to_e4m3x2(a, b) | (to_e4m3x2(c, d) << 16);
}
// Two codes to two halves (exact: every e4m3 value is an fp16 value).
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)codes));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint32_t codes) {
    const uint32_t h = e4m3x2_to_half2(codes);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
// Four codes times f, rounded to codes again.
__device__ __forceinline__ uint32_t rescale4(uint32_t codes, float f) {
    const float2 a = e4m3x2_to_f2(codes & 0xffffu), b = e4m3x2_to_f2(codes >> 16);
    return to_e4m3x4(a.x * f, a.y * f, b.x * f, b.y * f);
}

// The request whose rows [cu[b], cu[b + 1]) hold flat row t, or -1.  Every lane of a full warp
// calls with the same t; each round the 32 lanes cut the range of candidates 32-fold.
__device__ __forceinline__ int find_request(const int32_t *__restrict__ cu, int B, int t) {
    const int lane = threadIdx.x & 31;
    if (B <= 0) return -1;
    int lo = 0, n = B;  // b is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int i = lo + (lane + 1) * step;  // is b >= i ?
        const bool past = (lane + 1) * step < n && __ldg(cu + i) <= t;
        const int k = __popc(__ballot_sync(0xffffffffu, past));
        lo += k * step;
        n = min(step, n - k * step);
    }
    return __ldg(cu + lo) <= t && t < __ldg(cu + lo + 1) ? lo : -1;
}

} // namespace sas_fp8
