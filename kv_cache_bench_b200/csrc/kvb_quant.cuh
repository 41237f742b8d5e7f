// int8 quantization of fp32 values, shared by the page write path (kvb_pages.cu) and the append (kvb_step.cu).
#pragma once

#include "kvb_device.cuh"

namespace kvb_dev {

// Four values quantized with `scale` (0 when the scale is 0), packed low byte first:
// clamp(rint(x / scale), -127, 127) with the IEEE division of the reference. |x / scale| <= 127, so
// t = x * fl(1 / scale) is within 2^-16 of the exact quotient and fl(x / scale) within 2^-17 of it.
// When t is at least 2^-14 away from every half-integer, no rounding boundary lies between t and
// fl(x / scale), and the integer nearest t is the reference's value. t + 1.5 * 2^23 rounds t to that
// integer (ties to even) and holds it in its low mantissa bits: two full-rate additions instead of a
// round and a conversion. The fast path flags (in `near`) any value close to a boundary; the caller
// then redoes its values with quantize4_exact, which takes the division (rare: one test per run, not
// a branch per value). `rcp` = 1 / scale, finite.
__device__ __forceinline__ uint32_t quantize4_fast(const float4 v, float rcp, int& near) {
    constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float t = __fmul_rn(x[e], rcp);
        const float y = __fadd_rn(t, kMagic);
        const int q = min(max(__float_as_int(y) - 0x4B400000, -127), 127);
        near |= fabsf(__fsub_rn(t, __fsub_rn(y, kMagic))) >= 0.5f - 6.103515625e-05f;
        packed |= uint32_t(q & 255) << (8 * e);
    }
    return packed;
}

static __device__ __noinline__ uint32_t quantize4_exact(const float4 v, float scale) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int q = min(max(__float2int_rn(__fdiv_rn(x[e], scale)), -127), 127);
        packed |= uint32_t(q & 255) << (8 * e);
    }
    return packed;
}

__device__ __forceinline__ float finite_rcp(float scale) {
    const float r = 1.0f / scale;
    return scale > 0.f && r < 3.0e38f ? r : 0.f;
}

}  // namespace kvb_dev
