// Activations in 8 bits: e4m3 values with one power-of-two scale per row and block of 32 columns.
//
//   value = q * 2^k,   k = the smallest whole number with amax <= 448 * 2^k, kept in [-117, 119]
//
// stored as q[rows][D] and one byte k + 127 per block, scale[rows][ceil(D/32)].  amax is taken over the block's finite
// elements; an infinity or NaN becomes e4m3's NaN and leaves its neighbours as they are.  448 is e4m3's largest value, so
// nothing saturates (but magnitudes above 448 * 2^119 = 2.97e38).  The scale is a power of two rather than amax / 448
// because x * 2^-k is then exact - the conversion is the only rounding, at most half a step: 2^-4 relative, 2^(k-10)
// absolute under 2^(k-6) - and because a value in [-117, 119] always is a BF16 number, which the tensor cores take as it is.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include "ptx.cuh"

namespace ta {

constexpr int kQ8Block = 32;

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 t = unpack_bf16x2(w[i]);
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

// k + 127 of a block.  A mantissa above 0x600000 (1.75, that of 448) carries into the exponent.
__device__ __forceinline__ int q8_scale_byte(float amax) {
    const int k = int((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - (127 + 8);
    return min(max(k, -117), 119) + 127;
}
__device__ __forceinline__ float q8_step(int byte) { return __uint_as_float(uint32_t(byte) << 23); }           // 2^k
__device__ __forceinline__ float q8_inverse(int byte) { return __uint_as_float(uint32_t(254 - byte) << 23); }  // 2^-k

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return uint32_t(lo) | uint32_t(hi) << 16;
}
__device__ __forceinline__ void widen4(uint32_t w, float step, float* f) {
    uint32_t lo, hi;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(uint16_t(w)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(uint16_t(w >> 16)));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    f[0] = a.x * step; f[1] = a.y * step; f[2] = b.x * step; f[3] = b.y * step;
}
__device__ __forceinline__ void widen8(const uint2& q, int byte, float (&f)[8]) {
    const float step = q8_step(byte);
    widen4(q.x, step, f);
    widen4(q.y, step, f + 4);
}

// One block of 32 columns held by four neighbouring lanes, eight columns each (a lane past the row's end passes zeros).
// Returns this lane's eight bytes; `byte` is the block's scale.  All 32 lanes of the warp call it.
__device__ __forceinline__ uint2 narrow8(const float (&f)[8], int& byte) {
    auto quad_max = [](float v) {
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
        return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
    };
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) m = fmaxf(m, fabsf(f[e]));   // a NaN is passed over by fmaxf
    m = quad_max(m);
    if (!__any_sync(0xffffffffu, m == CUDART_INF_F)) {
        byte = q8_scale_byte(m);
        const float s = q8_inverse(byte);
        return make_uint2(e4m3x4(f[0] * s, f[1] * s, f[2] * s, f[3] * s), e4m3x4(f[4] * s, f[5] * s, f[6] * s, f[7] * s));
    }
    float g[8];
    m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        g[e] = fabsf(f[e]) < CUDART_INF_F ? f[e] : CUDART_NAN_F;
        m = fmaxf(m, fabsf(g[e]));
    }
    m = quad_max(m);
    byte = q8_scale_byte(m);
    const float s = q8_inverse(byte);
    return make_uint2(e4m3x4(g[0] * s, g[1] * s, g[2] * s, g[3] * s), e4m3x4(g[4] * s, g[5] * s, g[6] * s, g[7] * s));
}

}  // namespace ta
