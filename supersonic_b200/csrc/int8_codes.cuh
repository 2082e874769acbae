// Numbers into 8-bit codes under a scale, for the cache and for the rows of a product: code = rint(x / scale), value = code * scale.
#pragma once
#include "common.cuh"

constexpr float I8_LEAST_SCALE = 7.888609052210118e-31f;        // 2^-100: a block of zeros has a scale too
constexpr float I8_MOST = 1.7014118346046923e38f;               // 2^127: its largest code still stands for a finite number
__device__ __forceinline__ void i8_load8(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void i8_load8(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void i8_store8(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void i8_store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
// What of a number a code can stand for: NaN counts as zero, an infinity as 2^127 of its sign.  A maximum over magnitudes, taken in
// the order of their bits, is I8_WILD or more where that matters.
constexpr uint32_t I8_WILD = 0x7f000000u;
__device__ __forceinline__ float i8_finite(float x) { return x != x ? 0.f : fminf(fmaxf(x, -I8_MOST), I8_MOST); }
__device__ __forceinline__ uint32_t i8_magnitude(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

// Eight codes of eight numbers, rint(x / scale), and the values that the codes stand for; no |x| is above 127 scales.  The division
// is correctly rounded: x times the reciprocal is within 2e-5 of it (127 times two roundings), so only where that lies about half-way
// between two codes is there anything to divide for.  Adding 1.5 * 2^23 rounds to a whole number, whose low byte is the code.
__device__ __forceinline__ uint2 i8_encode8(float (&x)[8], float scale, float inverse) {
    constexpr float WHOLE = 12582912.f;
    float t[8], near = 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t[i] = fmaf(x[i], inverse, WHOLE);
        near = fminf(near, fabsf(fabsf(fmaf(x[i], inverse, WHOLE - t[i])) - 0.5f));
    }
    if (near < 1e-4f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = rintf(__fdiv_rn(x[i], scale)) + WHOLE;
    }
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        w[h] = __byte_perm(__byte_perm(__float_as_uint(t[4 * h]), __float_as_uint(t[4 * h + 1]), 0x0040),
                           __byte_perm(__float_as_uint(t[4 * h + 2]), __float_as_uint(t[4 * h + 3]), 0x0040), 0x5410);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(t[i] - WHOLE, scale);
    return make_uint2(w[0], w[1]);
}
