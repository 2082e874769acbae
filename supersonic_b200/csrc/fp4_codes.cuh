// Microscaled 4-bit floats (MXFP4): 32 neighbours along a row share a scale 2^(s - 127), s a byte; a number is a sign and one of
// 0 0.5 1 1.5 2 3 4 6 (codes 0-7, the sign in bit 3).  Two codes a byte, the earlier one in its low half.
//
// Scales lie as the tensor cores want them: 1,024 bytes hold 128 rows x 8 blocks (256 numbers of k), two halves of 4 blocks, in a half
// 16 bytes for each of 32 lanes, which are the 4 blocks of rows lane, lane + 32, lane + 64, lane + 96.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

constexpr int F4_BLOCK = 32;              // numbers a scale
constexpr int F4_KB = 256;                // numbers a k-block: 128 bytes of codes, one swizzle row
constexpr int F4_CHUNK = 1024;            // bytes of the scales of 128 rows x one k-block

__host__ __device__ __forceinline__ int f4_k_blocks(int k) { return (k + F4_KB - 1) / F4_KB; }
// Offset of the scale of row r's block b in a matrix whose rows have k_blocks k-blocks.
__host__ __device__ __forceinline__ size_t f4_scale_at(int r, int b, int k_blocks) {
    return ((size_t)(r >> 7) * k_blocks + (b >> 3)) * F4_CHUNK + ((b >> 2) & 1) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

// A block's scale byte from the bits of its largest magnitude: floor(log2 m) - 2, so that the largest is 4 to 8 (and 6 at most once
// it is a code); nothing below 2^-127.
__device__ __forceinline__ int f4_scale_byte(uint32_t most) { return max(0, (int)(most >> 23) - 2); }
__device__ __forceinline__ float f4_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float f4_scale(int byte) { return __uint_as_float(byte ? (uint32_t)byte << 23 : 0x00400000u); }

// What of a number a code can stand for: NaN counts as zero, an infinity as the largest finite number.  A maximum over magnitudes is
// F4_WILD or more where that matters.
constexpr uint32_t F4_WILD = 0x7f800000u;
__device__ __forceinline__ float f4_finite(float x) {
    return x != x ? 0.f : fminf(fmaxf(x, -3.4028234663852886e38f), 3.4028234663852886e38f);
}
template <int N> __device__ __forceinline__ uint32_t f4_most(const float (&x)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}
// Eight codes: x * inverse (a power of two: exact) to the nearest, ties to even codes, at most 6.
__device__ __forceinline__ uint32_t f4_encode8(const float* x, float inverse) {
    uint32_t w;
    asm("{\n.reg .b8 a, b, c, d;\n"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w) : "f"(x[0] * inverse), "f"(x[1] * inverse), "f"(x[2] * inverse), "f"(x[3] * inverse), "f"(x[4] * inverse),
                    "f"(x[5] * inverse), "f"(x[6] * inverse), "f"(x[7] * inverse));
    return w;
}
// One code, in the low four bits.
__device__ __forceinline__ uint32_t f4_encode1(float x) {
    uint32_t w;
    asm("{\n.reg .b8 a;\ncvt.rn.satfinite.e2m1x2.f32 a, %1, %2;\nmov.b32 %0, {a, 0, 0, 0};\n}" : "=r"(w) : "f"(0.f), "f"(x));
    return w;
}
// A warp's 32 numbers, one a lane, as a block: codes into ``row`` (of codes), the scale of row r's block; nothing from channel ``width`` on.
__device__ __forceinline__ void f4_put_block(float z, uint8_t* row, uint8_t* scales, int r, int k, int width, int k_blocks) {
    const int lane = threadIdx.x & 31;
    z = f4_finite(z);
    const int byte = f4_scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(z) & 0x7fffffffu));
    // a lane's code into its place among the eight of a word
    uint32_t w = f4_encode1(z * f4_inverse(byte)) << (4 * (lane & 7));
    w |= __shfl_xor_sync(0xffffffffu, w, 1);
    w |= __shfl_xor_sync(0xffffffffu, w, 2);
    w |= __shfl_xor_sync(0xffffffffu, w, 4);
    if (k < width) {
        if ((lane & 7) == 0) *reinterpret_cast<uint32_t*>(row + (k + lane) / 2) = w;
        if (lane == 0) scales[f4_scale_at(r, k / F4_BLOCK, k_blocks)] = (uint8_t)byte;
    }
}
// Eight codes' values times ``scale``.
__device__ __forceinline__ void f4_values8(uint32_t codes, float scale, float* v) {
    uint32_t h[4];
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\ncvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(h + i));
        v[2 * i] = f.x * scale;
        v[2 * i + 1] = f.y * scale;
    }
}

__device__ __forceinline__ void f4_load8(const __nv_bfloat16* p, float* x) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void f4_load8(const float* p, float* x) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void f4_store8(__nv_bfloat16* p, const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void f4_store8(float* p, const float* x) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// A row of a matrix whose rows are a gated unit's (gate rows, then up rows, ``inter`` each), as the products want them: 16 gate rows and
// the 16 up rows of the same columns side by side.  inter 0: rows as they are.
__host__ __device__ __forceinline__ int f4_laid_row(int r, int inter) {
    if (inter == 0) return r;
    const int up = r >= inter, i = up ? r - inter : r;
    return (i >> 4) * 32 + up * 16 + (i & 15);
}
