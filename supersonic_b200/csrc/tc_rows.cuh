// How the epilogues of the tcgen05 products write finished rows.
#pragma once
#include "common.cuh"

// A warp's 32 rows of WORDS 32-bit words each, a row a lane, to memory as whole runs: the rows meet in shared memory and go
// out several lanes a row, whole runs of memory an instruction instead of 16 bytes of each of 32 rows.  ``dst``: the warp's first
// row; ADD: float32 added in memory (red.global.add.v4.f32), which nobody waits for.
constexpr int TC_STAGE_LD = 36;                               // words a row (of 32 or less): eight rows start in eight groups of four banks
constexpr int TC_STAGE_BYTES = 4 * 32 * TC_STAGE_LD * 4;      // of the four epilogue warps

template <int WORDS, bool ADD>
__device__ __forceinline__ void tc_put_rows(float* stage, const uint32_t (&v)[WORDS], char* dst, size_t row_bytes, int rows) {
    constexpr int LD = WORDS + 4, PER = WORDS / 4, ROWS = 32 / PER;
    static_assert(LD <= TC_STAGE_LD, "");
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < WORDS; j += 4)
        *reinterpret_cast<uint4*>(stage + lane * LD + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    __syncwarp();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += ROWS) {
        const int r = r0 + lane / PER, c = lane % PER * 4;
        const float4 x = *reinterpret_cast<const float4*>(stage + r * LD + c);
        if (r < rows) {
            float4* at = reinterpret_cast<float4*>(dst + (size_t)r * row_bytes) + lane % PER;
            if (ADD) atomicAdd(at, x);
            else *at = x;
        }
    }
    __syncwarp();
}
