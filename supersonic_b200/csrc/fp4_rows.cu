// Rows into microscaled 4-bit floats, and back (the format: fp4_codes.cuh).
#include "fp4_codes.cuh"
#include "packed_call.cuh"
#include <algorithm>

typedef __nv_bfloat16 bf16;

constexpr int FR_THREADS = 256;
constexpr int FR_TURNS = 4;               // units a half-warp has in flight

// Where a row goes: row r of a matrix of several experts' rows, or (slot) pair r's row, a copy of its token's, in tiles of ``tile_rows``
// whose scales have runs of their own.
struct FrRows {
    int per_expert, inter;                 // rows of a matrix; of a gated unit's first, how many of them are gate rows
    const int* slot; int top, tile_rows;
};

// A unit is 128 numbers of a row: sixteen lanes of eight, four lanes a block, whose four scales are one word.  Units run over whole
// k-blocks; behind a row's end they write scales of zero.
template <typename T>
__global__ void __launch_bounds__(FR_THREADS)
fp4_quantize_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int rows, int K,
                    const FrRows to, int k_blocks, int* __restrict__ clear, int n_clear) {
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();                               // what was written before this launch is there: weights may be read ahead
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < n_clear; i += FR_THREADS) clear[i] = 0;
    const int lane = threadIdx.x & 15, per_row = 2 * k_blocks;
    const long long units = (long long)rows * per_row, step = (long long)gridDim.x * (FR_THREADS / 16);
    long long u = (long long)blockIdx.x * (FR_THREADS / 16) + (threadIdx.x >> 4);
    // the half-warps of a warp stay together: the loop ends for both at once
    for (long long first = u - ((threadIdx.x >> 4) & 1); first < units; first += FR_TURNS * step, u += FR_TURNS * step) {
        float v[FR_TURNS][8];
#pragma unroll
        for (int j = 0; j < FR_TURNS; ++j) {
            const long long unit = u + j * step;
            const int row = (int)(unit / per_row), k = (int)(unit - (long long)row * per_row) * 128 + lane * 8;
            const bool live = unit < units && k < K;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
            if (live) f4_load8(x + (to.slot ? row / to.top : row) * ldx + k, v[j]);
        }
#pragma unroll
        for (int j = 0; j < FR_TURNS; ++j) {
            const long long unit = u + j * step;
            const int row = (int)(unit / per_row), part = (int)(unit - (long long)row * per_row), k = part * 128 + lane * 8;
            uint32_t most = f4_most(v[j]);
            if (__any_sync(0xffffffffu, most >= F4_WILD)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = f4_finite(v[j][i]);
                most = f4_most(v[j]);
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int byte = f4_scale_byte(most);
            uint32_t word = (uint32_t)byte << (8 * (lane >> 2));
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            if (unit >= units) continue;
            long long at;                                      // row of the codes
            int run0 = 0, r;                                   // the matrix's first run of scales' rows, the row in it
            if (to.slot) {
                at = to.slot[row];
                if (at < 0) continue;
                const int tile = (int)at / to.tile_rows;
                r = tile * max(to.tile_rows, 128) + (int)at - tile * to.tile_rows;
            } else {
                const int expert = row / to.per_expert;
                r = f4_laid_row(row - expert * to.per_expert, to.inter);
                at = (long long)expert * to.per_expert + r;
                run0 = expert * ((to.per_expert + 127) >> 7);
            }
            if (k < K) *reinterpret_cast<uint32_t*>(codes + at * (K / 2) + k / 2) = f4_encode8(v[j], f4_inverse(byte));
            if (lane == 0)
                *reinterpret_cast<uint32_t*>(scales + (size_t)run0 * k_blocks * F4_CHUNK + f4_scale_at(r, part * 4, k_blocks)) = word;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(FR_THREADS)
fp4_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, long long ldo, int rows,
                  int K, int per_expert, int inter, int k_blocks) {
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int per_row = K / 8, tiles = (per_expert + 127) >> 7;
    const long long pieces = (long long)rows * per_row, step = (long long)gridDim.x * FR_THREADS;
    for (long long p = (long long)blockIdx.x * FR_THREADS + threadIdx.x; p < pieces; p += step) {
        const int row = (int)(p / per_row), k = (int)(p - (long long)row * per_row) * 8;
        const int expert = row / per_expert, r = f4_laid_row(row - expert * per_expert, inter);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + ((size_t)expert * per_expert + r) * (K / 2) + k / 2);
        const float s = f4_scale(scales[(size_t)expert * tiles * k_blocks * F4_CHUNK + f4_scale_at(r, k / F4_BLOCK, k_blocks)]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = f4_value(w >> (4 * i)) * s;
        f4_store8(out + row * ldo + k, v);
    }
}

static int fr_sizes(int rows, int K, int per_expert, int inter) {
    if (rows < 0 || K <= 0 || K % F4_BLOCK || per_expert <= 0 || rows % per_expert || (inter && (inter % 16 || per_expert != 2 * inter)))
        return SSB_ERR_BAD_SIZE;
    return 0;
}

template <typename T>
static int fr_quantize(const T* x, long long ldx, uint8_t* codes, uint8_t* scales, int rows, int K, const FrRows& to, int* clear, int n_clear,
                       cudaStream_t stream) {
    const int k_blocks = f4_k_blocks(K);
    const long long units = (long long)rows * 2 * k_blocks, per_block = FR_THREADS / 16;
    // a turn a thread until every SM has its eight blocks, then as many turns as it takes
    const int blocks = (int)std::min<long long>((units + per_block - 1) / per_block, 8 * ssb_sm_count());
    return ssb_launch(fp4_quantize_kernel<T>, dim3(blocks), dim3(FR_THREADS), 0, stream, true, x, ldx, codes, scales, rows, K, to, k_blocks,
                      clear, n_clear);
}

// x: rows x K, rows of 16-byte pieces; ``per_expert`` rows of them are a matrix; clear: words zeroed on the way.
SSB_API int ssb_fp4_quantize(const void* x, long long ldx, int dtype, void* codes, void* scales, int rows, int K, int per_expert, int inter,
                             int* clear, int n_clear, cudaStream_t stream) {
    const int rc = fr_sizes(rows, K, per_expert, inter);
    if (rc || rows == 0) return rc;
    if (((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15) return SSB_ERR_BAD_SIZE;
    const FrRows to{per_expert, inter, nullptr, 1, 128};
    if (dtype == SSB_BF16) return fr_quantize((const bf16*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, rows, K, to, clear, n_clear, stream);
    if (dtype == SSB_F32) return fr_quantize((const float*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, rows, K, to, clear, n_clear, stream);
    return SSB_ERR_BAD_DTYPE;
}

// The pairs' rows, pair p's from row p / top of x, to the rows that ``slot`` names (-1: none) in tiles of ``tile_rows``.
SSB_API int ssb_fp4_quantize_pairs(const void* x, long long ldx, int dtype, void* codes, void* scales, int pairs, int top, int K,
                                   const int* slot, int tile_rows, cudaStream_t stream) {
    const FrRows to{pairs, 0, slot, top, tile_rows};
    if (dtype == SSB_BF16) return fr_quantize((const bf16*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, pairs, K, to, nullptr, 0, stream);
    if (dtype == SSB_F32) return fr_quantize((const float*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, pairs, K, to, nullptr, 0, stream);
    return SSB_ERR_BAD_DTYPE;
}

SSB_API int ssb_fp4_values(const void* codes, const void* scales, void* out, long long ldo, int dtype, int rows, int K, int per_expert,
                           int inter, cudaStream_t stream) {
    const int rc = fr_sizes(rows, K, per_expert, inter);
    if (rc || rows == 0) return rc;
    if (((uintptr_t)out | (uintptr_t)codes | (uintptr_t)scales) & 15) return SSB_ERR_BAD_SIZE;
    const long long pieces = (long long)rows * (K / 8);
    const dim3 grid((unsigned)std::min<long long>((pieces + FR_THREADS - 1) / FR_THREADS, 16 * ssb_sm_count()));
    const uint8_t *c = (const uint8_t*)codes, *s = (const uint8_t*)scales;
    const int k_blocks = f4_k_blocks(K);
    if (dtype == SSB_BF16)
        return ssb_launch(fp4_values_kernel<bf16>, grid, dim3(FR_THREADS), 0, stream, true, c, s, (bf16*)out, ldo, rows, K, per_expert, inter, k_blocks);
    if (dtype == SSB_F32)
        return ssb_launch(fp4_values_kernel<float>, grid, dim3(FR_THREADS), 0, stream, true, c, s, (float*)out, ldo, rows, K, per_expert, inter, k_blocks);
    return SSB_ERR_BAD_DTYPE;
}

SSB_PACKED(ssb_fp4_quantize)
SSB_PACKED(ssb_fp4_values)
