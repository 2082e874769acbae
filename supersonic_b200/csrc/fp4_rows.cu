// Rows into microscaled 4-bit floats, and back (the format: fp4_codes.cuh).
#include "fp4_codes.cuh"
#include "packed_call.cuh"
#include <algorithm>
#include <climits>

typedef __nv_bfloat16 bf16;

constexpr int FR_THREADS = 256;
constexpr int FR_TURNS = 4;               // units of values that a half-warp has in flight

// Where a row goes: row r of a matrix of several experts' rows, or (slot) the rows of its ``top`` pairs, in tiles of 2^``tile_log`` whose
// scales have runs of their own.
struct FrRows {
    int per_expert, inter;                 // rows of a matrix; of a gated unit's first, how many of them are gate rows
    const int* slot; int top, tile_log;
};

// Where the units that a half-warp takes lie: unit u is part u % per_row of row u / per_row; from one turn to the next
// the half-warp goes on by ``rows`` rows and ``parts`` parts, so that nothing is divided on the way.
struct FrStep {
    int per_row, rows, parts;
    __device__ void next(int& row, int& part) const {
        row += rows;
        part += parts;
        if (part >= per_row) { part -= per_row; ++row; }
    }
};

// A unit is 16 V numbers of a row: sixteen lanes of V, 32 / V lanes a block, scales in words of four.  Units run over whole
// k-blocks; behind a row's end they write scales of zero.  TURNS units are in flight.
//
// Where there are many rows, fetches and instructions bound it (59 % of issue slots, 62 % of the ALU pipe's cycles, and fetches what most warps
// wait for; 144 instructions for 256 numbers of bfloat16 with V = 8, places and scale bytes more than half of them), so a lane takes sixteen
// numbers, two units in flight: 8,192 x 4,096 19.9 us (87 MB, 4.4 TB/s; eight numbers, one unit 23.7),
// 14,336 x 4,096 32 (40).  Few rows are a launch and a dependent fetch or two, on as many SMs as can be: 64 x 2,048 1.5 us (2.0 by sixteen),
// 512 x 2,048 1.9 (2.1); they cross at about 1,024 x 2,048 (2.6, 2.5).
template <typename T, int TURNS, int V, bool PAIRS>
__global__ void __launch_bounds__(FR_THREADS)
fp4_quantize_kernel(const T* __restrict__ x, long long ldx, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int rows, int K,
                    const FrRows to, const FrStep step, int k_blocks, int* __restrict__ clear, int n_clear, int early) {
    constexpr int PER = F4_BLOCK / V;                          // lanes a block
    const int lane = threadIdx.x & 15, u = blockIdx.x * (FR_THREADS / 16) + (threadIdx.x >> 4);
    int row = u / step.per_row, part = u - row * step.per_row;
    ssb_pdl_wait();
    if (early) ssb_pdl_launch_dependents();                    // what was written before this launch is there: weights may be read ahead
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < n_clear; i += FR_THREADS) clear[i] = 0;
    // the half-warps of a warp go on together: a later unit is in no earlier row
    while (__any_sync(0xffffffffu, row < rows)) {
        float v[TURNS][V];
        int at_row[TURNS], at_part[TURNS], slot[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
            at_row[j] = row;
            at_part[j] = part;
            const int k = (part * 16 + lane) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = 0.f;
            if (row < rows && k < K)
#pragma unroll
                for (int i = 0; i < V; i += 8) f4_load8(x + (long long)row * ldx + k + i, v[j] + i);
            slot[j] = PAIRS && row < rows && lane < to.top ? to.slot[row * to.top + lane] : -1;
            step.next(row, part);
        }
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
            const int k = (at_part[j] * 16 + lane) * V;
            uint32_t most = f4_most(v[j]);
            if (__any_sync(0xffffffffu, most >= F4_WILD)) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[j][i] = f4_finite(v[j][i]);
                most = f4_most(v[j]);
            }
#pragma unroll
            for (int o = 1; o < PER; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int byte = f4_scale_byte(most);
            uint32_t word = (uint32_t)byte << (8 * (lane / PER & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, PER);
            word |= __shfl_xor_sync(0xffffffffu, word, 2 * PER);
            if (!PAIRS && at_row[j] >= rows) continue;
            uint32_t code[V / 8];
#pragma unroll
            for (int i = 0; i < V; i += 8) code[i / 8] = f4_encode8(v[j] + i, f4_inverse(byte));
            for (int copy = 0; copy < (PAIRS ? to.top : 1); ++copy) {
                long long at = at_row[j];                      // row of the codes
                int run0 = 0, r = at_row[j];                   // the matrix's first run of scales' rows, the row in it
                if (PAIRS) {
                    at = __shfl_sync(0xffffffffu, slot[j], copy & 15, 16);
                    if (copy >= 16 && at_row[j] < rows) at = to.slot[at_row[j] * to.top + copy];
                    if (at < 0 || at_row[j] >= rows) continue;
                    const int tile = (int)at >> to.tile_log;
                    r = (tile << max(to.tile_log, 7)) + (int)at - (tile << to.tile_log);
                } else if (to.per_expert < rows || to.inter) {
                    const int expert = r / to.per_expert;
                    r = f4_laid_row(r - expert * to.per_expert, to.inter);
                    at = (long long)expert * to.per_expert + r;
                    run0 = expert * ((to.per_expert + 127) >> 7);
                }
                if (k < K) {
                    uint32_t* dst = reinterpret_cast<uint32_t*>(codes + at * (K / 2) + k / 2);
                    if (V == 8) *dst = code[0];
                    else *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[V / 8 - 1]);
                }
                if (lane % (4 * PER) == 0)
                    *reinterpret_cast<uint32_t*>(scales + (size_t)run0 * k_blocks * F4_CHUNK + f4_scale_at(r, k / F4_BLOCK, k_blocks)) = word;
            }
        }
    }
}

// The way back, units of 128 numbers: 14,336 x 4,096 to bfloat16 30.5 us (149 MB, 4.9 TB/s), with one unit in flight 32; 64 x 2,048 1.26 with
// one in flight, 1.7 with four.
template <typename T, int TURNS>
__global__ void __launch_bounds__(FR_THREADS)
fp4_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out, long long ldo, int rows,
                  int K, int per_expert, int inter, const FrStep step, int k_blocks) {
    const int lane = threadIdx.x & 15, u = blockIdx.x * (FR_THREADS / 16) + (threadIdx.x >> 4);
    int row = u / step.per_row, part = u - row * step.per_row;
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    while (row < rows) {
        uint32_t w[TURNS], byte[TURNS];
        int at_row[TURNS], at_part[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
            at_row[j] = row;
            at_part[j] = part;
            const int k = part * 128 + lane * 8;
            w[j] = byte[j] = 0;
            if (row < rows && k < K) {
                long long at = row;
                int run0 = 0, r = row;
                if (per_expert < rows || inter) {
                    const int expert = row / per_expert;
                    r = f4_laid_row(row - expert * per_expert, inter);
                    at = (long long)expert * per_expert + r;
                    run0 = expert * ((per_expert + 127) >> 7);
                }
                w[j] = *reinterpret_cast<const uint32_t*>(codes + at * (K / 2) + k / 2);
                byte[j] = scales[(size_t)run0 * k_blocks * F4_CHUNK + f4_scale_at(r, k / F4_BLOCK, k_blocks)];
            }
            step.next(row, part);
        }
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
            const int k = at_part[j] * 128 + lane * 8;
            float v[8];
            f4_values8(w[j], f4_scale((int)byte[j]), v);
            if (at_row[j] < rows && k < K) f4_store8(out + (long long)at_row[j] * ldo + k, v);
        }
    }
}

// Blocks of a launch over ``rows`` rows of ``per_row`` units of which a half-warp has ``turns`` in flight, and its step.
static FrStep fr_step(int rows, int per_row, int turns, int* blocks) {
    const long long units = (long long)rows * per_row, per_block = FR_THREADS / 16;
    *blocks = (int)std::min((units + per_block * turns - 1) / (per_block * turns), 8LL * ssb_sm_count());
    const long long step = *blocks * per_block;
    return FrStep{per_row, (int)(step / per_row), (int)(step % per_row)};
}
static int fr_sizes(int rows, int K, int per_expert, int inter) {
    if (rows < 0 || K <= 0 || K % F4_BLOCK || per_expert <= 0 || rows % per_expert || (inter && (inter % 16 || per_expert != 2 * inter)))
        return SSB_ERR_BAD_SIZE;
    return 0;
}

template <typename T>
static int fr_quantize(const T* x, long long ldx, uint8_t* codes, uint8_t* scales, int rows, int K, const FrRows& to, int* clear, int n_clear,
                       int early, cudaStream_t stream) {
    const int k_blocks = f4_k_blocks(K);
    int blocks;
    const bool wide = (long long)rows * k_blocks >= 4LL * (FR_THREADS / 16) * ssb_sm_count();
    const FrStep step = fr_step(rows, wide ? k_blocks : 2 * k_blocks, wide ? 2 : 1, &blocks);
    if ((long long)rows + step.rows * 4LL + 4 > INT_MAX) return SSB_ERR_BAD_SIZE;
    auto kernel = to.slot ? (wide ? fp4_quantize_kernel<T, 2, 16, true> : fp4_quantize_kernel<T, 1, 8, true>)
                          : (wide ? fp4_quantize_kernel<T, 2, 16, false> : fp4_quantize_kernel<T, 1, 8, false>);
    return ssb_launch(kernel, dim3(blocks), dim3(FR_THREADS), 0, stream, true,
                      x, ldx, codes, scales, rows, K, to, step, k_blocks, clear, n_clear, early);
}

// x: rows x K, rows of 16-byte pieces; ``per_expert`` rows of them are a matrix; clear: words zeroed on the way.  early: the next
// launch may begin meanwhile.
SSB_API int ssb_fp4_quantize(const void* x, long long ldx, int dtype, void* codes, void* scales, int rows, int K, int per_expert, int inter,
                             int* clear, int n_clear, int early, cudaStream_t stream) {
    const int rc = fr_sizes(rows, K, per_expert, inter);
    if (rc || rows == 0) return rc;
    if (((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15) return SSB_ERR_BAD_SIZE;
    const FrRows to{per_expert, inter, nullptr, 1, 7};
    if (dtype == SSB_BF16) return fr_quantize((const bf16*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, rows, K, to, clear, n_clear, early, stream);
    if (dtype == SSB_F32) return fr_quantize((const float*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, rows, K, to, clear, n_clear, early, stream);
    return SSB_ERR_BAD_DTYPE;
}

// The tokens' rows, each to the rows that its ``top`` pairs' ``slot`` names (-1: none) in tiles of ``tile_rows``.
SSB_API int ssb_fp4_quantize_pairs(const void* x, long long ldx, int dtype, void* codes, void* scales, int tokens, int top, int K,
                                   const int* slot, int tile_rows, cudaStream_t stream) {
    const FrRows to{tokens, 0, slot, top, tile_rows == 16 ? 4 : tile_rows == 64 ? 6 : 8};
    if (dtype == SSB_BF16) return fr_quantize((const bf16*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, tokens, K, to, nullptr, 0, 1, stream);
    if (dtype == SSB_F32) return fr_quantize((const float*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, tokens, K, to, nullptr, 0, 1, stream);
    return SSB_ERR_BAD_DTYPE;
}

template <typename T>
static int fr_values(const uint8_t* codes, const uint8_t* scales, T* out, long long ldo, int rows, int K, int per_expert, int inter,
                     cudaStream_t stream) {
    const long long units = (long long)rows * ((K + 127) / 128);
    // one unit a half-warp where more would leave SMs without work
    const int turns = units >= 4LL * (FR_THREADS / 16) * ssb_sm_count() ? FR_TURNS : 1;
    int blocks;
    const FrStep step = fr_step(rows, (K + 127) / 128, turns, &blocks);
    if ((long long)rows + step.rows * 4LL + 4 > INT_MAX) return SSB_ERR_BAD_SIZE;
    return ssb_launch(turns == 1 ? fp4_values_kernel<T, 1> : fp4_values_kernel<T, FR_TURNS>, dim3(blocks), dim3(FR_THREADS), 0, stream, true,
                      codes, scales, out, ldo, rows, K, per_expert, inter, step, f4_k_blocks(K));
}

SSB_API int ssb_fp4_values(const void* codes, const void* scales, void* out, long long ldo, int dtype, int rows, int K, int per_expert,
                           int inter, cudaStream_t stream) {
    const int rc = fr_sizes(rows, K, per_expert, inter);
    if (rc || rows == 0) return rc;
    if (((uintptr_t)out | (uintptr_t)codes | (uintptr_t)scales) & 15) return SSB_ERR_BAD_SIZE;
    const uint8_t *c = (const uint8_t*)codes, *sc = (const uint8_t*)scales;
    if (dtype == SSB_BF16) return fr_values(c, sc, (bf16*)out, ldo, rows, K, per_expert, inter, stream);
    if (dtype == SSB_F32) return fr_values(c, sc, (float*)out, ldo, rows, K, per_expert, inter, stream);
    return SSB_ERR_BAD_DTYPE;
}

SSB_PACKED(ssb_fp4_quantize)
SSB_PACKED(ssb_fp4_values)
