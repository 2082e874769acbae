// What the kernel of few rows (fp4_few.cu) is asked for.
#pragma once
#include "common.cuh"

constexpr int FW_MOST_PAIRS = 256;        // (token, choice) pairs that a block sorts for itself
enum { FW_STORE = 0, FW_GATED = 1, FW_ACT = 2 };

struct FwArgs {
    const uint8_t *w, *ws;                 // weights [experts][N][K / 2] and their scales
    const void* x; long long ldx; int dtype; const uint8_t* xs;       // rows, ldx elements apart; dtype -1: codes, with the scales xs
    void* out; uint8_t* out_scales; long long ldo; int is_f32, add;   // FW_STORE: rows of ldo elements; else codes, rows of ldo bytes, and their scales
    int M, N, K;                           // rows, rows of a weight matrix, numbers a row
    int kind; float limit; const float* row_scale; int inner_blocks;  // as FlOut's (fp4_linear.cu)
    const int* expert_of; int pairs, top, experts;                    // of a list: pair p's expert; its row of x is p / top (codes: p), of out p
    int k_warps, slots, k_blocks;          // the plan's
};

// The pairs (token, choice) by expert, in their order, for a block that has them to itself (pairs <= FW_MOST_PAIRS <= its threads): tile
// t, up to ROWS neighbours of one expert tile_expert[t], is pair_of[tile_first[t]], ..., tile_rows[t] of them.  Pairs whose expert is
// none are left out.  All threads call it; the number of tiles.
template <int ROWS>
__device__ __forceinline__ int fw_sort_pairs(const int* __restrict__ expert_of, int pairs, int experts, int* pair_of, int* tile_first,
                                             int* tile_rows, int* tile_expert) {
    const int tid = threadIdx.x;
    int e = -1, first = 0, place = 0, same = 0;
    if (tid < pairs) {
        e = expert_of[tid];
        if ((unsigned)e >= (unsigned)experts) e = -1;
        tile_first[tid] = e;
    }
    __syncthreads();
    if (e >= 0)
#pragma unroll 8
        for (int q = 0; q < pairs; ++q) {
            const int f = tile_first[q];
            first += f >= 0 && f < e;
            place += f == e && q < tid;
            same += f == e;
        }
    if (tid < FW_MOST_PAIRS) tile_rows[tid] = 0;
    __syncthreads();
    const bool starts = e >= 0 && place % ROWS == 0;
    const int rows = min(ROWS, same - place);
    if (e >= 0) pair_of[first + place] = tid;
    if (starts) tile_rows[first + place] = 1;
    __syncthreads();
    int before = 0;
    if (starts)
#pragma unroll 8
        for (int q = 0; q < first + place; ++q) before += tile_rows[q];
    const int tiles = __syncthreads_count(starts);
    if (starts) { tile_first[before] = first + place; tile_rows[before] = rows; tile_expert[before] = e; }
    __syncthreads();
    return tiles;
}

bool fw_takes(int M, int N, int K, int mode);
bool fw_takes_list(int pairs, int experts, int N, int K, int mode);
int fw_product(FwArgs a, int mode, cudaStream_t stream);
int fw_product_list(FwArgs a, int mode, cudaStream_t stream);
