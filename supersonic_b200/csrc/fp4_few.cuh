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

bool fw_takes(int M, int N, int K, int mode);
bool fw_takes_list(int pairs, int experts, int N, int K, int mode);
int fw_product(FwArgs a, int mode, cudaStream_t stream);
int fw_product_list(FwArgs a, int mode, cudaStream_t stream);
