// What the kernels of few rows (fp4_few.cu, fp4_step.cu) are asked for.
#pragma once
#include "common.cuh"

enum { FW_STORE = 0, FW_GATED = 1, FW_ACT = 2 };

struct FwArgs {
    const uint8_t *w, *ws;                 // weights [experts][N][K / 2] and their scales
    const void* x; long long ldx; int dtype; const uint8_t* xs;       // rows, ldx elements apart; dtype -1: codes, with the scales xs
    void* out; uint8_t* out_scales; long long ldo; int is_f32, add;   // FW_STORE: rows of ldo elements; else codes, rows of ldo bytes, and their scales
    int M, N, K;                           // rows, rows of a weight matrix, numbers a row
    int kind; float limit; const float* row_scale; int inner_blocks;  // as FlOut's (fp4_linear.cu)
    int k_warps, slots, k_blocks;          // the plan's
};

bool fw_takes(int M, int N, int K, int mode);
// early: the launch may begin, and read its weights, while the one in front of it still runs.
int fw_product(FwArgs a, int mode, bool early, cudaStream_t stream);
