// Products of a step's rows on tcgen05 in one launch (fp4_step.cu).
#pragma once
#include "fp4_few.cuh"

// Blocks that share a tile of 128 channels, or 0: the product is not for this kernel.
int fs_parts(int M, int N, int K);
// What the arguments say; x: codes, with the scales xs.  mode: FL_*.  early: as fw_product's.
int fs_product(FwArgs a, int mode, int parts, bool early, int* error_word, cudaStream_t stream);
