// What the kernels of attention over the 8-bit cache are given.
#pragma once
#include "common.cuh"

constexpr int IA_PAGE = 64;

struct IaArgs {
    const void* q;                // [rows, ldq]
    void* out;                    // [rows, ldo]
    float* lse;                   // [rows, n_q]
    const int8_t* k;
    const int8_t* v;
    const float* k_scale;
    const float* v_scale;
    float* weight;
    const int* page_table;
    const int* cu_new;
    const int* seq_start;
    const int* seq_slot;
    int ldq, ldo, rows, n_seqs, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, shift, window, weigh_last;    // 1 << shift tokens a scale
    float scale;
};

// Prompts of bfloat16 rows on tcgen05 (int8_attention_tc.cu): whether it takes these, and the launch.
bool ia_tc_takes(const IaArgs& a, int dtype, int max_new);
int ia_tc_launch(const IaArgs& a, int max_new, int* error_word, cudaStream_t stream);
