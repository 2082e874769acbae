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

// Prompts of bfloat16 rows on tcgen05 (int8_attention_tc.cu): whether it takes these, the float32 scratch it needs, and the launch.
bool ia_tc_takes(int dtype, int head_dim, int max_new, float scale);
long long ia_tc_scratch(int n_seqs, int rows, int max_new, int max_pages, int n_q, int n_kv, int head_dim);
int ia_tc_launch(const IaArgs& a, int max_new, float* scratch, int* error_word, cudaStream_t stream);
