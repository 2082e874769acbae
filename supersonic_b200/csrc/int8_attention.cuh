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
    int most_new = 0x7fffffff;    // rows that a sequence may have
    int most_start = 0;           // see ia_sequence
};

// A sequence of the step's batch as every kernel here takes it: the rows it has of those there are, its slot (negative: it has none, its
// rows are zeros) and the tokens before it.  A key lies in the table's 64 max_pages places, under a page id of the pool; one behind the
// table's end or under any other id is seen by nobody.  A start that lies farther behind the end than rows can tell is taken back to
// where they cannot (most_start): positions hold in 32 bits, and a single token spans the table's pages or its window's at most.
struct IaSeq { int row0, n_new, start, slot; };
__device__ __forceinline__ IaSeq ia_sequence(const IaArgs& a, int b) {
    const int row0 = a.cu_new[b], slot = a.seq_slot[b], start = a.seq_start[b];
    return IaSeq{row0, min(min(a.cu_new[b + 1], a.rows) - row0, a.most_new), min(start, a.most_start), slot < a.n_slots && start >= 0 ? slot : -1};
}
__device__ __forceinline__ bool ia_in_pool(const IaArgs& a, int page) { return page >= 0 && page < a.n_pages; }

// Prompts of bfloat16 rows on tcgen05 (int8_attention_tc.cu): whether it takes these, the float32 scratch it needs, and the launch.
bool ia_tc_takes(int dtype, int head_dim, int max_new, float scale);
long long ia_tc_scratch(int n_seqs, int rows, int max_new, int max_pages, int n_q, int n_kv, int head_dim);
int ia_tc_launch(const IaArgs& a, int max_new, float* scratch, int* error_word, cudaStream_t stream);
