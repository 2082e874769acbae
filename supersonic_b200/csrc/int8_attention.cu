// Attention over a cache in 8 bits (see int8_cache.cu), in packed sequences: row i of a sequence that held ``start`` tokens before
// the step sees the keys start + i - window < j <= start + i of its slot.
//   s_ij = scale * ks_j * (q_i . kc_j),   o_i = sum_j softmax_j(s_ij) * vs_j * vc_j,   lse_i = ln sum_j exp(s_ij)
// with codes kc, vc and their blocks' scales ks, vs.  The rows that keep account add exp(s_ij - lse_i), summed over the query
// heads of a kv head, to the weight of key j.
#include "common.cuh"
#include <math.h>

typedef __nv_bfloat16 bf16;

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
    int ldq, ldo, rows, n_seqs, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, block, window, weigh_last;
    float scale;
};

// Any head size that is a multiple of 16 up to 256: a warp a row and query head, words of four codes over its lanes.
template <typename T>
__global__ void __launch_bounds__(128)
int8_attention_plain_kernel(const IaArgs a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = a.head_dim / 4;
    const int row = blockIdx.x, head = blockIdx.y * 4 + warp;
    if (head >= a.n_q) return;
    const int kvh = head / (a.n_q / a.n_kv);
    int lo = 0, hi = a.n_seqs - 1;                               // the last sequence that begins at or before the row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu_new[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const int s = row < a.cu_new[a.n_seqs] && row >= a.cu_new[0] ? a.seq_slot[lo] : -1;
    const int at = a.seq_start[lo] + row - a.cu_new[lo];
    const int last = s < 0 || s >= a.n_slots ? -1 : min(at, a.max_pages * IA_PAGE - 1);
    const int from = a.window > 0 ? max(0, at - a.window + 1) : 0;
    float q[2][4], o[2][4] = {};
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            q[w][e] = lane + 32 * w < words ? ssb_to_float(((const T*)a.q)[(size_t)row * a.ldq + (size_t)head * a.head_dim + 4 * (lane + 32 * w) + e]) : 0.f;
    float m = -INFINITY, l = 0.f;
    for (int j = from; j <= last; ++j) {
        const int page = a.page_table[(size_t)s * a.max_pages + (j >> 6)];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t r = ((size_t)page * a.n_kv + kvh) * IA_PAGE + (j & 63);
        float d = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (lane + 32 * w < words) {
                const uint32_t c = reinterpret_cast<const uint32_t*>(a.k + r * a.head_dim)[lane + 32 * w];
#pragma unroll
                for (int e = 0; e < 4; ++e) d = fmaf(q[w][e], (float)(int8_t)(c >> (8 * e)), d);
            }
#pragma unroll
        for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
        d *= a.scale * a.k_scale[r / a.block];
        const float m_new = fmaxf(m, d), keep = m == -INFINITY ? 0.f : expf(m - m_new), p = expf(d - m_new);
        l = l * keep + p;
        m = m_new;
        const float pv = p * a.v_scale[r / a.block];
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (lane + 32 * w < words) {
                const uint32_t c = reinterpret_cast<const uint32_t*>(a.v + r * a.head_dim)[lane + 32 * w];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[w][e] = fmaf(pv, (float)(int8_t)(c >> (8 * e)), o[w][e] * keep);
            }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int w = 0; w < 2; ++w)
        if (lane + 32 * w < words)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                ((T*)a.out)[(size_t)row * a.ldo + (size_t)head * a.head_dim + 4 * (lane + 32 * w) + e] = ssb_from_float<T>(o[w][e] * inv);
    if (lane == 0 && a.lse) a.lse[(size_t)row * a.n_q + head] = l > 0.f ? m + logf(l) : -INFINITY;
}

// What the last rows of every sequence attend to: a warp a key, over those rows and the heads of the group; the key's weight is its
// alone to add to, so the sum has one order.
template <typename T>
__global__ void __launch_bounds__(128)
int8_weigh_plain_kernel(const IaArgs a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = a.head_dim / 4, group = a.n_q / a.n_kv;
    const int kvh = blockIdx.y, b = blockIdx.z, s = a.seq_slot[b];
    const int row0 = a.cu_new[b], n_new = a.cu_new[b + 1] - row0, start = a.seq_start[b];
    if (s < 0 || s >= a.n_slots || n_new <= 0) return;
    const int i0 = max(0, n_new - a.weigh_last);
    const int end = min(start + n_new, a.max_pages * IA_PAGE);
    const int begin = a.window > 0 ? max(0, start + i0 - a.window + 1) : 0;
    for (int j = begin + (int)blockIdx.x * 4 + warp; j < end; j += gridDim.x * 4) {
        const int page = a.page_table[(size_t)s * a.max_pages + (j >> 6)];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t r = ((size_t)page * a.n_kv + kvh) * IA_PAGE + (j & 63);
        const float ks = a.scale * a.k_scale[r / a.block];
        float sum = 0.f;
        for (int i = max(i0, j - start); i < n_new; ++i) {
            if (a.window > 0 && j <= start + i - a.window) break;
            for (int h = 0; h < group; ++h) {
                const size_t row = (size_t)(row0 + i), head = (size_t)(kvh * group + h);
                float d = 0.f;
                for (int w = lane; w < words; w += 32) {
                    const uint32_t c = reinterpret_cast<const uint32_t*>(a.k + r * a.head_dim)[w];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        d = fmaf(ssb_to_float(((const T*)a.q)[row * a.ldq + head * a.head_dim + 4 * w + e]), (float)(int8_t)(c >> (8 * e)), d);
                }
#pragma unroll
                for (int x = 16; x; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
                sum += expf(d * ks - a.lse[row * a.n_q + head]);
            }
        }
        if (lane == 0) a.weight[r] += sum;
    }
}

SSB_API int ssb_int8_attention_plain(const void* q, int ldq, int dtype, void* out, int ldo, float* lse, const void* k, const void* v,
                                     const float* k_scale, const float* v_scale, float* weight, const int* page_table, int n_slots,
                                     int max_pages, int n_pages, const int* cu_new, const int* seq_start, const int* seq_slot,
                                     int n_seqs, int rows, int n_q, int n_kv, int head_dim, int block, int window, int weigh_last,
                                     float scale, cudaStream_t stream) {
    if (n_seqs <= 0 || rows <= 0) return 0;
    if (head_dim % 16 || head_dim <= 0 || head_dim > 256 || n_kv <= 0 || n_q % n_kv || (block != 16 && block != 32 && block != 64) ||
        (n_q + 3) / 4 > 65535 || n_kv > 65535)
        return SSB_ERR_BAD_SIZE;
    if (weigh_last > 0 && (!weight || !lse || n_seqs > 65535)) return SSB_ERR_BAD_SIZE;
    const IaArgs a{q, out, lse, (const int8_t*)k, (const int8_t*)v, k_scale, v_scale, weight, page_table, cu_new, seq_start, seq_slot,
                   ldq, ldo, rows, n_seqs, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, block, window, weigh_last, scale};
    const dim3 grid(rows, (n_q + 3) / 4), wgrid(min((max_pages * IA_PAGE + 3) / 4, 512), n_kv, n_seqs);
    if (dtype == SSB_BF16) {
        int8_attention_plain_kernel<bf16><<<grid, 128, 0, stream>>>(a);
        if (weigh_last > 0) int8_weigh_plain_kernel<bf16><<<wgrid, 128, 0, stream>>>(a);
    } else if (dtype == SSB_F32) {
        int8_attention_plain_kernel<float><<<grid, 128, 0, stream>>>(a);
        if (weigh_last > 0) int8_weigh_plain_kernel<float><<<wgrid, 128, 0, stream>>>(a);
    } else {
        return SSB_ERR_BAD_DTYPE;
    }
    return ssb_launch_status();
}
