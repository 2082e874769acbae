// Feed-forward experts: which experts a token uses, the tokens of a step grouped by expert,
// matrix products per group, and the weighted sum of a token's expert outputs.
//
// A step's tokens each use `top` experts: P = T * top (token, choice) pairs.  A router fills
// expert_of[P] and pair_weight[P]; group_by_expert sorts the pairs by expert (row r of the sorted
// order is pair order[r]) and lists the row tiles of every expert, all on the device, so the
// launches that follow have sizes that depend on T alone and can be captured in a graph.  The
// grouped product walks that tile list: a block that finds its tile index beyond the count has
// nothing to do.  An expert's output rows are written per pair and summed per token in the order
// of the choices, so no result depends on the other tokens of the step.
#include "common.cuh"
#include "packed_call.cuh"
#include <math.h>

typedef __nv_bfloat16 bf16;

// ---------------------------------------------------------------------------------------
// table router: a token's experts are row token_id of an integer table, equal weights
// ---------------------------------------------------------------------------------------
__global__ void route_table_kernel(const int* __restrict__ token_ids, const int* __restrict__ table, int vocab,
                                   int top, int n_experts, int* __restrict__ expert_of,
                                   float* __restrict__ pair_weight, int n_pairs) {
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const int p = blockIdx.x * blockDim.x + threadIdx.x;
    if (p >= n_pairs) return;
    const int id = token_ids[p / top];
    int e = (id >= 0 && id < vocab) ? table[(size_t)id * top + p % top] : 0;
    if (e < 0 || e >= n_experts) e = 0;                  // the host refuses such tables; never index out of range
    expert_of[p] = e;
    pair_weight[p] = 1.0f / (float)top;
}

SSB_API int ssb_route_table(const int* token_ids, const int* table, int vocab, int top, int n_experts,
                            int* expert_of, float* pair_weight, int n_tokens, int pdl, cudaStream_t stream) {
    const long long n = (long long)n_tokens * top;
    if (n <= 0) return 0;
    if (n > (1ll << 30)) return SSB_ERR_BAD_SIZE;
    const int rc = ssb_launch(route_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, pdl != 0,
                              token_ids, table, vocab, top, n_experts, expert_of, pair_weight, (int)n);
    return rc ? rc : ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// sigmoid router with groups.  The logits z [tokens, ld] are float32 (a product of their own); s = sigmoid(z); an
// expert is chosen by s + correction among the experts of the `keep` best groups (the experts form `n_groups` equal
// groups of neighbours; a group's score is the sum of its two largest choice scores; the other groups' experts
// count as minus infinity); the `top` largest choice scores win, the lower index at equal scores; an expert's weight
// is its s (without the correction) times `scale`, not renormalized.  extra_col >= 0: the sigmoid of that column goes
// to extra_out[t] (the gate of a shared expert, whose row rides along in the product).  One warp per token: lanes
// over experts for the scores and for every pick, lanes over groups for the groups' scores.
// ---------------------------------------------------------------------------------------
constexpr int RG_THREADS = 128;

__global__ void __launch_bounds__(RG_THREADS)
route_sigmoid_groups_kernel(const float* __restrict__ z, int ld, const float* __restrict__ correction, int n_tokens,
                            int n_experts, int n_groups, int keep, int top, float scale, int extra_col,
                            int* __restrict__ expert_of, float* __restrict__ pair_weight, float* __restrict__ extra_out) {
    extern __shared__ float rg_smem[];                   // per warp: [n_experts] s, [n_experts] choice, [n_groups] group scores
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * (RG_THREADS / 32) + warp;
    if (t >= n_tokens) return;
    float* s_s = rg_smem + (size_t)warp * (2 * n_experts + n_groups);
    float* c_s = s_s + n_experts;
    float* g_s = c_s + n_experts;
    const float* zr = z + (size_t)t * ld;
    for (int e = lane; e < n_experts; e += 32) {
        const float sg = 1.0f / (1.0f + expf(-zr[e]));
        s_s[e] = sg;
        c_s[e] = sg + (correction ? correction[e] : 0.f);
    }
    if (extra_col >= 0 && lane == 0) extra_out[t] = 1.0f / (1.0f + expf(-zr[extra_col]));
    __syncwarp();
    const int per = n_experts / n_groups;
    if (keep < n_groups) {
        for (int g = lane; g < n_groups; g += 32) {
            float a = -INFINITY, b = -INFINITY;           // the two largest of the group
            for (int e = g * per; e < (g + 1) * per; ++e) {
                const float v = c_s[e];
                if (v > a) { b = a; a = v; } else if (v > b) b = v;
            }
            g_s[g] = per > 1 ? a + b : a;
        }
        __syncwarp();
        // a group stays if fewer than `keep` groups come before it (a larger score, or the same at a lower index)
        for (int g = lane; g < n_groups; g += 32) {
            int before = 0;
            for (int o = 0; o < n_groups; ++o) before += (g_s[o] > g_s[g] || (g_s[o] == g_s[g] && o < g)) ? 1 : 0;
            if (before >= keep)
                for (int e = g * per; e < (g + 1) * per; ++e) c_s[e] = -INFINITY;
        }
        __syncwarp();
    }
    for (int k = 0; k < top; ++k) {
        float bv = -INFINITY;
        int best = 0x7fffffff;
        for (int e = lane; e < n_experts; e += 32) {
            const float v = c_s[e];
            if (v > bv) { bv = v; best = e; }             // false for minus infinity and for a taken expert's NaN; rising e: the lower index stays
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oe = __shfl_xor_sync(0xffffffffu, best, o);
            if (ov > bv || (ov == bv && oe < best)) { bv = ov; best = oe; }
        }
        if (best == 0x7fffffff) {                         // fewer live experts than `top`: the lowest not yet taken, weight 0
            best = 0;
            for (int e = 0; e < n_experts; ++e) {
                bool taken = false;
                for (int j = 0; j < k; ++j) taken = taken || expert_of[(size_t)t * top + j] == e;
                if (!taken) { best = e; break; }
            }
            bv = -INFINITY;
        }
        if (lane == 0) {
            expert_of[(size_t)t * top + k] = best;
            pair_weight[(size_t)t * top + k] = bv == -INFINITY ? 0.f : s_s[best] * scale;
            c_s[best] = __int_as_float(0x7fc00000);       // taken
        }
        __syncwarp();
    }
}

SSB_API int ssb_route_sigmoid_groups(const float* z, int ld, const float* correction, int n_tokens, int n_experts,
                                     int n_groups, int keep, int top, float scale, int extra_col, int* expert_of,
                                     float* pair_weight, float* extra_out, int pdl, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (n_experts <= 0 || n_groups <= 0 || n_experts % n_groups || keep < 1 || keep > n_groups || top < 1 ||
        top > n_experts || n_experts > 2048 || ld < n_experts || extra_col >= ld || (extra_col >= 0 && extra_out == nullptr))
        return SSB_ERR_BAD_SIZE;
    const size_t smem = (size_t)(RG_THREADS / 32) * (2 * n_experts + n_groups) * sizeof(float);
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(route_sigmoid_groups_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    const int rc = ssb_launch(route_sigmoid_groups_kernel, dim3((n_tokens + RG_THREADS / 32 - 1) / (RG_THREADS / 32)),
                              dim3(RG_THREADS), smem, stream, pdl != 0, z, ld, correction, n_tokens, n_experts, n_groups, keep,
                              top, scale, extra_col, expert_of, pair_weight, extra_out);
    return rc ? rc : ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// softmax router.  s = softmax(z + bias) over all experts (float32; the bias is optional); the `top` experts with the largest scores win, the lower
// index at equal scores; an expert's weight is its s times `scale`, with `renormalize` divided by the sum of the
// chosen scores (+ 1e-20).  One warp per token, lanes over experts.
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(RG_THREADS)
route_softmax_kernel(float* __restrict__ z, int ld, const float* __restrict__ bias, int n_tokens, int n_experts, int top, int renormalize, float scale,
                     int clear, int* __restrict__ expert_of, float* __restrict__ pair_weight) {
    extern __shared__ float rs_smem[];                   // per warp: [n_experts] scores, [top] chosen scores
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * (RG_THREADS / 32) + warp;
    if (t >= n_tokens) return;
    float* s_s = rs_smem + (size_t)warp * (n_experts + top);
    float* w_s = s_s + n_experts;
    float* zr = z + (size_t)t * ld;
    float m = -INFINITY;
    for (int e = lane; e < n_experts; e += 32) {
        s_s[e] = zr[e] + (bias ? bias[e] : 0.f);
        m = fmaxf(m, s_s[e]);
    }
    if (clear)
        for (int e = lane; e < ld; e += 32) zr[e] = 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float sum = 0.f;
    for (int e = lane; e < n_experts; e += 32) {
        const float p = expf(s_s[e] - m);
        s_s[e] = p;
        sum += p;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = 1.0f / sum;
    for (int e = lane; e < n_experts; e += 32) s_s[e] *= inv;
    __syncwarp();
    float chosen = 0.f;
    for (int k = 0; k < top; ++k) {
        float bv = -1.0f;                                 // below every score; a taken expert's mark is lower still
        int best = 0x7fffffff;
        for (int e = lane; e < n_experts; e += 32) {
            const float v = s_s[e];
            if (v > bv) { bv = v; best = e; }             // rising e: the lower index stays at equal scores
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
            const int oe = __shfl_xor_sync(0xffffffffu, best, o);
            if (ov > bv || (ov == bv && oe < best)) { bv = ov; best = oe; }
        }
        if (best == 0x7fffffff) {                         // only where scores are not numbers: some expert in range, weight 0
            best = k;
            bv = 0.f;
        }
        chosen += bv;
        if (lane == 0) {
            expert_of[(size_t)t * top + k] = best;
            w_s[k] = bv;
            s_s[best] = -2.0f;                            // taken
        }
        __syncwarp();
    }
    const float f = renormalize ? scale / (chosen + 1e-20f) : scale;
    for (int k = lane; k < top; k += 32) pair_weight[(size_t)t * top + k] = w_s[k] * f;
}

// clear: the whole row of z (ld columns) is zeroed behind the read.
SSB_API int ssb_route_softmax(float* z, int ld, const float* bias, int n_tokens, int n_experts, int top, int renormalize, float scale, int clear,
                              int* expert_of, float* pair_weight, int pdl, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (n_experts <= 0 || top < 1 || top > n_experts || n_experts > 2048 || ld < n_experts) return SSB_ERR_BAD_SIZE;
    const size_t smem = (size_t)(RG_THREADS / 32) * (n_experts + top) * sizeof(float);
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(route_softmax_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    const int rc = ssb_launch(route_softmax_kernel, dim3((n_tokens + RG_THREADS / 32 - 1) / (RG_THREADS / 32)),
                              dim3(RG_THREADS), smem, stream, pdl != 0, z, ld, bias, n_tokens, n_experts, top, renormalize, scale,
                              clear, expert_of, pair_weight);
    return rc ? rc : ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// router by scores.  s = softmax(z) or sigmoid(z) over all experts, c = s + correction; the experts form `n_groups` equal groups of
// neighbours, a group's score is its largest c or the sum of its two largest; of the experts of the `keep` best groups the `top`
// largest c win, in order, the lower index (expert, group) at equal scores; an expert's weight is its s times `scale`, with
// `renormalize` divided by the sum of the chosen s (+ 1e-20).  A logit that is NaN counts as minus infinity, whose s is zero, an infinite one as the
// largest number; a c, or a sum of two, that is NaN counts as minus infinity.  Without correction the larger logit comes first, also where both have the same s.
//
// What is chosen is chosen by c in 64 bits.  c in 32 bits is within rs_near of it, so a warp (a token, its experts in registers)
// chooses in 32 bits and looks whether two neighbours of its order, the last chosen and the next among them, or a kept and a
// dropped group, are closer than that: only then (a token in a thousand) it computes the groups' scores, or the candidates', in 64
// bits.  Without correction c grows with z, and the order is z's own.  The chosen experts' weights are made in 32 bits: an exponential, a
// sum and a quotient, some 1e-7 of them.
// 8,192 tokens, 256 experts in 8 groups, 8 chosen by corrected sigmoids: 19 us; 1,400 instructions
// a token and what they wait for bound it (the logits' 8.4 MB take 1.3); registers for eight blocks an SM leave the forms of up to 512 experts
// stack frames of 120 to 176 bytes, spills among them (16 experts a lane: 308 bytes loaded).  Choosing round by round, a reduction over the warp for the largest and
// one for its expert, and with all scores of a close token in 64 bits, it took 34; in that form with the latter in local memory 49.
// ---------------------------------------------------------------------------------------
constexpr int RS_MOST_GROUPS = 32;
enum { RS_SOFTMAX = 0, RS_SIGMOID = 1 };

struct RsArgs {
    const float* z; int ld; const float* correction;
    int n_tokens, n_experts, n_groups, keep, top, kind, by_two, renormalize; float scale;
    int* expert_of; float* pair_weight;
};
// How far two c in 32 bits may be from the exact ones together: each s to 3.5e-7 (its exponential, its quotient, z - max rounded: where
// that is large, s is small), softmax's sum, which all have in common, to 1.2e-6 of it (16 additions in a row at most), c's rounding.
__device__ __forceinline__ float rs_near(float c) { return 2e-6f + 1e-6f * fabsf(c); }
__device__ __forceinline__ float rs_logit(float z) {
    return z != z || z == -INFINITY ? -INFINITY : fminf(fmaxf(z, -3.4028234663852886e38f), 3.4028234663852886e38f);
}
// A number's bits in an order that is the numbers'; 0 is below all of them, 1 (a NaN's) below minus infinity's.
__device__ __forceinline__ uint32_t rs_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);         // (both zeros are one)
    return x != x ? 1u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float rs_from_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// s in 64 bits; softmax's ``most`` and ``total`` from rs_exact_sum.
struct RsSum { double most, total; };
__device__ __forceinline__ double rs_exact(const RsArgs& a, const float* zr, int e, const RsSum& sum) {
    const double z = (double)rs_logit(zr[e]);
    double c = !(z > -INFINITY) ? 0.0 : a.kind == RS_SOFTMAX ? exp(z - sum.most) / sum.total : 1.0 / (1.0 + exp(-z));
    if (a.correction) c += (double)a.correction[e];
    return c != c ? -INFINITY : c;
}
__device__ __noinline__ RsSum rs_exact_sum(const RsArgs& a, const float* zr) {
    RsSum sum{-INFINITY, 0.0};
    if (a.kind != RS_SOFTMAX) return sum;
    const int lane = threadIdx.x & 31;
    float most = -INFINITY;
    for (int e = lane; e < a.n_experts; e += 32) most = fmaxf(most, rs_logit(zr[e]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    sum.most = (double)most;
    if (most > -INFINITY)
#pragma unroll 4
        for (int e = lane; e < a.n_experts; e += 32) sum.total += exp((double)rs_logit(zr[e]) - sum.most);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum.total += __shfl_xor_sync(0xffffffffu, sum.total, o);
    return sum;
}

// The groups that stay, where scores of 32 bits are too close: the lanes of each (bits), as the kernel below has them.
__device__ __noinline__ uint32_t rs_groups_exactly(const RsArgs& a, const float* zr, int log_share) {
    const int lane = threadIdx.x & 31, per = a.n_experts / a.n_groups, share = 1 << log_share, g = lane >> log_share;
    const RsSum sum = rs_exact_sum(a, zr);
    double first = -INFINITY, second = -INFINITY;
    if (g < a.n_groups)
#pragma unroll 4
        for (int i = lane & (share - 1); i < per; i += share) {
            const double c = rs_exact(a, zr, g * per + i, sum);
            second = fmax(second, fmin(first, c));
            first = fmax(first, c);
        }
    for (int o = share / 2; o > 0; o >>= 1) {
        const double f = __shfl_xor_sync(0xffffffffu, first, o), s = __shfl_xor_sync(0xffffffffu, second, o);
        second = fmax(fmin(first, f), fmax(second, s));
        first = fmax(first, f);
    }
    double mine = a.by_two && per > 1 ? first + second : first;
    if (mine != mine) mine = -INFINITY;
    int before = 0;
    for (int o = 0; o < a.n_groups; ++o) {
        const double other = __shfl_sync(0xffffffffu, mine, o << log_share);
        before += other > mine || (other == mine && o < g);
    }
    return __ballot_sync(0xffffffffu, g < a.n_groups && before < a.keep);
}
// The order of up to 32 candidates (``experts``, ascending), where scores of 32 bits are too close.
__device__ __noinline__ void rs_order_exactly(const RsArgs& a, const float* zr, const uint32_t* experts, int count, int* chosen) {
    const int lane = threadIdx.x & 31, e = lane < count ? (int)experts[lane] : 0;
    const RsSum sum = rs_exact_sum(a, zr);
    const double c = rs_exact(a, zr, e, sum);
    int place = 0;
    for (int i = 0; i < count; ++i) {
        const double other = __shfl_sync(0xffffffffu, c, i);
        place += other > c || (other == c && i < lane);
    }
    if (lane < count && place < a.top) chosen[place] = e;
}
// The choice among the experts of the groups that stay in 64 bits.  ``c``: room for all scores.
__device__ __noinline__ void rs_choose_exactly(const RsArgs& a, const float* zr, uint32_t stays, int log_share, double* c, int* chosen) {
    const int lane = threadIdx.x & 31, per = a.n_experts / a.n_groups;
    const RsSum sum = rs_exact_sum(a, zr);
    for (int e = lane; e < a.n_experts; e += 32) c[e] = rs_exact(a, zr, e, sum);
    __syncwarp();
    double last = INFINITY;
    int last_e = -1;
    for (int k = 0; k < a.top; ++k) {                     // the largest behind the last one chosen
        double best = -INFINITY;
        int best_e = 0x7fffffff;
        for (int e = lane; e < a.n_experts; e += 32) {
            const double v = c[e];
            if ((stays >> ((e / per) << log_share & 31) & 1) && (v < last || (v == last && e > last_e)) && (best_e == 0x7fffffff || v > best)) {
                best = v;
                best_e = e;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const double v = __shfl_xor_sync(0xffffffffu, best, o);
            const int e = __shfl_xor_sync(0xffffffffu, best_e, o);
            if (e != 0x7fffffff && (best_e == 0x7fffffff || v > best || (v == best && e < best_e))) { best = v; best_e = e; }
        }
        last = best;
        last_e = best_e;
        if (lane == 0) chosen[k] = best_e;
    }
    __syncwarp();
}

// A warp's shared memory: the experts' scores in 64 bits, or members of groups in 32, or a list of candidates; then the chosen.
constexpr int RS_LIST = 49;
__host__ __device__ __forceinline__ int rs_doubles(int n_experts, int n_groups, int top) {
    const int members = (n_experts + 4 * n_groups + 1) / 2;
    const int all = members > n_experts ? members : n_experts;
    return (all > RS_LIST ? all : RS_LIST) + (top + 1) / 2;
}

// A number in an order of 32 lanes' numbers, the largest first: the one that ``place`` others come before.
__device__ __forceinline__ uint32_t rs_sorted_at(uint32_t key, int place) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
        for (int o = k / 2; o > 0; o /= 2) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, key, o);
            key = ((lane & k) == 0) == ((lane & o) == 0) ? max(key, other) : min(key, other);
        }
    return __shfl_sync(0xffffffffu, key, place);
}

// PER: experts a lane (expert j * 32 + lane).  Eight blocks an SM where registers allow it: 8,192 tokens of 512 experts 32.6 us (39.6 as they
// come), of 256 18.6 (19.3; ten blocks 20.8).
template <int PER>
__global__ void __launch_bounds__(RG_THREADS, PER <= 16 ? 8 : 1)
route_scored_kernel(const RsArgs a) {
    // per warp: [n_experts] scores in 64 bits, over them in 32 bits groups' members, or 32 candidates and their order; [top] chosen
    extern __shared__ double rsc_smem[];
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * (RG_THREADS / 32) + warp;
    if (t >= a.n_tokens) return;
    const bool grouped = a.keep < a.n_groups;
    double* exact = rsc_smem + (size_t)warp * rs_doubles(a.n_experts, a.n_groups, a.top);
    float* member = (float*)exact;
    int* chosen = (int*)(exact + rs_doubles(a.n_experts, a.n_groups, 0));
    const float* zr = a.z + (size_t)t * a.ld;
    float z[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        z[j] = e < a.n_experts ? rs_logit(zr[e]) : -INFINITY;
    }
    float most = 0.f, inv = 1.f;
    if (a.kind == RS_SOFTMAX) {
        most = -INFINITY;
#pragma unroll
        for (int j = 0; j < PER; ++j) most = fmaxf(most, z[j]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        if (most > -INFINITY)
#pragma unroll
            for (int j = 0; j < PER; ++j) part[j & 3] += expf(z[j] - most);
        float total = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        inv = 1.f / total;
    }
    auto score = [&](float x) { return x == -INFINITY ? 0.f : a.kind == RS_SOFTMAX ? expf(x - most) * inv : 1.f / (1.f + expf(-x)); };
    // good enough to choose by, and to see what is close: its exponential is off by 2^-22 + |x| 2^-24 of itself, its quotient by 2^-22
    auto rough = [&](float x) { return x == -INFINITY ? 0.f : a.kind == RS_SOFTMAX ? __expf(x - most) * inv : __fdividef(1.f, 1.f + __expf(-x)); };
    uint32_t key[PER];                                   // of c, or without correction of z; 0: no expert, dropped or taken
    const int per = a.n_experts / a.n_groups;
    // as many lanes a group as there are for each: 32 / groups, down to a power of two
    const int log_share = a.n_groups <= 1 ? 5 : __clz(a.n_groups - 1) - 27;
    uint32_t stays = 0xffffffffu;
    // e / per of e < 2,048: half a step from a whole number at least, far more than the product is off
    const float per_inv = 1.f / (float)per;
    auto group_of = [&](int e) { return (int)(((float)e + 0.5f) * per_inv); };
    if (a.correction) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = j * 32 + lane;
            float c = e < a.n_experts ? rough(z[j]) + a.correction[e] : 0.f;
            c = c != c ? -INFINITY : c;
            key[j] = e < a.n_experts ? rs_key(c) : 0u;
            if (grouped && e < a.n_experts) member[e + 4 * group_of(e)] = c;
        }
    } else {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = j * 32 + lane;
            key[j] = e < a.n_experts ? rs_key(z[j]) : 0u;
            if (grouped && e < a.n_experts) member[e + 4 * group_of(e)] = a.by_two && per > 1 ? rough(z[j]) : z[j];
        }
    }
    if (grouped) {
        __syncwarp();
        // groups lie 4 words apart, so that their lanes meet no bank twice
        const int share = 1 << log_share, g = lane >> log_share;
        float first = -INFINITY, second = -INFINITY;
        if (g < a.n_groups)
            for (int i = lane & (share - 1); i < per; i += share) {
                const float c = member[g * (per + 4) + i];
                second = fmaxf(second, fminf(first, c));
                first = fmaxf(first, c);
            }
        for (int o = share / 2; o > 0; o >>= 1) {
            const float f = __shfl_xor_sync(0xffffffffu, first, o), s = __shfl_xor_sync(0xffffffffu, second, o);
            second = fmaxf(fminf(first, f), fmaxf(second, s));
            first = fmaxf(first, f);
        }
        float mine = a.by_two && per > 1 ? first + second : first;
        mine = mine != mine ? -INFINITY : mine;
        int before = 0;
        for (int o = 0; o < a.n_groups; ++o) {
            const float other = __shfl_sync(0xffffffffu, mine, o << log_share);
            before += other > mine || (other == mine && o < g);
        }
        const bool live = g < a.n_groups, kept = live && before < a.keep;
        const float worst_kept = rs_from_key(__reduce_min_sync(0xffffffffu, kept ? rs_key(mine) : 0xffffffffu));
        const float best_dropped = rs_from_key(__reduce_max_sync(0xffffffffu, live && !kept ? rs_key(mine) : 0u));
        stays = __ballot_sync(0xffffffffu, kept);
        // by the largest z alone nothing is rounded
        if ((a.correction || (a.by_two && per > 1)) && !(worst_kept - best_dropped > 2.f * rs_near(worst_kept)))
            stays = rs_groups_exactly(a, zr, log_share);
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (!(stays >> (group_of(j * 32 + lane) << log_share & 31) & 1)) key[j] = 0u;
        __syncwarp();
    }
    uint32_t mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) mine = max(mine, key[j]);
    // All of the top + 1 largest are at least the top + 1st of the lanes' largest.  What is that large (or could be) is few numbers more than
    // these: where there are 32 at most, a lane takes one, counts who comes before it, and its place is that.  (Else, and where lanes have two
    // experts each, round by round: 8,192 tokens of 64 experts, 6 chosen, 7.8 us so and 8.7 by candidates; of 256 below.)
    int count = 33;
    uint32_t* list = (uint32_t*)member;                  // [32] keys, [32] experts, [33] keys in order
    if (a.top < 32) {
        uint32_t least = rs_sorted_at(mine, a.top);
        if (a.correction && least > 1u) {
            const float c = rs_from_key(least);
            least = rs_key(c - 2.f * rs_near(c));
        }
        least = max(least, 1u);
        count = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const bool in = key[j] >= least;
            const uint32_t all = __ballot_sync(0xffffffffu, in);
            const int at = count + __popc(all & ((1u << lane) - 1));
            if (in && at < 32) { list[at] = key[j]; list[32 + at] = j * 32 + lane; }
            count += __popc(all);
        }
    }
    bool near = false;
    if (count <= 32) {
        list[64 + lane] = 0u;
        if (lane == 0) list[96] = 0u;
        __syncwarp();
        const uint32_t own = lane < count ? list[lane] : 0u;
        int place = 0;
        for (int i = 0; i < count; ++i) {                // equal keys lie in the order of their experts
            const uint32_t other = list[i];
            place += other > own || (other == own && i < lane);
        }
        if (lane < count) {
            list[64 + place] = own;
            if (place < a.top) chosen[place] = (int)list[32 + lane];
        }
        __syncwarp();
        if (a.correction) {
            const uint32_t here = list[64 + lane], next = list[65 + lane];
            const float c = rs_from_key(next);
            near = __any_sync(0xffffffffu, lane < a.top && next && !(rs_from_key(here) - c > rs_near(c)));
            if (near) rs_order_exactly(a, zr, list + 32, count, chosen);
        }
    } else {
        float before = INFINITY;
        for (int k = 0; k <= a.top; ++k) {               // one more than is chosen, to see how close it was
            const uint32_t best = __reduce_max_sync(0xffffffffu, mine);
            if (a.correction && best) {
                const float c = rs_from_key(best);
                near = near || !(before - c > rs_near(c));
                before = c;
            }
            if (k == a.top) break;
            int at = 0x7fffffff;                         // the lowest expert that has it
#pragma unroll
            for (int j = PER - 1; j >= 0; --j)
                if (key[j] == best) at = j * 32 + lane;
            at = __reduce_min_sync(0xffffffffu, at);
            mine = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (j * 32 + lane == at) key[j] = 0u;
                mine = max(mine, key[j]);
            }
            if (lane == 0) chosen[k] = at;
        }
        __syncwarp();
        if (near) rs_choose_exactly(a, zr, stays, log_share, exact, chosen);
    }
    __syncwarp();
    float sum = 0.f;
    for (int k = lane; k < a.top; k += 32) sum += score(rs_logit(zr[chosen[k]]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float f = a.renormalize ? a.scale / (sum + 1e-20f) : a.scale;
    for (int k = lane; k < a.top; k += 32) {
        const int e = chosen[k];
        a.expert_of[(size_t)t * a.top + k] = e;
        a.pair_weight[(size_t)t * a.top + k] = score(rs_logit(zr[e])) * f;
    }
}

template <int PER>
static int rs_launch(const RsArgs& a, int pdl, cudaStream_t stream) {
    const size_t smem = (size_t)(RG_THREADS / 32) * rs_doubles(a.n_experts, a.n_groups, a.top) * sizeof(double);
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(route_scored_kernel<PER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    const int rc = ssb_launch(route_scored_kernel<PER>, dim3((a.n_tokens + RG_THREADS / 32 - 1) / (RG_THREADS / 32)), dim3(RG_THREADS), smem,
                              stream, pdl != 0, a);
    return rc ? rc : ssb_launch_status();
}

SSB_API int ssb_route_scored(const float* z, int ld, const float* correction, int n_tokens, int n_experts, int n_groups, int keep, int top,
                             int kind, int by_two, int renormalize, float scale, int* expert_of, float* pair_weight, int pdl,
                             cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (n_experts <= 0 || n_experts > 2048 || n_groups <= 0 || n_groups > RS_MOST_GROUPS || n_experts % n_groups || keep < 1 || keep > n_groups ||
        top < 1 || top > keep * (n_experts / n_groups) || ld < n_experts || kind < RS_SOFTMAX || kind > RS_SIGMOID)
        return SSB_ERR_BAD_SIZE;
    const RsArgs a{z, ld, correction, n_tokens, n_experts, n_groups, keep, top, kind, by_two, renormalize, scale, expert_of, pair_weight};
    if (n_experts <= 64) return rs_launch<2>(a, pdl, stream);
    if (n_experts <= 256) return rs_launch<8>(a, pdl, stream);
    if (n_experts <= 512) return rs_launch<16>(a, pdl, stream);
    return rs_launch<64>(a, pdl, stream);
}
SSB_PACKED(ssb_route_scored)

// ---------------------------------------------------------------------------------------
// pairs sorted by expert.  One block: counts in shared memory, offsets and the tile list by one
// thread, then every pair takes the next free row of its expert.  The order inside a group is
// whatever the adds give; nothing downstream depends on it.
// meta: [0] number of tiles
// ---------------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024)
group_by_expert_kernel(const int* __restrict__ expert_of, int n_pairs, int n_experts, int tile_rows,
                       int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ tile_expert,
                       int* __restrict__ tile_row0, int* __restrict__ meta) {
    extern __shared__ int cnt[];                         // [n_experts] counts, then cursors
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    for (int e = threadIdx.x; e < n_experts; e += blockDim.x) cnt[e] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < n_pairs; p += blockDim.x) atomicAdd(&cnt[expert_of[p]], 1);
    __syncthreads();
    if (threadIdx.x == 0) {
        int row = 0, tile = 0;
        for (int e = 0; e < n_experts; ++e) {
            const int n = cnt[e];
            offsets[e] = row;
            cnt[e] = row;
            for (int r = 0; r < n; r += tile_rows) {
                tile_expert[tile] = e;
                tile_row0[tile] = row + r;
                ++tile;
            }
            row += n;
        }
        offsets[n_experts] = row;
        meta[0] = tile;
    }
    __syncthreads();
    for (int p = threadIdx.x; p < n_pairs; p += blockDim.x) order[atomicAdd(&cnt[expert_of[p]], 1)] = p;
}

SSB_API int ssb_group_by_expert(const int* expert_of, int n_pairs, int n_experts, int tile_rows, int* offsets,
                                int* order, int* tile_expert, int* tile_row0, int* meta, int pdl,
                                cudaStream_t stream) {
    if (n_pairs <= 0) return 0;
    if (n_experts <= 0 || n_experts > 8192 || tile_rows <= 0) return SSB_ERR_BAD_SIZE;
    const int rc = ssb_launch(group_by_expert_kernel, dim3(1), dim3(1024), (size_t)n_experts * sizeof(int), stream,
                              pdl != 0, expert_of, n_pairs, n_experts, tile_rows, offsets, order, tile_expert,
                              tile_row0, meta);
    return rc ? rc : ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// The same grouping over many blocks, with the rows of x copied into sorted order on the way (what the products that fetch
// whole boxes of rows read).  A block owns a run of neighbouring pairs.  It counts all pairs per expert and those before
// its own; an expert's first row is the sum of the counts of the experts before it, and a pair's place behind it is the
// number of pairs of its expert that come earlier: the order is stable, whatever the number of blocks.  Block 0 writes
// the offsets and the tile list.
// ---------------------------------------------------------------------------------------
constexpr int GR_THREADS = 256;

__global__ void __launch_bounds__(GR_THREADS)
group_gather_kernel(const int* __restrict__ expert_of, int n_pairs, int n_experts, int tile_rows, int chunk,
                    const uint4* __restrict__ x, int ldx, int top, int width, uint4* __restrict__ rows,
                    int* __restrict__ offsets, int* __restrict__ order, int* __restrict__ tile_expert,
                    int* __restrict__ tile_row0, int* __restrict__ meta) {
    extern __shared__ int gr_s[];                        // all [E], before [E], then [chunk] experts, [chunk] places
    int* all = gr_s;
    int* before = all + n_experts;
    int* mine = before + n_experts;
    int* place = mine + chunk;
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int lo = blockIdx.x * chunk, n = min(chunk, n_pairs - lo);
    for (int e = tid; e < 2 * n_experts; e += GR_THREADS) gr_s[e] = 0;
    __syncthreads();
    for (int p = tid; p < n_pairs; p += GR_THREADS) {
        const int e = expert_of[p];
        atomicAdd(&all[e], 1);
        if (p < lo) atomicAdd(&before[e], 1);
        if (p >= lo && p < lo + n) mine[p - lo] = e;
    }
    __syncthreads();
    if (warp == 0) {                                     // first rows (and tiles) of the experts, 32 at a time
        int row = 0, tile = 0;
        for (int e0 = 0; e0 < n_experts; e0 += 32) {
            const int e = e0 + lane, cnt = e < n_experts ? all[e] : 0, tiles = (cnt + tile_rows - 1) / tile_rows;
            int r = cnt, t = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int ru = __shfl_up_sync(0xffffffffu, r, o), tu = __shfl_up_sync(0xffffffffu, t, o);
                if (lane >= o) { r += ru; t += tu; }
            }
            const int first = row + r - cnt, tile0 = tile + t - tiles;
            if (e < n_experts) {
                before[e] += first;
                if (blockIdx.x == 0) {
                    offsets[e] = first;
                    for (int k = 0; k < tiles; ++k) {
                        tile_expert[tile0 + k] = e;
                        tile_row0[tile0 + k] = first + k * tile_rows;
                    }
                }
            }
            row += __shfl_sync(0xffffffffu, r, 31);
            tile += __shfl_sync(0xffffffffu, t, 31);
        }
        if (blockIdx.x == 0 && lane == 0) {
            offsets[n_experts] = row;
            meta[0] = tile;
        }
    }
    __syncthreads();
    for (int i = tid; i < n; i += GR_THREADS) {
        const int e = mine[i];
        int rank = 0;
        for (int j = 0; j < i; ++j) rank += mine[j] == e ? 1 : 0;
        const int at = before[e] + rank;
        place[i] = at;
        order[at] = lo + i;
    }
    if (rows == nullptr) return;
    __syncthreads();
    for (int i = warp; i < n; i += GR_THREADS / 32) {
        const uint4* src = x + (size_t)((lo + i) / top) * ldx;
        uint4* dst = rows + (size_t)place[i] * width;
#pragma unroll 4
        for (int c = lane; c < width; c += 32) dst[c] = src[c];
    }
}

// x [tokens, ldx] and rows [n_pairs, width] bfloat16 (columns and strides multiples of 8), or both null; chunk: pairs a block
SSB_API int ssb_group_gather(const int* expert_of, int n_pairs, int n_experts, int tile_rows, int chunk, const void* x, int ldx,
                             int top, int width, void* rows, int* offsets, int* order, int* tile_expert, int* tile_row0,
                             int* meta, int pdl, cudaStream_t stream) {
    if (n_pairs <= 0) return 0;
    if (n_experts <= 0 || n_experts > 2048 || tile_rows <= 0 || chunk < 1 || chunk > 4096 || top < 1) return SSB_ERR_BAD_SIZE;
    if (rows != nullptr && (x == nullptr || width % 8 || ldx % 8 || (((uintptr_t)x | (uintptr_t)rows) & 15))) return SSB_ERR_BAD_SIZE;
    const size_t smem = (size_t)(2 * n_experts + 2 * chunk) * sizeof(int);
    const int rc = ssb_launch(group_gather_kernel, dim3((n_pairs + chunk - 1) / chunk), dim3(GR_THREADS), smem, stream, pdl != 0,
                              expert_of, n_pairs, n_experts, tile_rows, chunk, (const uint4*)x, ldx / 8, top, width / 8,
                              (uint4*)rows, offsets, order, tile_expert, tile_row0, meta);
    return rc ? rc : ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// grouped product: for sorted row r of expert e, C[c_row(r), n] = sum_k A[a_row(r), k] W_e[n, k].
// a_row(r) = a_index ? a_index[r] / a_div : r;  c_row(r) = c_index ? c_index[r] : r.
// 64 x 64 tiles, the arithmetic of the plain matrix product (FMA sums of 16, added with compensation).
// ---------------------------------------------------------------------------------------
template <typename TA, typename TC>
__global__ void __launch_bounds__(256)
grouped_gemm_plain_kernel(const TA* __restrict__ A, int lda, const int* __restrict__ a_index, int a_div,
                          const TA* __restrict__ W, int ldw, long long w_expert, TC* __restrict__ C, int ldc,
                          const int* __restrict__ c_index, const int* __restrict__ offsets,
                          const int* __restrict__ tile_expert, const int* __restrict__ tile_row0,
                          const int* __restrict__ meta, int N, int K) {
    constexpr int BM = 64, BN = 64, BK = 16;
    __shared__ float As[BK][BM + 1];
    __shared__ float Ws[BK][BN + 1];
    __shared__ int a_rows[BM];
    if ((int)blockIdx.y >= meta[0]) return;
    const int e = tile_expert[blockIdx.y], r0 = tile_row0[blockIdx.y];
    const int r_end = min(offsets[e + 1], r0 + BM);
    const int tid = threadIdx.x;
    const int tx = tid % 16, ty = tid / 16;
    const int n0 = blockIdx.x * BN;
    W += (size_t)e * w_expert;
    if (tid < BM) {
        const int r = r0 + tid;
        a_rows[tid] = r < r_end ? (a_index ? a_index[r] / a_div : r) : -1;
    }
    __syncthreads();
    float acc[4][4], lost[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) { acc[i][j] = 0.f; lost[i][j] = 0.f; }
    for (int k0 = 0; k0 < K; k0 += BK) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int idx = tid + x * 256;
            const int r = idx / BK, c = idx % BK;
            const int k = k0 + c;
            const int m = a_rows[r], n = n0 + r;
            As[c][r] = (m >= 0 && k < K) ? ssb_to_float(A[(size_t)m * lda + k]) : 0.f;
            Ws[c][r] = (n < N && k < K) ? ssb_to_float(W[(size_t)n * ldw + k]) : 0.f;
        }
        __syncthreads();
        float part[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) part[i][j] = 0.f;
#pragma unroll
        for (int kk = 0; kk < BK; ++kk) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = As[kk][ty * 4 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = Ws[kk][tx * 4 + j];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(a[i], b[j], part[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y = __fsub_rn(part[i][j], lost[i][j]);
                const float t = __fadd_rn(acc[i][j], y);
                lost[i][j] = __fsub_rn(__fsub_rn(t, acc[i][j]), y);
                acc[i][j] = t;
            }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = r0 + ty * 4 + i;
        if (r >= r_end) continue;
        const size_t crow = c_index ? (size_t)c_index[r] : (size_t)r;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx * 4 + j;
            if (n < N) C[crow * ldc + n] = ssb_from_float<TC>(acc[i][j]);
        }
    }
}

SSB_API int ssb_grouped_gemm_plain(const void* A, int lda, const int* a_index, int a_div, const void* W, int ldw,
                                   long long w_expert, int in_dtype, void* C, int ldc, const int* c_index,
                                   int out_dtype, const int* offsets, const int* tile_expert, const int* tile_row0,
                                   const int* meta, int max_tiles, int N, int K, cudaStream_t stream) {
    if (max_tiles <= 0 || N <= 0) return 0;
    if (K <= 0 || max_tiles > 65535 || a_div <= 0) return SSB_ERR_BAD_SIZE;
    const dim3 grid((N + 63) / 64, max_tiles);
#define SSB_GG(TA, TC) \
    grouped_gemm_plain_kernel<TA, TC><<<grid, 256, 0, stream>>>((const TA*)A, lda, a_index, a_div, (const TA*)W, ldw, \
        w_expert, (TC*)C, ldc, c_index, offsets, tile_expert, tile_row0, meta, N, K)
    if (in_dtype == SSB_F32 && out_dtype == SSB_F32) SSB_GG(float, float);
    else if (in_dtype == SSB_BF16 && out_dtype == SSB_BF16) SSB_GG(bf16, bf16);
    else if (in_dtype == SSB_BF16 && out_dtype == SSB_F32) SSB_GG(bf16, float);
    else return SSB_ERR_BAD_DTYPE;
#undef SSB_GG
    return ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// residual[t, c] += sum_k pair_weight[t * top + k] * y[t * top + k, c], added in the order of k
// ---------------------------------------------------------------------------------------
template <typename T>
__global__ void expert_combine_kernel(float* __restrict__ residual, int ldr, const T* __restrict__ y, int ldy,
                                      const float* __restrict__ pair_weight, int top, int width, size_t total) {
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const size_t idx = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= total) return;
    const size_t t = idx / width;
    const int c = (int)(idx % width);
    float acc = 0.f;
    for (int k = 0; k < top; ++k)
        acc = fmaf(pair_weight[t * top + k], ssb_to_float(y[(t * top + k) * ldy + c]), acc);
    residual[t * ldr + c] += acc;
}

// The same sums in the same order, four columns a thread: bound by the pairs' rows, of which four are on their way at a time.
// 2,048 tokens of 6 experts, 2,048 columns: 38 us behind the products with a column a thread
// and two 64-bit divisions each, 25 so (the rows' 134 MB take 20).
template <typename T>
__global__ void __launch_bounds__(128)
expert_combine_vec_kernel(float* __restrict__ residual, int ldr, const T* __restrict__ y, int ldy,
                          const float* __restrict__ pair_weight, int top, int width) {
    constexpr int AHEAD = 4;
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const size_t t = blockIdx.x;
    const int c = (blockIdx.y * 128 + threadIdx.x) * 4;
    if (c >= width) return;
    float4* at = reinterpret_cast<float4*>(residual + t * ldr + c);
    float4 old = *at, acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* w = pair_weight + t * top;
    const T* src = y + t * top * (size_t)ldy + c;
    for (int k0 = 0; k0 < top; k0 += AHEAD) {
        float4 v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (k0 + k < top) {
                const T* p = src + (size_t)(k0 + k) * ldy;
                if constexpr (sizeof(T) == 4) {
                    v[k] = *reinterpret_cast<const float4*>(p);
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(p);
                    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
                    const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
                    v[k] = make_float4(lo.x, lo.y, hi.x, hi.y);
                }
            }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (k0 + k < top) {
                const float s = w[k0 + k];
                acc.x = fmaf(s, v[k].x, acc.x);
                acc.y = fmaf(s, v[k].y, acc.y);
                acc.z = fmaf(s, v[k].z, acc.z);
                acc.w = fmaf(s, v[k].w, acc.w);
            }
    }
    old.x += acc.x; old.y += acc.y; old.z += acc.z; old.w += acc.w;
    *at = old;
}

SSB_API int ssb_expert_combine(float* residual, int ldr, const void* y, int ldy, int y_dtype,
                               const float* pair_weight, int top, int n_tokens, int width, int pdl,
                               cudaStream_t stream) {
    const size_t total = (size_t)n_tokens * width;
    if (total == 0) return 0;
    if (top <= 0) return SSB_ERR_BAD_SIZE;
    const dim3 grid((unsigned)((total + 255) / 256));
    int rc;
    if (width % 4 == 0 && ldr % 4 == 0 && ldy % 4 == 0 && ((uintptr_t)residual & 15) == 0 &&
        ((uintptr_t)y & (y_dtype == SSB_F32 ? 15 : 7)) == 0 && width <= 65535 * 512 && (y_dtype == SSB_F32 || y_dtype == SSB_BF16)) {
        const dim3 pieces(n_tokens, (width / 4 + 127) / 128);
        rc = y_dtype == SSB_F32
            ? ssb_launch(expert_combine_vec_kernel<float>, pieces, dim3(128), 0, stream, pdl != 0, residual, ldr, (const float*)y, ldy, pair_weight, top, width)
            : ssb_launch(expert_combine_vec_kernel<bf16>, pieces, dim3(128), 0, stream, pdl != 0, residual, ldr, (const bf16*)y, ldy, pair_weight, top, width);
        return rc ? rc : ssb_launch_status();
    }
    if (y_dtype == SSB_F32)
        rc = ssb_launch(expert_combine_kernel<float>, grid, dim3(256), 0, stream, pdl != 0, residual, ldr,
                        (const float*)y, ldy, pair_weight, top, width, total);
    else if (y_dtype == SSB_BF16)
        rc = ssb_launch(expert_combine_kernel<bf16>, grid, dim3(256), 0, stream, pdl != 0, residual, ldr,
                        (const bf16*)y, ldy, pair_weight, top, width, total);
    else
        return SSB_ERR_BAD_DTYPE;
    return rc ? rc : ssb_launch_status();
}

// ---------------------------------------------------------------------------------------
// The same sum where it joins the stream through a norm of its own:
//     v = sum_k pair_weight[t, k] * y[t * top + k],   residual[t] += v / sqrt(mean(v^2) + eps) * w,
// and optionally the new stream rounded into next_out (what the next sublayer reads).  One block per token; the sums and
// the stream's row stay in registers for rows of up to 256 x 4 x CN_MAX columns in 16-byte pieces.
// ---------------------------------------------------------------------------------------
constexpr int CN_THREADS = 256;
constexpr int CN_MAX = 4;

__device__ __forceinline__ float cn_block_sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < CN_THREADS / 32; ++w) s += red[w];
    return s;
}

__device__ __forceinline__ void cn_store4(float* d, float4 o) { *reinterpret_cast<float4*>(d) = o; }
__device__ __forceinline__ void cn_store4(bf16* d, float4 o) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(o.x, o.y), b = __floats2bfloat162_rn(o.z, o.w);
    *reinterpret_cast<uint2*>(d) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <typename T>
__global__ void __launch_bounds__(CN_THREADS)
combine_rms_add_vec_kernel(float* __restrict__ residual, const float* __restrict__ y, const float* __restrict__ pair_weight,
                           int top, const float* __restrict__ w, float eps, int width, T* __restrict__ next_out) {
    __shared__ float red[CN_THREADS / 32];
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const size_t t = blockIdx.x;
    const int n4 = width / 4;
    const float4* y4 = reinterpret_cast<const float4*>(y + t * top * (size_t)width);
    float4* r4 = reinterpret_cast<float4*>(residual + t * width);
    const float4* w4 = reinterpret_cast<const float4*>(w);
    float4 v[CN_MAX], r[CN_MAX], g[CN_MAX];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < CN_MAX; ++i) {
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int c = threadIdx.x + i * CN_THREADS;
        if (c < n4) { r[i] = r4[c]; g[i] = w4[c]; }
    }
    for (int k = 0; k < top; ++k) {
        const float p = pair_weight[t * top + k];
#pragma unroll
        for (int i = 0; i < CN_MAX; ++i) {
            const int c = threadIdx.x + i * CN_THREADS;
            if (c < n4) {
                const float4 a = y4[(size_t)k * n4 + c];
                v[i].x = fmaf(p, a.x, v[i].x); v[i].y = fmaf(p, a.y, v[i].y);
                v[i].z = fmaf(p, a.z, v[i].z); v[i].w = fmaf(p, a.w, v[i].w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < CN_MAX; ++i)
        sq = fmaf(v[i].x, v[i].x, fmaf(v[i].y, v[i].y, fmaf(v[i].z, v[i].z, fmaf(v[i].w, v[i].w, sq))));
    const float inv = 1.0f / sqrtf(cn_block_sum(sq, red) / (float)width + eps);
#pragma unroll
    for (int i = 0; i < CN_MAX; ++i) {
        const int c = threadIdx.x + i * CN_THREADS;
        if (c >= n4) continue;
        float4 o;
        o.x = r[i].x + v[i].x * inv * g[i].x; o.y = r[i].y + v[i].y * inv * g[i].y;
        o.z = r[i].z + v[i].z * inv * g[i].z; o.w = r[i].w + v[i].w * inv * g[i].w;
        r4[c] = o;
        if (next_out != nullptr) {
            cn_store4(next_out + t * width + 4 * (size_t)c, o);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(CN_THREADS)
combine_rms_add_kernel(float* __restrict__ residual, const float* __restrict__ y, const float* __restrict__ pair_weight,
                       int top, const float* __restrict__ w, float eps, int width, T* __restrict__ next_out) {
    extern __shared__ float cn_row[];
    __shared__ float red[CN_THREADS / 32];
    ssb_pdl_launch_dependents();
    ssb_pdl_wait();
    const size_t t = blockIdx.x;
    float sq = 0.f;
    for (int c = threadIdx.x; c < width; c += CN_THREADS) {
        float v = 0.f;
        for (int k = 0; k < top; ++k) v = fmaf(pair_weight[t * top + k], y[(t * top + k) * width + c], v);
        cn_row[c] = v;
        sq = fmaf(v, v, sq);
    }
    const float inv = 1.0f / sqrtf(cn_block_sum(sq, red) / (float)width + eps);
    for (int c = threadIdx.x; c < width; c += CN_THREADS) {
        const float o = residual[t * width + c] + cn_row[c] * inv * w[c];
        residual[t * width + c] = o;
        if (next_out != nullptr) next_out[t * width + c] = ssb_from_float<T>(o);
    }
}

// residual [tokens, width], y [tokens * top, width], w [width], next_out [tokens, width] or null: all contiguous
SSB_API int ssb_combine_rms_add(float* residual, const float* y, const float* pair_weight, int top, const float* w, float eps,
                                int n_tokens, int width, void* next_out, int next_dtype, int pdl, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (top <= 0 || width <= 0 || (size_t)width * sizeof(float) > 200 * 1024) return SSB_ERR_BAD_SIZE;
    const bool vec = width % 4 == 0 && width <= CN_THREADS * 4 * CN_MAX &&
        (((uintptr_t)residual | (uintptr_t)y | (uintptr_t)w | (uintptr_t)next_out) & 15) == 0;
    const size_t smem = vec ? 0 : (size_t)width * sizeof(float);
    int rc;
#define SSB_CN(TYPE)                                                                                                  \
    {                                                                                                                 \
        auto kern = vec ? combine_rms_add_vec_kernel<TYPE> : combine_rms_add_kernel<TYPE>;                            \
        if (smem > 48 * 1024) {                                                                                       \
            cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);       \
            if (e != cudaSuccess) return (int)e;                                                                      \
        }                                                                                                             \
        rc = ssb_launch(kern, dim3(n_tokens), dim3(CN_THREADS), smem, stream, pdl != 0, residual, y, pair_weight,     \
                        top, w, eps, width, (TYPE*)next_out);                                                         \
    }
    if (next_out == nullptr || next_dtype == SSB_F32) SSB_CN(float)
    else if (next_dtype == SSB_BF16) SSB_CN(bf16)
    else return SSB_ERR_BAD_DTYPE;
#undef SSB_CN
    return rc ? rc : ssb_launch_status();
}
