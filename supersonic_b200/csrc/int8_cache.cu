// A cache entry in 8 bits: keys and values as int8 codes [pages, n_kv, 64, head_dim] with a float32 scale for every block of
// 16, 32 or 64 tokens and kv head [pages, n_kv, 64 / block], and, where a caller keeps account of it, the attention weight that
// every cached token has gathered [pages, n_kv, 64].  A value is code * scale.
//
// Here: the append (rotation of queries and keys, quantisation of keys and values), the read-back of values, and the eviction
// (which tokens stay, and their move to new pages).  Every quantity is computed with the correctly rounded float32 operations
// that the formulas name, one after another (no contraction into fused multiply-adds), so that codes do not depend on how a
// compiler orders them: a value that lies on the border of two codes falls the same way in every build.
//
// The reference keeps keys in int8 and values in int4 for one of its lanes, a scale per block of tokens and channel
// (kernels/certified_kv_bridge_cuda.cu:32-420); this cache has one scale per block of tokens and head, and both in int8.
#include "common.cuh"

typedef __nv_bfloat16 bf16;

constexpr float I8_LEAST_SCALE = 7.888609052210118e-31f;        // 2^-100: a block of zeros has a scale too
constexpr float I8_MOST = 1.7014118346046923e38f;               // 2^127: its largest code still stands for a finite number
constexpr int I8_PAGE = 64;

__device__ __forceinline__ void i8_load8(const bf16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void i8_load8(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void i8_store8(bf16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void i8_store8(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
// What of a number a code can stand for: NaN counts as zero, an infinity as 2^127 of its sign.
__device__ __forceinline__ float i8_finite(float x) { return x != x ? 0.f : fminf(fmaxf(x, -I8_MOST), I8_MOST); }
// Eight codes of eight numbers, and the values that the codes stand for.
__device__ __forceinline__ uint2 i8_encode8(float (&x)[8], float scale) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i], scale)), -127.f), 127.f);
        w[i >> 2] |= (uint32_t)(uint8_t)(int8_t)(int)c << (8 * (i & 3));
        x[i] = __fmul_rn(c, scale);
    }
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ int i8_code(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }
__device__ __forceinline__ uint32_t i8_rescale4(uint32_t w, float ratio) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (uint32_t)(uint8_t)(int8_t)(int)rintf(__fmul_rn((float)i8_code(w, i), ratio)) << (8 * i);
    return r;
}

struct I8Append {
    const void* qkv;              // [T, ldq]: query heads, key heads, value heads
    void* out;                    // [T, ldo]: queries rotated, keys and values as the cache holds them
    const float* cos_t;           // [positions, rot / 2], or null: nothing is rotated
    const float* sin_t;
    const int* pos;               // [T] position a query or key is rotated by
    const int* place;             // [T] place in the sequence's cache
    const int* slot;              // [T]
    const int* page_table;        // [slots, max_pages]
    int8_t* codes[2];             // keys, values
    float* scale[2];
    float* weight;                // or null
    int ldq, ldo, T, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, rot, positions, block, span;
};

constexpr int I8_APPEND_THREADS = 128;

// A block of the grid takes ``span`` rows of one head.  16 numbers of a head are a lane's: 8 of its pairs' first and 8 of their
// second members (or 16 that are not rotated), so a head of 128 is 8 lanes and the block works on 16 rows at a time.  A row that
// begins a run (of consecutive places in one scale block) has the whole run quantised by its block: the numbers stay in
// registers between the run's maximum and its codes, PASSES rows a lane.
template <typename T, int PASSES>
__global__ void __launch_bounds__(I8_APPEND_THREADS)
int8_append_kernel(const I8Append a) {
    const int head = blockIdx.y, hd = a.head_dim, lanes = hd / 16, at_once = I8_APPEND_THREADS / lanes;
    const int l = threadIdx.x % lanes, r_of = threadIdx.x / lanes, half = a.rot / 2;
    const bool turns = a.cos_t != nullptr && l < a.rot / 16 && head < a.n_q + a.n_kv;
    const int e0 = l < a.rot / 16 ? 8 * l : a.rot + 16 * (l - a.rot / 16), e1 = l < a.rot / 16 ? half + 8 * l : e0 + 8;
    const int row0 = blockIdx.x * a.span;
    const bool is_q = head < a.n_q;
    const int which = head >= a.n_q + a.n_kv, kvh = head - a.n_q - which * a.n_kv;
    __shared__ int run_len;
    __shared__ float warp_max[I8_APPEND_THREADS / 32];

    auto page_of = [&](int row) -> int {                      // or -1: a row without a place
        const int s = a.slot[row], p = a.place[row];
        if (s < 0 || s >= a.n_slots || p < 0 || (p >> 6) >= a.max_pages) return -1;
        const int page = a.page_table[(size_t)s * a.max_pages + (p >> 6)];
        return page < a.n_pages ? page : -1;
    };
    auto load = [&](int row, float (&x)[8], float (&y)[8]) {
        const T* src = (const T*)a.qkv + (size_t)row * a.ldq + (size_t)head * hd;
        i8_load8(src + e0, x);
        i8_load8(src + e1, y);
        if (turns) {
            const int p = a.pos[row];
            if (p >= 0 && p < a.positions) {
                float c[8], s[8];
                i8_load8(a.cos_t + (size_t)p * half + e0, c);
                i8_load8(a.sin_t + (size_t)p * half + e0, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = x[i], v = y[i];
                    x[i] = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(v, s[i]));
                    y[i] = __fadd_rn(__fmul_rn(u, s[i]), __fmul_rn(v, c[i]));
                }
            }
        }
    };
    auto store = [&](int row, const float (&x)[8], const float (&y)[8]) {
        T* dst = (T*)a.out + (size_t)row * a.ldo + (size_t)head * hd;
        i8_store8(dst + e0, x);
        i8_store8(dst + e1, y);
    };
    if (is_q) {
        for (int r = r_of; r < a.span && row0 + r < a.T; r += at_once) {
            if (page_of(row0 + r) < 0) continue;
            float x[8], y[8];
            load(row0 + r, x, y);
            store(row0 + r, x, y);
        }
        return;
    }
    for (int r = 0; r < a.span && row0 + r < a.T; ++r) {
        const int lead = row0 + r, page = page_of(lead);       // the same for the whole block
        if (page < 0) continue;
        const int p0 = a.place[lead], s0 = a.slot[lead], in_block = p0 & (a.block - 1);
        if (in_block != 0 && lead > 0 && a.slot[lead - 1] == s0 && a.place[lead - 1] == p0 - 1) continue;    // inside a run
        __syncthreads();
        if (threadIdx.x == 0) run_len = a.block - in_block;
        __syncthreads();
        if ((int)threadIdx.x < a.block - in_block) {
            const int row = lead + (int)threadIdx.x;
            if (row >= a.T || a.slot[row] != s0 || a.place[row] != p0 + (int)threadIdx.x) atomicMin(&run_len, (int)threadIdx.x);
        }
        __syncthreads();
        const int n = run_len;
        float x[PASSES][8], y[PASSES][8], most = 0.f;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = i * at_once + r_of;
            if (row < n) {
                load(lead + row, x[i], y[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[i][e] = i8_finite(x[i][e]);
                    y[i][e] = i8_finite(y[i][e]);
                    most = fmaxf(most, fmaxf(fabsf(x[i][e]), fabsf(y[i][e])));
                }
            }
        }
        most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));      // not negative: the order of its bits
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = most;
        const size_t head_at = (size_t)page * a.n_kv + kvh;
        const int per = I8_PAGE / a.block, in_page = p0 & (I8_PAGE - 1);
        float* scale_at = a.scale[which] + head_at * per + in_page / a.block;
        const float old = in_block ? *scale_at : 0.f;
        __syncthreads();                                       // and the old scale has been read
#pragma unroll
        for (int w = 0; w < I8_APPEND_THREADS / 32; ++w) most = fmaxf(most, warp_max[w]);
        const float now = fmaxf(fmaxf(old, __fmul_rn(most, 1.f / 127.f)), I8_LEAST_SCALE);
        int8_t* codes = a.codes[which] + (head_at * I8_PAGE + in_page) * hd;
        if (in_block && now > old) {                           // the block's earlier codes under the larger scale
            const float ratio = __fdiv_rn(old, now);
            for (int e = threadIdx.x; e < in_block * lanes; e += I8_APPEND_THREADS) {
                uint4* at = reinterpret_cast<uint4*>(codes - (size_t)in_block * hd) + e;
                uint4 v = *at;
                v.x = i8_rescale4(v.x, ratio); v.y = i8_rescale4(v.y, ratio); v.z = i8_rescale4(v.z, ratio); v.w = i8_rescale4(v.w, ratio);
                *at = v;
            }
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int row = i * at_once + r_of;
            if (row < n) {
                *reinterpret_cast<uint2*>(codes + (size_t)row * hd + e0) = i8_encode8(x[i], now);
                *reinterpret_cast<uint2*>(codes + (size_t)row * hd + e1) = i8_encode8(y[i], now);
                store(lead + row, x[i], y[i]);
            }
        }
        if (threadIdx.x == 0) *scale_at = now;
        if (a.weight && !which && (int)threadIdx.x < n) a.weight[head_at * I8_PAGE + in_page + threadIdx.x] = 0.f;
    }
}

SSB_API int ssb_int8_append(const void* qkv, int ldq, int dtype, void* out, int ldo, const float* cos_t, const float* sin_t,
                            int positions, int rot, const int* pos, const int* place, const int* slot, int T,
                            const int* page_table, int n_slots, int max_pages, void* k, void* v, float* k_scale, float* v_scale,
                            float* weight, int n_pages, int n_q, int n_kv, int head_dim, int block, cudaStream_t stream) {
    if (T <= 0) return 0;
    const int lanes = head_dim / 16;
    if (head_dim % 16 || lanes < 1 || lanes > 16 || (lanes & (lanes - 1)) || rot % 16 || rot > head_dim || n_kv <= 0 || n_q < 0 ||
        (block != 16 && block != 32 && block != 64) || n_q + 2 * n_kv > 65535)
        return SSB_ERR_BAD_SIZE;
    I8Append a{qkv, out, cos_t, sin_t, pos, place, slot, page_table, {(int8_t*)k, (int8_t*)v}, {k_scale, v_scale}, weight,
               ldq, ldo, T, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, rot, positions, block, 1};
    // a block a row while there are few; else as many rows as a scale block has, so that hardly a block finds nothing to do
    a.span = T <= 256 ? 1 : block;
    const int passes = (block * lanes + I8_APPEND_THREADS - 1) / I8_APPEND_THREADS;
    const dim3 grid((T + a.span - 1) / a.span, n_q + 2 * n_kv);
#define I8_APPEND(P_) \
    do { \
        if (dtype == SSB_BF16) int8_append_kernel<bf16, P_><<<grid, I8_APPEND_THREADS, 0, stream>>>(a); \
        else if (dtype == SSB_F32) int8_append_kernel<float, P_><<<grid, I8_APPEND_THREADS, 0, stream>>>(a); \
        else return SSB_ERR_BAD_DTYPE; \
    } while (0)
    if (passes <= 1) I8_APPEND(1);
    else if (passes <= 2) I8_APPEND(2);
    else if (passes <= 4) I8_APPEND(4);
    else I8_APPEND(8);
#undef I8_APPEND
    return ssb_launch_status();
}

// ---- values back ----------------------------------------------------------------------------------------------------
// out[b, i, head] = values of token i of sequence b, i < lengths[b] (and < most); 16 numbers a thread.
template <typename T>
__global__ void __launch_bounds__(256)
int8_read_kernel(const int8_t* __restrict__ k, const int8_t* __restrict__ v, const float* __restrict__ k_scale,
                 const float* __restrict__ v_scale, const int* __restrict__ page_table, int n_slots, int max_pages, int n_pages,
                 const int* __restrict__ seq_slot, const int* __restrict__ lengths, T* __restrict__ k_out, T* __restrict__ v_out,
                 int most, int n_kv, int head_dim, int block) {
    const int lanes = head_dim / 16, b = blockIdx.y, which = blockIdx.z;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;           // of the sequence's tokens, heads and lanes
    const int l = (int)(at % lanes), head = (int)(at / lanes % n_kv), i = (int)(at / lanes / n_kv);
    const int s = seq_slot[b], n = min(min(lengths[b], most), max_pages * I8_PAGE);
    if (s < 0 || s >= n_slots || i >= n) return;
    const int page = page_table[(size_t)s * max_pages + (i >> 6)];
    if (page < 0 || page >= n_pages) return;
    const size_t row = ((size_t)page * n_kv + head) * I8_PAGE + (i & 63);
    const float scale = (which ? v_scale : k_scale)[row / block];
    const uint4 c = reinterpret_cast<const uint4*>((which ? v : k) + row * head_dim)[l];
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    T* dst = (which ? v_out : k_out) + (((size_t)b * most + i) * n_kv + head) * head_dim + 16 * l;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn((float)i8_code(w[2 * h + (e >> 2)], e & 3), scale);
        i8_store8(dst + 8 * h, x);
    }
}

SSB_API int ssb_int8_read(const void* k, const void* v, const float* k_scale, const float* v_scale, const int* page_table,
                          int n_slots, int max_pages, int n_pages, const int* seq_slot, const int* lengths, int n_seqs, void* k_out,
                          void* v_out, int dtype, int most, int n_kv, int head_dim, int block, cudaStream_t stream) {
    if (n_seqs <= 0 || most <= 0) return 0;
    if (head_dim % 16 || head_dim <= 0 || n_kv <= 0 || (block != 16 && block != 32 && block != 64)) return SSB_ERR_BAD_SIZE;
    const long long blocks = ((long long)most * n_kv * (head_dim / 16) + 255) / 256;
    if (blocks > 0x7fffffffLL || n_seqs > 65535) return SSB_ERR_BAD_SIZE;
    const dim3 grid((unsigned)blocks, n_seqs, 2);
#define I8_READ(T_) \
    int8_read_kernel<T_><<<grid, 256, 0, stream>>>((const int8_t*)k, (const int8_t*)v, k_scale, v_scale, page_table, n_slots, max_pages, \
                                                   n_pages, seq_slot, lengths, (T_*)k_out, (T_*)v_out, most, n_kv, head_dim, block)
    if (dtype == SSB_BF16) I8_READ(bf16);
    else if (dtype == SSB_F32) I8_READ(float);
    else return SSB_ERR_BAD_DTYPE;
#undef I8_READ
    return ssb_launch_status();
}

// ---- eviction -------------------------------------------------------------------------------------------------------
// A number's rank as an unsigned integer: larger numbers have larger ranks, zeros of either sign one, NaN that of the lowest.
__device__ __forceinline__ uint32_t i8_rank(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int I8_SELECT_THREADS = 1024;

// kept[b, head] = the places that stay, in order: the first ``first``, the last ``recent``, and of the others the heaviest, equal
// ones by their place; -1 behind them.  One block a (sequence, kv head): the rank of the last one that stays is found from its
// highest byte to its lowest by counting, then one more pass writes places in order.
__global__ void __launch_bounds__(I8_SELECT_THREADS)
int8_select_kernel(const float* __restrict__ weight, const int* __restrict__ page_table, int n_slots, int max_pages, int n_pages,
                   const int* __restrict__ seq_slot, const int* __restrict__ lengths, int n_kv, int keep, int first, int recent,
                   int* __restrict__ kept) {
    const int b = blockIdx.x, head = blockIdx.y, s = seq_slot[b];
    const int n = s < 0 || s >= n_slots ? 0 : min(lengths[b], max_pages * I8_PAGE);
    int* dst = kept + ((size_t)b * n_kv + head) * keep;
    if (n <= keep) {
        for (int i = threadIdx.x; i < keep; i += I8_SELECT_THREADS) dst[i] = i < n ? i : -1;
        return;
    }
    const int* pt = page_table + (size_t)s * max_pages;
    auto rank_of = [&](int j) {
        const int page = pt[j >> 6];
        return page < 0 || page >= n_pages ? 0u : i8_rank(weight[((size_t)page * n_kv + head) * I8_PAGE + (j & 63)]);
    };
    __shared__ int count[256];
    __shared__ int chosen_digit, still;
    __shared__ int warp_sum[2][32];
    const int lo = first, hi = n - recent, want = keep - first - recent;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t prefix = 0;
    int left = want;                                           // of those with the prefix, how many stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (threadIdx.x < 256) count[threadIdx.x] = 0;
        __syncthreads();
        for (int j = lo + (int)threadIdx.x; j < hi; j += I8_SELECT_THREADS) {
            const uint32_t r = rank_of(j);
            if (shift == 24 || (r >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&count[(r >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int above = 0, d = 255;
            for (; d > 0 && above + count[d] < left; --d) above += count[d];
            chosen_digit = d;
            still = left - above;
        }
        __syncthreads();
        prefix |= (uint32_t)chosen_digit << shift;
        left = still;
        __syncthreads();
    }
    // want 0: the loop above ends at the largest rank with none of it to take
    int done = 0, equal = 0;                                   // places written, equal ones met
    for (int j0 = 0; j0 < n; j0 += I8_SELECT_THREADS) {
        const int j = j0 + (int)threadIdx.x;
        const bool sure = j < n && (j < lo || j >= hi);
        const uint32_t r = j < n && !sure ? rank_of(j) : 0u;
        const bool tie = j < n && !sure && r == prefix;
        const unsigned ties = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) warp_sum[0][warp] = __popc(ties);
        __syncthreads();
        int before = equal;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) before += warp_sum[0][w];
            equal += warp_sum[0][w];
        }
        before += __popc(ties & ((1u << lane) - 1));
        const bool stays = sure || (j < n && !sure && r > prefix) || (tie && before < left);
        const unsigned all = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) warp_sum[1][warp] = __popc(all);
        __syncthreads();
        int at = done;
        for (int w = 0; w < 32; ++w) {
            if (w < warp) at += warp_sum[1][w];
            done += warp_sum[1][w];
        }
        at += __popc(all & ((1u << lane) - 1));
        if (stays && at < keep) dst[at] = j;
        __syncthreads();
    }
}

constexpr int I8_MOVE_THREADS = 256;

// The kept tokens of one destination page and kv head: codes under the largest scale of their new block, weights beside them.
__global__ void __launch_bounds__(I8_MOVE_THREADS)
int8_move_kernel(int8_t* __restrict__ k, int8_t* __restrict__ v, float* __restrict__ k_scale, float* __restrict__ v_scale,
                 float* __restrict__ weight, const int* __restrict__ page_table, int n_slots, int max_pages, int n_pages,
                 const int* __restrict__ seq_slot, const int* __restrict__ new_table, int new_pages, int n_kv, int head_dim, int block,
                 int keep, const int* __restrict__ kept) {
    const int to = blockIdx.x, head = blockIdx.y, b = blockIdx.z, s = seq_slot[b];
    if (s < 0 || s >= n_slots) return;
    const int target = new_table[(size_t)b * new_pages + to];
    if (target < 0 || target >= n_pages) return;
    const int lanes = head_dim / 16, per = I8_PAGE / block;
    __shared__ long long from[I8_PAGE];                        // the row's place among all rows, or -1
    __shared__ float scale[2][I8_PAGE], now[2][4];
    if (threadIdx.x < I8_PAGE) {
        const int i = to * I8_PAGE + (int)threadIdx.x, j = i < keep ? kept[((size_t)b * n_kv + head) * keep + i] : -1;
        long long row = -1;
        if (j >= 0 && (j >> 6) < max_pages) {
            const int page = page_table[(size_t)s * max_pages + (j >> 6)];
            if (page >= 0 && page < n_pages) row = ((long long)page * n_kv + head) * I8_PAGE + (j & 63);
        }
        from[threadIdx.x] = row;
        scale[0][threadIdx.x] = row >= 0 ? k_scale[row / block] : 0.f;
        scale[1][threadIdx.x] = row >= 0 ? v_scale[row / block] : 0.f;
    }
    __syncthreads();
    const size_t head_at = (size_t)target * n_kv + head;
    if ((int)threadIdx.x < 2 * per) {
        const int which = threadIdx.x / per, blk = threadIdx.x % per;
        float m = 0.f;
        bool any = false;
        for (int i = blk * block; i < (blk + 1) * block; ++i) { m = fmaxf(m, scale[which][i]); any |= from[i] >= 0; }
        now[which][blk] = m;
        if (any) (which ? v_scale : k_scale)[head_at * per + blk] = m;
    }
    if (weight && threadIdx.x < I8_PAGE && from[threadIdx.x] >= 0) weight[head_at * I8_PAGE + threadIdx.x] = weight[from[threadIdx.x]];
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * I8_PAGE * lanes; e += I8_MOVE_THREADS) {
        const int which = e / (I8_PAGE * lanes), row = e / lanes % I8_PAGE, l = e % lanes;
        if (from[row] < 0) continue;
        int8_t* codes = which ? v : k;
        uint4 c = reinterpret_cast<const uint4*>(codes + (size_t)from[row] * head_dim)[l];
        const float m = now[which][row / block];
        if (scale[which][row] != m) {
            const float ratio = __fdiv_rn(scale[which][row], m);
            c.x = i8_rescale4(c.x, ratio); c.y = i8_rescale4(c.y, ratio); c.z = i8_rescale4(c.z, ratio); c.w = i8_rescale4(c.w, ratio);
        }
        reinterpret_cast<uint4*>(codes + (head_at * I8_PAGE + row) * head_dim)[l] = c;
    }
}

SSB_API int ssb_int8_evict(void* k, void* v, float* k_scale, float* v_scale, float* weight, const int* page_table, int n_slots,
                           int max_pages, int n_pages, const int* seq_slot, const int* lengths, int n_seqs, const int* new_table,
                           int new_pages, int n_kv, int head_dim, int block, int keep, int first, int recent, int* kept,
                           cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (head_dim % 16 || head_dim <= 0 || n_kv <= 0 || (block != 16 && block != 32 && block != 64) || keep <= 0 || first < 0 ||
        recent < 0 || (long long)first + recent > keep || (long long)new_pages * I8_PAGE < keep || n_seqs > 65535 || n_kv > 65535)
        return SSB_ERR_BAD_SIZE;
    int8_select_kernel<<<dim3(n_seqs, n_kv), I8_SELECT_THREADS, 0, stream>>>(weight, page_table, n_slots, max_pages, n_pages, seq_slot,
                                                                             lengths, n_kv, keep, first, recent, kept);
    int rc = ssb_launch_status();
    if (rc) return rc;
    int8_move_kernel<<<dim3((keep + I8_PAGE - 1) / I8_PAGE, n_kv, n_seqs), I8_MOVE_THREADS, 0, stream>>>(
        (int8_t*)k, (int8_t*)v, k_scale, v_scale, weight, page_table, n_slots, max_pages, n_pages, seq_slot, new_table, new_pages,
        n_kv, head_dim, block, keep, kept);
    return ssb_launch_status();
}
