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
#include "int8_codes.cuh"
#include "packed_call.cuh"
#include <algorithm>

typedef __nv_bfloat16 bf16;

constexpr int I8_PAGE = 64;

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
    int ldq, ldo, T, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, rot, positions, block, chunk, kv_blocks;
};

constexpr int I8_APPEND_WARPS = 4, I8_Q_HEADS = 8;

// 16 numbers of a head are a lane's: 8 of its pairs' first and 8 of their second members (or 16 that are not rotated), so a head of
// 128 is 8 lanes and a warp works on ROWS = 4 rows at a time.  Two kinds of warps:
//  * keys and values: ``chunk`` rows of one head.  A row that begins a run (consecutive places in one scale block) has the whole run
//    quantised by the warp that owns it, up to 4 ROWS rows in registers between their maximum and their codes, so nothing but the
//    warp's own reduction stands between (a block a run spent its time in barriers and in asking 16 rows one after another
//    whether they begin one: 18,000 rows of 48 heads 153 us).
//  * queries: ROWS rows of up to 8 heads, the rotation tables' rows read once for all of them.
// KV, Q: which kinds of warps the launch has; where there are many rows each kind has a launch of its own, and its own number of registers.
// 14,800 rows of 32 heads over 8 of 128 in bfloat16: 60 us for keys and values, 2.5 TB/s, bound by fetches one after another (places, rows,
// tables) under four warps a scheduler; 43 us for queries, 5.7 TB/s.
template <typename T, int LANES, bool KV, bool Q>
__global__ void __launch_bounds__(32 * I8_APPEND_WARPS, KV ? 4 : 8)
int8_append_kernel(const I8Append a) {
    constexpr int ROWS = 32 / LANES, KEEP = 4, HD = 16 * LANES;
    // queries that follow the keys' launch touch nothing of its, and what it waited for is there: they wait for it at their end, so
    // that they run beside its last blocks and whoever waits for them has waited for both
    if (KV) ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = lane % LANES, r_of = lane / LANES, half = a.rot / 2;
    const bool turned = a.cos_t != nullptr && l < a.rot / 16;
    const int e0 = l < a.rot / 16 ? 8 * l : a.rot + 16 * (l - a.rot / 16), e1 = l < a.rot / 16 ? half + 8 * l : e0 + 8;
    // the two kinds' blocks lie among one another in proportion
    int w = blockIdx.x * I8_APPEND_WARPS + (threadIdx.x >> 5);
    bool queries = !KV;
    if (KV && Q) {
        const long long before = (long long)blockIdx.x * a.kv_blocks / gridDim.x, then = (long long)(blockIdx.x + 1) * a.kv_blocks / gridDim.x;
        queries = then == before;
        w = (int)(queries ? blockIdx.x - before : before) * I8_APPEND_WARPS + (threadIdx.x >> 5);
    }

    auto page_of = [&](int s, int p) -> int {                 // or -1: no place
        if (s < 0 || s >= a.n_slots || p < 0 || (p >> 6) >= a.max_pages) return -1;
        const int page = a.page_table[(size_t)s * a.max_pages + (p >> 6)];
        return page < a.n_pages ? page : -1;
    };
    auto tables = [&](int p, float (&c)[8], float (&s)[8]) -> bool {
        if (!turned || p < 0 || p >= a.positions) return false;
        i8_load8(a.cos_t + (size_t)p * half + e0, c);
        i8_load8(a.sin_t + (size_t)p * half + e0, s);
        return true;
    };
    auto turn = [&](float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float u = x[i], v = y[i];
            x[i] = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(v, s[i]));
            y[i] = __fadd_rn(__fmul_rn(u, s[i]), __fmul_rn(v, c[i]));
        }
    };
    if (Q && queries) {
        const int blocks = (a.n_q + I8_Q_HEADS - 1) / I8_Q_HEADS, head0 = w % blocks * I8_Q_HEADS, row = w / blocks * ROWS + r_of;
        if (row < a.T) {
            const int sl = a.slot[row], pl = a.place[row];
            float c[8], s[8];
            const bool turns = tables(turned ? a.pos[row] : -1, c, s);
            const T* src = (const T*)a.qkv + (size_t)row * a.ldq;
            T* dst = (T*)a.out + (size_t)row * a.ldo;
            if (sl >= 0 && sl < a.n_slots && pl >= 0 && (pl >> 6) < a.max_pages)
#pragma unroll 4
                for (int h = head0; h < min(head0 + I8_Q_HEADS, a.n_q); ++h) {
                    float x[8], y[8];
                    i8_load8(src + h * HD + e0, x);
                    i8_load8(src + h * HD + e1, y);
                    if (turns) turn(x, y, c, s);
                    i8_store8(dst + h * HD + e0, x);
                    i8_store8(dst + h * HD + e1, y);
                }
        }
        if (!KV) ssb_pdl_wait();
        return;
    }
    if (!KV) return;
    const int kv_heads = 2 * a.n_kv, which = w % kv_heads / a.n_kv, kvh = w % a.n_kv, head = a.n_q + which * a.n_kv + kvh;
    const int row0 = w / kv_heads * a.chunk;
    if (row0 >= a.T) return;
    // a row a lane: its place, and whether it goes on from the row before it or begins a run
    int my_slot = -1, my_place = -1, my_pos = -1, my_page = -1;
    unsigned leads, goes_on;
    {
        const int row = row0 + lane;
        bool lead = false, on = false;
        if (lane < a.chunk && row < a.T) {
            my_slot = a.slot[row];
            my_place = a.place[row];
            my_pos = a.cos_t != nullptr && !which ? a.pos[row] : -1;
            on = row > 0 && (my_place & (a.block - 1)) != 0 && a.slot[row - 1] == my_slot && a.place[row - 1] == my_place - 1;
            lead = my_slot >= 0 && !on;
            my_page = page_of(my_slot, my_place);
        }
        leads = __ballot_sync(0xffffffffu, lead);
        goes_on = __ballot_sync(0xffffffffu, on);
    }
    for (; leads; leads &= leads - 1) {
        const int at = __ffs(leads) - 1, lead = row0 + at;
        const int s0 = __shfl_sync(0xffffffffu, my_slot, at), p0 = __shfl_sync(0xffffffffu, my_place, at);
        const int in_block = p0 & (a.block - 1), in_page = p0 & (I8_PAGE - 1), most_n = a.block - in_block;
        // rows that go on from the first: in the chunk by its lanes, behind it (a run may cross its end) by asking
        const unsigned after = at == 31 ? 0u : goes_on >> (at + 1);
        int n = 1 + (~after ? __ffs(~after) - 1 : 32);
        if (at + n >= a.chunk) {
            n = a.chunk - at;
            for (bool more = n < most_n; more;) {
                const int i = n + lane, row = lead + i;
                const unsigned on = __ballot_sync(0xffffffffu, i < most_n && row < a.T && a.slot[min(row, a.T - 1)] == s0 && a.place[min(row, a.T - 1)] == p0 + i);
                const int got = on == 0xffffffffu ? 32 : __ffs(~on) - 1;
                n += got;
                more = got == 32 && n < most_n;
            }
        }
        float x[KEEP][8], y[KEEP][8];
        uint32_t top = 0;
        bool wild = false;                                     // a number of the run is none, or too large
        auto load = [&](int first) {                           // rows first .. first + KEEP ROWS - 1 of the run
#pragma unroll
            for (int i = 0; i < KEEP; ++i) {
                const int row = first + i * ROWS + r_of;
                if (row < n) {
                    const T* src = (const T*)a.qkv + (size_t)(lead + row) * a.ldq + (size_t)head * HD;
                    i8_load8(src + e0, x[i]);
                    i8_load8(src + e1, y[i]);
                }
            }
            if (!which) {
#pragma unroll
                for (int i = 0; i < KEEP; ++i) {
                    const int row = first + i * ROWS + r_of, known = __shfl_sync(0xffffffffu, my_pos, (at + row) & 31);
                    float c[8], s[8];
                    if (row < n && tables(at + row < a.chunk ? known : turned ? a.pos[lead + row] : -1, c, s)) turn(x[i], y[i], c, s);
                }
            }
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
                if (first + i * ROWS + r_of < n) {
                    if (wild) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) { x[i][e] = i8_finite(x[i][e]); y[i][e] = i8_finite(y[i][e]); }
                    }
                    top = max(top, max(i8_magnitude(x[i]), i8_magnitude(y[i])));
                }
        };
        const int last = (n - 1) / (KEEP * ROWS) * (KEEP * ROWS);
        for (int first = 0; first <= last; first += KEEP * ROWS) load(first);
        // the page only now: the rows do not wait for its id
        const int page = __shfl_sync(0xffffffffu, my_page, at);
        if (page < 0) continue;
        const size_t head_at = (size_t)page * a.n_kv + kvh;
        const int per = I8_PAGE / a.block;
        float* scale_at = a.scale[which] + head_at * per + in_page / a.block;
        const float old = in_block ? *scale_at : 0.f;
        top = __reduce_max_sync(0xffffffffu, top);
        if (top >= I8_WILD) {
            wild = true;
            top = 0;
            for (int first = 0; first <= last; first += KEEP * ROWS) load(first);
            top = __reduce_max_sync(0xffffffffu, top);
        }
        const float most = __uint_as_float(top);
        const float now = fmaxf(fmaxf(old, __fmul_rn(most, 1.f / 127.f)), I8_LEAST_SCALE), inverse = 1.f / now;
        int8_t* codes = a.codes[which] + (head_at * I8_PAGE + in_page) * HD;
        if (in_block && now > old) {                           // the block's earlier codes under the larger scale
            const float ratio = __fdiv_rn(old, now);
            for (int e = lane; e < in_block * LANES; e += 32) {
                uint4* at = reinterpret_cast<uint4*>(codes - (size_t)in_block * HD) + e;
                uint4 v = *at;
                v.x = i8_rescale4(v.x, ratio); v.y = i8_rescale4(v.y, ratio); v.z = i8_rescale4(v.z, ratio); v.w = i8_rescale4(v.w, ratio);
                *at = v;
            }
        }
        for (int first = last; first >= 0; first -= KEEP * ROWS) {       // the last rows are still in registers
            if (first != last) load(first);
#pragma unroll
            for (int i = 0; i < KEEP; ++i) {
                const int row = first + i * ROWS + r_of;
                if (row < n) {
                    *reinterpret_cast<uint2*>(codes + (size_t)row * HD + e0) = i8_encode8(x[i], now, inverse);
                    *reinterpret_cast<uint2*>(codes + (size_t)row * HD + e1) = i8_encode8(y[i], now, inverse);
                    T* dst = (T*)a.out + (size_t)(lead + row) * a.ldo + (size_t)head * HD;
                    i8_store8(dst + e0, x[i]);
                    i8_store8(dst + e1, y[i]);
                }
            }
        }
        if (lane == 0) *scale_at = now;
        if (a.weight && !which)
            for (int i = lane; i < n; i += 32) a.weight[head_at * I8_PAGE + in_page + i] = 0.f;
    }
}

SSB_API int ssb_int8_append(const void* qkv, int ldq, int dtype, void* out, int ldo, const float* cos_t, const float* sin_t,
                            int positions, int rot, const int* pos, const int* place, const int* slot, int T,
                            const int* page_table, int n_slots, int max_pages, void* k, void* v, float* k_scale, float* v_scale,
                            float* weight, int n_pages, int n_q, int n_kv, int head_dim, int block, cudaStream_t stream) {
    if (T <= 0) return 0;
    if (rot % 16 || rot > head_dim || n_kv <= 0 || n_q < 0 || (block != 16 && block != 32 && block != 64)) return SSB_ERR_BAD_SIZE;
    I8Append a{qkv, out, cos_t, sin_t, pos, place, slot, page_table, {(int8_t*)k, (int8_t*)v}, {k_scale, v_scale}, weight,
               ldq, ldo, T, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, rot, positions, block};
    // A warp a row while there are few; else a chunk of rows, of which two or so begin a run; and a launch for each kind of warps where
    // there are so many that the keys' registers cost the queries more than a second launch.  32 heads over 8 of 128, us with one
    // launch of a row a warp, of chunks of 8, and two launches with chunks of 16: 2 x 256 tokens 9.7, -, 14.1; 4 x 256 16.0, 10.4, 18.5;
    // 4 x 512 31.4, 20.8, 26.3; 1,024 single tokens 29.6, 26.1, 39.9; 4 x 1,024 57.8, 38.2, 36.4; 16 x 1,024 -, 136, 116.
    const bool many = T > 2048;
    a.chunk = many ? std::min(block, 32) : T > 256 ? 8 : 1;
    const int rows = 32 / std::max(1, head_dim / 16);
    const long long kv = (long long)((T + a.chunk - 1) / a.chunk) * 2 * n_kv;
    const long long q = (long long)((T + rows - 1) / std::max(1, rows)) * ((n_q + I8_Q_HEADS - 1) / I8_Q_HEADS);
    const long long kv_blocks = (kv + I8_APPEND_WARPS - 1) / I8_APPEND_WARPS, blocks = kv_blocks + (q + I8_APPEND_WARPS - 1) / I8_APPEND_WARPS;
    if (blocks * I8_APPEND_WARPS > 0x7fffffffLL) return SSB_ERR_BAD_SIZE;
    a.kv_blocks = (int)kv_blocks;
    const dim3 threads(32 * I8_APPEND_WARPS), kv_grid((unsigned)((kv + I8_APPEND_WARPS - 1) / I8_APPEND_WARPS)),
        q_grid((unsigned)((q + I8_APPEND_WARPS - 1) / I8_APPEND_WARPS));
    int rc = 0;
#define I8_LAUNCH(T_, L_) \
    if (!many) return ssb_launch(int8_append_kernel<T_, L_, true, true>, dim3((unsigned)blocks), threads, 0, stream, true, a); \
    rc = ssb_launch(int8_append_kernel<T_, L_, true, false>, kv_grid, threads, 0, stream, true, a); \
    return rc || q == 0 ? rc : ssb_launch(int8_append_kernel<T_, L_, false, true>, q_grid, threads, 0, stream, true, a)
#define I8_APPEND(L_) \
    if (dtype == SSB_BF16) { I8_LAUNCH(bf16, L_); } \
    if (dtype == SSB_F32) { I8_LAUNCH(float, L_); } \
    return SSB_ERR_BAD_DTYPE
    switch (head_dim) {
        case 16: I8_APPEND(1);
        case 32: I8_APPEND(2);
        case 64: I8_APPEND(4);
        case 128: I8_APPEND(8);
        case 256: I8_APPEND(16);
    }
#undef I8_APPEND
#undef I8_LAUNCH
    return SSB_ERR_BAD_SIZE;
}

// ---- values back ----------------------------------------------------------------------------------------------------
// out[b, i, head] = values of token i of sequence b, i < lengths[b] (and < most); 16 numbers a thread.  4 x 4,096 tokens of 8 heads of
// 128 to bfloat16: 101 MB in 22 us, 4.6 TB/s.
template <typename T>
__global__ void __launch_bounds__(256)
int8_read_kernel(const int8_t* __restrict__ k, const int8_t* __restrict__ v, const float* __restrict__ k_scale,
                 const float* __restrict__ v_scale, const int* __restrict__ page_table, int n_slots, int max_pages, int n_pages,
                 const int* __restrict__ seq_slot, const int* __restrict__ lengths, T* __restrict__ k_out, T* __restrict__ v_out,
                 int most, int n_kv, int head_dim, int block) {
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int lanes = head_dim / 16, b = blockIdx.y;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;           // of the sequence's tokens, heads and lanes
    const int l = (int)(at % lanes), head = (int)(at / lanes % n_kv), i = (int)(at / lanes / n_kv);
    const int s = seq_slot[b], n = min(min(lengths[b], most), max_pages * I8_PAGE);
    if (s < 0 || s >= n_slots || i >= n) return;
    const int page = page_table[(size_t)s * max_pages + (i >> 6)];
    if (page < 0 || page >= n_pages) return;
    const size_t row = ((size_t)page * n_kv + head) * I8_PAGE + (i & 63);
    const uint4 c[2] = {reinterpret_cast<const uint4*>(k + row * head_dim)[l], reinterpret_cast<const uint4*>(v + row * head_dim)[l]};
    const float scale[2] = {k_scale[row / block], v_scale[row / block]};
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const uint32_t w[4] = {c[which].x, c[which].y, c[which].z, c[which].w};
        T* dst = (which ? v_out : k_out) + (((size_t)b * most + i) * n_kv + head) * head_dim + 16 * l;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __fmul_rn((float)i8_code(w[2 * h + (e >> 2)], e & 3), scale[which]);
            i8_store8(dst + 8 * h, x);
        }
    }
}

SSB_API int ssb_int8_read(const void* k, const void* v, const float* k_scale, const float* v_scale, const int* page_table,
                          int n_slots, int max_pages, int n_pages, const int* seq_slot, const int* lengths, int n_seqs, void* k_out,
                          void* v_out, int dtype, int most, int n_kv, int head_dim, int block, cudaStream_t stream) {
    if (n_seqs <= 0 || most <= 0) return 0;
    if (head_dim % 16 || head_dim <= 0 || n_kv <= 0 || (block != 16 && block != 32 && block != 64)) return SSB_ERR_BAD_SIZE;
    const long long blocks = ((long long)most * n_kv * (head_dim / 16) + 255) / 256;
    if (blocks > 0x7fffffffLL || n_seqs > 65535) return SSB_ERR_BAD_SIZE;
    const dim3 grid((unsigned)blocks, n_seqs);
#define I8_READ(T_) \
    return ssb_launch(int8_read_kernel<T_>, grid, dim3(256), 0, stream, true, (const int8_t*)k, (const int8_t*)v, k_scale, v_scale, \
                      page_table, n_slots, max_pages, n_pages, seq_slot, lengths, (T_*)k_out, (T_*)v_out, most, n_kv, head_dim, block)
    if (dtype == SSB_BF16) I8_READ(bf16);
    if (dtype == SSB_F32) I8_READ(float);
#undef I8_READ
    return SSB_ERR_BAD_DTYPE;
}

// ---- eviction -------------------------------------------------------------------------------------------------------
// A number's rank as an unsigned integer: larger numbers have larger ranks, zeros of either sign one, NaN that of the lowest.
__device__ __forceinline__ uint32_t i8_rank(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t u = __float_as_uint(__fadd_rn(x, 0.f));
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int I8_SELECT_THREADS = 512, I8_SELECT_WARPS = I8_SELECT_THREADS / 32, I8_BINS = 2048;
constexpr int I8_SELECT_KEEP = 16384;      // ranks a block keeps in shared memory; further ones are read again
// Ranks of no number, which go from that of minus infinity, 0x007fffff, to that of infinity, 0xff800000: of a place behind the end; of one
// whose page is not there, below every number; of one that stays whatever it weighs.
constexpr uint32_t I8_NEVER = 0u, I8_NOWHERE = 1u << 21, I8_SURE = 0xffffffffu;

__device__ __forceinline__ int4 i8_cluster_int4(const int* mine, unsigned rank) {
    uint32_t remote;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ int i8_cluster_int(const int* mine, unsigned rank) {
    return __float_as_int(ssb_cluster_f32(reinterpret_cast<const float*>(mine), rank));
}

// kept[b, head] = the places that stay, in order: the first ``first``, the last ``recent``, and of the others the heaviest, equal
// ones by their place; -1 behind them.  A cluster of 1, 4 or 8 blocks a (sequence, kv head), each with a run of whole pages of the
// sequence and each warp with a run of whole 128 places of its block's: the rank of the last one that stays is found 11, 11 and 10 bits
// at a time, by counting (every block adds the cluster's counts up for itself), then every warp writes its places behind those of the
// warps and blocks before it.  Ranks lie in shared memory, four places a lane and turn, and the loops over them stay loops: 32 ranks a
// thread in registers, every loop unrolled, is code that runs once, and took longer to fetch than to run (sequences of 700 tokens 9 us
// and 32).  What bounds it is the time of its phases one after another (fetching, three counts with the cluster's sums, two walks):
// 4 x 8 selections among 60,000 to 131,000 places 34 us, with a place a lane and turn 40; 12 MB of weights would be read in 2.
__global__ void __launch_bounds__(I8_SELECT_THREADS, 2)
int8_select_kernel(const float* __restrict__ weight, const int* __restrict__ page_table, int n_slots, int max_pages, int n_pages,
                   const int* __restrict__ seq_slot, const int* __restrict__ lengths, int n_kv, int keep, int first, int recent,
                   int cluster, int held, int* __restrict__ kept) {
    extern __shared__ __align__(16) uint32_t ranks[];
    __shared__ __align__(16) int count[I8_BINS], total[I8_BINS];
    __shared__ int warp_sum[2][32];
    __shared__ int chosen, still;
    __shared__ int mine[2];                                    // this block's ties and sure ones
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int rank_in = cluster > 1 ? (int)ssb_cluster_rank() : 0, pair = blockIdx.x / cluster, b = pair / n_kv, head = pair % n_kv;
    const int s = seq_slot[b], warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = s < 0 || s >= n_slots ? 0 : min(lengths[b], max_pages * I8_PAGE);
    int* dst = kept + ((size_t)b * n_kv + head) * keep;
    if (n <= keep) {                                           // the same for the whole cluster
        for (int i = rank_in * I8_SELECT_THREADS + threadIdx.x; i < keep; i += cluster * I8_SELECT_THREADS) dst[i] = i < n ? i : -1;
        return;
    }
    const int* pt = page_table + (size_t)s * max_pages;
    const int pages = (n + I8_PAGE - 1) / I8_PAGE, share = (pages + cluster - 1) / cluster * I8_PAGE;
    const int j0 = min(rank_in * share, n), j1 = min(j0 + share, n);        // this block's places
    const int lo = first, hi = n - recent;                     // places that have to be chosen from
    const int per_warp = ((j1 - j0 + I8_SELECT_WARPS - 1) / I8_SELECT_WARPS + 127) / 128 * 128, w0 = min(j0 + warp * per_warp, j1), w1 = min(w0 + per_warp, j1);
    const bool wide = ((uintptr_t)weight & 15) == 0;
    auto fetch = [&](int j) -> uint4 {                         // of four places, which share a page
        if (j >= w1) return make_uint4(I8_NEVER, I8_NEVER, I8_NEVER, I8_NEVER);
        const int page = pt[j >> 6];
        const bool there = page >= 0 && page < n_pages;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there) {
            const float* at = weight + ((size_t)page * n_kv + head) * I8_PAGE + (j & 63);
            f = wide ? *reinterpret_cast<const float4*>(at) : make_float4(at[0], at[1], at[2], at[3]);
        }
        auto rank = [&](int i, float x) { return i >= w1 ? I8_NEVER : i < lo || i >= hi ? I8_SURE : there ? i8_rank(x) : I8_NOWHERE; };
        return make_uint4(rank(j, f.x), rank(j + 1, f.y), rank(j + 2, f.z), rank(j + 3, f.w));
    };
    for (int i = threadIdx.x; i < I8_BINS; i += I8_SELECT_THREADS) count[i] = 0;
    const int kept_in = min(held / I8_SELECT_WARPS / 128 * 128, per_warp);   // of the warp's places, in shared memory
    uint32_t* own = ranks + warp * kept_in;
#pragma unroll 4
    for (int j = w0 + 4 * lane; j < min(w0 + kept_in, w1); j += 128) *reinterpret_cast<uint4*>(own + (j - w0)) = fetch(j);
    __syncthreads();
    // f(first place, ranks) for each four of the lane's places, 128 of the warp's at a time
    auto each = [&](auto&& f) {
        for (int j = w0 + 4 * lane; j - 4 * lane < w1; j += 128)
            f(j, j >= w1 ? make_uint4(I8_NEVER, I8_NEVER, I8_NEVER, I8_NEVER) : j - w0 < kept_in ? *reinterpret_cast<const uint4*>(own + (j - w0)) : fetch(j));
    };

    uint32_t prefix = 0;                                       // the bits found so far
    int left = keep - first - recent;                          // of those with the prefix, how many stay
    for (int shift = left > 0 ? 21 : -1; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
        const int bits = shift == 0 ? 10 : 11;
        const uint32_t above = shift == 21 ? 0u : ~0u << (shift + bits);
        auto counted = [&](uint32_t r) {
            if (((r ^ prefix) & above) == 0 && r - 1u < I8_SURE - 1u) atomicAdd(&count[(r >> shift) & ((1 << bits) - 1)], 1);
        };
        each([&](int, const uint4& r) { counted(r.x); counted(r.y); counted(r.z); counted(r.w); });
        if (cluster > 1) ssb_cluster_sync(); else __syncthreads();
        // four bins a thread, the highest first: how many lie above them.  In a cluster every block adds up its share of the bins over
        // the blocks and fetches the other shares' totals (each adding all of them up for itself moved 64 KB a block and pass through
        // the cluster: 24 us of a pass over 131,000 places)
        constexpr int EACH = I8_BINS / I8_SELECT_THREADS;
        static_assert(EACH == 4, "a 16-byte load a thread");
        const int top = I8_BINS - 1 - EACH * (int)threadIdx.x, share_bins = I8_BINS / cluster;
        int4 four = *reinterpret_cast<const int4*>(count + top - 3);
        if (cluster > 1) {
            if ((int)threadIdx.x * 4 < share_bins) {
                const int at = rank_in * share_bins + 4 * (int)threadIdx.x;
                int4 sum = make_int4(0, 0, 0, 0);
                for (int r = 0; r < cluster; ++r) {
                    const int4 v = i8_cluster_int4(count + at, r);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                *reinterpret_cast<int4*>(total + at) = sum;
            }
            ssb_cluster_sync();
            four = i8_cluster_int4(total + top - 3, (top - 3) / share_bins);
        }
        const int c[EACH] = {four.w, four.z, four.y, four.x}, mine_sum = four.x + four.y + four.z + four.w;
        int incl = mine_sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_sum[0][warp] = incl;
        __syncthreads();
        if (warp == 0) {
            int v = lane < I8_SELECT_WARPS ? warp_sum[0][lane] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            warp_sum[1][lane] = v;
        }
        if (threadIdx.x == 0) { chosen = 0; still = 0; }
        __syncthreads();
        int over = (warp ? warp_sum[1][warp - 1] : 0) + incl - mine_sum;        // in the bins above these
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (over < left && over + c[i] >= left) { chosen = top - i; still = left - over; }
            over += c[i];
        }
        __syncthreads();
        prefix |= (uint32_t)chosen << shift;
        left = still;
        for (int i = threadIdx.x; i < I8_BINS; i += I8_SELECT_THREADS) count[i] = 0;        // nobody reads them any more
        __syncthreads();
    }
    if (left == 0) prefix = I8_SURE - 1;                       // none that has to be chosen stays
    // how many tie and how many stay for sure; then those before this block and warp
    int ties = 0, sures = 0;
    each([&](int, const uint4& r) {
        ties += (r.x == prefix) + (r.y == prefix) + (r.z == prefix) + (r.w == prefix);
        sures += (r.x > prefix) + (r.y > prefix) + (r.z > prefix) + (r.w > prefix);
    });
    ties = __reduce_add_sync(0xffffffffu, ties);
    sures = __reduce_add_sync(0xffffffffu, sures);
    if (lane == 0) { warp_sum[0][warp] = ties; warp_sum[1][warp] = sures; }
    __syncthreads();
    if (threadIdx.x < 2) {
        int sum = 0;
        for (int w = 0; w < I8_SELECT_WARPS; ++w) sum += warp_sum[threadIdx.x][w];
        mine[threadIdx.x] = sum;
    }
    if (cluster > 1) ssb_cluster_sync();
    int ties_before = 0, sures_before = 0;
    for (int r = 0; r < rank_in; ++r) { ties_before += i8_cluster_int(mine, r); sures_before += i8_cluster_int(mine + 1, r); }
    for (int w = 0; w < warp; ++w) { ties_before += warp_sum[0][w]; sures_before += warp_sum[1][w]; }
    each([&](int j, const uint4& r) {
        auto packed = [&](uint32_t x) { return (x > prefix ? 1 : 0) + (x == prefix ? 1 << 16 : 0); };
        const int four = packed(r.x) + packed(r.y) + packed(r.z) + packed(r.w);
        int incl = four;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        int sure_at = sures_before + ((incl - four) & 0xffff), tie_at = ties_before + ((incl - four) >> 16);
        auto put = [&](int i, uint32_t x) {
            const int at = sure_at + min(tie_at, left);
            if ((x > prefix || (x == prefix && tie_at < left)) && at < keep) dst[at] = i;
            sure_at += x > prefix;
            tie_at += x == prefix;
        };
        put(j, r.x); put(j + 1, r.y); put(j + 2, r.z); put(j + 3, r.w);
        incl = __shfl_sync(0xffffffffu, incl, 31);
        sures_before += incl & 0xffff;
        ties_before += incl >> 16;
    });
    if (cluster > 1) ssb_cluster_sync();                       // no block leaves while another may read its counts
}

constexpr int I8_MOVE_THREADS = 256;

// The kept tokens of one destination page and kv head: codes under the largest scale of their new block, weights beside them; zeros of
// a token whose page id names no page.  A thread's pieces of codes are on their way while the block's scales are compared.  4 x 8 times
// 4,096 tokens of 128: 67 MB in 25 us, 2.7 TB/s; bound by fetches that wait for one another (the place, its page, the codes and scale
// under it).
template <int LANES>
__global__ void __launch_bounds__(I8_MOVE_THREADS)
int8_move_kernel(int8_t* __restrict__ k, int8_t* __restrict__ v, float* __restrict__ k_scale, float* __restrict__ v_scale,
                 float* __restrict__ weight, const int* __restrict__ page_table, int n_slots, int max_pages, int n_pages,
                 const int* __restrict__ seq_slot, const int* __restrict__ new_table, int new_pages, int n_kv, int block, int keep,
                 const int* __restrict__ kept) {
    constexpr int PIECES = (2 * I8_PAGE * LANES + I8_MOVE_THREADS - 1) / I8_MOVE_THREADS;
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    // what does not wait for anything else is asked for together
    const int to = blockIdx.x, head = blockIdx.y, b = blockIdx.z, mine = to * I8_PAGE + (int)threadIdx.x;
    const int s = seq_slot[b], target = new_table[(size_t)b * new_pages + to];
    const int j = threadIdx.x < I8_PAGE && mine < keep ? kept[((size_t)b * n_kv + head) * keep + mine] : -1;
    if (s < 0 || s >= n_slots || target < 0 || target >= n_pages) return;
    const int per = I8_PAGE / block;
    __shared__ long long from[I8_PAGE];                        // the row's place among all rows, -1: nothing is kept there, or -2: kept, but in no page
    __shared__ float scale[2][I8_PAGE];
    const size_t head_at = (size_t)target * n_kv + head;
    if (threadIdx.x < I8_PAGE) {
        long long row = -1;
        if (j >= 0) {
            row = -2;
            const int page = page_table[(size_t)s * max_pages + (j >> 6)];
            if (page >= 0 && page < n_pages) row = ((long long)page * n_kv + head) * I8_PAGE + (j & 63);
        }
        from[threadIdx.x] = row;
    }
    __syncthreads();
    uint4 c[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int e = threadIdx.x + i * I8_MOVE_THREADS, which = e / (I8_PAGE * LANES), row = e / LANES % I8_PAGE;
        if (e < 2 * I8_PAGE * LANES && from[row] >= 0)
            c[i] = reinterpret_cast<const uint4*>((which ? v : k) + (size_t)from[row] * (16 * LANES))[e % LANES];
    }
    if (threadIdx.x < 2 * I8_PAGE) {                           // four warps: 32 rows of keys or values each, whose maxima blocks of 16 share
        const int which = threadIdx.x / I8_PAGE, row = threadIdx.x % I8_PAGE;
        const float mine = from[row] >= 0 ? (which ? v_scale : k_scale)[from[row] / block] : 0.f;
        scale[which][row] = mine;
    } else if (weight && threadIdx.x < 3 * I8_PAGE) {
        const int row = threadIdx.x - 2 * I8_PAGE;
        if (from[row] >= 0) weight[head_at * I8_PAGE + row] = weight[from[row]];
    }
    const bool homeless = __syncthreads_or(threadIdx.x < I8_PAGE && from[threadIdx.x % I8_PAGE] == -2);
    auto largest = [&](int which, int first) {
        float m = 0.f;
        for (int r = first; r < first + block; r += 4) {
            const float4 f = *reinterpret_cast<const float4*>(&scale[which][r]);
            m = fmaxf(fmaxf(m, fmaxf(f.x, f.y)), fmaxf(f.z, f.w));
        }
        return m;
    };
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int e = threadIdx.x + i * I8_MOVE_THREADS, which = e / (I8_PAGE * LANES), row = e / LANES % I8_PAGE;
        if (e >= 2 * I8_PAGE * LANES || from[row] < 0) continue;
        const int first = row / block * block;
        const float m = largest(which, first);
        if (e % LANES == 0 && row == first) (which ? v_scale : k_scale)[head_at * per + row / block] = m;        // the block's first row is kept if any is
        if (scale[which][row] != m) {
            const float ratio = __fdiv_rn(scale[which][row], m);
            c[i].x = i8_rescale4(c[i].x, ratio); c[i].y = i8_rescale4(c[i].y, ratio);
            c[i].z = i8_rescale4(c[i].z, ratio); c[i].w = i8_rescale4(c[i].w, ratio);
        }
        reinterpret_cast<uint4*>((which ? v : k) + (head_at * I8_PAGE + row) * (16 * LANES))[e % LANES] = c[i];
    }
    if (homeless)
        for (int e = threadIdx.x; e < 2 * I8_PAGE * LANES; e += I8_MOVE_THREADS) {
            const int which = e / (I8_PAGE * LANES), row = e / LANES % I8_PAGE, first = row / block * block;
            if (from[row] != -2) continue;
            reinterpret_cast<uint4*>((which ? v : k) + (head_at * I8_PAGE + row) * (16 * LANES))[e % LANES] = make_uint4(0, 0, 0, 0);
            if (e % LANES == 0 && row == first) (which ? v_scale : k_scale)[head_at * per + row / block] = largest(which, first);
            if (e % LANES == 0 && weight && !which) weight[head_at * I8_PAGE + row] = 0.f;
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
    // blocks a (sequence, kv head) by the longest sequence there can be.  us of selecting 512 and moving them with 1, 4 and 8 blocks (a
    // place a lane and turn): 8 x 4,000 places 32.8, 32.5 and 48; 8 x 8,000 38.8, 35.2 and 51; 8 x 32,000 117, 45 and 62; 64,000 179,
    // 35.7 and 33.3; 4 x 131,000 503, 122 and 83.  Above 65,536 the ranks of four blocks' places do not fit their shared memory.
    const long long longest = (long long)max_pages * I8_PAGE;
    const int cluster = longest <= 4096 ? 1 : longest <= 65536 ? 4 : 8;
    // a warp's share of a block's places, in whole 128, as the kernel has it for the longest
    const long long block_most = ((long long)max_pages + cluster - 1) / cluster * I8_PAGE, warp_most = ((block_most + I8_SELECT_WARPS - 1) / I8_SELECT_WARPS + 127) / 128 * 128;
    const int held = (int)std::min<long long>(I8_SELECT_KEEP, warp_most * I8_SELECT_WARPS);
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(int8_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, I8_SELECT_KEEP * 4);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    if ((long long)n_seqs * n_kv * cluster > 0x7fffffffLL) return SSB_ERR_BAD_SIZE;
    int rc = ssb_launch_cluster(int8_select_kernel, dim3(n_seqs * n_kv * cluster), dim3(I8_SELECT_THREADS), (size_t)held * 4, stream, true, cluster,
                                (const float*)weight, page_table, n_slots, max_pages, n_pages, seq_slot, lengths, n_kv, keep, first, recent, cluster,
                                held, kept);
    if (rc) return rc;
#define I8_MOVE(L_) \
    return ssb_launch(int8_move_kernel<L_>, dim3((keep + I8_PAGE - 1) / I8_PAGE, n_kv, n_seqs), dim3(I8_MOVE_THREADS), 0, stream, true, \
                      (int8_t*)k, (int8_t*)v, k_scale, v_scale, weight, page_table, n_slots, max_pages, n_pages, seq_slot, new_table, \
                      new_pages, n_kv, block, keep, (const int*)kept)
    switch (head_dim) {
        case 16: I8_MOVE(1);
        case 32: I8_MOVE(2);
        case 64: I8_MOVE(4);
        case 128: I8_MOVE(8);
        case 256: I8_MOVE(16);
    }
#undef I8_MOVE
    return SSB_ERR_BAD_SIZE;
}

SSB_PACKED(ssb_int8_append)
SSB_PACKED(ssb_int8_read)
SSB_PACKED(ssb_int8_evict)
