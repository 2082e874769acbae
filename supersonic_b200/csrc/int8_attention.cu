// Attention over a cache in 8 bits (see int8_cache.cu), in packed sequences: row i of a sequence that held ``start`` tokens before
// the step sees the keys start + i - window < j <= start + i of its slot.
//   s_ij = scale * ks_j * (q_i . kc_j),   o_i = sum_j softmax_j(s_ij) * vs_j * vc_j,   lse_i = ln sum_j exp(s_ij)
// with codes kc, vc and their blocks' scales ks, vs.  The rows that keep account add exp(s_ij - lse_i), summed over the query
// heads of a kv head, to the weight of key j.
#include "int8_attention.cuh"
#include "packed_call.cuh"
#include "tc_helpers.cuh"
#include <cuda_fp16.h>
#include <math.h>
#include <algorithm>
#include <atomic>
#include <type_traits>

typedef __nv_bfloat16 bf16;

// ---- head sizes other than 64 and 128, and more than 32 query heads a kv head -------------------------------------------
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
    const IaSeq seq = ia_sequence(a, lo);
    const int s = row >= seq.row0 && row < seq.row0 + seq.n_new ? seq.slot : -1, at = seq.start + row - seq.row0;
    const int last = s < 0 ? -1 : (int)min((long long)at, (long long)a.max_pages * IA_PAGE - 1);
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
        if (!ia_in_pool(a, page)) continue;
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
        d *= a.scale * a.k_scale[r >> a.shift];
        const float m_new = fmaxf(m, d), keep = m == -INFINITY ? 0.f : expf(m - m_new), p = expf(d - m_new);
        l = l * keep + p;
        m = m_new;
        const float pv = p * a.v_scale[r >> a.shift];
#pragma unroll
        for (int w = 0; w < 2; ++w)
            if (lane + 32 * w < words) {
                const uint32_t c = reinterpret_cast<const uint32_t*>(a.v + r * a.head_dim)[lane + 32 * w];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[w][e] = fmaf(pv, (float)(int8_t)(c >> (8 * e)), o[w][e] * keep);
            }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int w = 0; w < 2; ++w)
        if (lane + 32 * w < words)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                ((T*)a.out)[(size_t)row * a.ldo + (size_t)head * a.head_dim + 4 * (lane + 32 * w) + e] = ssb_from_float<T>(o[w][e] * inv);
    if (lane == 0 && a.lse) a.lse[(size_t)row * a.n_q + head] = l == 0.f ? -INFINITY : m + logf(l);
}

// What the last rows of every sequence attend to: a warp a key, over those rows and the heads of the group; the key's weight is its
// alone to add to, so the sum has one order.
template <typename T>
__global__ void __launch_bounds__(128)
int8_weigh_plain_kernel(const IaArgs a) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = a.head_dim / 4, group = a.n_q / a.n_kv;
    const int kvh = blockIdx.y;
    const auto [row0, n_new, start, s] = ia_sequence(a, blockIdx.z);
    if (s < 0 || n_new <= 0) return;
    const int i0 = max(0, n_new - a.weigh_last);
    const int end = (int)min((long long)start + n_new, (long long)a.max_pages * IA_PAGE);
    const int begin = a.window > 0 ? max(0, start + i0 - a.window + 1) : 0;
    for (int j = begin + (int)blockIdx.x * 4 + warp; j < end; j += gridDim.x * 4) {
        const int page = a.page_table[(size_t)s * a.max_pages + (j >> 6)];
        if (!ia_in_pool(a, page)) continue;
        const size_t r = ((size_t)page * a.n_kv + kvh) * IA_PAGE + (j & 63);
        const float ks = a.scale * a.k_scale[r >> a.shift];
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

// ---- tensor cores, a page at a time ---------------------------------------------------------------------------------
// Rows of a step that share a kv head (the query heads of its group, and up to 2^tts neighbouring tokens) are the columns, the 16
// keys of a warp what is summed over.  Scores take the codes as they are, in products of 8-bit integers (m16n8k32): a query goes
// times the power of two that brings its largest element to 2^29 .. 2^30, is rounded to a whole number (which keeps all of a
// float32 and more), and its four bytes, as digits -128 .. 127, are rows of the A operand, 8 columns' two digits an instruction; K
// is the B operand as it lies in memory.  The sums are exact and are put together in float32.  O^T = V^T P^T is in float16
// (m16n8k16): codes are whole numbers up to 127, which float16 holds exactly; probabilities are rounded to its 11 bits, or (WIDE,
// float32 rows) go in two halves.  The scores' registers are the B operand's, so nothing moves between lanes.
// The scales stay outside the products: a key's goes onto the score; a value's, f * 2^x, into the exponent (x) and onto the
// probability (f), with the running maximum taken over score + x, so that float16 holds what is summed.  The sum of weights takes x
// back in float32: all keys count in it whose values' scales are within 2^90 of one another.  The maximum is rounded up to a whole
// number, in the log2 domain: taking x and it off a score then costs no bits.
//
// Value codes become float16 in registers: 1024 + (code + 128) is a float16 whose low byte is the code with its sign bit turned, so
// two keys' four codes take two exclusive-ors, six byte permutations and four subtractions.  Which key is which column or k of
// the products, and which dims its k-steps, is free as long as both operands agree: chosen so that every lane reads whole 16-byte
// pieces of a row, a quarter-warp from 8 banks' groups (head size 128).
//
// The launch's work is its pages: tiles of rows x pages that they see, dealt out evenly over the blocks wherever a tile ends (a
// block finds its range from the batch's integers alone).  A tile that lies in one block's range is finished there; pieces of
// others go to scratch, and int8_finish_kernel puts them together in the order of the keys.  Nothing is left from one launch
// to the next.
constexpr int IR_THREADS = 128, IR_WARPS = 4, IR_SEQS = 1024, IR_STAGES = 3;
// What beginning and ending a tile costs, in pages.  us with 0, 1, 3, 6, 8 and 11: 64 sequences of 1 to 8,192 135, 130, 110, 102.6, 105
// and 109; 32 of 20 to 4,000 (64 dims) 51, 39, 31, 29.9, 30.9 and 32.7; 64 of 2,000 with 3, 6 and 11 58.4, 59.8 and 60.7.
constexpr int IR_EXTRA = 6;
constexpr long long IR_KEPT_MOST = 1LL << 26;  // floats
constexpr float IR_NONE = -1e30f;               // a maximum over no key: finite, so that nothing below needs to ask for it
constexpr int IR_SIDE = 12;                  // beside a stage's page: its scales of keys and of values, and its id
constexpr int IR_LEAST_X = -80, IR_MOST_X = 120;
constexpr float IR_NO_PAGE = -1.f;           // in the place of the scales of a page id that names no page

// What the dealing needs: tokens a tile (1 << tts), the window, and the batch with the units before each sequence.
struct IrBatch {
    const IaSeq* seqs;
    const long long* cum;                // [n_seqs + 1]
    int n_seqs, n_kv, tts, window;
    bool one_tile;                       // a sequence's rows are one tile, however many
    int extra;                           // what beginning and ending a tile costs, in pages: units without a page before its first

    // sum over i < t of floor(max(0, a + i * 2^tts) / 64)
    __device__ long long floors(long long t, long long a) const {
        if (a < 0) {
            const long long skip = min(t, (-a + (1 << tts) - 1) >> tts);
            t -= skip;
            a += skip << tts;
            if (a < 0) return 0;
        }
        const int gs = 6 - tts;
        auto ramp = [&](long long m) { const long long q = m >> gs; return (q * (q - 1) / 2 << gs) + q * (m & ((1 << gs) - 1)); };
        const long long r0 = (a & 63) >> tts;
        return (a >> 6) * t + ramp(r0 + t) - ramp(r0);
    }
    __device__ int tiles(const IaSeq& s) const { return s.slot < 0 || s.n_new <= 0 ? 0 : one_tile ? 1 : (s.n_new + (1 << tts) - 1) >> tts; }
    // units of the first t tiles of a sequence: the pages that each sees, and the extra ones
    __device__ long long units_before(const IaSeq& s, long long t) const {
        if (one_tile) return t * (((s.start + s.n_new - 1) >> 6) - first_page(s, 0) + 1 + extra);
        return t * (1 + extra) + floors(t, (long long)s.start + (1 << tts) - 1) - (window > 0 ? floors(t, (long long)s.start - window + 1) : 0);
    }
    __device__ int first_page(const IaSeq& s, int tile) const {
        const long long lo = (long long)s.start + ((long long)tile << tts) - window + 1;
        return window > 0 && lo > 0 ? (int)(lo >> 6) : 0;
    }
};

// A run of pages of one tile and kv head: what of it lies in a block's range.
struct IrSegment {
    int b, kvh, tile, page, n;           // pages page .. page + n - 1 of the sequence (n may be 0)
    long long first, last, at, next;     // the units of the tile's first and last page, the segment's first, and the one behind it
    bool begins, whole;                  // has the tile's first page; all of them
};

__device__ __forceinline__ IrSegment ir_locate(const IrBatch& B, long long u, long long end) {
    int lo = 0, hi = B.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (B.cum[mid] <= u) lo = mid; else hi = mid - 1;
    }
    const IaSeq s = B.seqs[lo];
    IrSegment g;
    g.b = lo;
    const int tiles = B.tiles(s);
    const long long per = tiles == 1 ? B.units_before(s, 1) : (B.cum[lo + 1] - B.cum[lo]) / B.n_kv;
    long long r = u - B.cum[lo];
    // r / per, below n_kv: by float32, and put right
    int h = (int)((float)r / (float)per);
    while (h > 0 && h * per > r) --h;
    while ((h + 1) * per <= r) ++h;
    g.kvh = h;
    r -= h * per;
    int t0 = 0, t1 = tiles - 1;          // the last tile that begins at or before the unit
    while (t0 < t1) {
        const int mid = (t0 + t1 + 1) >> 1;
        if (B.units_before(s, mid) <= r) t0 = mid; else t1 = mid - 1;
    }
    const long long before = t0 ? B.units_before(s, t0) : 0, units = (tiles == 1 ? per : B.units_before(s, t0 + 1)) - before;
    g.tile = t0;
    g.first = u - (r - before) + B.extra;
    g.last = g.first + units - B.extra - 1;
    const long long from = max(u, g.first);
    g.at = from;
    g.next = min(g.last + 1, end);
    g.n = (int)max(0LL, g.next - from);
    g.page = B.first_page(s, t0) + (int)(from - g.first);
    g.begins = from == g.first;
    g.whole = g.begins && g.next == g.last + 1;
    return g;
}

// Reads the batch and sums its units up; every thread of the block gets the total.
__device__ __forceinline__ long long ir_read_batch(const IaArgs& a, int s0, int n_seqs, IrBatch& B, IaSeq* seqs, long long* cum,
                                                   long long* warp_total, int last = 0) {
    for (int b = threadIdx.x; b < n_seqs; b += IR_THREADS) {
        const IaSeq s = ia_sequence(a, s0 + b);
        const int skip = last > 0 && s.n_new > last ? s.n_new - last : 0;    // with ``last``, that many last rows only
        seqs[b] = IaSeq{s.row0 + skip, s.n_new - skip, s.start + skip, s.slot};
    }
    __syncthreads();
    const int per = (n_seqs + IR_THREADS - 1) / IR_THREADS, b0 = (int)threadIdx.x * per, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto units_of = [&](int b) { return b < n_seqs ? B.units_before(seqs[b], B.tiles(seqs[b])) * B.n_kv : 0LL; };
    long long local = 0;
    for (int i = 0; i < per; ++i) local += units_of(b0 + i);
    long long incl = local;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) warp_total[warp] = incl;
    __syncthreads();
    long long base = 0, total = 0;
    for (int w = 0; w < IR_WARPS; ++w) {
        if (w < warp) base += warp_total[w];
        total += warp_total[w];
    }
    long long running = base + incl - local;
    for (int i = 0; i < per; ++i)
        if (b0 + i < n_seqs) { cum[b0 + i] = running; running += units_of(b0 + i); }
    if (threadIdx.x == 0) cum[n_seqs] = total;
    __syncthreads();
    B.seqs = seqs;
    B.cum = cum;
    B.n_seqs = n_seqs;
    return total;
}
// Where block c's units begin; no more blocks are dealt to than there are units, so that none of those is left without.
__device__ __forceinline__ long long ir_begin(long long total, int c, int blocks) { return total * min(c, blocks) / blocks; }
__device__ __forceinline__ int ir_dealt(long long total) { return (int)max(1LL, min((long long)gridDim.x, total)); }
__device__ __forceinline__ int ir_owner(long long unit, long long total, int blocks) { return (int)(((unit + 1) * blocks - 1) / total); }

__device__ __forceinline__ float ir_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ir_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ir_mma8(int (&c)[4], const uint4& a, uint32_t b0, uint32_t b1, bool first) {
    if (first)
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(0));
    else
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t ir_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// The bytes of ``w`` that ``sel`` puts into the low byte of each half (codes with their sign bit turned), as float16 codes.
__device__ __forceinline__ uint32_t ir_codes(uint32_t w, uint32_t sel) {
    const uint32_t v = __byte_perm(w, 0x64646464u, sel);
    const uint32_t bias = 0x64806480u;                            // 1024 + 128
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Byte offset of 16-byte piece c of row r of a page tile as the TMA unit leaves it (rows of 128 or 64 bytes with the swizzle of
// that width).
template <int HD> __device__ __forceinline__ uint32_t ir_at(int r, int c) {
    return HD == 128 ? (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)) : (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
// Column g of eight keys is key ir_key_of(g) of them: a lane's columns 2 t, 2 t + 1 are keys t and t + 4.
__device__ __forceinline__ int ir_key_of(int g) { return (g >> 1) + 4 * (g & 1); }

// Words of a column tile's queries: for each 64 dims and half of 16-byte pieces two pairs of digits, four words a lane.
template <int HD> constexpr int ir_q_words() { return HD / 64 * 2 * 2 * 32 * 4; }

// Scores of a warp's 16 keys: of column 8 i + g with keys t, t + 4, t + 8, t + 12.
template <int HD, int NT>
__device__ __forceinline__ void ir_scores(const unsigned char* keys, const uint32_t* qs, int warp, int lane, float (&s)[NT][4]) {
    const int g = lane >> 2, t = lane & 3, r0 = 16 * warp + ir_key_of(g);
    constexpr int H = HD / 64;
    uint4 k[2][H];
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j) k[j][h] = *reinterpret_cast<const uint4*>(keys + ir_at<HD>(r0 + 8 * j, 4 * h + t));
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        int sum[2][2][4];                                        // [pair of digits][eight keys]
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    const uint4 q = reinterpret_cast<const uint4*>(qs)[(((i * H + h) * 2 + half) * 2 + d) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        ir_mma8(sum[d][j], q, half ? k[j][h].z : k[j][h].x, half ? k[j][h].w : k[j][h].y, h == 0 && half == 0);
                }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = e >> 1, c = e & 1;
            s[i][e] = fmaf((float)(sum[0][j][c] * 256 + sum[0][j][c + 2]), 65536.f, (float)(sum[1][j][c] * 256 + sum[1][j][c + 2]));
        }
    }
}

// Query columns c0 .. c0 + 8 NT - 1 of a (sequence, kv head) as digits of the products' A operand, and each column's factor (scale *
// log2 e over its power of two; no number for a column that holds one that is not finite).  Column c: token c / group of the
// tile, head c % group.
template <int HD, int NT, bool WIDE>
__device__ __forceinline__ void ir_queries(const IaArgs& a, int row0, int n_tokens, int kvh, int c0, uint32_t* qs, float* qf) {
    using T = typename std::conditional<WIDE, float, bf16>::type;
    constexpr int LANES = HD / 8;                                // lanes a column, 8 elements each
    const int group = a.n_q / a.n_kv, l = threadIdx.x % LANES;
#pragma unroll
    for (int pass = 0; pass < (8 * NT * LANES + IR_THREADS - 1) / IR_THREADS; ++pass) {
        const int col = pass * (IR_THREADS / LANES) + threadIdx.x / LANES, c = c0 + col, token = c / group;
        float x[8] = {};
        if (col < 8 * NT && token < n_tokens) {
            const T* src = (const T*)a.q + (size_t)(row0 + token) * a.ldq + (size_t)(kvh * group + c % group) * HD + 8 * l;
            if constexpr (WIDE) {
                const float4 u = reinterpret_cast<const float4*>(src)[0], v = reinterpret_cast<const float4*>(src)[1];
                x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
            } else {
                const uint4 v = *reinterpret_cast<const uint4*>(src);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
            }
        }
        uint32_t most = 0;                                       // magnitudes in the order of their bits: no number is above infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int up = most ? min(29 - ((int)(most >> 23) - 127), 126) : 0;
        const float times = __uint_as_float((uint32_t)(127 + up) << 23), back = __uint_as_float((uint32_t)(127 - up) << 23);
        if (col < 8 * NT) {
            const int piece = l >> 1, lane = (col & 7) * 4 + (piece & 3);
            uint32_t n[8], w[4][2];                              // digit, four elements
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = ((uint32_t)__float2int_rn(x[i] * times) + 0x00808080u) ^ 0x00808080u;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t sel = 0x0040u + 0x11u * d;     // byte d of two words
                    w[d][i] = __byte_perm(__byte_perm(n[4 * i], n[4 * i + 1], sel), __byte_perm(n[4 * i + 2], n[4 * i + 3], sel), 0x5410);
                }
            uint4* at = reinterpret_cast<uint4*>(qs) + ((((col >> 3) * (HD / 64) + (piece >> 2)) * 2 + (l & 1)) * 2) * 32 + lane;
            at[0] = make_uint4(w[3][0], w[2][0], w[3][1], w[2][1]);
            at[32] = make_uint4(w[1][0], w[0][0], w[1][1], w[0][1]);
            if (l == 0) qf[col] = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : a.scale * 1.4426950408889634f * back;
        }
    }
}

// mbar_wait, asking once before the clock is read.
__device__ __forceinline__ bool ir_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    uint32_t ok;
    asm volatile("{\n.reg .pred P1;\nmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2;\nselp.b32 %0, 1, 0, P1;\n}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok || mbar_wait(bar, parity, abort_flag);
}

// Pages on their way into the ring: warp 0 asks for them, up to IR_STAGES - 1 ahead of the warps that work.
template <int HD, bool VALUES> constexpr int ir_stage_bytes() { return (VALUES ? 2 : 1) * 64 * HD; }

struct IrFeed {
    IrSegment seg;
    long long next, end;                 // the unit behind the segment
    int left, ids, ids_from, issued;     // pages of the segment not yet asked for; page ids of 32 pages, one a lane
    int stage, lap;                      // where the next page goes
};

template <int HD, bool VALUES>
__device__ __forceinline__ bool ir_feed(const IaArgs& a, const IrBatch& B, IrFeed& f, unsigned char* stages, float* scales, uint32_t full0,
                                        uint32_t empty0, const CUtensorMap& map_k, const CUtensorMap& map_v, volatile int* abort_flag) {
    const int lane = threadIdx.x & 31, per = 64 >> a.shift;
    while (f.left == 0) {
        if (f.next >= f.end) return true;
        f.seg = ir_locate(B, f.next, f.end);
        f.next = f.seg.next;
        f.left = f.seg.n;
        f.ids_from = -1;
    }
    const IaSeq s = B.seqs[f.seg.b];
    const int i = f.seg.n - f.left;
    if (f.ids_from < 0 || i - f.ids_from >= 32) {
        // a tile that is not full may count a page behind the sequence's last: the last again, which no row of it sees; one that starts
        // behind the table counts pages there, which are none
        const int page = f.seg.page + i + lane;
        const int named = a.page_table[(size_t)s.slot * a.max_pages + min(min(page, (s.start + s.n_new - 1) >> 6), a.max_pages - 1)];
        f.ids = page < a.max_pages && ia_in_pool(a, named) ? named : -1;
        f.ids_from = i;
    }
    const int named = __shfl_sync(0xffffffffu, f.ids, i - f.ids_from), id = max(named, 0);      // of no page: any, unseen
    const int st = f.stage;
    bool ok = true;
    if (lane == 0) ok = ir_wait(empty0 + 8 * st, f.lap ^ 1, abort_flag);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (!ok) return false;
    const size_t head = (size_t)id * a.n_kv + f.seg.kvh;
    if (named < 0) {
        if (lane < 2 * per) scales[IR_SIDE * st + lane] = IR_NO_PAGE;
        __syncwarp();                                              // before lane 0's arrival at the barrier, below
    } else if (lane < 2 * per) {
        const float* src = (lane < per ? a.k_scale : a.v_scale) + head * per + (lane & (per - 1));
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(scales + IR_SIDE * st + lane)), "l"(src) : "memory");
    }
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full0 + 8 * st) : "memory");
    if (lane == 0) {
        if (!VALUES) scales[IR_SIDE * st + 8] = __int_as_float(named);
        const uint32_t dst = smem_u32(stages + st * ir_stage_bytes<HD, VALUES>());
        mbar_expect_tx(full0 + 8 * st, ir_stage_bytes<HD, VALUES>());
        tma_load_2d(dst, &map_k, full0 + 8 * st, 0, (int)(head * 64));
        if (VALUES) tma_load_2d(dst + 64 * HD, &map_v, full0 + 8 * st, 0, (int)(head * 64));
    }
    if (++f.stage == IR_STAGES) { f.stage = 0; f.lap ^= 1; }
    ++f.issued;
    --f.left;
    return true;
}

template <int HD> constexpr int ir_acc_ld() { return HD + 4; }
template <int HD, int NT> constexpr int ir_work_words() {
    return 8 * NT * ir_acc_ld<HD>() > NT * ir_q_words<HD>() ? 8 * NT * ir_acc_ld<HD>() : NT * ir_q_words<HD>();
}
template <int HD, int NT> constexpr size_t ir_smem(int n_seqs) {
    return 1024 + (size_t)IR_STAGES * ir_stage_bytes<HD, true>() + (size_t)ir_work_words<HD, NT>() * 4 + IR_STAGES * IR_SIDE * 4 + 2 * IR_STAGES * 8 + (size_t)n_seqs * (sizeof(IaSeq) + 8) + 8;
}
// floats of a piece: a column's sums, its maximum and its sum of weights
template <int HD, int NT> constexpr int ir_piece() { return 8 * NT * (HD + 2); }

template <typename T> __device__ __forceinline__ void ir_store4(T* p, float4 v);
template <> __device__ __forceinline__ void ir_store4<float>(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
template <> __device__ __forceinline__ void ir_store4<bf16>(bf16* p, float4 v) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}
// What a column's result is written as.
template <int HD, bool WIDE>
__device__ __forceinline__ void ir_put(const IaArgs& a, const IaSeq& s, int tile, int tts, int kvh, int col, int d, float4 o, float m, float l, float offset) {
    using T = typename std::conditional<WIDE, float, bf16>::type;
    const int group = a.n_q / a.n_kv, token = (tile << tts) + col / group, head = kvh * group + col % group;
    if (col / group >= (1 << tts) || token >= s.n_new) return;
    const size_t row = (size_t)(s.row0 + token);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    ir_store4<T>((T*)a.out + row * a.ldo + (size_t)head * HD + d, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (d == 0 && a.lse) a.lse[row * a.n_q + head] = l == 0.f ? -INFINITY : (m - offset + log2f(l)) * 0.6931471805599453f;
}

// Single tokens and few rows.  64 sequences of 1 to 8,192 tokens, 32 heads over 8 of 128, bfloat16: 102 us with the joining, 5.5 TB/s, bound by the pages
// in flight (three a block, four blocks an SM); 16 of 8,000, 32 over 8 of 64, float32: 45 us, 3 TB/s, by instructions (a page has half
// the bytes there, and probabilities go in two halves).  NT, tiles of 8 columns: the fewest that hold the group (and up to 4 where
// neighbouring tokens fill them): 8 x 4,000 single tokens of a group of 4 with 1, 2 and 4 tiles 28, 38 and 57 us, four new tokens 39, 39
// and 58.
template <int HD, int NT, bool WIDE>
__global__ void __launch_bounds__(IR_THREADS, NT == 1 ? 4 : 2)
int8_rows_kernel(const IaArgs a, int s0, int n_seqs, int tts, float* __restrict__ pieces, float* __restrict__ kept, int* __restrict__ error_word,
                 const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    // probabilities are summed times 2^OFFSET and may exceed that by 2^LAZY before the reference maximum is moved; with f below 2
    // and both in float16, 2^(OFFSET + LAZY + 1) stays below 2^16
    constexpr float OFFSET = WIDE ? 13.f : 2.f, LAZY = WIDE ? 1.f : 12.f;
    constexpr int C = 8 * NT, ACC_LD = ir_acc_ld<HD>(), TILES = HD / 16;
    using T = typename std::conditional<WIDE, float, bf16>::type;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* stages = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    // a segment's queries, and when all its pages are worked on its sums [column][ACC_LD]
    float* acc = (float*)(stages + IR_STAGES * ir_stage_bytes<HD, true>());
    uint32_t* qs = (uint32_t*)acc;
    float* scales = acc + ir_work_words<HD, NT>();                                // [stage][keys' | values' | page id]
    uint64_t* bars = (uint64_t*)(scales + IR_STAGES * IR_SIDE);                         // full, empty
    long long* cum = (long long*)(bars + 2 * IR_STAGES);
    IaSeq* seqs = (IaSeq*)(cum + n_seqs + 1);
    __shared__ float warp_m[IR_WARPS][C], warp_l[IR_WARPS][C], qf[C];
    __shared__ long long warp_total[IR_WARPS];
    __shared__ int sm_abort[2];
    volatile int* abort_flag = sm_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + IR_STAGES);
    const int block_at = (16 * warp) >> a.shift;                   // the warp's keys have one scale
    if (threadIdx.x == 0) {
        for (int i = 0; i < IR_STAGES; ++i) { mbar_init(full0 + 8 * i, 33); mbar_init(empty0 + 8 * i, IR_WARPS); }
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    IrBatch B{nullptr, nullptr, 0, a.n_kv, tts, a.window, false, IR_EXTRA};
    // dependents may start once all that came before this launch is done: they read the batch and the pages ahead of their own wait
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const long long total = ir_read_batch(a, s0, n_seqs, B, seqs, cum, warp_total);
    const int blocks = ir_dealt(total);
    const long long begin = ir_begin(total, blockIdx.x, blocks), end = ir_begin(total, blockIdx.x + 1, blocks);
    const int group = a.n_q / a.n_kv;

    // sequences without a slot: zeros
    for (int b = blockIdx.x; b < n_seqs; b += gridDim.x)
        if (seqs[b].slot < 0)
            for (int e = threadIdx.x; e < seqs[b].n_new * a.n_q * (HD / 4); e += IR_THREADS) {
                const int d = e % (HD / 4) * 4, head = e / (HD / 4) % a.n_q;
                const size_t row = (size_t)(seqs[b].row0 + e / (HD / 4) / a.n_q);
                ir_store4<T>((T*)a.out + row * a.ldo + (size_t)head * HD + d, make_float4(0.f, 0.f, 0.f, 0.f));
                if (d == 0 && a.lse) a.lse[row * a.n_q + head] = -INFINITY;
            }

    IrFeed feed{};
    feed.next = begin;
    feed.end = end;
    bool ok = true;
    if (warp == 0)
        for (int i = 0; ok && i < IR_STAGES - 1; ++i)
            ok = ir_feed<HD, true>(a, B, feed, stages, scales, full0, empty0, map_k, map_v, abort_flag);
    int st = 0, lap = 0;                                           // the stage of the page that comes next
    for (long long u = begin; u < end;) {
        const IrSegment seg = ir_locate(B, u, end);
        if (seg.n == 0) { u = seg.next; continue; }
        const IaSeq s = seqs[seg.b];
        const int token0 = seg.tile << tts, n_tokens = min(1 << tts, s.n_new - token0);
        ir_queries<HD, NT, WIDE>(a, s.row0 + token0, n_tokens, seg.kvh, 0, qs, qf);
        __syncthreads();
        // a column's last and first visible key, and those that all columns see
        int hi[NT], lo[NT];
        float m[NT], l[NT], factor[NT], o[TILES][NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int token = (8 * i + g) / group;
            hi[i] = token < n_tokens ? s.start + token0 + token : -1;
            lo[i] = a.window > 0 ? hi[i] - a.window + 1 : 0;
            m[i] = IR_NONE;
            l[i] = 0.f;
            factor[i] = qf[8 * i + g];
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;
        const int all_hi = s.start + token0, all_lo = a.window > 0 ? s.start + token0 + n_tokens - a.window : 0;
        for (int p = 0; p < seg.n; ++p, lap ^= st == IR_STAGES - 1, st = st == IR_STAGES - 1 ? 0 : st + 1) {
            if (warp == 0 && ok)
                ok = ir_feed<HD, true>(a, B, feed, stages, scales, full0, empty0, map_k, map_v, abort_flag);
            if (ok) ok = __all_sync(0xffffffffu, ir_wait(full0 + 8 * st, lap, abort_flag));
            if (!ok) {                                             // give up, but meet the others at the segment's end
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                continue;
            }
            const unsigned char* keys = stages + st * ir_stage_bytes<HD, true>();
            const unsigned char* values = keys + 64 * HD;
            const int key0 = (seg.page + p) * 64 + 16 * warp;
            const float ks = scales[IR_SIDE * st + block_at], vs = scales[IR_SIDE * st + (64 >> a.shift) + block_at];
            float sc[NT][4];
            ir_scores<HD, NT>(keys, qs, warp, lane, sc);
            // vs = f 2^x; what is no scale belongs to keys that nobody sees, and x = -inf leaves nothing of a page that is none
            const int x = min(max((int)(__float_as_uint(vs) >> 23 & 255) - 127, IR_LEAST_X), IR_MOST_X);
            const float fx = vs == IR_NO_PAGE ? -INFINITY : (float)x, down = __uint_as_float((uint32_t)(127 - x) << 23), f = fabsf(vs) < 3e38f ? vs * down : 0.f;
            const bool inside = key0 >= all_lo && key0 + 15 <= all_hi;
            float worst = -INFINITY;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const float by = factor[i] * ks;
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[i][e] *= by;
                if (!inside) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (key0 + t + 4 * e > hi[i] || key0 + t + 4 * e < lo[i]) sc[i][e] = -INFINITY;
                }
                worst = fmaxf(worst, fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])) - (m[i] - fx));
            }
            if (__any_sync(0xffffffffu, worst > LAZY)) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    float top = fmaxf(fmaxf(sc[i][0], sc[i][1]), fmaxf(sc[i][2], sc[i][3])) + fx;
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float now = fmaxf(m[i], ceilf(top)), alpha = ir_ex2(m[i] - now);
                    m[i] = now;
                    l[i] *= alpha;
                    const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);    // columns 2 t, 2 t + 1
#pragma unroll
                    for (int k = 0; k < TILES; ++k) { o[k][i][0] *= a0; o[k][i][1] *= a1; o[k][i][2] *= a0; o[k][i][3] *= a1; }
                }
            }
            if (NT == 1 && kept && g < group)                      // the scores as they are, for what accounts for them
                *reinterpret_cast<float4*>(kept + (((seg.at + p) * IR_WARPS + warp) * group + g) * 16 + 4 * t) = make_float4(sc[0][0], sc[0][1], sc[0][2], sc[0][3]);
            uint32_t p_hi[NT][2], p_lo[NT][2];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const float ref = m[i] - fx - OFFSET;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = ir_ex2(sc[i][e] - ref);
                l[i] = fmaf((v[0] + v[1]) + (v[2] + v[3]), down, l[i]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {                      // keys t, t + 4, then t + 8, t + 12
                    const float v0 = v[2 * h] * f, v1 = v[2 * h + 1] * f;
                    p_hi[i][h] = ir_half2(v0, v1);
                    if (WIDE) {
                        const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&p_hi[i][h]));
                        p_lo[i][h] = ir_half2(v0 - r.x, v1 - r.y);
                    }
                }
            }
            // values of keys t, t + 4, t + 8, t + 12 of the warp: HD / 8 dims of this lane each
            constexpr int WORDS = HD / 32;
            uint32_t vw[4][WORDS];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 16 * warp + t + 4 * j;
                if (HD == 128) {
                    const uint4 c = *reinterpret_cast<const uint4*>(values + ir_at<HD>(r, g));
                    vw[j][0] = c.x; vw[j][1] = c.y; vw[j][WORDS - 2] = c.z; vw[j][WORDS - 1] = c.w;
                } else {
                    const uint2 c = *reinterpret_cast<const uint2*>(values + ir_at<HD>(r, g >> 1) + 8 * (g & 1));
                    vw[j][0] = c.x; vw[j][1] = c.y;
                }
            }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                const uint32_t u0 = vw[0][w] ^ 0x80808080u, u1 = vw[1][w] ^ 0x80808080u, u2 = vw[2][w] ^ 0x80808080u, u3 = vw[3][w] ^ 0x80808080u;
#pragma unroll
                for (int h = 0; h < 2; ++h) {                      // two of the word's four dims: one tile of the products
                    const uint32_t lo2 = __byte_perm(u0, u1, h ? 0x7362 : 0x5140), hi2 = __byte_perm(u2, u3, h ? 0x7362 : 0x5140);
                    const uint32_t a0 = ir_codes(lo2, 0x4140), a1 = ir_codes(lo2, 0x4342), a2 = ir_codes(hi2, 0x4140), a3 = ir_codes(hi2, 0x4342);
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        if (WIDE) ir_mma(o[2 * w + h][i], a0, a1, a2, a3, p_lo[i][0], p_lo[i][1]);
                        ir_mma(o[2 * w + h][i], a0, a1, a2, a3, p_hi[i][0], p_hi[i][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty0 + 8 * st) : "memory");
        }
        // the warps' parts: a column's maximum and sum of weights, then its sums, warp after warp; dims (HD / 8) g + 2 k, + 1 of
        // the head lie at 16 k + 2 g
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) { warp_m[warp][8 * i + g] = m[i]; warp_l[warp][8 * i + g] = l[i]; }
        }
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < IR_WARPS; ++w) {
            if (warp == w) {
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int c = 8 * i + 2 * t + e;
                        const float by = ir_ex2(warp_m[w][c] - fmaxf(fmaxf(warp_m[0][c], warp_m[1][c]), fmaxf(warp_m[2][c], warp_m[3][c])));
#pragma unroll
                        for (int k = 0; k < TILES; ++k) {
                            float2* at = reinterpret_cast<float2*>(acc + c * ACC_LD + 16 * k + 2 * g);
                            const float2 was = w ? *at : make_float2(0.f, 0.f);
                            *at = make_float2(fmaf(o[k][i][e], by, was.x), fmaf(o[k][i][e + 2], by, was.y));
                        }
                    }
            }
            __syncthreads();
        }
        float* piece = pieces + (size_t)(2 * blockIdx.x + seg.begins) * ir_piece<HD, NT>();
        for (int e = threadIdx.x; e < C * (HD / 4); e += IR_THREADS) {
            const int c = e / (HD / 4), d = e % (HD / 4) * 4;
            const float top = fmaxf(fmaxf(warp_m[0][c], warp_m[1][c]), fmaxf(warp_m[2][c], warp_m[3][c]));
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < IR_WARPS; ++w) sum = fmaf(warp_l[w][c], ir_ex2(warp_m[w][c] - top), sum);
            const float* at = acc + c * ACC_LD + 16 * (d % (HD / 8) / 2) + 2 * (d / (HD / 8));
            const float2 x = *reinterpret_cast<const float2*>(at), y = *reinterpret_cast<const float2*>(at + 16);
            const float4 v = make_float4(x.x, x.y, y.x, y.y);
            if (seg.whole) {
                ir_put<HD, WIDE>(a, s, seg.tile, tts, seg.kvh, c, d, v, top, sum, OFFSET);
            } else {
                *reinterpret_cast<float4*>(piece + c * HD + d) = v;
                if (d == 0) { piece[C * HD + c] = top; piece[C * HD + C + c] = sum; }
            }
        }
        __syncthreads();                                           // the queries of the next segment go where the sums were
        u = seg.next;
    }
    if (!ok && warp == 0)                                          // let issued copies land before the block ends
        for (int i = max(0, feed.issued - IR_STAGES); i < feed.issued; ++i)
            mbar_wait(full0 + 8 * (i % IR_STAGES), (i / IR_STAGES) & 1, abort_flag + 1);
}

// Tiles whose pages lay in several blocks' ranges: block c, whose range may begin in the middle of one and end in another, takes its share
// of each one's sums, half a block a tile: a column's four dims a thread where there are many, else several threads with a part of
// the pieces each, put together by shuffles.  (A tile a block, whichever had its first page: one sequence of 4,000 tokens, whose 8
// tiles are 74 pieces each, 34 us instead of 15.)
template <int HD, int NT, bool WIDE>
__global__ void __launch_bounds__(IR_THREADS)
int8_finish_kernel(const IaArgs a, int s0, int n_seqs, int tts, const float* __restrict__ pieces) {
    constexpr float OFFSET = WIDE ? 13.f : 2.f;
    constexpr int C = 8 * NT, HALF = IR_THREADS / 2;
    extern __shared__ unsigned char smem_raw[];
    long long* cum = (long long*)smem_raw;
    IaSeq* seqs = (IaSeq*)(cum + n_seqs + 1);
    __shared__ long long warp_total[IR_WARPS];
    __shared__ float others[2][6][32];
    IrBatch B{nullptr, nullptr, 0, a.n_kv, tts, a.window, false, IR_EXTRA};
    ssb_pdl_launch_dependents();
    const long long total = ir_read_batch(a, s0, n_seqs, B, seqs, cum, warp_total);
    const int blocks = ir_dealt(total), c = blockIdx.x, half = threadIdx.x / HALF, thread = threadIdx.x % HALF, lane = threadIdx.x & 31;
    const long long begin = ir_begin(total, c, blocks), end = ir_begin(total, c + 1, blocks);
    // every block waits for the pieces, those without a share too: whoever waits for this launch has waited for them
    if (begin >= end) { ssb_pdl_wait(); return; }
    const IrSegment seg = ir_locate(B, half ? end - 1 : begin, end);
    const IaSeq s = seqs[seg.b];
    const int c0 = ir_owner(seg.first, total, blocks), c1 = ir_owner(seg.last, total, blocks), n_pieces = c1 - c0 + 1;
    const int live = min(C, min(1 << tts, s.n_new - (seg.tile << tts)) * (a.n_q / a.n_kv)) * (HD / 4);
    int e0 = (int)((long long)live * (c - c0) / n_pieces), e1 = (int)((long long)live * (c - c0 + 1) / n_pieces);
    if (half ? seg.first - B.extra <= begin : seg.last >= end - 1) (half ? e0 : e1) = (e0 + e1) / 2;        // both halves have this tile
    ssb_pdl_wait();
    if (n_pieces < 2 || c < c0 || c > c1) return;              // the same for the whole half
    auto piece = [&](int i) { return pieces + (size_t)(2 * i + (i == c0)) * ir_piece<HD, NT>(); };
    for (; e0 < e1; e0 += HALF) {
        const int n = min(HALF, e1 - e0), width = n > 32 ? HALF : n > 1 ? 1 << (32 - __clz(n - 1)) : 1, groups = HALF / width;
        const int e = e0 + min(thread % width, n - 1), col = e / (HD / 4), d = e % (HD / 4) * 4;
        float top = IR_NONE, sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int AT_ONCE = 4;                                 // pieces asked for together
        for (int i0 = c0 + thread / width; i0 <= c1; i0 += AT_ONCE * groups) {
            float pm[AT_ONCE], pl[AT_ONCE];
            float4 pv[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float* p = piece(min(i0 + i * groups, c1));
                pm[i] = i0 + i * groups <= c1 ? __ldcg(p + C * HD + col) : IR_NONE;
                pl[i] = __ldcg(p + C * HD + C + col);
                pv[i] = __ldcg(reinterpret_cast<const float4*>(p + col * HD + d));
            }
            const float now = fmaxf(top, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]))), keep = ir_ex2(top - now);
            v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep; sum *= keep;
            top = now;
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                const float by = i0 + i * groups <= c1 ? ir_ex2(pm[i] - now) : 0.f;
                v.x = fmaf(pv[i].x, by, v.x); v.y = fmaf(pv[i].y, by, v.y); v.z = fmaf(pv[i].z, by, v.z); v.w = fmaf(pv[i].w, by, v.w);
                sum = fmaf(pl[i], by, sum);
            }
        }
        auto add = [&](float t, float l, float x, float y, float z, float w) {
            const float now = fmaxf(top, t), keep = ir_ex2(top - now), by = ir_ex2(t - now);
            top = now;
            sum = sum * keep + l * by;
            v.x = v.x * keep + x * by; v.y = v.y * keep + y * by; v.z = v.z * keep + z * by; v.w = v.w * keep + w * by;
        };
        for (int o = width; o < 32; o <<= 1)
            add(__shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, sum, o), __shfl_xor_sync(0xffffffffu, v.x, o),
                __shfl_xor_sync(0xffffffffu, v.y, o), __shfl_xor_sync(0xffffffffu, v.z, o), __shfl_xor_sync(0xffffffffu, v.w, o));
        if (groups > 1) {                                          // the half's two warps
            float (&o)[6][32] = others[half];
            if (thread >= 32) { o[0][lane] = top; o[1][lane] = sum; o[2][lane] = v.x; o[3][lane] = v.y; o[4][lane] = v.z; o[5][lane] = v.w; }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(HALF) : "memory");
            if (thread < 32) add(o[0][lane], o[1][lane], o[2][lane], o[3][lane], o[4][lane], o[5][lane]);
        }
        if (thread < n) ir_put<HD, WIDE>(a, s, seg.tile, tts, seg.kvh, col, d, v, top, sum, OFFSET);
    }
}

// What single tokens attend to, from the scores that int8_rows_kernel kept: a page a warp, a lane four keys of every second head.  A row
// whose sum is no number makes the weights of the keys that it sees none, as the formula has it (eviction ranks those lowest).
// 16 sequences of 8,000, 32 heads over 8: 17 MB of scores in 13 us.
__global__ void __launch_bounds__(IR_THREADS)
int8_account_kernel(const IaArgs a, int s0, int n_seqs, const float* __restrict__ kept) {
    extern __shared__ unsigned char smem_raw[];
    long long* cum = (long long*)smem_raw;
    IaSeq* seqs = (IaSeq*)(cum + n_seqs + 1);
    __shared__ long long warp_total[IR_WARPS];
    IrBatch B{nullptr, nullptr, 0, a.n_kv, 0, a.window, false, IR_EXTRA};
    const long long total = ir_read_batch(a, s0, n_seqs, B, seqs, cum, warp_total);
    const int blocks = ir_dealt(total), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.n_q / a.n_kv;
    const long long begin = ir_begin(total, blockIdx.x, blocks), end = ir_begin(total, blockIdx.x + 1, blocks);
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    for (long long u = begin; u < end;) {
        const IrSegment seg = ir_locate(B, u, end);
        u = seg.next;
        const IaSeq s = seqs[seg.b];
        if (seg.n == 0) continue;
        // lanes 0 - 15 take heads 0, 2, .., the others 1, 3, ..: of up to 8
        float ref[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = 2 * i + (lane >> 4);
            ref[i] = h < group ? a.lse[(size_t)s.row0 * a.n_q + seg.kvh * group + h] * 1.4426950408889634f : INFINITY;
        }
        const int part = (lane & 15) >> 2, t = lane & 3;
        auto pages = [&](auto none) {                              // whether a row saw nothing or has no number for its sum: -inf, which it does not see, counts 0
#pragma unroll (decltype(none)::value ? 1 : 2)
            for (int p = warp; p < seg.n; p += IR_WARPS) {
                const float* src = kept + (seg.at + p) * (IR_WARPS * 16) * group;
                const int id = a.page_table[(size_t)s.slot * a.max_pages + min(seg.page + p, a.max_pages - 1)];
                const bool there = seg.page + p < a.max_pages && ia_in_pool(a, id);
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int h = 2 * i + (lane >> 4);
                    if (h < group) {
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(src + (part * group + h) * 16 + 4 * t));
                        auto weight = [&](float x) { return decltype(none)::value && x == -INFINITY ? 0.f : ir_ex2(x - ref[i]); };
                        sum.x += weight(v.x); sum.y += weight(v.y); sum.z += weight(v.z); sum.w += weight(v.w);
                    }
                }
                sum.x += __shfl_xor_sync(0xffffffffu, sum.x, 16); sum.y += __shfl_xor_sync(0xffffffffu, sum.y, 16);
                sum.z += __shfl_xor_sync(0xffffffffu, sum.z, 16); sum.w += __shfl_xor_sync(0xffffffffu, sum.w, 16);
                // keys t, t + 4, t + 8, t + 12 of 16: the lower half adds the first two, the upper the others; one addition a key, so in
                // one order, and nobody waits for it
                float* w = a.weight + ((size_t)id * a.n_kv + seg.kvh) * 64 + 16 * part + t + (lane & 16 ? 8 : 0);
                const float x = lane & 16 ? sum.z : sum.x, y = lane & 16 ? sum.w : sum.y;
                if (there && x != 0.f) atomicAdd(w, x);
                if (there && y != 0.f) atomicAdd(w + 4, y);
            }
        };
        if (__all_sync(0xffffffffu, ref[0] > -INFINITY && ref[1] > -INFINITY && ref[2] > -INFINITY && ref[3] > -INFINITY)) pages(std::false_type{});
        else pages(std::true_type{});
    }
}

// What the last rows of every sequence attend to, from their lse: the keys once more, 8 NT of the (row, head) columns at a time, QB
// such batches beside each page.  A key belongs to one block, which adds its columns' probabilities up in one order and then to the
// key's weight.
template <int HD, int NT, int QB> constexpr size_t ir_weigh_smem(int n_seqs) {
    return 1024 + (size_t)IR_STAGES * ir_stage_bytes<HD, false>() + (size_t)QB * NT * ir_q_words<HD>() * 4 + IR_STAGES * IR_SIDE * 4 +
           2 * IR_STAGES * 8 + (size_t)n_seqs * (sizeof(IaSeq) + 8) + 8;
}
template <int HD, int NT, int QB, bool WIDE>
__global__ void __launch_bounds__(IR_THREADS)
int8_weigh_kernel(const IaArgs a, int s0, int n_seqs, int column0, int* __restrict__ error_word, const __grid_constant__ CUtensorMap map_k) {
    constexpr int C = 8 * NT, Q_WORDS = NT * ir_q_words<HD>();
    extern __shared__ unsigned char smem_raw[];
    unsigned char* stages = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint32_t* qs = (uint32_t*)(stages + IR_STAGES * ir_stage_bytes<HD, false>());
    float* scales = (float*)(qs + QB * Q_WORDS);
    uint64_t* bars = (uint64_t*)(scales + IR_STAGES * IR_SIDE);
    long long* cum = (long long*)(bars + 2 * IR_STAGES);
    IaSeq* seqs = (IaSeq*)(cum + n_seqs + 1);
    __shared__ float qf[QB * C], lse2[QB * C];
    __shared__ int last_of[QB * C];                                // the last key a column sees
    __shared__ long long warp_total[IR_WARPS];
    __shared__ int sm_abort[2];
    volatile int* abort_flag = sm_abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, group = a.n_q / a.n_kv;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + IR_STAGES);
    const int block_at = (16 * warp) >> a.shift;                   // the warp's keys have one scale
    if (threadIdx.x == 0) {
        for (int i = 0; i < IR_STAGES; ++i) { mbar_init(full0 + 8 * i, 33); mbar_init(empty0 + 8 * i, IR_WARPS); }
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    IrBatch B{nullptr, nullptr, 0, a.n_kv, 0, a.window, true, IR_EXTRA};
    const long long total = ir_read_batch(a, s0, n_seqs, B, seqs, cum, warp_total, a.weigh_last);
    const int blocks = ir_dealt(total);
    const long long begin = ir_begin(total, blockIdx.x, blocks), end = ir_begin(total, blockIdx.x + 1, blocks);
    IrFeed feed{};
    feed.next = begin;
    feed.end = end;
    bool ok = true;
    if (warp == 0)
        for (int i = 0; ok && i < IR_STAGES - 1; ++i)
            ok = ir_feed<HD, false>(a, B, feed, stages, scales, full0, empty0, map_k, map_k, abort_flag);
    ssb_pdl_wait();                                                // the rows' lse
    int st = 0, lap = 0;
    for (long long u = begin; u < end;) {
        const IrSegment seg = ir_locate(B, u, end);
        if (seg.n == 0) { u = seg.next; continue; }
        const IaSeq s = seqs[seg.b];
        __syncthreads();                                           // the segment before is done with its queries
        const int batches = min(QB, (s.n_new * group - column0 + C - 1) / C);      // may be none
        for (int q = 0; q < batches; ++q)
            ir_queries<HD, NT, WIDE>(a, s.row0, s.n_new, seg.kvh, column0 + q * C, qs + q * Q_WORDS, qf + q * C);
        for (int c = threadIdx.x; c < batches * C; c += IR_THREADS) {
            const int token = (column0 + c) / group;
            last_of[c] = s.start + token;
            lse2[c] = token < s.n_new ? a.lse[(size_t)(s.row0 + token) * a.n_q + seg.kvh * group + (column0 + c) % group] * 1.4426950408889634f : INFINITY;
        }
        __syncthreads();
        for (int p = 0; p < seg.n; ++p, lap ^= st == IR_STAGES - 1, st = st == IR_STAGES - 1 ? 0 : st + 1) {
            if (warp == 0 && ok)
                ok = ir_feed<HD, false>(a, B, feed, stages, scales, full0, empty0, map_k, map_k, abort_flag);
            if (ok) ok = __all_sync(0xffffffffu, ir_wait(full0 + 8 * st, lap, abort_flag));
            if (!ok) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                continue;
            }
            const unsigned char* keys = stages + st * ir_stage_bytes<HD, false>();
            const int key0 = (seg.page + p) * 64 + 16 * warp;
            const float ks = scales[IR_SIDE * st + block_at];
            const bool inside = key0 + 15 <= s.start + column0 / group && (a.window <= 0 || key0 > s.start + s.n_new - 1 - a.window);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};                   // keys t, t + 4, t + 8, t + 12
#pragma unroll 1
            for (int q = 0; q < batches; ++q) {
                float sc[NT][4];
                ir_scores<HD, NT>(keys, qs + q * Q_WORDS, warp, lane, sc);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const int c = q * C + 8 * i + g, at = last_of[c];
                    const float by = qf[c] * ks, ref = lse2[c];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = ir_ex2(sc[i][e] * by - ref);
                        const int key = key0 + t + 4 * e;
                        if (inside || (key <= at && (a.window <= 0 || key > at - a.window))) sum[e] += v;
                    }
                }
            }
            const int id = __float_as_int(scales[IR_SIDE * st + 8]);
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty0 + 8 * st) : "memory");
            // over the columns: eight lanes' four sums, two of them handed over at each of the first two steps
            const bool up2 = lane & 16, up1 = lane & 8;
            float x0 = up2 ? sum[2] : sum[0], x1 = up2 ? sum[3] : sum[1];
            x0 += __shfl_xor_sync(0xffffffffu, up2 ? sum[0] : sum[2], 16);
            x1 += __shfl_xor_sync(0xffffffffu, up2 ? sum[1] : sum[3], 16);
            float x = up1 ? x1 : x0;
            x += __shfl_xor_sync(0xffffffffu, up1 ? x0 : x1, 8);
            x += __shfl_xor_sync(0xffffffffu, x, 4);
            const int key = key0 + t + 4 * (2 * up2 + up1);
            if (!(lane & 4) && id >= 0 && key < s.start + s.n_new && x != 0.f)
                atomicAdd(a.weight + ((size_t)id * a.n_kv + seg.kvh) * 64 + (key & 63), x);
        }
        u = seg.next;
    }
    if (!ok && warp == 0)
        for (int i = max(0, feed.issued - IR_STAGES); i < feed.issued; ++i)
            mbar_wait(full0 + 8 * (i % IR_STAGES), (i / IR_STAGES) & 1, abort_flag + 1);
}

// ---- host side --------------------------------------------------------------------------------------------------------
static int ir_map(CUtensorMap* map, const void* codes, long long rows, int head_dim) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return SSB_ERR_UNSUPPORTED;
    if (rows > 0x7fffffffLL) return SSB_ERR_BAD_SIZE;
    cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)head_dim};
    cuuint32_t box[2] = {(cuuint32_t)head_dim, 64};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : SSB_ERR_BAD_SIZE;
}

// Blocks of a kernel that the device holds at once, at ``smem`` bytes a block.
template <typename K> static int ir_resident(K kernel, size_t smem) {
    int each = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kernel, IR_THREADS, smem) != cudaSuccess || each < 1) each = 1;
    return each * ssb_sm_count();
}
template <typename K> static int ir_configure(K kernel, size_t smem) {
    return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
}

struct IrPlan { int nt, tts, blocks; size_t piece; long long kept; };      // floats of a piece; of the scores that are kept

// Blocks of a launch over n_seqs sequences, or -1.  Host threads may ask at the same time for different sizes, and what a thread is told
// does not depend on who asked before: its scratch is sized by it.  Nothing here allocates or locks, so nothing is thrown.
template <int HD, int NT, bool WIDE> static int ir_blocks(int n_seqs) {
    constexpr int DEVICES = 8;                                     // of any others every call asks the driver
    static std::atomic<int> known[DEVICES][IR_SEQS + 1];           // 0: not asked yet
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) { cudaGetLastError(); return -1; }
    std::atomic<int>* at = device < DEVICES ? &known[device][n_seqs] : nullptr;
    int blocks = at ? at->load(std::memory_order_acquire) : 0;
    if (blocks == 0) {
        if (ir_configure(int8_rows_kernel<HD, NT, WIDE>, ir_smem<HD, NT>(IR_SEQS)) != 0) { cudaGetLastError(); return -1; }
        blocks = ir_resident(int8_rows_kernel<HD, NT, WIDE>, ir_smem<HD, NT>(n_seqs));
        if (at) at->store(blocks, std::memory_order_release);
    }
    return blocks;
}
#define IR_EACH(HD_, NT_, WIDE_, WHAT_) \
    do { \
        if (HD_ == 64) { \
            if (WIDE_) { if (NT_ == 1) { WHAT_(64, 1, true); } else if (NT_ == 2) { WHAT_(64, 2, true); } else { WHAT_(64, 4, true); } } \
            else { if (NT_ == 1) { WHAT_(64, 1, false); } else if (NT_ == 2) { WHAT_(64, 2, false); } else { WHAT_(64, 4, false); } } \
        } else { \
            if (WIDE_) { if (NT_ == 1) { WHAT_(128, 1, true); } else if (NT_ == 2) { WHAT_(128, 2, true); } else { WHAT_(128, 4, true); } } \
            else { if (NT_ == 1) { WHAT_(128, 1, false); } else if (NT_ == 2) { WHAT_(128, 2, false); } else { WHAT_(128, 4, false); } } \
        } \
    } while (0)

static bool ir_takes(int n_q, int n_kv, int head_dim) { return (head_dim == 64 || head_dim == 128) && n_q / n_kv <= 32; }

static IrPlan ir_plan(bool wide, int n_seqs, int rows, int max_new, int max_pages, int n_q, int n_kv, int head_dim, int window,
                      int weigh_last) {
    IrPlan p{};
    const int group = n_q / n_kv;
    const long long most = (long long)max_new * group;
    p.nt = most <= 8 ? 1 : most <= 16 ? 2 : 4;
    while (p.tts < 6 && (1 << p.tts) < max_new && (2 << p.tts) * group <= 8 * p.nt) ++p.tts;
    const int n = std::min(n_seqs, IR_SEQS);
#define IR_BLOCKS(H_, N_, W_) { p.blocks = ir_blocks<H_, N_, W_>(n); p.piece = ir_piece<H_, N_>(); }
    IR_EACH(head_dim, p.nt, wide, IR_BLOCKS);
#undef IR_BLOCKS
    const long long units = ((long long)(rows >> p.tts) + n_seqs) * n_kv * max_pages;
    p.blocks = (int)std::min<long long>(p.blocks, std::max(1LL, units));
    // single tokens that keep account: their scores are kept, a sixteenth to an eighth of what the pages hold, where that has a
    // bound (of the longest sequence there can be) that a scratch may have; else the keys are read once more.  16 sequences of 8,192,
    // 32 heads of 64 in float32: 59 us so, 73 with the keys read again.
    const long long spans = window > 0 ? (window + 62LL) / IA_PAGE + 1 : max_pages;      // pages a token sees at most
    const long long kept = (long long)n * n_kv * (spans + IR_EXTRA) * 64 * group;
    p.kept = weigh_last > 0 && max_new == 1 && p.nt == 1 && kept <= IR_KEPT_MOST ? kept : 0;
    return p;
}

static long long ir_scratch(const IrPlan& p) { return 2LL * p.blocks * (long long)p.piece + p.kept; }

// float32 elements of scratch that the launch needs.
SSB_API long long ssb_int8_attention_scratch(int dtype, int n_seqs, int rows, int max_new, int max_pages, int n_q, int n_kv, int head_dim,
                                             int window, int weigh_last, float scale) {
    if (n_seqs <= 0 || rows <= 0 || n_kv <= 0 || !ir_takes(n_q, n_kv, head_dim)) return 0;
    if (ia_tc_takes(dtype, head_dim, max_new, scale)) return ia_tc_scratch(n_seqs, rows, max_new, max_pages, n_q, n_kv, head_dim);
    const IrPlan p = ir_plan(dtype == SSB_F32, n_seqs, rows, max_new, max_pages, n_q, n_kv, head_dim, window, weigh_last);
    return p.blocks < 0 ? 0 : ir_scratch(p);
}

template <int HD, int NT, bool WIDE>
static int ir_rows(IaArgs a, const IrPlan& p, float* pieces, int* error_word, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
    float* kept = p.kept ? pieces + 2LL * p.blocks * (long long)p.piece : nullptr;
    if (kept) a.most_new = 1;                                      // which is what there is room for
    for (int s0 = 0; s0 < a.n_seqs; s0 += IR_SEQS) {
        const int n = std::min(IR_SEQS, a.n_seqs - s0);
        // not as a dependent of what came before: blocks that wait beside another launch's are dealt to SMs unevenly (64 sequences of
        // 1 to 8,192 tokens, one call behind another: 111 us, 162 as dependents, when a tile's cost was counted as 3 pages)
        int rc = ssb_launch(int8_rows_kernel<HD, NT, WIDE>, dim3(p.blocks), dim3(IR_THREADS), ir_smem<HD, NT>(n), stream, false, a, s0, n, p.tts,
                            pieces, kept, error_word, mk, mv);
        if (rc) return rc;
        rc = ssb_launch(int8_finish_kernel<HD, NT, WIDE>, dim3(p.blocks), dim3(IR_THREADS), (size_t)n * (sizeof(IaSeq) + 8) + 8, stream, true,
                        a, s0, n, p.tts, (const float*)pieces);
        if (rc) return rc;
        if (kept)
            rc = ssb_launch(int8_account_kernel, dim3(p.blocks), dim3(IR_THREADS), (size_t)n * (sizeof(IaSeq) + 8) + 8, stream, true, a, s0, n,
                            (const float*)kept);
        if (rc) return rc;
    }
    return 0;
}

template <int HD, int NT, int QB, bool WIDE>
static int ir_weigh(const IaArgs& a, int max_new, int* error_word, const CUtensorMap& mk, bool chained, cudaStream_t stream) {
    static int blocks = 0;
    if (blocks == 0) {
        const int rc = ir_configure(int8_weigh_kernel<HD, NT, QB, WIDE>, ir_weigh_smem<HD, NT, QB>(IR_SEQS));
        if (rc) return rc;
        blocks = ir_resident(int8_weigh_kernel<HD, NT, QB, WIDE>, ir_weigh_smem<HD, NT, QB>(64));
    }
    const long long columns = (long long)std::min(a.weigh_last, max_new) * (a.n_q / a.n_kv);
    for (int s0 = 0; s0 < a.n_seqs; s0 += IR_SEQS) {
        const int n = std::min(IR_SEQS, a.n_seqs - s0);
        const int grid = (int)std::min<long long>(blocks, (long long)n * a.n_kv * a.max_pages);
        for (long long c = 0; c < columns; c += 8 * NT * QB) {
            const int rc = ssb_launch(int8_weigh_kernel<HD, NT, QB, WIDE>, dim3(grid), dim3(IR_THREADS), ir_weigh_smem<HD, NT, QB>(n),
                                      stream, chained && s0 == 0 && c == 0, a, s0, n, (int)c, error_word, mk);
            if (rc) return rc;
        }
    }
    return 0;
}

static int ia_weigh(const IaArgs& a, bool wide, int max_new, int* error_word, const CUtensorMap& mk, cudaStream_t stream) {
    const long long columns = (long long)std::min(a.weigh_last, max_new) * (a.n_q / a.n_kv);
#define IR_WEIGH(N_, B_) \
    return a.head_dim == 64 ? (wide ? ir_weigh<64, N_, B_, true>(a, max_new, error_word, mk, true, stream) : ir_weigh<64, N_, B_, false>(a, max_new, error_word, mk, true, stream)) \
                            : (wide ? ir_weigh<128, N_, B_, true>(a, max_new, error_word, mk, true, stream) : ir_weigh<128, N_, B_, false>(a, max_new, error_word, mk, true, stream))
    if (columns <= 8) IR_WEIGH(1, 1);
    IR_WEIGH(4, 4);
#undef IR_WEIGH
}

SSB_API int ssb_int8_attention(const void* q, int ldq, int dtype, void* out, int ldo, float* lse, const void* k, const void* v,
                               const float* k_scale, const float* v_scale, float* weight, const int* page_table, int n_slots,
                               int max_pages, int n_pages, const int* cu_new, const int* seq_start, const int* seq_slot,
                               int n_seqs, int rows, int max_new, int n_q, int n_kv, int head_dim, int block, int window, int weigh_last,
                               float scale, float* scratch, long long scratch_size, int* error_word, cudaStream_t stream) {
    if (n_seqs <= 0 || rows <= 0) return 0;
    if (head_dim % 16 || head_dim <= 0 || head_dim > 256 || n_kv <= 0 || n_q % n_kv || (block != 16 && block != 32 && block != 64) ||
        (n_q + 3) / 4 > 65535 || n_kv > 65535 || max_new <= 0 || max_pages <= 0 || n_pages <= 0 || !error_word)
        return SSB_ERR_BAD_SIZE;
    if (weigh_last > 0 && (!weight || !lse)) return SSB_ERR_BAD_SIZE;
    if (dtype != SSB_BF16 && dtype != SSB_F32) return SSB_ERR_BAD_DTYPE;
    IaArgs a{q, out, lse, (const int8_t*)k, (const int8_t*)v, k_scale, v_scale, weight, page_table, cu_new, seq_start, seq_slot,
                   ldq, ldo, rows, n_seqs, n_slots, max_pages, n_pages, n_q, n_kv, head_dim, block == 16 ? 4 : block == 32 ? 5 : 6, window, weigh_last, scale};
    a.most_start = (int)std::min((long long)max_pages * IA_PAGE - 1 + std::max(window, 0), 0x7fffff00LL - rows);
    if (!ir_takes(n_q, n_kv, head_dim)) {
        if (weigh_last > 0 && n_seqs > 65535) return SSB_ERR_BAD_SIZE;
        const dim3 grid(rows, (n_q + 3) / 4), wgrid(std::min((max_pages * IA_PAGE + 3) / 4, 512), n_kv, n_seqs);
        if (dtype == SSB_BF16) {
            int8_attention_plain_kernel<bf16><<<grid, 128, 0, stream>>>(a);
            if (weigh_last > 0) int8_weigh_plain_kernel<bf16><<<wgrid, 128, 0, stream>>>(a);
        } else {
            int8_attention_plain_kernel<float><<<grid, 128, 0, stream>>>(a);
            if (weigh_last > 0) int8_weigh_plain_kernel<float><<<wgrid, 128, 0, stream>>>(a);
        }
        return ssb_launch_status();
    }
    const bool wide = dtype == SSB_F32, prompt = ia_tc_takes(dtype, head_dim, max_new, scale);
    CUtensorMap mk, mv;
    int rc = prompt && weigh_last <= 0 ? 0 : ir_map(&mk, k, (long long)n_pages * n_kv * 64, head_dim);
    if (rc) return rc;
    if (prompt) {
        if (ldq % 8 || ldo % 8 || (((uintptr_t)q | (uintptr_t)out) & 15)) return SSB_ERR_BAD_SIZE;
        if (scratch_size < ia_tc_scratch(n_seqs, rows, max_new, max_pages, n_q, n_kv, head_dim)) return SSB_ERR_BAD_SIZE;
        rc = ia_tc_launch(a, max_new, scratch, error_word, stream);
        if (rc || weigh_last <= 0) return rc;
        return ia_weigh(a, wide, max_new, error_word, mk, stream);
    }
    rc = ir_map(&mv, v, (long long)n_pages * n_kv * 64, head_dim);
    if (rc) return rc;
    if (!scratch) return SSB_ERR_BAD_SIZE;
    const IrPlan p = ir_plan(wide, n_seqs, rows, max_new, max_pages, n_q, n_kv, head_dim, window, weigh_last);
    if (p.blocks < 0) return SSB_ERR_UNSUPPORTED;
    if (scratch_size < ir_scratch(p)) return SSB_ERR_BAD_SIZE;
#define IR_ROWS(H_, N_, W_) rc = ir_rows<H_, N_, W_>(a, p, scratch, error_word, mk, mv, stream)
    IR_EACH(head_dim, p.nt, wide, IR_ROWS);
#undef IR_ROWS
    return rc || weigh_last <= 0 || p.kept ? rc : ia_weigh(a, wide, max_new, error_word, mk, stream);
}

SSB_PACKED(ssb_int8_attention)
