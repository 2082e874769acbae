// Attention of prompts over the 8-bit cache on the fifth-generation tensor cores: bfloat16 rows, head sizes 64 and 128.
//
// A unit of work is two tiles of 128 query rows that share a kv head (two query heads of the group over the same rows, or
// neighbouring row tiles), or one tile where there are fewer units than SMs; a block stays for many units.  Scores S = Q K^T and
// outputs O += P V are tcgen05.mma into tensor memory, 128 keys (two pages) a turn, P from tensor memory, as in the attention over
// bfloat16 pages (prefill_attention_tc.cu).  What is different here:
//
// * Keys and values come as codes.  Four warps fetch a turn's codes into registers one turn ahead, 16 bytes a lane, and write them
//   to shared memory as the operands: keys as bfloat16 beside bfloat16 queries, values as float16 beside float16 probabilities (a
//   code is a whole number up to 127: exact in both), in the 128-byte swizzle that the tensor cores read.  bfloat16: a byte behind
//   0x43 is 128 + its low seven bits, or 128 or 256 by its sign alone, and the code is their difference.  float16: a byte with its
//   sign bit turned behind 0x64 is 1,024 + 128 + the code.
// * Scales stay out of the products.  16 keys have one scale of keys, which multiplies their scores where the softmax scales them
//   anyway, and one of values, whose logarithm goes into the exponent: 2^(s ks + log2 vs - m) is a probability times its value's
//   scale, at no instruction more than the probability alone; a group's sum is divided by vs once before it counts in the
//   denominator.  The maximum m is over s ks + log2 vs, so float16 holds what is summed; the denominator
//   has all keys whose values' scales are within 2^90 of one another.
//
// A row's reference moves only when a maximum is 2^12 above it (float16 holds up to 2^16), and only then is O rescaled; what lies
// 2^-14 below the reference is rounded to 2^-25 of it, and a sum is at least 2^-12 of the largest.  Every mbarrier wait is bounded.
#include "int8_attention.cuh"
#include "packed_f32.cuh"
#include "tc_helpers.cuh"
#include <cuda_fp16.h>
#include <math.h>
#include <algorithm>

typedef __nv_bfloat16 bf16;

constexpr int IT_BM = 128, IT_BN = 128;    // query rows a tile, keys a turn
constexpr int IT_SEQS = 512;               // sequences a launch: their table lies in shared memory
constexpr int IT_SCALES = 4;               // turns whose scales are kept
constexpr float IT_LAZY = 12.f;            // how far, in the log2 domain, a maximum may rise above its row's reference
constexpr float IT_LEAST = 7.888609052210118e-31f;
struct ItTile { int row, head, p0, rows, turns; };
struct ItUnit { int turns, kb_lo, kvh, slot, last, part; ItTile tile[2]; };       // no turns: the block is done; last: the sequence's last key in the table; part: of the keys, or -1: all
__host__ __device__ constexpr int it_threads(int tiles) { return 256 + 128 * tiles; }
constexpr int IT_BARS = 6 + 8 + 6 + IT_SCALES;
__host__ __device__ constexpr size_t it_smem(int tiles, int hd) {
    return (size_t)tiles * IT_BM * hd * 2 + 2 * 2 * IT_BN * hd * 2 + IT_SEQS * (sizeof(IaSeq) + 4) + IT_SCALES * 8 * 16 + 2 * sizeof(ItUnit) +
           IT_BARS * 8 + 32 + 1024;
}
// Registers a thread of the three kinds of warps: 4 that control, 4 that convert, 4 a tile that take the softmax.
__host__ __device__ constexpr int it_blocks(int tiles, int hd) { return tiles == 1 && hd == 64 ? 2 : 1; }       // an SM
constexpr int IT_REGS_CONTROL = 48;
__host__ __device__ constexpr int it_regs_convert(int tiles, int hd) { return it_blocks(tiles, hd) == 2 ? 72 : 96; }
__host__ __device__ constexpr int it_regs_softmax(int tiles, int hd) { return it_blocks(tiles, hd) == 2 ? 120 : tiles == 2 ? 184 : 232; }

// The turns of a unit: items (row tile, head of the group) TILES * level and, with two tiles, the one behind it.  Keys begin at the
// page that the first tile of the pair sees first, for a tile that is alone too: a row's turns, and with them its sums, are the same in
// a unit of either size.  All of it in the ``pages`` of the table, of which a tile has one at least.
template <int TILES> struct ItSpan {
    int kb_lo, most, nb[TILES];          // first page; turns of the longer tile; of each
    __device__ ItSpan(int start, int n_new, int group, int window, int pages, int level) : kb_lo(0), most(0) {
        const int n_items = ((n_new + IT_BM - 1) / IT_BM) * group;
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
            const int item = TILES * level + x, tile = item / group;
            const int p0 = start + tile * IT_BM, rows = item < n_items ? min(IT_BM, n_new - tile * IT_BM) : 0;
            if (x == 0) {
                const int first = start + (item & ~1) / group * IT_BM;
                kb_lo = (window > 0 && first - window + 1 > 0) ? min((first - window + 1) >> 6, pages - 1) : 0;
            }
            nb[x] = rows > 0 ? (min((p0 + rows - 1) >> 6, pages - 1) - kb_lo + 2) >> 1 : 0;
            most = max(most, nb[x]);
        }
    }
};
// Where there are fewer units than SMs a unit's turns are cut into up to ``parts`` runs of ``each`` turns, four at least, that are units
// of their own; int8_join_kernel puts them together.
struct ItCut {
    int parts, each;
    __device__ ItCut(int turns, int most_parts) {
        parts = min(most_parts, max(1, turns / 4));
        each = (turns + parts - 1) / parts;
        parts = (turns + each - 1) / max(1, each);
    }
};

__device__ __forceinline__ void it_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// A from tensor memory (8 columns a step of 16 keys), B's descriptor 128 units (16 rows of 128 bytes) a step: four steps.
__device__ __forceinline__ void it_mma_ts_x4(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b32 a1, a2, a3;\n.reg .b64 b1, b2, b3;\n"
                 "setp.ne.b32 p, %4, 0;\nsetp.eq.b32 q, %5, 0;\n"
                 "add.u32 a1, %1, 8;\nadd.u32 a2, %1, 16;\nadd.u32 a3, %1, 24;\n"
                 "add.u64 b1, %2, 128;\nadd.u64 b2, %2, 256;\nadd.u64 b3, %2, 384;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, {%5, %5, %5, %5}, q;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, {%5, %5, %5, %5}, q;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, {%5, %5, %5, %5}, q;\n}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void it_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void it_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void it_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void it_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void it_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float it_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// MN-major operand (values: [key][dim], dim contiguous) in 64-column boxes 8 KB apart, rows of 128 bytes with the 128-byte swizzle.
__device__ __forceinline__ uint64_t it_desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (512ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// Codes pass through a block once: not by way of its L1, which is what shared memory leaves of it.
__device__ __forceinline__ uint4 it_load_once(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// Two codes of a word as bfloat16 or float16.
__device__ __forceinline__ uint32_t it_bf16(uint32_t w, uint32_t sel) {
    const uint32_t y = __byte_perm(w, 0x43434343u, sel), a = y & 0xff7fff7fu, b = y & 0xff80ff80u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint32_t it_f16(uint32_t turned, uint32_t sel) {
    const uint32_t y = __byte_perm(turned, 0x64646464u, sel), bias = 0x64806480u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&y), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&d);
}
template <bool KEYS> __device__ __forceinline__ uint4 it_operand(uint32_t w0, uint32_t w1) {      // eight codes
    if (KEYS) return make_uint4(it_bf16(w0, 0x4140), it_bf16(w0, 0x4342), it_bf16(w1, 0x4140), it_bf16(w1, 0x4342));
    w0 ^= 0x80808080u;
    w1 ^= 0x80808080u;
    return make_uint4(it_f16(w0, 0x4140), it_f16(w0, 0x4342), it_f16(w1, 0x4140), it_f16(w1, 0x4342));
}

// 4 x 2,048 tokens, 32 heads over 8: of 128 207 us, 664 TFLOP/s, of 64 184 us; 500 behind 16,001, of 128 197 us, 676 TFLOP/s, of 64 181.
// No unit is busy for more than 40 % of the time: a tile's scores, softmax and outputs wait for one another.
template <int HD, int TILES>
__global__ void __launch_bounds__(it_threads(TILES), it_blocks(TILES, HD))
int8_attention_tc_kernel(const IaArgs a, const __grid_constant__ CUtensorMap map_q, int s0, int n_seqs, int levels, int parts,
                         float* __restrict__ part_o, float2* __restrict__ part_ml, int* __restrict__ error_word) {
    constexpr uint32_t TMEM_COLS = 256 * TILES, S0 = 0, O0 = IT_BN * TILES;       // scores, later probabilities; outputs behind them
    constexpr int HALVES = HD / 64;
    constexpr uint32_t Q_BYTES = IT_BM * HD * 2, PAGE_BYTES = 64 * HD * 2, KV_BYTES = 2 * PAGE_BYTES;
    constexpr int PIECES = IT_BN * HD / 16 / 128;                 // 16-byte pieces of a turn's keys (or values) a converting lane has
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    unsigned char* q_s = smem;
    unsigned char* kv_s = smem + TILES * Q_BYTES;                 // two stages of [keys of two pages | values of two pages]
    float4* scales = (float4*)(kv_s + 4 * KV_BYTES);              // [turn & 3][group of 16 keys]: ks scale log2 e, log2 vs, 1 / vs
    IaSeq* seqs = (IaSeq*)(scales + IT_SCALES * 8);
    int* units_of = (int*)(seqs + IT_SEQS);                       // units of a sequence for one kv head
    ItUnit* units = (ItUnit*)(units_of + IT_SEQS);                // the one that is computed and the next
    uint64_t* bars = (uint64_t*)(units + 2);
    const uint32_t q_full = smem_u32(bars), q_empty = q_full + 8, u_full0 = q_full + 16, u_empty0 = q_full + 32, k_full0 = q_full + 48,
                   v_full0 = k_full0 + 16, k_empty0 = v_full0 + 16, v_empty0 = k_empty0 + 16, s_full0 = v_empty0 + 16, p_full0 = s_full0 + 16,
                   o_full0 = p_full0 + 16, c_full0 = o_full0 + 16;
    uint32_t* tmem_slot = (uint32_t*)(bars + IT_BARS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);   // [0]: a role gave up; [1]: stays zero
    const int group = a.n_q / a.n_kv, window = a.window;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    ssb_pdl_wait();
    ssb_pdl_launch_dependents();                                 // dependents read the batch and the pages ahead of their own wait
    for (int b = threadIdx.x; b < n_seqs; b += it_threads(TILES)) {
        const IaSeq q = ia_sequence(a, s0 + b);
        seqs[b] = q;
        // (row tile, head of the group) items, heads fastest, TILES a unit
        units_of[b] = q.slot < 0 || q.n_new <= 0 ? 0 : min(levels, (((q.n_new + IT_BM - 1) / IT_BM) * group + TILES - 1) / TILES);
    }
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(u_full0 + 8 * i, 1); mbar_init(u_empty0 + 8 * i, 1 + 4 + 4 * TILES);
            mbar_init(k_full0 + 8 * i, 4); mbar_init(v_full0 + 8 * i, 4);
            mbar_init(k_empty0 + 8 * i, 1); mbar_init(v_empty0 + 8 * i, 1);
            mbar_init(s_full0 + 8 * i, 1); mbar_init(p_full0 + 8 * i, 4); mbar_init(o_full0 + 8 * i, 1);
        }
        for (int i = 0; i < IT_SCALES; ++i) mbar_init(c_full0 + 8 * i, 1);
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // sequences without a slot: zeros
    for (int b = blockIdx.x; b < n_seqs; b += gridDim.x)
        if (seqs[b].slot < 0)
            for (int e = threadIdx.x; e < seqs[b].n_new * a.n_q * (HD / 8); e += it_threads(TILES)) {
                const int piece = e % (HD / 8), head = e / (HD / 8) % a.n_q;
                const size_t row = (size_t)(seqs[b].row0 + e / (HD / 8) / a.n_q);
                *reinterpret_cast<uint4*>((bf16*)a.out + row * a.ldo + (size_t)head * HD + 8 * piece) = make_uint4(0, 0, 0, 0);
                if (piece == 0 && a.lse) a.lse[row * a.n_q + head] = -INFINITY;
            }

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(IT_REGS_CONTROL));
        if (warp == 0) {
            // The units of the launch go from the latest position to the first, over sequences and kv heads; a block takes every
            // gridDim.x-th of them, forwards and backwards in turn.
            int base = 0, level = levels - 1;                    // units before this level's
            int n_units = 0, taken = 0;                          // units published, and looked at (some have no turn)
            bool ok = true;
            while (ok) {
                const int all = taken * (int)gridDim.x + ((taken & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
                const int u = all / parts, part = all - u * parts;
                ++taken;
                while (level >= 0) {
                    int here = 0, next = 0;                      // levels next..level are reached by the same sequences
                    for (int c = 0; c < n_seqs; c += 32) {
                        const int v = c + lane < n_seqs ? units_of[c + lane] : 0;
                        here += __popc(__ballot_sync(0xffffffffu, v > level));
                        next = max(next, __reduce_max_sync(0xffffffffu, v > level ? 0 : v));
                    }
                    const int run = level - next + 1, span = here * a.n_kv;
                    const int skip = span ? min((u - base) / span, run) : run;
                    base += skip * span;
                    level -= skip;
                    if (skip < run) break;
                }
                const int slot = n_units & 1;
                ItUnit& unit = units[slot];
                int nb_max = 0, kb_lo = 0, kvh = 0, q_tiles = 0;
                int t_head[TILES], t_row[TILES], nb[TILES];
                ok = __all_sync(0xffffffffu, mbar_wait(u_empty0 + 8 * slot, ((n_units >> 1) & 1) ^ 1, abort_flag));
                if (!ok) break;
                if (level >= 0) {
                    int member = (u - base) / a.n_kv, b = 0;
                    kvh = (u - base) - member * a.n_kv;
                    for (int c = 0; c < n_seqs; c += 32) {
                        unsigned has = __ballot_sync(0xffffffffu, c + lane < n_seqs && units_of[c + lane] > level);
                        const int n = __popc(has);
                        if (member < n) {
                            for (; member > 0; --member) has &= has - 1;
                            b = c + __ffs(has) - 1;
                            break;
                        }
                        member -= n;
                    }
                    const IaSeq q = seqs[b];
                    const ItSpan<TILES> span(q.start, q.n_new, group, window, a.max_pages, level);
                    const ItCut cut(span.most, parts);
                    const int skip = part * cut.each;
                    if (skip >= span.most) continue;             // fewer parts than others have
                    kb_lo = span.kb_lo + 2 * skip;
#pragma unroll
                    for (int x = 0; x < TILES; ++x) {
                        const int item = TILES * level + x, tile = item / group;
                        t_head[x] = kvh * group + item % group;
                        t_row[x] = q.row0 + tile * IT_BM;
                        nb[x] = min(max(span.nb[x] - skip, 0), cut.each);
                        nb_max = max(nb_max, nb[x]);
                        q_tiles += nb[x] > 0;
                        if (lane == 0) unit.tile[x] = ItTile{t_row[x], t_head[x], q.start + tile * IT_BM, min(IT_BM, q.n_new - tile * IT_BM), nb[x]};
                    }
                    if (lane == 0) unit.part = cut.parts > 1 ? part : -1;
                    if (lane == 0) { unit.slot = q.slot; unit.last = (int)min((long long)q.start + q.n_new, (long long)a.max_pages * IA_PAGE) - 1; }
                }
                if (lane == 0) {
                    unit.turns = nb_max;
                    unit.kb_lo = kb_lo;
                    unit.kvh = kvh;
                    it_arrive(u_full0 + 8 * slot);               // release: the unit is read behind a wait for it
                }
                if (nb_max == 0) break;
                if (lane == 0) {
                    ok = mbar_wait(q_empty, (n_units & 1) ^ 1, abort_flag);
                    if (ok) {
                        mbar_expect_tx(q_full, q_tiles * Q_BYTES);
#pragma unroll
                        for (int x = 0; x < TILES; ++x)
                            if (nb[x] > 0) {
#pragma unroll
                                for (int h = 0; h < HALVES; ++h)
                                    tma_load_2d(smem_u32(q_s) + x * Q_BYTES + h * (Q_BYTES / HALVES), &map_q, q_full, t_head[x] * HD + 64 * h, t_row[x]);
                            }
                        ++n_units;
                    }
                }
                n_units = __shfl_sync(0xffffffffu, n_units, 0);
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if (lane == 0) {
                if (!ok) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); }
                if (*abort_flag && n_units > 0) mbar_wait(q_full, (n_units - 1) & 1, abort_flag + 1);      // let issued copies land
            }
        } else if (warp == 1 && lane == 0) {
            // S: D float32, A and B bfloat16 K-major, M 128, N 128.  PV: A and B float16, B MN-major (bit 16), N head size.
            const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(IT_BN >> 3) << 17) | ((uint32_t)(IT_BM >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(IT_BM >> 4) << 24);
            const uint64_t q_desc = smem_desc(smem_u32(q_s)), k_desc = smem_desc(smem_u32(kv_s)), v_desc = it_desc_mn(smem_u32(kv_s) + KV_BYTES);
            int turns = 0, mine[TILES] = {};                     // turns of the units before, and of their tiles
            bool ok = true;
            auto issue_s = [&](int x, int turn) {                // scores of a turn of tile x
                const int s = turn & 1;
                if (!mbar_wait(k_full0 + 8 * s, (turn >> 1) & 1, abort_flag)) { ok = false; return; }
                tc_fence_after();
                const uint64_t da = q_desc + (uint64_t)(x * (Q_BYTES >> 4)), db = k_desc + (uint64_t)(s * (2 * KV_BYTES >> 4));
#pragma unroll
                for (int h = 0; h < HALVES; ++h)                 // 64 dims a box, four steps of 16; descriptors count in units of 16 bytes
                    tc_mma_x4(tmem + S0 + x * IT_BN, da + h * (Q_BYTES / HALVES >> 4), db + h * (KV_BYTES / HALVES >> 4), idesc_s, h ? 1u : 0u);
                tc_commit(s_full0 + 8 * x);
            };
            for (int n = 0; ok; ++n) {
                if (!mbar_wait(u_full0 + 8 * (n & 1), (n >> 1) & 1, abort_flag)) { ok = false; break; }
                const ItUnit& unit = units[n & 1];
                const int nb_max = unit.turns;
                if (nb_max == 0) break;
                int nb[TILES];
#pragma unroll
                for (int x = 0; x < TILES; ++x) nb[x] = unit.tile[x].turns;
                it_arrive(u_empty0 + 8 * (n & 1));
                ok = mbar_wait(q_full, n & 1, abort_flag);
                // A turn's scores go where the probabilities of the turn (or the unit) before lay: the tensor cores take their
                // work in the order of issue.
                for (int j = -1; j < nb_max && ok; ++j) {
                    const int s = (turns + j) & 1;
#pragma unroll
                    for (int x = 0; x < TILES; ++x) {
                        if (ok && j >= 0 && j < nb[x]) {
                            ok = mbar_wait(p_full0 + 8 * x, (mine[x] + j) & 1, abort_flag) &&
                                 mbar_wait(v_full0 + 8 * s, ((turns + j) >> 1) & 1, abort_flag);
                            if (ok) {
                                tc_fence_after();
#pragma unroll
                                for (int pg = 0; pg < 2; ++pg)   // a page: four steps of 16 keys
                                    it_mma_ts_x4(tmem + O0 + x * HD, tmem + S0 + x * IT_BN + pg * 32,
                                                 v_desc + (uint64_t)(s * (2 * KV_BYTES >> 4) + pg * (PAGE_BYTES >> 4)), idesc_o, (j > 0 || pg > 0) ? 1u : 0u);
                                tc_commit(o_full0 + 8 * x);
                            }
                        }
                        if (ok && j + 1 < nb[x]) issue_s(x, turns + j + 1);
                    }
                    if (!ok) break;
                    if (j >= 0) tc_commit(v_empty0 + 8 * s);
                    if (j + 1 < nb_max) tc_commit(k_empty0 + 8 * ((turns + j + 1) & 1));    // keys are free when their scores are made
                    if (j + 2 == nb_max) tc_commit(q_empty);
                }
                turns += nb_max;
#pragma unroll
                for (int x = 0; x < TILES; ++x) mine[x] += nb[x];
            }
            if (!ok) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); }
        }
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(it_regs_convert(TILES, HD)));
        const int id = threadIdx.x - 128;
        const int per = 64 >> a.shift;
        const int row_of = id / (HD / 16), c = id % (HD / 16);    // of the pieces id, id + 128, ...: rows 128 / (HD / 16) apart
        constexpr int ROWS = 128 / (HD / 16);
        int turn = 0;                                            // counted on over the units
        bool ok = true;
        for (int n = 0; ok; ++n) {
            ok = __all_sync(0xffffffffu, mbar_wait(u_full0 + 8 * (n & 1), (n >> 1) & 1, abort_flag));
            if (!ok) break;
            const ItUnit& unit = units[n & 1];
            const int nb = unit.turns, kb_lo = unit.kb_lo, kvh = unit.kvh, last = unit.last;
            const int* pt = a.page_table + (size_t)max(unit.slot, 0) * a.max_pages;
            __syncwarp();
            if (nb == 0) break;
            if (lane == 0) it_arrive(u_empty0 + 8 * (n & 1));
            // a page past the sequence's last one (odd page counts) is the last one again: its groups have no scale
            auto page_at = [&](int j, int pg) { return pt[min(kb_lo + 2 * j + pg, last >> 6)]; };
            uint4 kr[PIECES], vr[PIECES];
            float ks = 0.f, vs = 0.f;
            bool there = false;
            int ids[2] = {page_at(0, 0), page_at(0, 1)}, ahead[2];
            auto fetch = [&](uint4 (&r)[PIECES], const int8_t* codes, const int (&p)[2]) {
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {               // the first half of the pieces is the first page's
                    const int pg = i / (PIECES / 2), row = (i % (PIECES / 2)) * ROWS + row_of;
                    r[i] = it_load_once(codes + (((size_t)(ia_in_pool(a, p[pg]) ? p[pg] : 0) * a.n_kv + kvh) * 64 + row) * HD + 16 * c);
                }
            };
            auto fetch_scales = [&](const int (&p)[2]) {
                if (id < 8) {
                    const int page = p[id >> 2];
                    const size_t at = ((size_t)page * a.n_kv + kvh) * per + (((id & 3) * 16) >> a.shift);
                    there = ia_in_pool(a, page);
                    ks = there ? a.k_scale[at] : 0.f;
                    vs = there ? a.v_scale[at] : 0.f;
                }
            };
            fetch(kr, a.k, ids);
            fetch_scales(ids);
            fetch(vr, a.v, ids);
            for (int j = 0; j < nb; ++j, ++turn) {
                const int s = turn & 1;
                const uint32_t free = ((turn >> 1) & 1) ^ 1;
                const bool more = j + 1 < nb;
                if (more) { ahead[0] = page_at(j + 1, 0); ahead[1] = page_at(j + 1, 1); }
                unsigned char* k_dst = kv_s + s * 2 * KV_BYTES;
                unsigned char* v_dst = k_dst + KV_BYTES;
                auto put = [&](unsigned char* dst, const uint4& w, int row_bytes_at, int row, auto keys) {
                    // 16 codes: two of the eight 16-byte pieces of a row of 64; the second box's lanes write theirs the other way round
                    constexpr bool KEYS = decltype(keys)::value;
                    const uint4 x = it_operand<KEYS>(w.x, w.y), y = it_operand<KEYS>(w.z, w.w);
                    const int f = 2 * (c & 3), flip = (c >> 2) & 1;
                    unsigned char* at = dst + row_bytes_at;
                    *reinterpret_cast<uint4*>(at + (((f + flip) ^ (row & 7)) << 4)) = flip ? y : x;
                    *reinterpret_cast<uint4*>(at + (((f + 1 - flip) ^ (row & 7)) << 4)) = flip ? x : y;
                };
                ok = __all_sync(0xffffffffu, mbar_wait(k_empty0 + 8 * s, free, abort_flag));
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {               // keys: [box][key], a K-major tile of 128 rows a box
                    const int row = (i / (PIECES / 2)) * 64 + (i % (PIECES / 2)) * ROWS + row_of;
                    put(k_dst, kr[i], (c >> 2) * (KV_BYTES / HALVES) + row * 128, row, std::true_type{});
                }
                if (id < 8) {
                    // groups that begin behind the sequence's last key, or whose page is none, have no scale: what is added to their
                    // scores leaves nothing of them
                    const bool has = there && (kb_lo + 2 * j) * 64 + 16 * id <= last;
                    const float v1 = has ? fmaxf(vs, IT_LEAST) : 1.f, k1 = has ? fmaxf(ks * (a.scale * 1.4426950408889634f), 1e-37f) : 1.f;
                    scales[(turn & (IT_SCALES - 1)) * 8 + id] = make_float4(k1, has ? log2f(v1) : -INFINITY, 1.f / v1, 0.f);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if (warp == 4) it_arrive(c_full0 + 8 * (turn & (IT_SCALES - 1)));
                    it_arrive(k_full0 + 8 * s);
                }
                if (more) { fetch(kr, a.k, ahead); fetch_scales(ahead); }
                ok = __all_sync(0xffffffffu, mbar_wait(v_empty0 + 8 * s, free, abort_flag));
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {               // values: [page][box][key]
                    const int row = (i % (PIECES / 2)) * ROWS + row_of;
                    put(v_dst, vr[i], (i / (PIECES / 2)) * PAGE_BYTES + (c >> 2) * 8192 + row * 128, row, std::false_type{});
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) it_arrive(v_full0 + 8 * s);
                if (more) fetch(vr, a.v, ahead);
            }
        }
        if (!ok && lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(it_regs_softmax(TILES, HD)));
        // softmax and output: one query row per thread; warps 8-11 tile 0, warps 12-15 tile 1
        const int x = TILES == 1 ? 0 : (warp - 8) >> 2;
        const int quarter = warp & 3;                            // the lanes of tensor memory this warp may touch
        const int r = quarter * 32 + lane;
        const uint32_t t_s = tmem + ((uint32_t)(quarter * 32) << 16) + S0 + x * IT_BN;
        const uint32_t t_o = tmem + ((uint32_t)(quarter * 32) << 16) + O0 + x * HD;
        const uint32_t s_full = s_full0 + 8 * x, p_full = p_full0 + 8 * x, o_full = o_full0 + 8 * x;
        int turn = 0, turns = 0;                                 // of the tile, and of the units, counted on
        bool ok = true;
        for (int n = 0; ok; ++n) {
            ok = __all_sync(0xffffffffu, mbar_wait(u_full0 + 8 * (n & 1), (n >> 1) & 1, abort_flag));
            if (!ok) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                break;
            }
            const int nb_max = units[n & 1].turns;
            if (nb_max == 0) break;
            const int kb_lo = units[n & 1].kb_lo;
            const ItTile tile = units[n & 1].tile[x];
            const int part = units[n & 1].part;
            __syncwarp();
            if (lane == 0) it_arrive(u_empty0 + 8 * (n & 1));
            const int n_mine = tile.turns, p0 = tile.p0, pos = p0 + r;
            const int before = turns;
            turns += nb_max;
            if (n_mine <= 0) continue;
            float m_ref = -INFINITY, l_run = 0.f;
            for (int j = 0; j < n_mine; ++j, ++turn) {
                const int ring = (before + j) & (IT_SCALES - 1);
                bool w = mbar_wait(s_full, turn & 1, abort_flag) && mbar_wait(c_full0 + 8 * ring, ((before + j) / IT_SCALES) & 1, abort_flag);
                w = __all_sync(0xffffffffu, w);
                if (!w) { ok = false; break; }
                tc_fence_after();
                const float4* sc = scales + ring * 8;
                const int key0 = (kb_lo + 2 * j) * 64;
                const bool edge = key0 + IT_BN - 1 > p0 || window > 0;   // on the diagonal or at a window's edge
                const int hi = pos - key0;                       // keys 0..hi of the turn are seen
                const int lo = window > 0 ? hi - window + 1 : 0;
                // Two rounds over the scores, 32 at a time from tensor memory: their maximum, then their probabilities, written over
                // scores that both rounds are done with.  Both are loops: unrolled, the warps' roles together outgrew the
                // instruction cache, and times moved by a quarter with any change to the code.
                auto scores = [&](int q, uint32_t (&v)[32]) {
                    it_ld32(t_s + q * 32, v);
                    it_ld_wait();
                    if (edge) {
                        const int top = hi - q * 32, bottom = lo - q * 32;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i > top || i < bottom) v[i] = 0xff800000u;
                    }
                };
                float m_new = m_ref;
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    uint32_t v[32];
                    scores(q, v);
#pragma unroll
                    for (int gr = 0; gr < 2; ++gr) {
                        const float4 f = sc[q * 2 + gr];
                        float mx = __uint_as_float(v[gr * 16]);
#pragma unroll
                        for (int i = 1; i < 15; i += 2) mx = fmaxf(fmaxf(mx, __uint_as_float(v[gr * 16 + i])), __uint_as_float(v[gr * 16 + i + 1]));
                        mx = fmaxf(mx, __uint_as_float(v[gr * 16 + 15]));
                        m_new = fmaxf(m_new, fmaf(mx, f.x, f.y));
                    }
                }
                // The reference moves when a maximum is 2^12 above it, in the warp's 32 rows together; what was summed follows
                if (__any_sync(0xffffffffu, m_new > m_ref + IT_LAZY)) {
                    if (j > 0) {
                        ok = __all_sync(0xffffffffu, mbar_wait(o_full, (turn - 1) & 1, abort_flag));
                        if (!ok) break;
                        tc_fence_after();
                        const float alpha = m_new == -INFINITY ? 1.f : it_ex2(m_ref - m_new);
#pragma unroll 1
                        for (int i = 0; i < HD / 32; ++i) {
                            uint32_t o[32];
                            it_ld32(t_o + i * 32, o);
                            it_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                            it_st32(t_o + i * 32, o);
                        }
                        l_run *= alpha;
                    }
                    m_ref = m_new;
                }
                const float ref = m_ref == -INFINITY ? 0.f : m_ref;
#pragma unroll 1
                for (int q = 0; q < 4; ++q) {
                    uint32_t v[32], packed[16];
                    scores(q, v);
#pragma unroll
                    for (int gr = 0; gr < 2; ++gr) {
                        const float4 f = sc[q * 2 + gr];
                        const unsigned long long by = f2_twice(f.x), at = f2_twice(f.y - ref);
                        unsigned long long sum = 0;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const unsigned long long e = f2_fma(f2_pair(__uint_as_float(v[gr * 16 + i]), __uint_as_float(v[gr * 16 + i + 1])), by, at);
                            const float pa = it_ex2(f2_lo(e)), pb = it_ex2(f2_hi(e));
                            sum = f2_add(sum, f2_pair(pa, pb));
                            const __half2 p = __floats2half2_rn(pa, pb);
                            packed[gr * 8 + i / 2] = *reinterpret_cast<const uint32_t*>(&p);
                        }
                        l_run = fmaf(f2_lo(sum) + f2_hi(sum), f.z, l_run);
                    }
                    it_st16(t_s + q * 16, packed);
                }
                it_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) it_arrive(p_full);
            }
            if (ok) {
                bool w = mbar_wait(o_full, (turn - 1) & 1, abort_flag);
                ok = __all_sync(0xffffffffu, w);
            }
            if (!ok) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
            } else {
                tc_fence_after();
                const size_t row = (size_t)(tile.row + r);
                if (part >= 0) {                                 // a part: sums as they are, the reference and the sum of weights
                    const size_t at = ((size_t)part * a.rows + row) * a.n_q + tile.head;
#pragma unroll 1
                    for (int i = 0; i < HD / 32; ++i) {
                        uint32_t o[32];
                        it_ld32(t_o + i * 32, o);
                        it_ld_wait();
                        if (r < tile.rows) {
#pragma unroll
                            for (int q = 0; q < 8; ++q)
                                *reinterpret_cast<uint4*>(part_o + at * HD + i * 32 + 4 * q) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
                        }
                    }
                    if (r < tile.rows) part_ml[at] = make_float2(m_ref, l_run);
                    continue;
                }
                const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
                uint4* dst = reinterpret_cast<uint4*>((bf16*)a.out + row * a.ldo + (size_t)tile.head * HD);
#pragma unroll
                for (int i = 0; i < HD / 32; ++i) {
                    uint32_t o[32];
                    it_ld32(t_o + i * 32, o);
                    it_ld_wait();
                    if (r < tile.rows) {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t v[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(o[8 * q + 2 * e]) * inv, __uint_as_float(o[8 * q + 2 * e + 1]) * inv);
                                v[e] = *reinterpret_cast<const uint32_t*>(&y);
                            }
                            dst[i * 4 + q] = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    }
                }
                if (a.lse && r < tile.rows)
                    a.lse[row * a.n_q + tile.head] = l_run == 0.f ? -INFINITY : (m_ref + log2f(l_run)) * 0.6931471805599453f;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Rows whose keys were cut into parts: a thread four dims of a row's head.  500 rows of 32 heads of 64: 10 us, by the parts' fetches.
template <int HD, int TILES>
__global__ void __launch_bounds__(256)
int8_join_kernel(const IaArgs a, int s0, int n_seqs, int parts, const float* __restrict__ part_o, const float2* __restrict__ part_ml) {
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    const int d = (int)(e % (HD / 4)) * 4, head = (int)(e / (HD / 4) % a.n_q);
    const long long row_of = e / (HD / 4) / a.n_q;
    if (row_of >= a.rows) return;
    const int row = (int)row_of, group = a.n_q / a.n_kv;
    int lo = s0, hi = s0 + n_seqs - 1;                           // the last sequence that begins at or before the row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.cu_new[mid] <= row) lo = mid; else hi = mid - 1;
    }
    const auto [row0, n_new, start, slot] = ia_sequence(a, lo);
    if (slot < 0 || row < row0 || row >= row0 + n_new) return;
    const int item = (row - row0) / IT_BM * group + head % group;
    const ItSpan<TILES> span(start, n_new, group, a.window, a.max_pages, item / TILES);
    const ItCut cut(span.most, parts);
    if (cut.parts <= 1) return;
    const int turns = TILES == 2 && (item & 1) ? span.nb[TILES - 1] : span.nb[0];
    const int mine = (turns + cut.each - 1) / cut.each;          // parts that reach the row's tile
    float m = -INFINITY, l = 0.f;
    for (int p = 0; p < mine; ++p) m = fmaxf(m, __ldcg(part_ml + ((size_t)p * a.rows + row) * a.n_q + head).x);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < mine; ++p) {
        const size_t at = ((size_t)p * a.rows + row) * a.n_q + head;
        const float2 ml = __ldcg(part_ml + at);
        const float4 v = __ldcg(reinterpret_cast<const float4*>(part_o + at * HD + d));
        const float by = ml.x == -INFINITY ? ml.y : it_ex2(ml.x - m);       // a part that saw nothing has a sum of 0, one of no numbers none
        o.x = fmaf(v.x, by, o.x); o.y = fmaf(v.y, by, o.y); o.z = fmaf(v.z, by, o.z); o.w = fmaf(v.w, by, o.w);
        l = fmaf(ml.y, by, l);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * inv, o.y * inv), y = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>((bf16*)a.out + (size_t)row * a.ldo + (size_t)head * HD + d) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    if (d == 0 && a.lse) a.lse[(size_t)row * a.n_q + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// From 17 or 33 new tokens of a sequence on, by the head size.  us with the kernel of rows and with this one, 32 heads over 8: of 128,
// 16 x 2,000 tokens and 12 new 91 and 99, 16 new 92 and 99, 24 new 126 and 99; 4,000 tokens and 16 new 27 and 30, 24 new 33 and 31; of 64,
// 16 x 8,000 and 16 new 170 and 330, 32 new 317 and 330; 16,000 and 24 new 46 and 50, 32 new 54 and 50.  (What one sequence holds is not
// known here: with few keys, 64 x 300 tokens, this one is ahead from 12 new on.)
bool ia_tc_takes(int dtype, int head_dim, int max_new, float scale) {
    return dtype == SSB_BF16 && (head_dim == 64 || head_dim == 128) && max_new > (head_dim == 128 ? 16 : 32) && scale > 0.f;
}

// Tiles a unit, and parts that a unit's keys are cut into at most.
struct ItPlan { int tiles, levels, parts; };
static ItPlan it_plan(int n_seqs, int rows, int max_new, int max_pages, int n_q, int n_kv, int head_dim) {
    const int group = n_q / n_kv, sms = ssb_sm_count(), items = ((max_new + IT_BM - 1) / IT_BM) * group;
    const long long turns = (max_pages + 1) / 2;                 // of the longest sequence there can be
    // parts of four turns at least, in a scratch of up to 256 MB
    const long long most = std::min({turns / 4, 16LL, (1LL << 26) / ((long long)rows * n_q * (head_dim + 2))});
    // Of one or two tiles a unit and the numbers of parts, what is done first: rounds of the SMs times the turns of a part, and three
    // more for its beginning and end.  A turn of two tiles is 1.65 of one's at head size 128; at 64, where single tiles run two blocks
    // an SM, the same, and one that has its SM to itself 0.78.  us with one tile and with two, heads x size: 500 tokens behind 16,001,
    // 32 x 64 184 and 181, 32 x 128 314 and 196; 300 behind 3,000, 8 x 64 23.3 and 28.2, 8 x 128 27.8 and 33.8; two of 600 behind
    // 1,000, 32 x 128 90 and 98, 32 x 64 67 and 73; four of 2,048, 32 x 128 323 and 206, 32 x 64 192 and 184.
    ItPlan p{};
    double best = 0;
    for (int tiles = 2; tiles >= 1; --tiles) {
        const int levels = (items + tiles - 1) / tiles;
        // units there can be: every sequence may end in a tile and a unit that is not full
        const long long units = std::min((long long)n_kv * n_seqs * levels, n_kv * (((long long)rows / IT_BM + n_seqs) * group / tiles + n_seqs));
        const long long slots = (long long)sms * it_blocks(tiles, head_dim);
        for (long long n = 1; n <= std::max(1LL, most); ++n) {
            const double turn = tiles == 2 ? (head_dim == 128 ? 1.65 : 1.0) : head_dim == 64 && units * n <= sms ? 0.78 : 1.0;
            const double cost = (double)((units * n + slots - 1) / slots) * (double)((turns + n - 1) / n + 3) * turn;
            if (p.parts == 0 || cost < best) { best = cost; p = ItPlan{tiles, levels, (int)n}; }
        }
    }
    return p;
}
// float32 elements that parts are kept in.
long long ia_tc_scratch(int n_seqs, int rows, int max_new, int max_pages, int n_q, int n_kv, int head_dim) {
    const ItPlan p = it_plan(n_seqs, rows, max_new, max_pages, n_q, n_kv, head_dim);
    return p.parts > 1 ? (long long)p.parts * rows * n_q * (head_dim + 2) : 0;
}

template <int HD, int TILES>
static int it_launch(const IaArgs& a, const CUtensorMap& mq, int s0, int n, const ItPlan& p, long long grid, float* scratch, int* error_word,
                     cudaStream_t stream) {
    constexpr size_t smem = it_smem(TILES, HD);
    static bool configured = false;
    if (!configured) {
        cudaFuncAttributes attr;
        cudaError_t e = cudaFuncGetAttributes(&attr, int8_attention_tc_kernel<HD, TILES>);
        // what the softmax warps take must be what the others give: a kernel built with fewer registers a thread would wait for good
        if (e == cudaSuccess && attr.numRegs * it_threads(TILES) < 128 * (IT_REGS_CONTROL + it_regs_convert(TILES, HD) + TILES * it_regs_softmax(TILES, HD)))
            return SSB_ERR_UNSUPPORTED;
        if (e == cudaSuccess) e = cudaFuncSetAttribute(int8_attention_tc_kernel<HD, TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    float* part_o = scratch;
    float2* part_ml = p.parts > 1 ? reinterpret_cast<float2*>(scratch + (size_t)p.parts * a.rows * a.n_q * HD) : nullptr;
    const int rc = ssb_launch(int8_attention_tc_kernel<HD, TILES>, dim3((unsigned)grid), dim3(it_threads(TILES)), smem, stream, true, a, mq, s0, n,
                              p.levels, p.parts, part_o, part_ml, error_word);
    if (rc || p.parts == 1) return rc;
    return ssb_launch(int8_join_kernel<HD, TILES>, dim3((unsigned)(((long long)a.rows * a.n_q * (HD / 4) + 255) / 256)), dim3(256), 0, stream, true,
                      a, s0, n, p.parts, (const float*)part_o, (const float2*)part_ml);
}

int ia_tc_launch(const IaArgs& a, int max_new, float* scratch, int* error_word, cudaStream_t stream) {
    CUtensorMap mq;
    int rc = make_map(&mq, a.q, a.rows, a.n_q * a.head_dim, a.ldq, IT_BM);
    if (rc) return rc;
    const ItPlan p = it_plan(a.n_seqs, a.rows, max_new, a.max_pages, a.n_q, a.n_kv, a.head_dim);
    if (p.parts > 1 && !scratch) return SSB_ERR_BAD_SIZE;
    const int group = a.n_q / a.n_kv, sms = ssb_sm_count(), tiles = p.tiles;
    for (int s0 = 0; s0 < a.n_seqs; s0 += IT_SEQS) {
        const int n = std::min(IT_SEQS, a.n_seqs - s0);
        // a block for every SM, and no more than there can be units
        const long long units = std::min((long long)a.n_kv * n * p.levels, a.n_kv * (((long long)a.rows / IT_BM + n) * group / tiles + n)) * p.parts;
        const long long grid = std::min((long long)sms * it_blocks(tiles, a.head_dim), units);
        if (a.head_dim == 64) rc = tiles == 1 ? it_launch<64, 1>(a, mq, s0, n, p, grid, scratch, error_word, stream) : it_launch<64, 2>(a, mq, s0, n, p, grid, scratch, error_word, stream);
        else rc = tiles == 1 ? it_launch<128, 1>(a, mq, s0, n, p, grid, scratch, error_word, stream) : it_launch<128, 2>(a, mq, s0, n, p, grid, scratch, error_word, stream);
        if (rc) return rc;
    }
    return 0;
}
