// Products of matrices in microscaled 4-bit floats (the format: fp4_codes.cuh): out[m, n] (+)= sum_k x[m, k] w[n, k], on the
// fifth-generation tensor cores (tcgen05 kind::mxf4 with a scale for every 32 numbers).  Codes and scales arrive by TMA, codes with the
// 128-byte swizzle (a k-block of 256 numbers is one swizzle row), scales as they lie; scales go on to tensor memory (tcgen05.cp, each
// 128 rows x 4 blocks to four columns, in all four lane quarters), where the instructions read them.  Products of codes and their scales
// are exact; sums are float32 in tensor memory.
//
// Two kernels here (and one for up to 16 rows in fp4_few.cu, one for up to 32 in fp4_step.cu):
//  * where the weights' bytes or the number of tiles is what bounds it: weights on the M side (128 of them a tile), rows of x on the
//    N side, and the k-blocks of all tiles dealt out over the SMs, in equal parts of tiles or wherever a tile ends; the same for experts,
//    whose tiles of rows a list in memory names;
//  * many rows: tiles of 256 x 256 on pairs of SMs (cta_group::2).
//
// What becomes of the sums: stored, added in float32, or (an inner row of a feed-forward) through an activation or a gated unit's inner
// step and into 4 bits at once, from the float32 sums.
#include "fp4_codes.cuh"
#include "fp4_few.cuh"
#include "fp4_step.cuh"
#include "packed_call.cuh"
#include "per_device.h"
#include "fp4_tc.cuh"
#include <algorithm>

typedef __nv_bfloat16 bf16;

struct FlOut {
    void* out;                     // FL_STORE: rows of ldo elements; else codes, rows of ldo bytes
    uint8_t* scales;               // FL_GATED, FL_ACT: of the codes
    const int* index;              // where a row goes (experts: the pair of a sorted row), or null
    const float* row_scale;        // FL_GATED: a factor for each row's results, or null
    int ldo, is_f32, add, M, N;    // rows of x, rows of a weight matrix
    int kind;                      // FL_GATED: ssb_gate's kind; FL_ACT: ssb_activate's
    float limit;                   // of ssb_gate, or the factor behind ssb_activate
    int inner_blocks;              // FL_GATED, FL_ACT: k-blocks of the codes that are written
};
// The experts' tiles of rows: tile t holds up to BN rows of expert tile_expert[t], sorted rows tile_row0[t] onwards, which lie at rows
// t * BN onwards of x (and of codes that are written); meta[0] tiles.  Null: rows as they are.
struct FlTiles {
    const int* offsets; const int* tile_expert; const int* tile_row0; const int* meta;
    // it was there before the launch in front of this one let others begin, so weights come beside that one (16 tokens of 64 experts 51.8 us;
    // behind it 52.4)
    int ready;
};

// The launch's work is tiles x k-blocks, dealt out evenly: block c takes units U c / G .. U (c + 1) / G - 1, tiles in order, a tile's
// k-blocks in order, so that every SM streams the same bytes whatever the sizes.  A tile that lies in one block's range is finished
// there; of any other the blocks write their sums to memory (at most two such pieces a block) and the one whose piece arrives last adds
// them up, in the order of k.
struct FlRange {
    long long units, begin, end;
    int k_blocks, blocks;
    // no more blocks than units: each of them then has some, as whoever adds up a tile's pieces expects
    __device__ FlRange(long long units_, int k_blocks_, int c, int blocks_) : units(units_), k_blocks(k_blocks_), blocks(blocks_) {
        begin = c < blocks ? units * c / blocks : units;
        end = c < blocks ? units * (c + 1) / blocks : units;
    }
    __device__ int owner(long long unit) const { return (int)(((unit + 1) * blocks - 1) / units); }       // the block that takes it
};

template <int BN, int STAGES> constexpr int fl_columns() { return fl_power(2 * BN + 16 * STAGES); }
template <int BN, int STAGES> constexpr size_t fl_smem() {
    return (size_t)STAGES * ((FL_BM + BN) * FL_ROW + 2 * FL_CHUNK) + FL_INNER_ROWS * FL_INNER_LD * 4 + (2 * STAGES + 4) * 8 + 32 + 1024;
}

template <int BN, int STAGES, int MODE, bool LIST>
__global__ void __launch_bounds__(FL_THREADS, 1)
fp4_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws,
                  const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs, const FlOut o, const FlTiles list,
                  int m_tiles, int n_tiles, int k_blocks, int* __restrict__ arrived, float* __restrict__ pieces, int* __restrict__ error_word) {
    constexpr uint32_t W_BYTES = FL_BM * FL_ROW, X_BYTES = BN * FL_ROW, STAGE_BYTES = W_BYTES + X_BYTES + 2 * FL_CHUNK;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* inner = (float*)(smem + STAGES * STAGE_BYTES);           // [FL_INNER_ROWS][FL_INNER_LD]
    uint64_t* bars = (uint64_t*)(inner + FL_INNER_ROWS * FL_INNER_LD);      // full[STAGES], empty[STAGES], acc_full[2], acc_empty[2]
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * STAGES + 4);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);     // [0]: a role gave up; [1]: stays zero
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
    const uint32_t acc_full0 = smem_u32(bars + 2 * STAGES), acc_empty0 = smem_u32(bars + 2 * STAGES + 2);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(acc_full0 + 8 * i, 1); mbar_init(acc_empty0 + 8 * i, 4); }
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(fl_columns<BN, STAGES>()) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const bool late = LIST && !list.ready;                         // nothing can be fetched before the launch in front has ended
    if (late) { ssb_pdl_wait(); ssb_pdl_launch_dependents(); }
    // a tile's place: dense, tiles of rows go fastest; of a list, tiles of channels
    const int listed = LIST ? list.meta[0] : m_tiles;
    const long long units = (long long)listed * n_tiles * k_blocks;
    // of a list as many blocks as tiles, or equal parts of tiles, where there are no more tiles than blocks
    const int list_tiles = listed * n_tiles, blocks = (int)gridDim.x;
    const FlRange range(units, k_blocks, blockIdx.x,
                        !LIST || list_tiles > blocks || list_tiles == 0 ? blocks : list_tiles * max(1, min(blocks / list_tiles, k_blocks / 4)));
    auto place = [&](int tile, int& m, int& n) {
        if (LIST) { m = tile / n_tiles; n = tile - m * n_tiles; }
        else { n = tile / m_tiles; m = tile - n * m_tiles; }
    };

    if (warp == 0) {
        if (lane == 0) {
            const int all = (int)(range.end - range.begin), ahead = late ? 0 : min(STAGES, all);
            const int tile0 = (int)(range.begin / k_blocks);
            const int kb_first = (int)(range.begin - (long long)tile0 * k_blocks);
            int tile = tile0, kb = kb_first, m, n, e = 0;
            auto begin = [&]() {
                place(tile, m, n);
                if (LIST) e = list.tile_expert[m];
            };
            auto next = [&]() {
                if (++kb == k_blocks) { kb = 0; ++tile; if ((long long)tile * k_blocks < range.end) begin(); }
            };
            auto weights = [&](int s) {
                const uint32_t dst = smem_u32(smem + s * STAGE_BYTES);
                mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                tma_load_2d(dst, &map_w, full0 + 8 * s, kb * FL_ROW, e * o.N + n * FL_BM);
                tma_load_2d(dst + W_BYTES + X_BYTES, &map_ws, full0 + 8 * s, 0, (e * n_tiles + n) * k_blocks + kb);
            };
            if (all > 0) begin();
            // the first stages' weights are nobody's output: they come while the rows are still being quantised
            for (int s = 0; s < ahead; ++s, next()) weights(s);
            if (!late) { ssb_pdl_wait(); ssb_pdl_launch_dependents(); }
            tile = tile0; kb = kb_first;
            if (all > 0) begin();
            int c = 0, s = 0;
            uint32_t lap = 1;
            for (; c < all; ++c, next()) {
                if (c >= ahead) {
                    if (!mbar_wait(empty0 + 8 * s, lap, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); break;
                    }
                    weights(s);
                }
                const uint32_t x_dst = smem_u32(smem + s * STAGE_BYTES) + W_BYTES;
                tma_load_2d(x_dst, &map_x, full0 + 8 * s, kb * FL_ROW, m * BN);
                tma_load_2d(x_dst + X_BYTES + FL_CHUNK, &map_xs, full0 + 8 * s, 0, (LIST ? m : m * BN >> 7) * k_blocks + kb);
                if (++s == STAGES) { s = 0; lap ^= 1; }
            }
            if (*abort_flag)                                       // let copies that were issued land before the block ends
                for (int i = max(0, c - STAGES); i < c; ++i)
                    mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, abort_flag + 1);
        }
    } else if (warp == 1) {
        if (!late) ssb_pdl_wait();                                 // what follows spins on barriers
        constexpr uint32_t idesc0 = fl_idesc(FL_BM, BN, 0), idesc1 = fl_idesc(FL_BM, BN, 1);
        const bool issues = fl_elect();
        const uint64_t w_desc = smem_desc(smem_u32(smem)), x_desc = smem_desc(smem_u32(smem) + W_BYTES);
        bool ok = true;
        int i = 0, s = 0;
        uint32_t lap = 0;
        for (long long u = range.begin; u < range.end && ok; ++i) {
            const int tile = (int)(u / k_blocks), kb0 = (int)(u - (long long)tile * k_blocks);
            const int n = (int)min((long long)(k_blocks - kb0), range.end - u), buf = i & 1;
            int m, unused;
            place(tile, m, unused);
            const int rows_at = LIST || BN == 128 ? 0 : (m * BN & 127) / 32;          // 32 rows' scales a column
            ok = mbar_wait(acc_empty0 + 8 * buf, ((i >> 1) & 1) ^ 1, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break; }
            tc_fence_after();
            for (int j = 0; j < n; ++j) {
                ok = mbar_wait(full0 + 8 * s, lap, abort_flag);
                if (!__all_sync(0xffffffffu, ok)) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break; }
                tc_fence_after();
                // a stage has columns of its own for its scales, so what reads them is done when they are written again
                const uint32_t s_addr = smem_u32(smem) + s * STAGE_BYTES + W_BYTES + X_BYTES, scales = tmem + 2 * BN + 16 * s;
                const uint32_t step = s * (STAGE_BYTES >> 4);
                if (issues) {
                    fl_copy_scales(scales, s_addr);
                    fl_copy_scales(scales + 4, s_addr + 512);
                    fl_copy_scales(scales + 8, s_addr + FL_CHUNK);
                    fl_copy_scales(scales + 12, s_addr + FL_CHUNK + 512);
                    fl_mma_x4(tmem + buf * BN, w_desc + step, x_desc + step, idesc0, idesc1, scales, scales + 8 + rows_at, scales + 4,
                              scales + 12 + rows_at, j > 0 ? 1u : 0u);
                    tc_commit(empty0 + 8 * s);
                }
                __syncwarp();
                if (++s == STAGES) { s = 0; lap ^= 1; }
            }
            if (ok && issues) tc_commit(acc_full0 + 8 * buf);
            __syncwarp();
            u += n;
        }
    } else {
        if (!late) ssb_pdl_wait();
        constexpr int CH = 16;                                    // rows of x at a time
        const int quarter = warp & 3, in_tile = quarter * 32 + lane, who = threadIdx.x - 64;
        int i = 0;
        for (long long u = range.begin; u < range.end; ++i) {
            const int tile = (int)(u / k_blocks), kb0 = (int)(u - (long long)tile * k_blocks);
            const int n = (int)min((long long)(k_blocks - kb0), range.end - u), buf = i & 1;
            int mt, nt;
            place(tile, mt, nt);
            const int m0 = mt * BN, col = nt * FL_BM + in_tile;    // the tile's first row of x, this thread's output channel
            u += n;
            // all that does not wait for the sums comes before them
            int rows, sorted0 = 0;
            if (LIST) { sorted0 = list.tile_row0[mt]; rows = min(list.offsets[list.tile_expert[mt] + 1] - sorted0, BN); }
            else rows = min(BN, o.M - m0);
            const long long first = (long long)tile * k_blocks;
            const int c0_block = n == k_blocks ? 0 : range.owner(first), c1_block = n == k_blocks ? 0 : range.owner(first + k_blocks - 1);
            __syncwarp();
            // the four warps meet below: they go on together or not at all
            if (fl_any_of_four(!mbar_wait(acc_full0 + 8 * buf, (i >> 1) & 1, abort_flag))) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
            // a block's pieces: of the tile that its range begins in the middle of (or that is all it has), and of its last; four
            // rows' sums of a channel lie together
            auto sums_of = [&](int c) { return reinterpret_cast<float4*>(pieces) + (size_t)(2 * c + (c == c0_block)) * (BN / 4) * FL_BM + in_tile; };
            bool mine = true;                                      // whether this block writes the tile's results
            if (n < k_blocks) {
                float4* dst = sums_of(blockIdx.x);
#pragma unroll 1
                for (int c0 = 0; c0 < rows; c0 += CH) {
                    float sum[CH];
                    fl_ld16(acc + c0, sum);
#pragma unroll
                    for (int e = 0; e < CH; e += 4)
                        if (c0 + e < rows) dst[(size_t)((c0 + e) / 4) * FL_BM] = make_float4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
                }
                __threadfence();
                fl_any_of_four(false);
                bool last = false;
                if (threadIdx.x == 64) {
                    last = atomicAdd(arrived + c0_block, n) + n == k_blocks;
                    if (last) arrived[c0_block] = 0;               // as it was, for the next launch that counts here
                }
                mine = fl_any_of_four(last);
                if (mine) __threadfence();
            }
#pragma unroll 1
            for (int c0 = 0; mine && c0 < rows; c0 += CH) {        // rows of x
                const int live = col < o.N ? rows - c0 : 0;
                const size_t at = (size_t)(m0 + c0) * o.ldo + col;
                float was[CH];
                __syncwarp();
                if (MODE == FL_STORE && o.add)
#pragma unroll
                    for (int e = 0; e < CH; ++e) was[e] = e < live ? ((const float*)o.out)[at + (size_t)e * o.ldo] : 0.f;
                float sum[CH];
                if (n == k_blocks) {
                    fl_ld16(acc + c0, sum);
                } else {
#pragma unroll
                    for (int e = 0; e < CH; ++e) sum[e] = 0.f;
#pragma unroll 4
                    for (int c = c0_block; c <= c1_block; ++c) {
                        const float4* src = sums_of(c) + (size_t)(c0 / 4) * FL_BM;
#pragma unroll
                        for (int e = 0; e < CH; e += 4) {
                            const float4 v = c0 + e < rows ? __ldcg(src + (size_t)(e / 4) * FL_BM) : make_float4(0.f, 0.f, 0.f, 0.f);
                            sum[e] += v.x; sum[e + 1] += v.y; sum[e + 2] += v.z; sum[e + 3] += v.w;
                        }
                    }
                }
                if (MODE == FL_STORE) {
                    if (o.index) {
#pragma unroll
                        for (int e = 0; e < CH; ++e)
                            if (e < live) ((float*)o.out)[(size_t)o.index[sorted0 + c0 + e] * o.ldo + col] = sum[e];
                    } else if (!o.is_f32) {
#pragma unroll
                        for (int e = 0; e < CH; ++e)
                            if (e < live) ((bf16*)o.out)[at + (size_t)e * o.ldo] = __float2bfloat16_rn(sum[e]);
                    } else {
#pragma unroll
                        for (int e = 0; e < CH; ++e)
                            if (e < live) ((float*)o.out)[at + (size_t)e * o.ldo] = o.add ? sum[e] + was[e] : sum[e];
                    }
                } else {
                    fl_inner_tile<MODE>(sum, inner, quarter, lane, who, c0, m0, LIST ? mt * 128 : m0, rows, nt, n_tiles, o.N, o.kind, o.limit,
                                        o.row_scale, (uint8_t*)o.out, o.ldo, o.scales, o.inner_blocks);      // a listed tile's scales are 128 rows'
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) fl_arrive(acc_empty0 + 8 * buf);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(fl_columns<BN, STAGES>()) : "memory");
    }
}

// Tiles of 256 rows x 256 channels on pairs of SMs: each block fetches 128 rows and 128 channels a k-block, its rows' scales and those
// of all 256 channels; the leader issues the pair's instructions, each block's tensor memory gets its 128 rows.  Tensor memory has 512
// columns: two accumulators of 256 that share 128 of them, and five times 24 for a k-block's scales.  An epilogue begins with the
// columns that the next tile wants, and hands them over as soon as they are in registers.
//
// Scales come to tensor memory through the registers of four warps (tcgen05.st), which fetch them some k-blocks ahead: tcgen05.cp runs
// in order with the products and took 0.19 us of a k-block's 0.66 (six of them; 8,192 x 14,336 x 4,096: 266 us); through shared memory
// by TMA they stand behind the codes that were asked for before them (357 us), and by cp.async a k-block takes these warps 850 clocks.
//
// 8,192 x 14,336 x 4,096: 179 us (201 with rows to codes), 5.4 PFLOP/s, the tensor pipe busy 73 % of the cycles, at 1,965 MHz; where calls
// follow one another for half a second the power cap takes the clock to some 1,500 MHz, and a call 229 us.  Bound by codes on their way from L2 (two sides of
// 256 a tile, some 46 bytes a clock and SM) and by results on theirs (without them 35 us less).
//
// Results leave in runs of 128 bytes, which takes the place of a sixth stage of codes (of 64 bytes with six: 8,192 x 14,336 x 4,096 209 us
// for 206, 2,048 tokens' experts 159 for 151).
//
// Tiles go in bands of ``group_m`` row tiles, row tiles fastest; of experts (LIST), a list's tile of rows with all its channels.  Bands of
// 32 where there are many tiles of channels, of 16 where there are few: 8,192 x 14,336 x 4,096 181 us (by 16 191), 16,384 x 28,672 x 2,048
// 405 (426); 8,192 x 4,096 x 14,336 187 (179), 32,768 x 4,096 x 4,096 210 (205).
constexpr int FL_PAIR_STAGES = 5;
constexpr int FL_PAIR_STAGE_BYTES = 2 * FL_BM * FL_ROW;
constexpr int FL_PAIR_SETS = 5;           // k-blocks whose scales are in tensor memory
constexpr int FL_PAIR_AHEAD = 3;          // and in registers, on their way
constexpr int FL_PAIR_ACC = 128;          // columns from the first accumulator to the second
constexpr int FL_PAIR_SCALES = 384;       // scales' first column
constexpr int FL_PAIR_WARPS = 14;         // 0: TMA, 1: MMA + tensor memory, 2-5: scales, 6-13: epilogue
constexpr int FL_PAIR_PUT = 32 * 36;      // words in which an epilogue warp's rows meet
constexpr int FL_PAIR_BARS = 2 * FL_PAIR_STAGES + FL_PAIR_SETS + 3;
static_assert(FL_PAIR_SETS <= FL_PAIR_STAGES, "a set's last products are told by the stage that they freed, which must not have been freed again");
constexpr size_t FL_PAIR_SMEM = (size_t)FL_PAIR_STAGES * FL_PAIR_STAGE_BYTES + 8 * FL_PAIR_PUT * 4 + FL_PAIR_BARS * 8 + 24 + 1024;

// A lane's 32 words of its row, a warp's rows in runs of 128 bytes through ``stage``; ``at``: the lane's row of dst.
template <bool ADD>
__device__ __forceinline__ void fl_put_rows(float* stage, const uint32_t* v, char* dst, size_t row_bytes, int at, int rows) {
    constexpr int WORDS = 32, LD = WORDS + 4, PER = WORDS / 4, ROWS = 32 / PER;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < WORDS; j += 4)
        *reinterpret_cast<uint4*>(stage + lane * LD + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    __syncwarp();
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += ROWS) {
        const int r = r0 + lane / PER, c = lane % PER * 4, row = __shfl_sync(0xffffffffu, at, r);
        const float4 x = *reinterpret_cast<const float4*>(stage + r * LD + c);
        if (r < rows) {
            float4* to = reinterpret_cast<float4*>(dst + (size_t)row * row_bytes) + lane % PER;
            if (ADD) atomicAdd(to, x);
            else *to = x;
        }
    }
    __syncwarp();
}

template <int MODE, bool LIST>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(32 * FL_PAIR_WARPS, 1)
fp4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const uint8_t* __restrict__ xs,
                const uint8_t* __restrict__ ws, int x_runs, const FlOut o, const FlTiles list, int m_tiles, int n_tiles, int k_blocks,
                int group_m, int* __restrict__ error_word) {
    constexpr int BN = 256, STAGES = FL_PAIR_STAGES;
    constexpr uint32_t X_BYTES = FL_BM * FL_ROW, W_BYTES = FL_BM * FL_ROW, STAGE_BYTES = FL_PAIR_STAGE_BYTES;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* put = (float*)(smem + STAGES * STAGE_BYTES);
    uint64_t* bars = (uint64_t*)(put + 8 * FL_PAIR_PUT);            // full, empty [STAGES], ready [SETS], acc_full[2], free
    uint32_t* tmem_slot = (uint32_t*)(bars + FL_PAIR_BARS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();                        // 0: the leader
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
    const uint32_t ready0 = smem_u32(bars + 2 * STAGES);            // scales are in both blocks' tensor memory: at the leader, as full
    const uint32_t acc_full0 = ready0 + 8 * FL_PAIR_SETS, free0 = acc_full0 + 16;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < FL_PAIR_SETS; ++s) mbar_init(ready0 + 8 * s, 8);
        for (int i = 0; i < 2; ++i) mbar_init(acc_full0 + 8 * i, 1);
        mbar_init(free0, 16);
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync_all();   // both blocks' barriers are initialised before either signals the other
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    ssb_pdl_wait();       // rows, scales and a list are there
    if (threadIdx.x == 0) ssb_pdl_launch_dependents();
    const int tiles = (LIST ? list.meta[0] : m_tiles) * n_tiles;
    auto tile_at = [&](int tile, int& m, int& n) {
        if (LIST) { m = tile / n_tiles; n = tile - m * n_tiles; return; }
        const int band = tile / (group_m * n_tiles), in_band = tile - band * group_m * n_tiles, rows = min(group_m, m_tiles - band * group_m);
        m = band * group_m + in_band % rows;
        n = in_band / rows;
    };

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t leader_full0 = cluster_map(full0, 0);
            int c = 0;
            for (int tile = pair; tile < tiles && !*abort_flag; tile += n_pairs) {
                int m, n;
                tile_at(tile, m, n);
                const int e = LIST ? list.tile_expert[m] : 0;
                const int mt = 2 * m + (int)rank, n0 = e * o.N + n * BN + (int)rank * FL_BM;
                for (int kb = 0; kb < k_blocks; ++kb, ++c) {
                    const int s = c % STAGES;
                    const uint32_t x_dst = smem_u32(smem + s * STAGE_BYTES), bar = leader_full0 + 8 * s;
                    if (!mbar_wait(empty0 + 8 * s, ((c / STAGES) & 1) ^ 1, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); break;
                    }
                    if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * (X_BYTES + W_BYTES));
                    tma_load_2d_pair(x_dst, &map_x, bar, kb * FL_ROW, mt * FL_BM);
                    tma_load_2d_pair(x_dst + X_BYTES, &map_w, bar, kb * FL_ROW, n0);
                }
            }
            if (*abort_flag) {
                // let issued copies land: the leader sees both blocks' codes on its barriers, the other block gives them time
                if (rank == 0) {
                    for (int i = max(0, c - STAGES); i < c; ++i)
                        mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, abort_flag + 1);
                } else {
                    const long long t0 = clock64();
                    while (clock64() - t0 < 2000000LL) __nanosleep(1000);
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            constexpr uint32_t idesc0 = fl_idesc(256, BN, 0), idesc1 = fl_idesc(256, BN, 1);
            const bool issues = fl_elect();
            const uint64_t x_desc = smem_desc(smem_u32(smem)), w_desc = smem_desc(smem_u32(smem) + X_BYTES);
            bool ok = true;
            int i = 0, s = 0, set = 0;
            uint32_t lap = 0, set_lap = 0;
            for (int tile = pair; tile < tiles && ok; tile += n_pairs, ++i) {
                const uint32_t acc = tmem + (i & 1) * FL_PAIR_ACC;
                if (i > 0) ok = mbar_wait(free0, (i - 1) & 1, abort_flag);            // both epilogues have the shared columns
                if (!__all_sync(0xffffffffu, ok)) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break; }
                for (int kb = 0; kb < k_blocks; ++kb) {
                    ok = mbar_wait(ready0 + 8 * set, set_lap, abort_flag) && mbar_wait(full0 + 8 * s, lap, abort_flag);
                    if (!__all_sync(0xffffffffu, ok)) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break; }
                    tc_fence_after();
                    const uint32_t x_sc = tmem + FL_PAIR_SCALES + set * 24, w_sc = x_sc + 8, step = s * (STAGE_BYTES >> 4);
                    if (issues) {
                        fl_mma_pair_x4(acc, x_desc + step, w_desc + step, idesc0, idesc1, x_sc, w_sc, x_sc + 4, w_sc + 8, kb > 0 ? 1u : 0u);
                        tc_commit_pair(empty0 + 8 * s, 3);          // the stage is free in both blocks
                    }
                    __syncwarp();
                    if (++s == STAGES) { s = 0; lap ^= 1; }
                    if (++set == FL_PAIR_SETS) { set = 0; set_lap ^= 1; }
                }
                if (ok && issues) tc_commit_pair(acc_full0 + 8 * (i & 1), 3);
                __syncwarp();
            }
        }
    } else if (warp < 6) {
        // a lane's 16 bytes of each 512 are four columns of its lane, in this warp's quarter of the lanes as in the others
        const uint32_t leader_ready0 = cluster_map(ready0, 0), columns = tmem + FL_PAIR_SCALES + ((uint32_t)(warp & 3) << 21);
        const int runs = (o.N + FL_BM - 1) / FL_BM;                 // of a weight matrix's scales
        // what is fetched next: k-block in_kb of tile in_tile; of rows x, of channels 0-127 a, 128-255 b, blocks 0-3 and 4-7
        struct { uint4 x0, x1, a0, a1, b0, b1; } w[FL_PAIR_AHEAD];
        int in_tile = pair, in_kb = 0;
        const uint8_t *src_x = xs, *src_a = ws, *src_b = ws;
        bool live_x = false, live_b = false;                        // behind the last run: zeros
        auto load = [&](auto& to) {
            if (in_tile >= tiles) return;
            if (in_kb == 0) {
                int m, n;
                tile_at(in_tile, m, n);
                const int run_x = 2 * m + (int)rank, run_w = (LIST ? list.tile_expert[m] : 0) * runs + 2 * n;
                live_x = run_x < x_runs;
                live_b = 2 * n + 1 < runs;
                src_x = xs + (size_t)(live_x ? run_x : 0) * k_blocks * FL_CHUNK + lane * 16;
                src_a = ws + (size_t)run_w * k_blocks * FL_CHUNK + lane * 16;
                src_b = live_b ? src_a + (size_t)k_blocks * FL_CHUNK : src_a;
            }
            const size_t at = (size_t)in_kb * FL_CHUNK;
            auto get = [&](const uint8_t* p, bool live) { return live ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0); };
            to.x0 = get(src_x + at, live_x); to.x1 = get(src_x + at + 512, live_x);
            to.a0 = get(src_a + at, true); to.a1 = get(src_a + at + 512, true);
            to.b0 = get(src_b + at, live_b); to.b1 = get(src_b + at + 512, live_b);
            if (++in_kb == k_blocks) { in_kb = 0; in_tile += n_pairs; }
        };
#pragma unroll
        for (int q = 0; q < FL_PAIR_AHEAD; ++q) load(w[q]);
        const int my_tiles = pair < tiles ? (tiles - pair + n_pairs - 1) / n_pairs : 0, all = my_tiles * k_blocks;
        bool ok = true;
        for (int c0 = 0; c0 < all && ok; c0 += FL_PAIR_AHEAD) {
#pragma unroll
            for (int q = 0; q < FL_PAIR_AHEAD; ++q) {
                const int c = c0 + q, set = c % FL_PAIR_SETS, before = c - FL_PAIR_SETS;
                if (c >= all || !ok) continue;
                // the set's last products are done
                if (before >= 0) ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * (before % STAGES), (before / STAGES) & 1, abort_flag));
                if (!ok) {
                    if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); }
                    continue;
                }
                tc_fence_after();
                fl_st8(columns + set * 24, w[q].x0, w[q].x1);       // rows: blocks 0-3, 4-7
                fl_st8(columns + set * 24 + 8, w[q].a0, w[q].b0);   // blocks 0-3: channels 0-127, 128-255
                fl_st8(columns + set * 24 + 16, w[q].a1, w[q].b1);  // blocks 4-7
                load(w[q]);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) fl_arrive_leader(leader_ready0 + 8 * set);
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 6) >> 2;
        float* stage = put + (warp - 6) * FL_PAIR_PUT;
        const uint32_t leader_free = cluster_map(free0, 0);
        int i = 0;
        for (int tile = pair; tile < tiles; tile += n_pairs, ++i) {
            int m, n;
            tile_at(tile, m, n);
            // this warp's 32 rows: the first of them in the matrix (among a list's tiles) and how many there are
            const int in_tile = (int)rank * FL_BM + quarter * 32, row0 = m * BN + in_tile, row = row0 + lane, buf = i & 1;
            int rows = o.M - row0, to = row;
            if (LIST) {
                const int first = list.tile_row0[m];
                rows = min(list.offsets[list.tile_expert[m] + 1] - first, BN) - in_tile;
                if (o.index && lane < rows) to = o.index[first + in_tile + lane];
            }
            const float row_scale = MODE == FL_GATED && o.row_scale && lane < rows ? o.row_scale[row] : 1.f;
            bool ok = mbar_wait(acc_full0 + 8 * buf, (i >> 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * FL_PAIR_ACC + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
            for (int j = 0; j < 2; ++j) {
                const int g = half + 2 * (j ^ buf ^ 1);              // the shared 128 columns first
                uint32_t r[2][32];
                tc_ld32(acc + g * 64, r[0]);
                tc_ld32(acc + g * 64 + 32, r[1]);
                if (j == 0) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) fl_arrive_leader(leader_free);
                }
                if (rows <= 0) continue;
                if (MODE == FL_STORE && !o.is_f32 && n * BN + g * 64 + 64 <= o.N) {
                    uint32_t packed[32];
#pragma unroll
                    for (int e = 0; e < 64; e += 2) {
                        const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(r[e >> 5][e & 31]), __uint_as_float(r[e >> 5][(e & 31) + 1]));
                        packed[e / 2] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    fl_put_rows<false>(stage, packed, (char*)((bf16*)o.out + n * BN + g * 64), (size_t)o.ldo * 2, to, rows);
                } else if (MODE == FL_STORE) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int col = n * BN + g * 64 + h * 32;
                        if (col >= o.N) continue;
                        if (o.is_f32) {
                            if (col + 32 <= o.N) {
                                char* dst = (char*)((float*)o.out + col);
                                if (o.add) fl_put_rows<true>(stage, r[h], dst, (size_t)o.ldo * 4, to, rows);
                                else fl_put_rows<false>(stage, r[h], dst, (size_t)o.ldo * 4, to, rows);
                            } else if (lane < rows) {
                                float* dst = (float*)o.out + (size_t)to * o.ldo + col;
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (col + e < o.N) dst[e] = o.add ? dst[e] + __uint_as_float(r[h][e]) : __uint_as_float(r[h][e]);
                            }
                        } else if (lane < rows) {
                            bf16* dst = (bf16*)o.out + (size_t)to * o.ldo + col;
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (col + e < o.N) dst[e] = __float2bfloat16_rn(__uint_as_float(r[h][e]));
                        }
                    }
                } else {
                    // a lane holds 64 sums of its row: a block of 32 inner channels (16 gate, 16 up, twice), or two of them
                    constexpr int BLOCKS = MODE == FL_GATED ? 1 : 2;
                    const int width = MODE == FL_GATED ? o.N / 2 : o.N;
#pragma unroll
                    for (int h = 0; h < BLOCKS; ++h) {
                        float v[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            v[e] = MODE == FL_GATED ? ssb_gate_fast(__uint_as_float(r[e >> 4][e & 15]), __uint_as_float(r[e >> 4][16 + (e & 15)]), o.kind, o.limit) * row_scale
                                                    : ssb_activate(__uint_as_float(r[h][e]), o.kind) * o.limit;
                        uint32_t most = f4_most(v);
                        if (most >= F4_WILD) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = f4_finite(v[e]);
                            most = f4_most(v);
                        }
                        const int byte = f4_scale_byte(most), k = (n * 4 + g) * 32 * BLOCKS + h * 32;
                        const float inverse = f4_inverse(byte);
                        if (lane < rows && k < width) {
                            *reinterpret_cast<uint4*>((uint8_t*)o.out + (size_t)row * o.ldo + k / 2) =
                                make_uint4(f4_encode8(v, inverse), f4_encode8(v + 8, inverse), f4_encode8(v + 16, inverse), f4_encode8(v + 24, inverse));
                            o.scales[f4_scale_at(row, k / F4_BLOCK, o.inner_blocks)] = (uint8_t)byte;
                        }
                    }
                    // behind the last channel: scales of zero up to a whole k-block
                    if (j == 0 && half == 0 && n == n_tiles - 1 && lane < rows)
                        for (int b = width / F4_BLOCK; b < 8 * o.inner_blocks; ++b) o.scales[f4_scale_at(row, b, o.inner_blocks)] = 0;
                }
            }
        }
    }
    tc_fence_before();
    cluster_sync_all();   // neither block leaves while the other may still read its shared memory or signal it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
    cluster_sync_all();
}

// ---- host side --------------------------------------------------------------------------------------------------------
struct FlPlan {
    int bn, m_tiles, n_tiles, blocks;      // bn 0: tiles on pairs
    size_t pieces;                         // bytes
};
// What a product is expected to take, in microseconds, by a fit to measured times of all forms over 1 .. 1,024 rows and 4 to 117
// million weights (of the pairs' kernel with a sixth stage, which its results' runs have taken since):
//  * a block of the streaming kernel takes 3.8 + 0.046 a row, and 0.37 a k-block of 128 weight rows whatever its rows; pieces of split
//    tiles 2.2 and, each, 0.1 + 0.01 a row;
//  * a pair 6.5, 0.43 a k-block of 256 x 256 and 0.03 for each tile beside it.
// At 2,048 x 2,048: 48 rows by tiles of 64 that are whole 9.1, in 2 parts 10.7; at 4,096 x 14,336: 64 rows by 64 in 2 parts 20.4, in 4 16.7,
// dealt out over all SMs 20.8; 128 rows by 64 in 2 parts 20.7, by 128 in 4 22.2, on pairs 30; at 14,336 x 4,096: 64 rows by 64 14.0, 128
// by 128 17.2, on pairs 15.7; 1,024 rows by 128 70, on pairs 35.  As they are taken now, rows to codes among them, weights from memory and
// from L2: 14,336 x 4,096 64 rows 12.0 and 10.3, 128 17.2 and 14.2, 300 23.9 and 21.3, 1,024 39.5 and 39.3; 4,096 x 14,336 64 rows 16.2 and
// 15.0, 128 20.2 and 19.8; 28,672 x 4,096 8 rows 16.7 and 14.1.  Tiles of 16 and 32 rows are only where one holds all rows: the next one's
// scales would begin between the columns that a product can name (and only where there are more tiles than SMs: else fp4_step.cu).
static FlPlan fl_plan(int M, int N, int K) {
    const int sms = ssb_sm_count(), k_blocks = f4_k_blocks(K);
    FlPlan best{};
    double least = 0;
    auto consider = [&](double cost, int bn, int m_tiles, int n_tiles, int blocks) {
        if (best.m_tiles && cost >= least) return;
        least = cost;
        best = FlPlan{bn, m_tiles, n_tiles, blocks, (size_t)blocks * 2 * bn * FL_BM * 4};
    };
    for (int bn = M <= 16 ? 16 : M <= 32 ? 32 : 64; bn <= 128; bn *= 2) {
        const int m_tiles = (M + bn - 1) / bn, n_tiles = (N + FL_BM - 1) / FL_BM, rows = std::min(bn, M);
        const long long tiles = (long long)m_tiles * n_tiles, units = tiles * k_blocks;
        const double block = 3.8 + 0.046 * rows, piece = 0.1 + 0.01 * rows;
        if (tiles <= sms)
            for (int parts = 1; parts <= std::min(sms / (int)tiles, k_blocks); ++parts)
                consider(block + 0.37 * ((k_blocks + parts - 1) / parts) + (parts > 1 ? 2.2 + piece * parts : 0), bn, m_tiles, n_tiles, (int)tiles * parts);
        const int any = (int)std::min<long long>(sms, units);
        const double share = (double)tiles / any;
        consider(block + 0.37 * ((double)units / any) + 3.7 + piece * std::max(2.0, 1 / share) + share * (0.7 + 0.046 * rows), bn, m_tiles, n_tiles, any);
        if (M <= bn) break;
    }
    if (M > 64) {
        const int m_tiles = (M + 255) / 256, n_tiles = (N + 255) / 256, pairs = sms / 2;
        const long long tiles = (long long)m_tiles * n_tiles;
        consider(6.5 + 0.43 * (double)((tiles + pairs - 1) / pairs) * k_blocks + 0.03 * (double)std::min<long long>(tiles, pairs), 0, m_tiles, n_tiles, 0);
    }
    return best;
}
static size_t fl_round(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr int FL_COUNTERS = 256;          // of a launch: one for each of its blocks

// Scratch of a product of M rows by N x K weights: codes and scales of the rows (of rows that come as numbers), pieces of tiles.
struct FlScratch {
    size_t codes, scales, pieces, all;
    FlScratch(int M, int K, bool numbers, size_t piece_bytes) {
        codes = 0;
        scales = numbers ? fl_round((size_t)M * (K / 2)) : 0;
        pieces = scales + (numbers ? (size_t)((M + 127) / 128) * f4_k_blocks(K) * F4_CHUNK : 0);
        all = pieces + std::max<size_t>(piece_bytes, 16);
    }
};
// The kernel of few rows takes products where there is little to read (its time here, and with their rows' launch the other's, by tiles of
// 16 on clusters): 1 x 2,048 x 2,048 3.5 us (5.2), 8 rows 3.9 (5.4), 16 rows 5.7 (5.9); 1 x 4,096 x 4,096 5.2 (7.2), 8 rows 7.2 (7.2);
// 1 x 6,144 x 4,096 7.3 (7.9), 8 rows 9.2 (8.0).  Inner rows are put into 4 bits a block of 32 at a time, which is fewer and longer strips
// of weights: 1 x 2,048 x 2,048 5.1 (5.3), 8 rows 5.8 (5.7), 16 rows 8.6 (6.4); 1 x 4,096 x 4,096 7.0 (7.3); 1 x 1,024 x 8,192 11.5 (8.0).
constexpr long long FL_FEW_NUMBERS = 32768, FL_FEW_INNER = 16384;
static bool fl_few(int M, int N, int K, int mode) {
    if ((long long)N * K > (M <= 4 ? 24 << 20 : M <= 8 ? 16 << 20 : 4 << 20)) return false;
    if (mode == FL_STORE ? (long long)M * K > FL_FEW_NUMBERS : K > 4096 || (long long)M * K > FL_FEW_INNER) return false;
    return fw_takes(M, N, K, mode);
}

// Twice the bytes of scratch that a product needs, and one if it needs counters.  numbers: rows come as numbers; mode: FL_*.
SSB_API long long ssb_fp4_product_scratch(int M, int N, int K, int numbers, int mode) {
    if (M <= 0 || N <= 0 || K <= 0 || fl_few(M, N, K, mode)) return 0;
    if (fs_parts(M, N, K)) return numbers ? 2 * (long long)FlScratch(M, K, true, 0).all : 0;
    return 2 * (long long)FlScratch(M, K, numbers != 0, fl_plan(M, N, K).pieces).all + 1;
}

template <int BN, int STAGES, int MODE, bool LIST>
static int fl_stream(const CUtensorMap& mw, const CUtensorMap& mws, const CUtensorMap& mx, const CUtensorMap& mxs, const FlOut& o,
                     const FlTiles& list, int m_tiles, int n_tiles, int blocks, int K, bool early, int* counters, float* pieces,
                     int* error_word, cudaStream_t stream) {
    constexpr size_t smem = fl_smem<BN, STAGES>();
    static_assert(smem <= 227 * 1024, "");
    static SsbPerDevice<bool> set;
    bool* configured = set.here();
    if (!configured) return SSB_ERR_UNSUPPORTED;
    if (!*configured) {
        cudaError_t e = cudaFuncSetAttribute(fp4_stream_kernel<BN, STAGES, MODE, LIST>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        *configured = true;
    }
    return ssb_launch(fp4_stream_kernel<BN, STAGES, MODE, LIST>, dim3(blocks), dim3(FL_THREADS), smem, stream, early, mw, mws, mx, mxs, o, list,
                      m_tiles, n_tiles, f4_k_blocks(K), counters, pieces, error_word);
}

template <int MODE, bool LIST>
static int fl_pair(const CUtensorMap& mx, const CUtensorMap& mw, const void* xs, const void* ws, int x_runs, const FlOut& o,
                   const FlTiles& list, int m_tiles, int n_tiles, int K, int* error_word, cudaStream_t stream) {
    static_assert(FL_PAIR_SMEM <= 227 * 1024, "");
    auto kernel = fp4_pair_kernel<MODE, LIST>;
    static SsbPerDevice<int> found;
    int* max_pairs = found.here();
    if (!max_pairs) return SSB_ERR_UNSUPPORTED;
    if (!*max_pairs) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FL_PAIR_SMEM);
        if (e != cudaSuccess) return (int)e;
        const int sms = ssb_sm_count();
        // how many pairs the device holds at once (a GPC with an odd SM left over holds one fewer)
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sms & ~1);
        cfg.blockDim = dim3(32 * FL_PAIR_WARPS);
        cfg.dynamicSmemBytes = FL_PAIR_SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters <= 0) {
            cudaGetLastError();
            clusters = sms / 2;
        }
        *max_pairs = std::min(clusters, sms / 2);
    }
    const int pairs = (int)std::min<long long>((long long)m_tiles * n_tiles, *max_pairs);
    return ssb_launch(kernel, dim3(2 * pairs), dim3(32 * FL_PAIR_WARPS), FL_PAIR_SMEM, stream, true, mx, mw, (const uint8_t*)xs,
                      (const uint8_t*)ws, x_runs, o, list, m_tiles,
                      n_tiles, f4_k_blocks(K), std::min(n_tiles >= 32 ? 32 : 16, m_tiles), error_word);
}

template <int MODE>
static int fl_dense(const void* x, const void* xs, const void* w, const void* ws, const FlOut& o, int K, bool early, int* counters,
                    float* pieces, const FlPlan& p, int* error_word, cudaStream_t stream) {
    const int k_blocks = f4_k_blocks(K);
    CUtensorMap mw, mws, mx, mxs;
    int rc = fl_map(&mx, x, o.M, K / 2, p.bn ? p.bn : FL_BM);
    if (!rc) rc = fl_map(&mw, w, o.N, K / 2, FL_BM);
    if (!rc) rc = fl_scale_map(&mxs, xs, (long long)((o.M + 127) / 128) * k_blocks);
    if (!rc) rc = fl_scale_map(&mws, ws, (long long)((o.N + 127) / 128) * k_blocks);
    if (rc) return rc;
    const FlTiles none{};
    switch (p.bn) {
        case 16: return fl_stream<16, 5, MODE, false>(mw, mws, mx, mxs, o, none, p.m_tiles, p.n_tiles, p.blocks, K, early, counters, pieces, error_word, stream);
        case 32: return fl_stream<32, 9, MODE, false>(mw, mws, mx, mxs, o, none, p.m_tiles, p.n_tiles, p.blocks, K, early, counters, pieces, error_word, stream);
        case 64: return fl_stream<64, 8, MODE, false>(mw, mws, mx, mxs, o, none, p.m_tiles, p.n_tiles, p.blocks, K, early, counters, pieces, error_word, stream);
        case 128: return fl_stream<128, 6, MODE, false>(mw, mws, mx, mxs, o, none, p.m_tiles, p.n_tiles, p.blocks, K, early, counters, pieces, error_word, stream);
    }
    return fl_pair<MODE, false>(mx, mw, xs, ws, (o.M + 127) / 128, o, none, p.m_tiles, p.n_tiles, K, error_word, stream);
}

SSB_API int ssb_fp4_quantize(const void* x, long long ldx, int dtype, void* codes, void* scales, int rows, int K, int per_expert, int inter,
                             int* clear, int n_clear, int early, cudaStream_t stream);
SSB_API int ssb_fp4_quantize_pairs(const void* x, long long ldx, int dtype, void* codes, void* scales, int tokens, int top, int K,
                                   const int* slot, int tile_rows, cudaStream_t stream);

// A product of dense weights.  x: rows of dtype (ldx elements apart), which are quantised first, or (dtype -1) codes with the scales xs.
// settled: the weights were written before the launch in front of this call began; else a product that nothing is quantised for waits for
// all that is in front of it (behind a launch that quantises rows they are there: that one waited).
// scratch: ssb_fp4_product_scratch bytes.  counters: FL_COUNTERS words (``n_clear`` of them and behind them are zeroed on the way where x
// is quantised; else the launch needs them zero); the launch leaves them zero.
template <int MODE>
static int fl_product(const void* x, long long ldx, int dtype, const void* xs, const void* w, const void* ws, const FlOut& o, int K,
                      int settled, void* scratch, int* counters, int n_clear, int* error_word, cudaStream_t stream) {
    if (o.M < 0 || o.N <= 0 || K <= 0 || K % F4_BLOCK || o.N % 8 || dtype > SSB_BF16) return SSB_ERR_BAD_SIZE;
    if (((uintptr_t)x | (uintptr_t)xs | (uintptr_t)w | (uintptr_t)ws | (uintptr_t)o.out | (uintptr_t)o.scales | (uintptr_t)scratch) & 15) return SSB_ERR_BAD_SIZE;
    if (o.M == 0) return 0;
    const bool few = fl_few(o.M, o.N, K, MODE);
    const int parts = few ? 0 : fs_parts(o.M, o.N, K);
    if (!error_word || (!few && dtype >= 0 && !scratch) || (!few && !parts && (!scratch || !counters))) return SSB_ERR_BAD_SIZE;
    char* base = (char*)scratch;
    if (few || parts) {
        if (parts && dtype >= 0) {
            const FlScratch at(o.M, K, true, 0);
            const int rc = ssb_fp4_quantize(x, ldx, dtype, base + at.codes, base + at.scales, o.M, K, o.M, 0, nullptr, 0, 1, stream);
            if (rc) return rc;
            x = base + at.codes;
            xs = base + at.scales;
        }
        FwArgs a{};
        a.w = (const uint8_t*)w; a.ws = (const uint8_t*)ws;
        a.x = x; a.ldx = ldx; a.dtype = dtype; a.xs = (const uint8_t*)xs;
        a.out = o.out; a.out_scales = o.scales; a.ldo = o.ldo; a.is_f32 = o.is_f32; a.add = o.add;
        a.M = o.M; a.N = o.N; a.K = K;
        a.kind = o.kind; a.limit = o.limit; a.row_scale = o.row_scale; a.inner_blocks = o.inner_blocks;
        return few ? fw_product(a, MODE, settled, stream) : fs_product(a, MODE, parts, settled || dtype >= 0, error_word, stream);
    }
    const FlPlan p = fl_plan(o.M, o.N, K);
    if (p.blocks > FL_COUNTERS) return SSB_ERR_UNSUPPORTED;
    const FlScratch at(o.M, K, dtype >= 0, p.pieces);
    if (dtype >= 0) {
        const int rc = ssb_fp4_quantize(x, ldx, dtype, base + at.codes, base + at.scales, o.M, K, o.M, 0, counters, n_clear, 1, stream);
        if (rc) return rc;
        x = base + at.codes;
        xs = base + at.scales;
    }
    return fl_dense<MODE>(x, xs, w, ws, o, K, settled || dtype >= 0, counters, (float*)(base + at.pieces), p, error_word, stream);
}

SSB_API int ssb_fp4_linear(const void* x, long long ldx, int dtype, const void* xs, const void* w, const void* ws, void* out, int ldo,
                           int out_dtype, int M, int N, int K, int add, int settled, void* scratch, int* counters, int* error_word, cudaStream_t stream) {
    if ((out_dtype != SSB_F32 && out_dtype != SSB_BF16) || (add && out_dtype != SSB_F32)) return SSB_ERR_BAD_DTYPE;
    const FlOut o{out, nullptr, nullptr, nullptr, ldo, out_dtype == SSB_F32, add, M, N, 0, 0.f, 0};
    return fl_product<FL_STORE>(x, ldx, dtype, xs, w, ws, o, K, settled, scratch, counters, FL_COUNTERS, error_word, stream);
}

// The inner rows of a feed-forward in 4 bits.  gated: w holds 16 gate rows and their 16 up rows in turn, N = 2 x inner channels, kind and
// limit as ssb_gate's; else kind as ssb_activate's and limit a factor.  counters: as above, and as many behind them for the product that
// reads the inner rows.
SSB_API int ssb_fp4_inner(const void* x, long long ldx, int dtype, const void* xs, const void* w, const void* ws, void* codes, void* scales,
                          int M, int N, int K, int gated, int kind, float limit, const float* row_scale, int settled, void* scratch,
                          int* counters, int* error_word, cudaStream_t stream) {
    const int inner = gated ? N / 2 : N;
    if (inner % F4_BLOCK || (gated && N % 2) || kind < 0 || kind > 2 || (row_scale && !gated)) return SSB_ERR_BAD_SIZE;
    const FlOut o{codes, (uint8_t*)scales, nullptr, row_scale, inner / 2, 0, 0, M, N, kind, limit, f4_k_blocks(inner)};
    return gated ? fl_product<FL_GATED>(x, ldx, dtype, xs, w, ws, o, K, settled, scratch, counters, 2 * FL_COUNTERS, error_word, stream)
                 : fl_product<FL_ACT>(x, ldx, dtype, xs, w, ws, o, K, settled, scratch, counters, 2 * FL_COUNTERS, error_word, stream);
}

// ---- experts ----------------------------------------------------------------------------------------------------------
// Pairs (token, choice) by expert, one block.  A warp has a run of neighbouring pairs and counts of its own: it counts them by expert, the
// counts of the warps before it say where its pairs go, and it places them.  ``slot``: where a pair's row goes among tiles of BN rows
// (-1: its expert is none), ``order``: the pair of a sorted row.  RANKED: an expert's pairs keep their order.  Which of its tiles a pair is in
// may then decide where its sums are cut, so lists whose tiles are cut are ranked; where every tile is whole (on SM pairs) the order inside a
// warp's run is whatever the adds give, and nothing that leaves the call depends on it.  12,288 pairs of 64 experts: 13 us, steps one
// after another on one SM (loaded twice and summed by a thread an expert 15; counts that all warps share 16; ranks by match.any 26).  Ranked, a call for 700 tokens with 3 of 256 experts takes 54.9 us for 53.4, for 85
// with 6 of 64 37.5 as before: by ballots over the bits of an expert's number, and no further than the run goes (every unrolled turn that is
// passed over is instructions to be fetched, 2 us in all).
constexpr int FL_GROUP_WARPS = 32;
// Words from one warp's counts to the next's: an odd number, so that an expert's counts lie in as many banks.
__host__ __device__ __forceinline__ int fl_group_stride(int experts, int n_warps) { return n_warps > 1 ? experts | 1 : experts; }

template <bool RANKED>
__global__ void __launch_bounds__(32 * FL_GROUP_WARPS)
fp4_group_kernel(const int* __restrict__ expert_of, int pairs, int experts, int bn, int* __restrict__ offsets, int* __restrict__ order,
                 int* __restrict__ slot, int* __restrict__ tile_expert, int* __restrict__ tile_row0, int* __restrict__ meta,
                 int* __restrict__ clear, int n_clear, int n_warps) {
    extern __shared__ int counts[];                                // [n_warps] rows of ``stride`` for the experts; two more: first row, first tile
    const int stride = fl_group_stride(experts, n_warps);
    int *row0 = counts + n_warps * stride, *tile0 = row0 + stride;
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run = (pairs + n_warps - 1) / n_warps;
    const int lo = min(pairs, warp * run), hi = warp < n_warps ? min(pairs, lo + run) : lo;
    for (int i = threadIdx.x; i < n_clear; i += blockDim.x) clear[i] = 0;
    for (int e = threadIdx.x; e < n_warps * stride; e += blockDim.x) counts[e] = 0;
    __syncthreads();
    int* mine = counts + min(warp, n_warps - 1) * stride;
    constexpr int AHEAD = 16;                                      // loads in flight, kept where they are a warp's whole run
    int es[AHEAD];
    auto load = [&](int p0) {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int p = p0 + 32 * q + lane, e = p < hi ? expert_of[p] : -1;
            es[q] = (unsigned)e < (unsigned)experts ? e : -1;
        }
    };
    for (int p0 = lo; p0 < hi; p0 += 32 * AHEAD) {
        load(p0);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q)
            if (es[q] >= 0) atomicAdd(mine + es[q], 1);
    }
    __syncthreads();
    for (int e = warp; e < experts; e += FL_GROUP_WARPS) {         // an expert's counts become the rows before each warp's
        const int n = lane < n_warps ? counts[lane * stride + e] : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int before = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += before;
        }
        if (lane < n_warps) counts[lane * stride + e] = sum - n;
        if (lane == 31) row0[e] = sum;
    }
    __syncthreads();
    if (warp == 0) {
        int row = 0, tile = 0;
        for (int e0 = 0; e0 < experts; e0 += 32) {
            const int e = e0 + lane, n = e < experts ? row0[e] : 0, t = (n + bn - 1) / bn;
            int r_sum = n, t_sum = t;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int r = __shfl_up_sync(0xffffffffu, r_sum, d), q = __shfl_up_sync(0xffffffffu, t_sum, d);
                if (lane >= d) { r_sum += r; t_sum += q; }
            }
            if (e < experts) {
                row0[e] = row + r_sum - n;
                tile0[e] = tile + t_sum - t;
                offsets[e + 1] = row + r_sum;                      // where an expert's rows end
            }
            row += __shfl_sync(0xffffffffu, r_sum, 31);
            tile += __shfl_sync(0xffffffffu, t_sum, 31);
        }
        if (lane == 0) { offsets[0] = 0; meta[0] = tile; }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x)
        for (int t = tile0[e], end = e + 1 < experts ? tile0[e + 1] : meta[0]; t < end; ++t) {
            tile_expert[t] = e;
            tile_row0[t] = row0[e] + (t - tile0[e]) * bn;
        }
    const int bits = 32 - __clz(experts - 1);
    for (int p0 = lo; p0 < hi; p0 += 32 * AHEAD) {
        if (run > 32 * AHEAD) load(p0);
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            if (RANKED && p0 + 32 * q >= hi) break;
            const int e = es[q], p = p0 + 32 * q + lane;
            int to = -1, i = 0;
            if (RANKED) {                                          // the first lane of each expert counts for all of them
                uint32_t same = __ballot_sync(0xffffffffu, e >= 0);          // the lanes of this one's expert, bit by bit of its number
                for (int b = 0; b < bits; ++b) {
                    const bool set = e >> b & 1;
                    const uint32_t all = __ballot_sync(0xffffffffu, set);
                    same &= set ? all : ~all;
                }
                const int first = e >= 0 ? __ffs(same) - 1 : lane;
                if (lane == first && e >= 0) {
                    i = mine[e];
                    mine[e] = i + __popc(same);
                }
                i = __shfl_sync(0xffffffffu, i, first) + __popc(same & ((1u << lane) - 1));
                __syncwarp();
            } else if (e >= 0) {
                i = atomicAdd(mine + e, 1);
            }
            if (e >= 0) {
                to = tile0[e] * bn + i;                            // an expert's tiles are neighbours
                order[row0[e] + i] = p;
            }
            if (p < hi) slot[p] = to;
        }
    }
}

constexpr int FL_SORTED_PAIRS = 256;      // (token, choice) pairs that a block sorts for itself
// The pairs (token, choice) by expert, in their order, for a block that has them to itself (pairs <= FL_SORTED_PAIRS <= its threads): tile
// t, up to ROWS neighbours of one expert tile_expert[t], is pair_of[tile_first[t]], ..., tile_rows[t] of them.  Pairs whose expert is
// none are left out.  All threads call it; the number of tiles.
template <int ROWS>
__device__ __forceinline__ int fl_sort_pairs(const int* __restrict__ expert_of, int pairs, int experts, int* pair_of, int* tile_first,
                                             int* tile_rows, int* tile_expert) {
    const int tid = threadIdx.x;
    int e = -1, first = 0, place = 0, same = 0;
    if (tid < pairs) {
        e = expert_of[tid];
        if ((unsigned)e >= (unsigned)experts) e = -1;
        tile_first[tid] = e;
    }
    __syncthreads();
    if (e >= 0)
#pragma unroll 8
        for (int q = 0; q < pairs; ++q) {
            const int f = tile_first[q];
            first += f >= 0 && f < e;
            place += f == e && q < tid;
            same += f == e;
        }
    if (tid < FL_SORTED_PAIRS) tile_rows[tid] = 0;
    __syncthreads();
    const bool starts = e >= 0 && place % ROWS == 0;
    const int rows = min(ROWS, same - place);
    if (e >= 0) pair_of[first + place] = tid;
    if (starts) tile_rows[first + place] = 1;
    __syncthreads();
    int before = 0;
    if (starts)
#pragma unroll 8
        for (int q = 0; q < first + place; ++q) before += tile_rows[q];
    const int tiles = __syncthreads_count(starts);
    if (starts) { tile_first[before] = first + place; tile_rows[before] = rows; tile_expert[before] = e; }
    __syncthreads();
    return tiles;
}


// Tiles of up to FL_SORTED_PAIRS pairs beside their rows into 4 bits, in one launch: every block sorts the pairs for itself, and takes
// k-blocks of rows by its warps (a lane eight numbers, four lanes a block).  One token's experts (64 of 2,048 x 1,408, 6 chosen) 17.2 us, by
// the two launches of many pairs 20.1; 16 tokens' 52.0 and 54.5.
template <typename T, int BN>
__global__ void __launch_bounds__(256)
fp4_place_kernel(const int* __restrict__ expert_of, int pairs, int experts, int top, const T* __restrict__ x, long long ldx, int K, int k_blocks,
                 uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, int* __restrict__ offsets, int* __restrict__ order,
                 int* __restrict__ tile_expert, int* __restrict__ tile_row0, int* __restrict__ meta, int* __restrict__ clear, int n_clear) {
    __shared__ int pair_of[FL_SORTED_PAIRS], first_of[FL_SORTED_PAIRS], rows_of[FL_SORTED_PAIRS], expert[FL_SORTED_PAIRS];
    static_assert(FL_SORTED_PAIRS == 256, "a thread a pair");
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = fl_sort_pairs<BN>(expert_of, pairs, experts, pair_of, first_of, rows_of, expert);
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < n_clear; i += 256) clear[i] = 0;
        for (int t = threadIdx.x; t < tiles; t += 256) {
            tile_expert[t] = expert[t];
            tile_row0[t] = first_of[t];
            // where an expert's rows end, which is all that the products ask of it
            if (t + 1 == tiles || expert[t + 1] != expert[t]) offsets[expert[t] + 1] = first_of[t] + rows_of[t];
        }
        if (threadIdx.x < pairs) order[threadIdx.x] = pair_of[threadIdx.x];
        if (threadIdx.x == 0) meta[0] = tiles;
    }
    const int sorted = tiles ? first_of[tiles - 1] + rows_of[tiles - 1] : 0;
    for (int task = blockIdx.x * 8 + warp; task < sorted * k_blocks; task += gridDim.x * 8) {
        const int i = task / k_blocks, kb = task - i * k_blocks, k = kb * F4_KB + lane * 8, pair = pair_of[i];
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = 0.f;
        if (k < K) f4_load8(x + (size_t)(pair / top) * ldx + k, v);
        int t = 0;                                                   // its tile
        for (int base = 0; base < tiles; base += 32) {
            const int q = base + lane;
            const uint32_t hit = __ballot_sync(0xffffffffu, q < tiles && first_of[q] <= i);
            t += __popc(hit);
        }
        --t;
        const int r = i - first_of[t];
        uint32_t most = f4_most(v);
        if (__any_sync(0xffffffffu, most >= F4_WILD)) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = f4_finite(v[q]);
            most = f4_most(v);
        }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int byte = f4_scale_byte(most);
        uint32_t word = (uint32_t)byte << (8 * ((lane & 15) >> 2));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if (k < K) *reinterpret_cast<uint32_t*>(codes + (size_t)(t * BN + r) * (K / 2) + k / 2) = f4_encode8(v, f4_inverse(byte));
        if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(scales + f4_scale_at(t * 128 + r, kb * 8 + (lane >> 4) * 4, k_blocks)) = word;
    }
}

// out[t] (+)= sum over the choices j, in their order, of weight[t, j] * y[t, j]; choices of no expert count nothing.
template <typename T>
__global__ void __launch_bounds__(256)
fp4_combine_kernel(const float* __restrict__ y, const int* __restrict__ expert_of, int experts, const float* __restrict__ weight,
                   T* __restrict__ out, long long ldo, int tokens, int top, int width, int add) {
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();
    const int per_row = width / 8;
    const long long pieces = (long long)tokens * per_row, step = (long long)gridDim.x * blockDim.x;
    for (long long p = (long long)blockIdx.x * blockDim.x + threadIdx.x; p < pieces; p += step) {
        const int t = (int)(p / per_row), c = (int)(p - (long long)t * per_row) * 8;
        float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int j0 = 0; j0 < top; j0 += 4) {                      // four choices in flight
            float v[4][8], w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int pair = t * top + j0 + q;
                w[q] = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[q][i] = 0.f;
                if (j0 + q < top && (unsigned)expert_of[pair] < (unsigned)experts) {
                    w[q] = weight[pair];
                    f4_load8(y + (size_t)pair * width + c, v[q]);
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] = fmaf(w[q], v[q][i], sum[i]);
        }
        T* dst = out + t * ldo + c;
        if (add) {
            float v[8];
            f4_load8(dst, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += v[i];
        }
        f4_store8(dst, sum);
    }
}

// Rows a tile, by how many an expert has on average.  Tiles of 16 where most experts fill one; tiles on SM pairs where an expert fills
// more; between them, where sums are long enough to hide the larger tile's epilogue, tiles of 64.  Microseconds, all measured with tiles of
// 16 / 64 / 256:  64 experts of 2,048 x 1,408, 6 a token: a mean of 6 rows 72 / 80 / 89, of 12 82 / 103 / 93, of 18 103 / 115 / 95, of 48
// 172 / 165 / 104;  256 of 7,168 x 512: 16 rows 521 / 653 / 564, 24 692 / 798 / 606;  16 of 4,096 x 6,400: 4 rows 121 / 122 / 155, 12
// 142 / 131 / 158, 32 263 / 152 / 161, 48 353 / 176 / 167;  8 of 4,096 x 14,336: 12 rows 154 / 139 / 176, 32 304 / 161 / 178, 48 374 /
// 181 / 179.  (Of 32: 5 to 10 % less than these where a mean of 12 to 20 meets sums of some 3,000, nothing elsewhere; of 128: never least.)
static int fl_list_rows(int tokens, int top, int experts, int K, int inter) {
    const long long mean = (long long)tokens * top / experts;
    if (tokens <= 16 || mean <= 8) return 16;
    if (K >= 4096 && inter >= 4096) return mean <= 40 ? 64 : 256;
    return mean <= 16 ? 16 : 256;
}
struct FlExperts {
    int bn, tiles, blocks;                 // rows a tile, tiles at most, blocks of a product
    size_t counters, offsets, order, slot, tile_expert, tile_row0, meta, x, xs, z, zs, y, pieces, all;
    FlExperts(int tokens, int top, int experts, int K, int inter) {
        const int pairs = tokens * top;
        bn = fl_list_rows(tokens, top, experts, K, inter);
        tiles = pairs / bn + std::min(experts, pairs);
        blocks = ssb_sm_count();
        const size_t rows = (size_t)tiles * bn, chunks = (size_t)tiles * (bn > 128 ? 2 : 1) * F4_CHUNK;
        size_t at = 0;
        auto take = [&](size_t bytes) { const size_t was = at; at += fl_round(bytes); return was; };
        counters = take(2 * FL_COUNTERS * 4);
        offsets = take((size_t)(experts + 1) * 4);
        order = take((size_t)pairs * 4);
        slot = take((size_t)pairs * 4);
        tile_expert = take((size_t)tiles * 4);
        tile_row0 = take((size_t)tiles * 4);
        meta = take(4);
        x = take(rows * (K / 2));
        xs = take(chunks * f4_k_blocks(K));
        z = take(rows * (inter / 2));
        zs = take(chunks * f4_k_blocks(inter));
        y = take((size_t)pairs * K * 4);
        pieces = bn < 256 ? take((size_t)blocks * 2 * bn * FL_BM * 4) : at;
        all = at;
    }
};
SSB_API long long ssb_fp4_experts_scratch(int tokens, int top, int experts, int K, int inter) {
    if (tokens <= 0 || top <= 0 || experts <= 0 || K <= 0 || inter <= 0) return 0;
    return (long long)FlExperts(tokens, top, experts, K, inter).all;
}

template <int MODE>
static int fl_listed(const void* x, const void* xs, const void* w, const void* ws, const FlOut& o, const FlTiles& list, const FlExperts& at,
                     int experts, int K, int* counters, float* pieces, int* error_word, cudaStream_t stream) {
    const int k_blocks = f4_k_blocks(K), n_tiles = (o.N + FL_BM - 1) / FL_BM;
    CUtensorMap mw, mws, mx, mxs;
    int rc = fl_map(&mx, x, (long long)at.tiles * at.bn, K / 2, std::min(at.bn, FL_BM));
    if (!rc) rc = fl_map(&mw, w, (long long)experts * o.N, K / 2, FL_BM);
    if (!rc) rc = fl_scale_map(&mxs, xs, (long long)at.tiles * (at.bn > 128 ? 2 : 1) * k_blocks);
    if (!rc) rc = fl_scale_map(&mws, ws, (long long)experts * n_tiles * k_blocks);
    if (rc) return rc;
    if (at.bn == 16)
        return fl_stream<16, 5, MODE, true>(mw, mws, mx, mxs, o, list, 0, n_tiles, at.blocks, K, true, counters, pieces, error_word, stream);
    if (at.bn == 64)
        return fl_stream<64, 8, MODE, true>(mw, mws, mx, mxs, o, list, 0, n_tiles, at.blocks, K, true, counters, pieces, error_word, stream);
    return fl_pair<MODE, true>(mx, mw, xs, ws, 2 * at.tiles, o, list, at.tiles, (o.N + 255) / 256, K, error_word, stream);
}

// out[t] (+)= sum_j weight[t, j] E(x_t) of expert expert_of[t, j]; w1: [experts][N1][K], w2: [experts][K][inter].
SSB_API int ssb_fp4_experts(const void* x, long long ldx, int dtype, const int* expert_of, const float* weight, const void* w1, const void* ws1,
                            const void* w2, const void* ws2, void* out, long long ldo, int out_dtype, int tokens, int top, int experts, int K,
                            int inter, int gated, int kind, float limit, int add, void* scratch, int* error_word, cudaStream_t stream) {
    if (tokens < 0 || top <= 0 || experts <= 0 || experts > 4096 || K <= 0 || K % F4_BLOCK || inter <= 0 || inter % F4_BLOCK || kind < 0 || kind > 2 ||
        !scratch || !error_word || (long long)tokens * top > (1 << 24)) return SSB_ERR_BAD_SIZE;          // 4,096: of the grouping's shared memory
    if (((uintptr_t)x | (uintptr_t)w1 | (uintptr_t)ws1 | (uintptr_t)w2 | (uintptr_t)ws2 | (uintptr_t)out | (uintptr_t)scratch) & 15) return SSB_ERR_BAD_SIZE;
    if ((dtype != SSB_F32 && dtype != SSB_BF16) || (out_dtype != SSB_F32 && out_dtype != SSB_BF16) || (add && out_dtype != SSB_F32)) return SSB_ERR_BAD_DTYPE;
    if (tokens == 0) return 0;
    const FlExperts at(tokens, top, experts, K, inter);
    char* base = (char*)scratch;
    const int pairs = tokens * top, N1 = gated ? 2 * inter : inter;
    float* y = (float*)(base + at.y);
    int rc;
    if (at.blocks > FL_COUNTERS) return SSB_ERR_UNSUPPORTED;
    auto ints = [&](size_t o) { return (int*)(base + o); };
    if (pairs <= FL_SORTED_PAIRS && at.bn == 16) {
        const int k_blocks = f4_k_blocks(K);
        const dim3 grid((unsigned)std::min(ssb_sm_count(), (pairs * k_blocks + 7) / 8));
        auto place = [&](auto kernel, auto* numbers) {
            return ssb_launch(kernel, grid, dim3(256), 0, stream, true, expert_of, pairs, experts, top, numbers, ldx, K, k_blocks,
                              (uint8_t*)(base + at.x), (uint8_t*)(base + at.xs), ints(at.offsets), ints(at.order), ints(at.tile_expert),
                              ints(at.tile_row0), ints(at.meta), ints(at.counters), 2 * FL_COUNTERS);
        };
        rc = dtype == SSB_BF16 ? place(fp4_place_kernel<bf16, 16>, (const bf16*)x) : place(fp4_place_kernel<float, 16>, (const float*)x);
    } else {
        // as many warps as shared memory has room for their counts
        const int n_warps = std::max(1, std::min(FL_GROUP_WARPS, 48 * 1024 / (4 * (experts | 1)) - 2));
        rc = ssb_launch(at.bn < 256 ? fp4_group_kernel<true> : fp4_group_kernel<false>, dim3(1), dim3(32 * FL_GROUP_WARPS), (size_t)fl_group_stride(experts, n_warps) * (n_warps + 2) * 4, stream, true, expert_of, pairs,
                        experts, at.bn, ints(at.offsets), ints(at.order), ints(at.slot), ints(at.tile_expert), ints(at.tile_row0), ints(at.meta),
                        ints(at.counters), 2 * FL_COUNTERS, n_warps);
        if (!rc) rc = ssb_fp4_quantize_pairs(x, ldx, dtype, base + at.x, base + at.xs, tokens, top, K, ints(at.slot), at.bn, stream);
    }
    if (rc) return rc;
    FlTiles list{ints(at.offsets), ints(at.tile_expert), ints(at.tile_row0), ints(at.meta), 0};
    float* pieces = (float*)(base + at.pieces);
    const FlOut first{base + at.z, (uint8_t*)(base + at.zs), nullptr, nullptr, inter / 2, 0, 0, tokens, N1, kind, limit, f4_k_blocks(inter)};
    rc = gated ? fl_listed<FL_GATED>(base + at.x, base + at.xs, w1, ws1, first, list, at, experts, K, ints(at.counters), pieces, error_word, stream)
               : fl_listed<FL_ACT>(base + at.x, base + at.xs, w1, ws1, first, list, at, experts, K, ints(at.counters), pieces, error_word, stream);
    if (rc) return rc;
    list.ready = 1;                                                // the first product waited for it
    const FlOut second{y, nullptr, ints(at.order), nullptr, K, 1, 0, tokens, K, 0, 0.f, 0};
    rc = fl_listed<FL_STORE>(base + at.z, base + at.zs, w2, ws2, second, list, at, experts, inter, ints(at.counters) + FL_COUNTERS, pieces, error_word, stream);
    if (rc) return rc;
    const dim3 grid((unsigned)std::min<long long>(((long long)tokens * (K / 8) + 255) / 256, 8 * ssb_sm_count()));
    if (out_dtype == SSB_BF16)
        return ssb_launch(fp4_combine_kernel<bf16>, grid, dim3(256), 0, stream, true, (const float*)y, expert_of, experts, weight, (bf16*)out, ldo, tokens, top, K, add);
    return ssb_launch(fp4_combine_kernel<float>, grid, dim3(256), 0, stream, true, (const float*)y, expert_of, experts, weight, (float*)out, ldo, tokens, top, K, add);
}

SSB_PACKED(ssb_fp4_linear)
SSB_PACKED(ssb_fp4_inner)
SSB_PACKED(ssb_fp4_experts)
