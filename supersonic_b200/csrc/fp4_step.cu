// Products of a step's rows (up to 32, in 4 bits) in microscaled 4-bit floats on tcgen05 (the format: fp4_codes.cuh).  As in the streaming
// kernel the weights are on the M side, 128 of them a tile; here a tile's k-blocks are shared by the blocks of a cluster, which put their
// sums into the first one's shared memory, and it adds them up in the order of k: nothing goes through memory, and nothing counts there.
// 8 x 4,096 x 14,336 (rows in 4 bits) 8.1 us from memory, 3.8 TB/s, 7.5 where the weights are in L2; 16 x 2,048 x 8,192 5.5 and 5.0;
// 16 x 16,384 x 2,048 4.6 and 3.9; by the streaming kernel, with pieces in memory and counters, 12.3, 9.2 and 8.5.  A launch's start, the
// first stages and the sums' meeting are some 4 us of each.
//
// Rows that come as numbers are quantised by a launch in front, which the first weights come beside: 10.7 us from memory and 8.9 from L2;
// 7.7 and 7.2; 7.8 and 6.0.  By warps of every block, a k-block at a time into its stage, it took longer: 8 x 4,096 x 14,336 15.2 us for
// 11.2 from memory, 16 x 2,048 x 8,192 18.3 for 8.2.
#include "fp4_codes.cuh"
#include "fp4_few.cuh"
#include "fp4_step.cuh"
#include "fp4_tc.cuh"
#include "per_device.h"
#include <algorithm>

typedef __nv_bfloat16 bf16;

constexpr int FS_STAGES = 5;
constexpr int FS_MOST_SUMS = 96;          // rows of sums that a cluster's first block gets: three others, 32 each

template <int BN> constexpr int fs_columns() { return fl_power(BN + 16 * FS_STAGES); }
template <int BN> constexpr int fs_stage() { return FL_BM * FL_ROW + BN * FL_ROW + 2 * (int)FL_CHUNK; }
template <int BN> constexpr size_t fs_smem(int sums) {
    return (size_t)FS_STAGES * fs_stage<BN>() + FL_INNER_ROWS * FL_INNER_LD * 4 + (size_t)sums * FL_BM * 4 + (2 * FS_STAGES + 1) * 8 + 24 + 1024;
}

template <int BN, int MODE>
__global__ void __launch_bounds__(FL_THREADS, 1)
fp4_step_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_x,
                const __grid_constant__ CUtensorMap map_xs, const FwArgs a, int parts, int* __restrict__ error_word) {
    constexpr int STAGES = FS_STAGES;
    constexpr uint32_t W_BYTES = FL_BM * FL_ROW, X_BYTES = BN * FL_ROW, STAGE_BYTES = fs_stage<BN>();
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* inner = (float*)(smem + STAGES * STAGE_BYTES);           // [FL_INNER_ROWS][FL_INNER_LD]
    float* sums = inner + FL_INNER_ROWS * FL_INNER_LD;              // [parts - 1][M][FL_BM]: the other blocks'
    uint64_t* bars = (uint64_t*)(sums + (size_t)(parts - 1) * a.M * FL_BM);          // full[STAGES], empty[STAGES], acc_full
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * STAGES + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);      // [0]: a role gave up; [1]: stays zero
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES), acc_full = smem_u32(bars + 2 * STAGES);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        mbar_init(acc_full, 1);
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(fs_columns<BN>()) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync_all();                                             // the first block is there when the others write to it
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    bool good = false;                                              // (the epilogue's four warps) the sums are there
    const int part = (int)(blockIdx.x % parts), n = (int)(blockIdx.x / parts);
    const int kb0 = a.k_blocks * part / parts, all = a.k_blocks * (part + 1) / parts - kb0;          // this block's k-blocks

    if (warp == 0) {
        if (lane == 0) {
            const int ahead = min(STAGES, all);
            auto weights = [&](int s, int kb) {
                const uint32_t dst = smem_u32(smem + s * STAGE_BYTES);
                mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                tma_load_2d(dst, &map_w, full0 + 8 * s, kb * FL_ROW, n * FL_BM);
                tma_load_2d(dst + W_BYTES + X_BYTES, &map_ws, full0 + 8 * s, 0, n * a.k_blocks + kb);
            };
            for (int s = 0; s < ahead; ++s) weights(s, kb0 + s);    // nobody's output: before what is in front of this launch has ended
            ssb_pdl_wait();
            ssb_pdl_launch_dependents();
            int c = 0;
            for (; c < all; ++c) {
                const int s = c % STAGES;
                if (c >= ahead) {
                    if (!mbar_wait(empty0 + 8 * s, ((c / STAGES) & 1) ^ 1, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); break;
                    }
                    weights(s, kb0 + c);
                }
                const uint32_t x_dst = smem_u32(smem + s * STAGE_BYTES) + W_BYTES;
                tma_load_2d(x_dst, &map_x, full0 + 8 * s, (kb0 + c) * FL_ROW, 0);
                tma_load_2d(x_dst + X_BYTES + FL_CHUNK, &map_xs, full0 + 8 * s, 0, kb0 + c);
            }
            if (*abort_flag)                                        // let copies that were issued land before the block ends
                for (int i = max(0, c - STAGES); i < c; ++i)
                    mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, abort_flag + 1);
        }
    } else if (warp == 1) {
        ssb_pdl_wait();                                             // what follows spins on barriers
        constexpr uint32_t idesc0 = fl_idesc(FL_BM, BN, 0), idesc1 = fl_idesc(FL_BM, BN, 1);
        const bool issues = fl_elect();
        const uint64_t w_desc = smem_desc(smem_u32(smem)), x_desc = smem_desc(smem_u32(smem) + W_BYTES);
        bool ok = true;
        int s = 0;
        uint32_t lap = 0;
        for (int c = 0; c < all; ++c) {
            ok = mbar_wait(full0 + 8 * s, lap, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break; }
            tc_fence_after();
            // a stage has columns of its own for its scales, so what reads them is done when they are written again
            const uint32_t s_addr = smem_u32(smem) + s * STAGE_BYTES + W_BYTES + X_BYTES, scales = tmem + BN + 16 * s;
            const uint32_t step = s * (STAGE_BYTES >> 4);
            if (issues) {
                fl_copy_scales(scales, s_addr);
                fl_copy_scales(scales + 4, s_addr + 512);
                fl_copy_scales(scales + 8, s_addr + FL_CHUNK);
                fl_copy_scales(scales + 12, s_addr + FL_CHUNK + 512);
                fl_mma_x4(tmem, w_desc + step, x_desc + step, idesc0, idesc1, scales, scales + 8, scales + 4, scales + 12, c > 0 ? 1u : 0u);
                tc_commit(empty0 + 8 * s);
            }
            __syncwarp();
            if (++s == STAGES) { s = 0; lap ^= 1; }
        }
        if (ok && issues) tc_commit(acc_full);
    } else {
        ssb_pdl_wait();
        const int in_tile = (warp & 3) * 32 + lane;
        if (fl_any_of_four(!mbar_wait(acc_full, 0, abort_flag))) {
            if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
        } else {
            good = true;
        }
        if (good && part > 0) {
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const uint32_t to = cluster_map(smem_u32(sums), 0) + (uint32_t)(((part - 1) * a.M * FL_BM + in_tile) * 4);
#pragma unroll 1
            for (int c0 = 0; c0 < a.M; c0 += 16) {
                float sum[16];
                fl_ld16(acc + c0, sum);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c0 + e < a.M)
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + (uint32_t)((c0 + e) * FL_BM * 4)), "f"(sum[e]) : "memory");
            }
            tc_fence_before();
        }
    }
    __syncwarp();
    if (parts > 1) cluster_sync_all();
    if (part == 0 && good) {
        tc_fence_after();
        const int quarter = warp & 3, in_tile = quarter * 32 + lane, who = threadIdx.x - 64, col = n * FL_BM + in_tile;
        const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
        for (int c0 = 0; c0 < a.M; c0 += 16) {
            const int live = col < a.N ? a.M - c0 : 0;
            const size_t at = (size_t)c0 * a.ldo + col;
            float was[16], sum[16];
            if (MODE == FL_STORE && a.add)
#pragma unroll
                for (int e = 0; e < 16; ++e) was[e] = e < live ? ((const float*)a.out)[at + (size_t)e * a.ldo] : 0.f;
            __syncwarp();
            fl_ld16(acc + c0, sum);
            for (int p = 1; p < parts; ++p)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (c0 + e < a.M) sum[e] += sums[((p - 1) * a.M + c0 + e) * FL_BM + in_tile];
            if (MODE == FL_STORE) {
                if (a.is_f32) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (e < live) ((float*)a.out)[at + (size_t)e * a.ldo] = a.add ? sum[e] + was[e] : sum[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (e < live) ((bf16*)a.out)[at + (size_t)e * a.ldo] = __float2bfloat16_rn(sum[e]);
                }
            } else {
                fl_inner_tile<MODE>(sum, inner, quarter, lane, who, c0, 0, 0, a.M, n, (a.N + FL_BM - 1) / FL_BM, a.N, a.kind, a.limit, a.row_scale,
                                    (uint8_t*)a.out, a.ldo, a.out_scales, a.inner_blocks);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(fs_columns<BN>()) : "memory");
    }
}

// Blocks that share a tile, or 0: the product is not for this kernel.  Four, two or one, by what is left of the k-blocks (0.37 us each) and
// what the sums' meeting costs, which grows with the rows.  One, two, four blocks, with the rows' launch before them: 8 x 2,048 x 2,048 6.0, 5.7,
// 5.4 us, 32 rows 6.9, 7.1, 7.5; 8 x 4,096 x 4,096 9.0, 7.5, 7.2, 32 rows 9.8, 8.9, 9.6; 8 x 2,048 x 8,192 13.7, 9.8, 7.9, eight blocks 11.3;
// 16 x 4,096 x 14,336 21.3, 14.1, 11.7.
int fs_parts(int M, int N, int K) {
    const int sms = ssb_sm_count(), tiles = (N + FL_BM - 1) / FL_BM, k_blocks = f4_k_blocks(K);
    if (M > 32 || tiles > sms) return 0;
    const double meeting[3] = {0, 1.0 + 0.02 * M, 1.3 + 0.06 * M};
    int best = 1;
    double least = 1e30;
    for (int i = 0, p = 1; i < 3 && tiles * p <= sms && p <= k_blocks; ++i, p *= 2) {
        const double cost = 0.37 * ((k_blocks + p - 1) / p) + meeting[i];
        if (cost < least) { least = cost; best = p; }
    }
    return best;
}

// (``early`` is no field of FwArgs: with one int more there, the kernels that store took 91 registers for 145 and 0.3 to 0.8 us longer for their
// ends, 32 x 2,048 x 8,192 7.2 us for 6.3.)
template <int BN, int MODE>
static int fs_launch(const CUtensorMap& mw, const CUtensorMap& mws, const CUtensorMap& mx, const CUtensorMap& mxs, const FwArgs& a, int parts,
                     bool early, int* error_word, cudaStream_t stream) {
    static_assert(fs_smem<BN>(FS_MOST_SUMS) <= 227 * 1024, "");
    auto kernel = fp4_step_kernel<BN, MODE>;
    static SsbPerDevice<bool> set;
    bool* configured = set.here();
    if (!configured) return SSB_ERR_UNSUPPORTED;
    if (!*configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fs_smem<BN>(FS_MOST_SUMS));
        if (e != cudaSuccess) return (int)e;
        *configured = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.N + FL_BM - 1) / FL_BM * parts);
    cfg.blockDim = dim3(FL_THREADS);
    cfg.dynamicSmemBytes = fs_smem<BN>((parts - 1) * a.M);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = early ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, mw, mws, mx, mxs, a, parts, error_word);
}

template <int BN>
static int fs_mode(const CUtensorMap& mw, const CUtensorMap& mws, const CUtensorMap& mx, const CUtensorMap& mxs, const FwArgs& a, int mode,
                   int parts, bool early, int* error_word, cudaStream_t stream) {
    return mode == FL_STORE ? fs_launch<BN, FL_STORE>(mw, mws, mx, mxs, a, parts, early, error_word, stream)
           : mode == FL_GATED ? fs_launch<BN, FL_GATED>(mw, mws, mx, mxs, a, parts, early, error_word, stream)
                              : fs_launch<BN, FL_ACT>(mw, mws, mx, mxs, a, parts, early, error_word, stream);
}

int fs_product(FwArgs a, int mode, int parts, bool early, int* error_word, cudaStream_t stream) {
    a.k_blocks = f4_k_blocks(a.K);
    const int bn = a.M <= 16 ? 16 : 32;
    CUtensorMap mw, mws, mx, mxs;
    int rc = fl_map(&mw, a.w, a.N, a.K / 2, FL_BM);
    if (!rc) rc = fl_scale_map(&mws, a.ws, (long long)((a.N + 127) / 128) * a.k_blocks);
    if (!rc) rc = fl_map(&mx, a.x, a.M, a.K / 2, bn);
    if (!rc) rc = fl_scale_map(&mxs, a.xs, a.k_blocks);
    if (rc) return rc;
    return bn == 16 ? fs_mode<16>(mw, mws, mx, mxs, a, mode, parts, early, error_word, stream) : fs_mode<32>(mw, mws, mx, mxs, a, mode, parts, early, error_word, stream);
}
