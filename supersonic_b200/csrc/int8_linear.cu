// Matrix products in 8-bit integers: out[m, n] (+)= (sum_k xc[m, k] wc[n, k]) * sx[m] * sw[n], with the rows of x quantised as they
// come (sx = max |x_row| * (1/127), xc = rint(x / sx)) and weights that lie in codes with a scale per output channel.  The sums are
// exact: 32-bit integers up to k = 132,096 (127 * 128 * k < 2^31, of weights down to -128), which is checked.  So a result has the same bits whatever
// kernel, cut of k or batch it was computed in.
//
// Three launches' worth of code, two launches a call: the rows' codes; then one of two products on the fifth-generation tensor
// cores (tcgen05 kind::i8, operands by TMA with the 128-byte swizzle, 32-bit sums in tensor memory):
//  * where the weights' bytes or the number of tiles is what bounds it: weights on the M side (128 of them a tile), rows of x on the
//    N side, and the k-blocks of all tiles dealt out over the SMs, in equal parts of tiles or wherever a tile ends;
//  * many rows: tiles of 256 x 256 on pairs of SMs (cta_group::2).
//
// The reference's 8-bit lane of this architecture multiplies int8 weights by activations of the model's type
// (crates/runner/src/llama31_engine.rs:289-430).
#include "int8_codes.cuh"
#include "packed_call.cuh"
#include "tc_helpers.cuh"
#include "tc_rows.cuh"
#include <algorithm>

typedef __nv_bfloat16 bf16;

constexpr int IL_MOST_K = 132096;

// ---- rows to codes ------------------------------------------------------------------------------------------------
// rint(x / s), the division correctly rounded (as in i8_encode8).
__device__ __forceinline__ int il_code(float x, float s, float inverse) {
    const float y = x * inverse;
    float c = rintf(y);
    if (fabsf(fabsf(y - c) - 0.5f) < 1e-4f) c = rintf(__fdiv_rn(x, s));
    return (int)c;
}
__device__ __forceinline__ uint32_t il_block_max(uint32_t m, uint32_t* warp_max) {
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < warps ? warp_max[lane] : 0u);
}

// The launch's first block zeroes the product's counters: one for each of its blocks, a hundred or so.
__device__ __forceinline__ void il_clear(int* clear, int n_clear) {
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < n_clear; i += blockDim.x) clear[i] = 0;
}

// A block a row, 8 numbers a thread and turn, all of them in registers between the row's maximum and its codes (NV turns).
// ``clear``: words that the product counts in, zeroed here.  8,192 x 4,096 in bfloat16: 24 us, 4.2 TB/s.
template <typename T, int NV>
__global__ void __launch_bounds__(1024)
int8_quantize_kernel(const T* __restrict__ x, int ldx, int8_t* __restrict__ codes, int ldc, float* __restrict__ scale, int K,
                     int* __restrict__ clear, int n_clear) {
    __shared__ uint32_t warp_max[2][32];
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();                               // what was written before this launch is there: weights may be read ahead
    const int row = blockIdx.x;
    il_clear(clear, n_clear);
    float v[NV][8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int k = 8 * (threadIdx.x + j * blockDim.x);
        if (k < K) i8_load8(x + (size_t)row * ldx + k, v[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (8 * (int)(threadIdx.x + j * blockDim.x) < K) top = max(top, i8_magnitude(v[j]));
    top = il_block_max(top, warp_max[0]);
    if (top >= I8_WILD) {                                      // the same for the whole block
        top = 0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (8 * (int)(threadIdx.x + j * blockDim.x) < K) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[j][e] = i8_finite(v[j][e]);
                top = max(top, i8_magnitude(v[j]));
            }
        top = il_block_max(top, warp_max[1]);
    }
    const float s = fmaxf(__fmul_rn(__uint_as_float(top), 1.f / 127.f), I8_LEAST_SCALE), inverse = 1.f / s;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int k = 8 * (threadIdx.x + j * blockDim.x);
        if (k < K) *reinterpret_cast<uint2*>(codes + (size_t)row * ldc + k) = i8_encode8(v[j], s, inverse);
    }
    if (threadIdx.x == 0) scale[row] = s;
}

// Rows of any alignment and length: read twice.
template <typename T>
__global__ void __launch_bounds__(256)
int8_quantize_any_kernel(const T* __restrict__ x, int ldx, int8_t* __restrict__ codes, int ldc, float* __restrict__ scale, int K,
                         int* __restrict__ clear, int n_clear) {
    __shared__ uint32_t warp_max[2][32];
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();                               // what was written before this launch is there: weights may be read ahead
    const T* src = x + (size_t)blockIdx.x * ldx;
    il_clear(clear, n_clear);
    uint32_t top = 0;
    for (int k = threadIdx.x; k < K; k += 256) top = max(top, __float_as_uint(fabsf(i8_finite(ssb_to_float(src[k])))));
    const float s = fmaxf(__fmul_rn(__uint_as_float(il_block_max(top, warp_max[0])), 1.f / 127.f), I8_LEAST_SCALE), inverse = 1.f / s;
    for (int k = threadIdx.x; k < K; k += 256)
        codes[(size_t)blockIdx.x * ldc + k] = (int8_t)il_code(i8_finite(ssb_to_float(src[k])), s, inverse);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
}

template <typename T>
static int quantize_rows(const T* x, int ldx, int8_t* codes, int ldc, float* scale, int rows, int K, int* clear, int n_clear,
                         cudaStream_t stream) {
    const bool whole = K % 8 == 0 && ldc % 8 == 0 && ((uintptr_t)codes & 7) == 0 && ((size_t)ldx * sizeof(T)) % 16 == 0 &&
                       ((uintptr_t)x & 15) == 0 && K <= 8 * 4 * 1024;
    if (!whole) {
        return ssb_launch(int8_quantize_any_kernel<T>, dim3(rows), dim3(256), 0, stream, true, x, ldx, codes, ldc, scale, K, clear, n_clear);
    }
    const int vectors = K / 8;
    // few rows: as many threads as there are vectors, for the shortest way through; many: two vectors a thread (x 2,048 x 4,096 with
    // the product, us so and with as many threads as vectors: 64 rows 13.6 and 13.4, 4,096 rows 43.2 and 44.1)
    const int threads = std::min(1024, std::max(32, ((rows > 256 ? (vectors + 1) / 2 : vectors) + 31) / 32 * 32));
    const int nv = (vectors + threads - 1) / threads;
    if (nv == 1) return ssb_launch(int8_quantize_kernel<T, 1>, dim3(rows), dim3(threads), 0, stream, true, x, ldx, codes, ldc, scale, K, clear, n_clear);
    if (nv == 2) return ssb_launch(int8_quantize_kernel<T, 2>, dim3(rows), dim3(threads), 0, stream, true, x, ldx, codes, ldc, scale, K, clear, n_clear);
    return ssb_launch(int8_quantize_kernel<T, 4>, dim3(rows), dim3(threads), 0, stream, true, x, ldx, codes, ldc, scale, K, clear, n_clear);
}

SSB_API int ssb_int8_quantize_rows(const void* x, int ldx, int dtype, void* codes, int ldc, float* scale, int rows, int K,
                                   cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (K <= 0) return SSB_ERR_BAD_SIZE;
    if (dtype == SSB_BF16) return quantize_rows((const bf16*)x, ldx, (int8_t*)codes, ldc, scale, rows, K, nullptr, 0, stream);
    if (dtype == SSB_F32) return quantize_rows((const float*)x, ldx, (int8_t*)codes, ldc, scale, rows, K, nullptr, 0, stream);
    return SSB_ERR_BAD_DTYPE;
}

// ---- the products -----------------------------------------------------------------------------------------------------
constexpr int IL_BK = 128;                // codes a k-block: one swizzle row of 128 bytes, four instructions of 32
constexpr int IL_BM = 128;
constexpr int IL_THREADS = 192;           // warp 0: TMA, warp 1: MMA + tensor memory, warps 2-5: epilogue

// D 32-bit integer, A and B signed 8-bit, both K-major
__host__ __device__ constexpr uint32_t il_idesc(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void il_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// A k-block: four instructions of 32 codes (32 bytes along the swizzled row: 2 descriptor units).
__device__ __forceinline__ void il_mma_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 a1, a2, a3, b1, b2, b3;\n"
                 "setp.ne.b32 p, %4, 0;\nsetp.eq.b32 q, %5, 0;\n"
                 "add.u64 a1, %1, 2;\nadd.u64 a2, %1, 4;\nadd.u64 a3, %1, 6;\n"
                 "add.u64 b1, %2, 2;\nadd.u64 b2, %2, 4;\nadd.u64 b3, %2, 6;\n"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], a1, b1, %3, {%5, %5, %5, %5}, q;\n"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], a2, b2, %3, {%5, %5, %5, %5}, q;\n"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], a3, b3, %3, {%5, %5, %5, %5}, q;\n}"
                 ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
__device__ __forceinline__ void il_mma_pair_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 a1, a2, a3, b1, b2, b3;\n"
                 "setp.ne.b32 p, %4, 0;\nsetp.eq.b32 q, %5, 0;\n"
                 "add.u64 a1, %1, 2;\nadd.u64 a2, %1, 4;\nadd.u64 a3, %1, 6;\n"
                 "add.u64 b1, %2, 2;\nadd.u64 b2, %2, 4;\nadd.u64 b3, %2, 6;\n"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], a1, b1, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, q;\n"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], a2, b2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, q;\n"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], a3, b3, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, q;\n}"
                 ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
template <int N> __device__ __forceinline__ void il_ld16(uint32_t taddr, int (&r)[N], int i) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[i + 0]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7]),
                   "=r"(r[i + 8]), "=r"(r[i + 9]), "=r"(r[i + 10]), "=r"(r[i + 11]), "=r"(r[i + 12]), "=r"(r[i + 13]), "=r"(r[i + 14]), "=r"(r[i + 15])
                 : "r"(taddr) : "memory");
}
// N columns of the lane's row of tensor memory.
template <int N> __device__ __forceinline__ void il_ld(uint32_t taddr, int (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 16) il_ld16(taddr + i, r, i);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float il_result(int sum, float sx, float sw) { return __fmul_rn(__fmul_rn((float)sum, sx), sw); }

// Whether any thread of the four epilogue warps says so; all of them meet here (barrier 1).
__device__ __forceinline__ bool il_any_of_four(bool mine) {
    uint32_t any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.or.pred q, 1, 128, p;\nselp.b32 %0, 1, 0, q;\n}"
                 : "=r"(any) : "r"((uint32_t)mine) : "memory");
    return any != 0;
}

struct IlOut {
    void* out;
    const float* sx;               // [M]
    const float* sw;               // [N]
    int ldo, is_f32, add, M, N;
};

// The rows of x on the N side, BN a tile.  The launch's work is tiles x k-blocks, dealt out evenly: block c takes units
// U c / G .. U (c + 1) / G - 1, tiles in order, a tile's k-blocks in order, so that every SM streams the same bytes whatever the
// sizes.  A tile that lies in one block's range is finished there; of any other the blocks write their sums to memory (at most two
// such pieces a block) and the one whose piece arrives last adds them up.  8 rows x 4,096 x 14,336: 17.1 us with the rows' codes, 3.5
// TB/s; x 28,672 x 4,096: 26 us, 4.5 TB/s; bound by what comes before the first and after the last product, in between by memory.
struct IlRange {
    long long units, begin, end;
    int k_blocks, blocks;
    __device__ IlRange(int tiles, int k_blocks_, int c, int blocks_) : units((long long)tiles * k_blocks_), k_blocks(k_blocks_), blocks(blocks_) {
        begin = units * c / blocks;
        end = units * (c + 1) / blocks;
    }
    __device__ int owner(long long unit) const { return (int)(((unit + 1) * blocks - 1) / units); }       // the block that takes it
};

template <int BN> constexpr int il_columns() { return 2 * BN < 32 ? 32 : 2 * BN; }
template <int BN, int STAGES> constexpr size_t il_smem() {
    return (size_t)STAGES * (IL_BM + BN) * IL_BK + 4 * BN * 4 + (2 * STAGES + 4) * 8 + 32 + 1024;
}

template <int BN, int STAGES>
__global__ void __launch_bounds__(IL_THREADS, 1)
int8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const IlOut o, int m_tiles,
                   int tiles, int k_blocks, int* __restrict__ arrived, int* __restrict__ pieces, int* __restrict__ error_word) {
    constexpr uint32_t W_BYTES = IL_BM * IL_BK, X_BYTES = BN * IL_BK, STAGE_BYTES = W_BYTES + X_BYTES;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* row_scales = (float*)(smem + STAGES * STAGE_BYTES);      // of a tile's rows, an epilogue warp's own
    uint64_t* bars = (uint64_t*)(row_scales + 4 * BN);              // full[STAGES], empty[STAGES], acc_full[2], acc_empty[2]
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * STAGES + 4);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);     // [0]: a role gave up; [1]: stays zero
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
    const uint32_t acc_full0 = smem_u32(bars + 2 * STAGES), acc_empty0 = smem_u32(bars + 2 * STAGES + 2);
    const IlRange range(tiles, k_blocks, blockIdx.x, gridDim.x);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(acc_full0 + 8 * i, 1); mbar_init(acc_empty0 + 8 * i, 4); }
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(il_columns<BN>()) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            // the first stages' weights are nobody's output: they come while the rows are still being quantised
            const int all = (int)(range.end - range.begin), ahead = min(STAGES, all);
            // a unit's place: channels of W, rows of x, k; the next one's
            const int tile0 = (int)(range.begin / k_blocks), m_first = tile0 % m_tiles, n_first = tile0 / m_tiles;
            const int kb_first = (int)(range.begin - (long long)tile0 * k_blocks);
            auto next = [&](int& kb, int& m, int& n) {
                if (++kb == k_blocks) { kb = 0; if (++m == m_tiles) { m = 0; ++n; } }
            };
            int kb = kb_first, m = m_first, n = n_first;
            for (int s = 0; s < ahead; ++s, next(kb, m, n)) {
                mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                tma_load_2d(smem_u32(smem + s * STAGE_BYTES), &map_w, full0 + 8 * s, kb * IL_BK, n * IL_BM);
            }
            ssb_pdl_wait();
            kb = kb_first; m = m_first; n = n_first;
            int c = 0, s = 0;
            uint32_t lap = 1;
            for (; c < all; ++c, next(kb, m, n)) {
                const uint32_t w_dst = smem_u32(smem + s * STAGE_BYTES);
                if (c >= ahead) {
                    if (!mbar_wait(empty0 + 8 * s, lap, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); break;
                    }
                    mbar_expect_tx(full0 + 8 * s, STAGE_BYTES);
                    tma_load_2d(w_dst, &map_w, full0 + 8 * s, kb * IL_BK, n * IL_BM);
                }
                tma_load_2d(w_dst + W_BYTES, &map_x, full0 + 8 * s, kb * IL_BK, m * BN);
                if (++s == STAGES) { s = 0; lap ^= 1; }
            }
            if (*abort_flag)                                       // let copies that were issued land before the block ends
                for (int i = max(0, c - STAGES); i < c; ++i)
                    mbar_wait(full0 + 8 * (i % STAGES), (i / STAGES) & 1, abort_flag + 1);
        }
    } else if (warp == 1) {
        ssb_pdl_wait();                                            // what follows spins on barriers
        if (lane == 0) {
            constexpr uint32_t idesc = il_idesc(IL_BM, BN);
            bool ok = true;
            int i = 0, s = 0;
            uint32_t lap = 0;
            for (long long u = range.begin; u < range.end && ok; ++i) {
                const int kb0 = (int)(u % k_blocks), n = (int)min((long long)(k_blocks - kb0), range.end - u);
                const int buf = i & 1;
                if (!mbar_wait(acc_empty0 + 8 * buf, ((i >> 1) & 1) ^ 1, abort_flag)) {
                    *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break;
                }
                tc_fence_after();
                for (int j = 0; j < n; ++j) {
                    if (!mbar_wait(full0 + 8 * s, lap, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break;
                    }
                    tc_fence_after();
                    const uint32_t w_addr = smem_u32(smem + s * STAGE_BYTES);
                    il_mma_x4(tmem + buf * BN, smem_desc(w_addr), smem_desc(w_addr + W_BYTES), idesc, j > 0 ? 1u : 0u);
                    tc_commit(empty0 + 8 * s);
                    if (++s == STAGES) { s = 0; lap ^= 1; }
                }
                if (ok) tc_commit(acc_full0 + 8 * buf);
                u += n;
            }
        }
    } else {
        ssb_pdl_wait();
        constexpr int CH = 16;                                    // columns at a time
        const int quarter = warp & 3, in_tile = quarter * 32 + lane;
        float* scales = row_scales + quarter * BN;
        int i = 0;
        for (long long u = range.begin; u < range.end; ++i) {
            const int tile = (int)(u / k_blocks), kb0 = (int)(u - (long long)tile * k_blocks);
            const int n = (int)min((long long)(k_blocks - kb0), range.end - u), buf = i & 1;
            const int m0 = tile % m_tiles * BN, col = tile / m_tiles * IL_BM + in_tile;       // this thread's output channel
            u += n;
            // all that does not wait for the sums comes before them: scales, and which blocks have pieces of the tile
            const int rows = min(BN, o.M - m0);
            for (int r = lane; r < rows; r += 32) scales[r] = o.sx[m0 + r];
            const float sw = col < o.N ? o.sw[col] : 0.f;
            const long long first = (long long)tile * k_blocks;
            const int c0_block = n == k_blocks ? 0 : range.owner(first), c1_block = n == k_blocks ? 0 : range.owner(first + k_blocks - 1);
            __syncwarp();
            // the four warps meet below: they go on together or not at all
            if (il_any_of_four(!mbar_wait(acc_full0 + 8 * buf, (i >> 1) & 1, abort_flag))) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * BN + ((uint32_t)(quarter * 32) << 16);
            // a block's pieces: of the tile that its range begins in the middle of (or that is all it has), and of its last; four
            // columns of a channel lie together
            auto piece = [&](int c) { return reinterpret_cast<int4*>(pieces) + (size_t)(2 * c + (c == c0_block)) * (BN / 4) * IL_BM + in_tile; };
            bool mine = true;                                      // whether this block writes the tile's results
            if (n < k_blocks) {
                int4* dst = piece(blockIdx.x);
#pragma unroll 1
                for (int c0 = 0; c0 < rows; c0 += CH) {
                    int sum[CH];
                    il_ld<CH>(acc + c0, sum);
#pragma unroll
                    for (int e = 0; e < CH; e += 4)
                        if (c0 + e < rows) dst[(size_t)((c0 + e) / 4) * IL_BM] = make_int4(sum[e], sum[e + 1], sum[e + 2], sum[e + 3]);
                }
                __threadfence();
                il_any_of_four(false);
                mine = il_any_of_four(threadIdx.x == 64 && atomicAdd(arrived + c0_block, n) + n == k_blocks);
                if (mine) __threadfence();
            }
#pragma unroll 1
            for (int c0 = 0; mine && c0 < rows; c0 += CH) {        // rows of x
                const int live = col < o.N ? rows - c0 : 0;
                const size_t at = (size_t)(m0 + c0) * o.ldo + col;
                float was[CH];
                if (o.add)
#pragma unroll
                    for (int e = 0; e < CH; ++e) was[e] = e < live ? ((const float*)o.out)[at + (size_t)e * o.ldo] : 0.f;
                int sum[CH];
                if (n == k_blocks) {
                    il_ld<CH>(acc + c0, sum);
                } else {
#pragma unroll
                    for (int e = 0; e < CH; ++e) sum[e] = 0;
#pragma unroll 4
                    for (int c = c0_block; c <= c1_block; ++c) {
                        const int4* src = piece(c) + (size_t)(c0 / 4) * IL_BM;
#pragma unroll
                        for (int e = 0; e < CH; e += 4) {
                            const int4 v = c0 + e < rows ? __ldcg(src + (size_t)(e / 4) * IL_BM) : make_int4(0, 0, 0, 0);
                            sum[e] += v.x; sum[e + 1] += v.y; sum[e + 2] += v.z; sum[e + 3] += v.w;
                        }
                    }
                }
                float y[CH];
#pragma unroll
                for (int e = 0; e < CH; ++e) y[e] = il_result(sum[e], scales[c0 + e], sw);
                if (!o.is_f32) {
#pragma unroll
                    for (int e = 0; e < CH; ++e)
                        if (e < live) ((bf16*)o.out)[at + (size_t)e * o.ldo] = __float2bfloat16_rn(y[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < CH; ++e)
                        if (e < live) ((float*)o.out)[at + (size_t)e * o.ldo] = o.add ? y[e] + was[e] : y[e];
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) il_arrive(acc_empty0 + 8 * buf);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(il_columns<BN>()) : "memory");
    }
}

// Tiles of 256 rows x 256 channels on pairs of SMs: each block fetches 128 rows and 128 channels a k-block (32 KB for 512 clocks of
// products), the leader issues the pair's instructions, each block's tensor memory gets its 128 rows.  The epilogue of a tile runs
// beside the products of the next (two regions of 256 columns).  Tiles go in bands of ``group_m`` row tiles, row tiles fastest.
// 8,192 x 28,672 x 4,096: 608 us by itself, 3.16 POP/s, at the power cap.
constexpr int IL_PAIR_STAGES = 6;
constexpr size_t IL_PAIR_SMEM = (size_t)IL_PAIR_STAGES * 2 * IL_BM * IL_BK + TC_STAGE_BYTES + (2 * IL_PAIR_STAGES + 4) * 8 + 16 + 1024;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(IL_THREADS, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const IlOut o, int m_tiles,
                 int n_tiles, int k_blocks, int group_m, int* __restrict__ error_word) {
    constexpr int BN = 256, STAGES = IL_PAIR_STAGES;
    constexpr uint32_t X_BYTES = IL_BM * IL_BK, W_BYTES = IL_BM * IL_BK, STAGE_BYTES = X_BYTES + W_BYTES;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* put = (float*)(smem + STAGES * STAGE_BYTES);
    uint64_t* bars = (uint64_t*)(smem + STAGES * STAGE_BYTES + TC_STAGE_BYTES);
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * STAGES + 4);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();                        // 0: the leader
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1, tiles = m_tiles * n_tiles;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + STAGES);
    const uint32_t acc_full0 = smem_u32(bars + 2 * STAGES), acc_empty0 = smem_u32(bars + 2 * STAGES + 2);
    auto tile_at = [&](int tile, int& m, int& n) {
        const int band = tile / (group_m * n_tiles), in_band = tile - band * group_m * n_tiles, rows = min(group_m, m_tiles - band * group_m);
        m = band * group_m + in_band % rows;
        n = in_band / rows;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(acc_full0 + 8 * i, 1); mbar_init(acc_empty0 + 8 * i, 8); }
        abort_flag[0] = 0;
        abort_flag[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * BN) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync_all();   // both blocks' barriers are initialised before either signals the other
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        ssb_pdl_wait();
        if (lane == 0) {
            const uint32_t leader_full0 = cluster_map(full0, 0);
            int c = 0;
            for (int tile = pair; tile < tiles && !*abort_flag; tile += n_pairs) {
                int m, n;
                tile_at(tile, m, n);
                const int m0 = (2 * m + (int)rank) * IL_BM, n0 = n * BN + (int)rank * IL_BM;
                for (int kb = 0; kb < k_blocks; ++kb, ++c) {
                    const int s = c % STAGES;
                    const uint32_t x_dst = smem_u32(smem + s * STAGE_BYTES);
                    if (!mbar_wait(empty0 + 8 * s, ((c / STAGES) & 1) ^ 1, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_PRODUCER); break;
                    }
                    if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2 * STAGE_BYTES);
                    tma_load_2d_pair(x_dst, &map_x, leader_full0 + 8 * s, kb * IL_BK, m0);
                    tma_load_2d_pair(x_dst + X_BYTES, &map_w, leader_full0 + 8 * s, kb * IL_BK, n0);
                }
            }
            if (*abort_flag) {
                // let issued copies land: the leader sees both blocks' bytes on its barriers, the other block gives them time
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
        ssb_pdl_wait();
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = il_idesc(256, BN);
            bool ok = true;
            int c = 0, i = 0;
            for (int tile = pair; tile < tiles && ok; tile += n_pairs, ++i) {
                const int buf = i & 1;
                if (!mbar_wait(acc_empty0 + 8 * buf, ((i >> 1) & 1) ^ 1, abort_flag)) {    // both epilogues have drained this region
                    *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break;
                }
                tc_fence_after();
                for (int kb = 0; kb < k_blocks && ok; ++kb, ++c) {
                    const int s = c % STAGES;
                    if (!mbar_wait(full0 + 8 * s, (c / STAGES) & 1, abort_flag)) {
                        *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_MMA); ok = false; break;
                    }
                    tc_fence_after();
                    const uint32_t x_addr = smem_u32(smem + s * STAGE_BYTES);
                    il_mma_pair_x4(tmem + buf * BN, smem_desc(x_addr), smem_desc(x_addr + X_BYTES), idesc, kb > 0 ? 1u : 0u);
                    tc_commit_pair(empty0 + 8 * s, 3);              // the stage is free in both blocks
                }
                if (ok) tc_commit_pair(acc_full0 + 8 * buf, 3);
            }
        }
    } else {
        ssb_pdl_wait();
        const int quarter = warp & 3;
        float* stage = put + quarter * 32 * TC_STAGE_LD;
        const uint32_t leader_acc_empty0 = cluster_map(acc_empty0, 0);
        int i = 0;
        for (int tile = pair; tile < tiles; tile += n_pairs, ++i) {
            int m, n;
            tile_at(tile, m, n);
            const int row0 = (2 * m + (int)rank) * IL_BM + quarter * 32, row = row0 + lane, rows = o.M - row0, buf = i & 1;
            const float sx = row < o.M ? o.sx[row] : 0.f;
            bool ok = mbar_wait(acc_full0 + 8 * buf, (i >> 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                if (lane == 0) { *abort_flag = 1; atomicCAS(error_word, 0, TC_ERR_EPILOGUE); }
                break;
            }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < BN / 32; ++c) {
                uint32_t r[32];
                tc_ld32(tmem + buf * BN + ((uint32_t)(quarter * 32) << 16) + c * 32, r);
                const int col = n * BN + c * 32;
                if (rows <= 0 || col >= o.N) continue;
                const float sw = col + lane < o.N ? o.sw[col + lane] : 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(il_result((int)r[e], sx, __shfl_sync(0xffffffffu, sw, e)));
                const bool whole = col + 32 <= o.N;
                if (o.is_f32) {
                    if (whole) {
                        char* dst = (char*)((float*)o.out + (size_t)row0 * o.ldo + col);
                        if (o.add) tc_put_rows<32, true>(stage, r, dst, (size_t)o.ldo * 4, rows);
                        else tc_put_rows<32, false>(stage, r, dst, (size_t)o.ldo * 4, rows);
                    } else if (row < o.M) {
                        float* dst = (float*)o.out + (size_t)row * o.ldo + col;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e < o.N) dst[e] = o.add ? dst[e] + __uint_as_float(r[e]) : __uint_as_float(r[e]);
                    }
                } else {
                    uint32_t packed[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const __nv_bfloat162 p = __floats2bfloat162_rn(__uint_as_float(r[e]), __uint_as_float(r[e + 1]));
                        packed[e / 2] = *reinterpret_cast<const uint32_t*>(&p);
                    }
                    if (whole) {
                        tc_put_rows<16, false>(stage, packed, (char*)((bf16*)o.out + (size_t)row0 * o.ldo + col), (size_t)o.ldo * 2, rows);
                    } else if (row < o.M) {
                        bf16* dst = (bf16*)o.out + (size_t)row * o.ldo + col;
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (col + e < o.N) dst[e] = __float2bfloat16_rn(__uint_as_float(r[e]));
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(leader_acc_empty0 + 8 * buf);
        }
    }
    tc_fence_before();
    cluster_sync_all();   // neither block leaves while the other may still read its shared memory or signal it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * BN) : "memory");
    }
    cluster_sync_all();
}

// ---- host side --------------------------------------------------------------------------------------------------------
static int il_map(CUtensorMap* map, const void* base, int rows, int cols, int ld, int box_rows) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return SSB_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {IL_BK, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : SSB_ERR_BAD_SIZE;
}

struct IlPlan {
    int bn, m_tiles, n_tiles, blocks;      // bn 0: tiles on pairs
    size_t counters, pieces;               // in scratch, behind the rows' scales (bytes)
};
// The kernel, its tile and its blocks, by what they are estimated to take (us; k-blocks of 128 codes):
//  * a block of the streaming kernel 0.36 a k-block, 0.45 with 128 rows a tile, 0.6 where those are all there are (nothing then shares
//    a fetch of weights); beginning and ending 9; the pieces of a tile 0.012 a piece and row, and 4 where tiles are cut wherever a
//    block's share ends instead of into equal parts;
//  * a pair 0.37 a k-block of 256 x 256, 8 for beginning and ending, 0.09 a tile that begins cold.
// Parts have four k-blocks at least, eight in tiles of 64 rows and more, whose pieces are larger.  us measured on both sides, rows x
// channels x k: shares that end anywhere and equal parts, 1 x 16,384 x 2,048 12.4 and 9.6, 8 x 4,096 x 4,096 10.2 and 8.8, 72 x 16,384
// x 2,048 21.3 and 14.2; parts of four and of eight, 1 x 2,048 x 2,048 7.0 and 8.4, 72 x 1,024 x 4,096 (64 rows a tile) 13.9 and 13.0;
// tiles of 64 rows, of 128, and pairs, 72 x 28,672 x 4,096 45, 36 and 36, 128 x 1,024 x 4,096 13.8, 19.3 and 18.8, 128 x 28,672 x 4,096
// 49, 45 and 38, 256 x 4,096 x 14,336 47, 41 and 50, 512 x 4,096 x 4,096 29, 33 and 22.  Tiles of 256 rows in the streaming kernel were
// behind one of these everywhere (256 x 4,096 x 14,336 49).
static IlPlan il_plan(int M, int N, int K) {
    const int sms = ssb_sm_count(), k_blocks = (K + IL_BK - 1) / IL_BK;
    IlPlan best{};
    double least = 0;
    auto consider = [&](double cost, int bn, int m_tiles, int n_tiles, int blocks) {
        if (best.m_tiles && cost >= least) return;
        least = cost;
        best = IlPlan{bn, m_tiles, n_tiles, blocks, (size_t)blocks * 4, (size_t)blocks * 2 * bn * IL_BM * 4};
    };
    for (int bn = M <= 16 ? 16 : M <= 32 ? 32 : 64; bn <= 128; bn *= 2) {
        const int m_tiles = (M + bn - 1) / bn, n_tiles = (N + IL_BM - 1) / IL_BM;
        const long long tiles = (long long)m_tiles * n_tiles, units = tiles * k_blocks;
        const double each = bn < 128 ? 0.36 : m_tiles == 1 ? 0.6 : 0.45;
        const double piece = 0.012 * std::min(bn, M);
        const int any = (int)std::min<long long>(sms, std::max(1LL, units / 4));
        consider(9 + each * (double)((units + any - 1) / any) + 4 + piece * (double)((any + tiles - 1) / tiles), bn, m_tiles, n_tiles, any);
        if (tiles <= sms) {
            const int parts = std::min(sms / (int)tiles, std::max(1, k_blocks / (bn <= 32 ? 4 : 8)));
            consider(9 + each * ((k_blocks + parts - 1) / parts) + (parts > 1 ? piece * parts : 0), bn, m_tiles, n_tiles, (int)tiles * parts);
        }
        if (M <= bn) break;
    }
    if (M > 64) {
        const int m_tiles = (M + 255) / 256, n_tiles = (N + 255) / 256, pairs = sms / 2;
        const long long tiles = (long long)m_tiles * n_tiles;
        consider(8 + 0.37 * (double)((tiles + pairs - 1) / pairs) * k_blocks + 0.09 * (double)std::min<long long>(tiles, pairs), 0, m_tiles, n_tiles, 0);
    }
    return best;
}
static size_t il_round(size_t n) { return (n + 127) & ~(size_t)127; }

// Bytes of scratch a product needs: codes and scales of the rows, counters, pieces of tiles.
SSB_API long long ssb_int8_linear_scratch(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const IlPlan p = il_plan(M, N, K);
    return (long long)(il_round((size_t)M * K) + il_round((size_t)M * 4) + il_round(p.counters) + p.pieces);
}

template <int BN, int STAGES>
static int il_stream(const CUtensorMap& mw, const CUtensorMap& mx, const IlOut& o, const IlPlan& p, int K, int* counters, int* pieces,
                     int* error_word, cudaStream_t stream) {
    constexpr size_t smem = il_smem<BN, STAGES>();
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(int8_stream_kernel<BN, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        configured = true;
    }
    return ssb_launch(int8_stream_kernel<BN, STAGES>, dim3(p.blocks), dim3(IL_THREADS), smem, stream, true, mw, mx, o, p.m_tiles,
                      p.m_tiles * p.n_tiles, (K + IL_BK - 1) / IL_BK, counters, pieces, error_word);
}

SSB_API int ssb_int8_linear(const void* x, int ldx, int dtype, const void* w, int ldw, const float* sw, void* out, int ldo,
                            int out_dtype, int M, int N, int K, int add, void* scratch, int* error_word, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || K % 16 || K > IL_MOST_K || ldw % 16 || N % 8 || (add && out_dtype != SSB_F32) || !scratch || !error_word) return SSB_ERR_BAD_SIZE;
    if (((uintptr_t)w | (uintptr_t)scratch | (uintptr_t)out) & 15) return SSB_ERR_BAD_SIZE;
    if (out_dtype != SSB_F32 && out_dtype != SSB_BF16) return SSB_ERR_BAD_DTYPE;
    const IlPlan p = il_plan(M, N, K);
    int8_t* codes = (int8_t*)scratch;
    float* sx = (float*)(codes + il_round((size_t)M * K));
    int* counters = (int*)((char*)sx + il_round((size_t)M * 4));
    int* pieces = (int*)((char*)counters + il_round(p.counters));
    int rc = SSB_ERR_BAD_DTYPE;
    if (dtype == SSB_BF16) rc = quantize_rows((const bf16*)x, ldx, codes, K, sx, M, K, counters, (int)(p.counters / 4), stream);
    else if (dtype == SSB_F32) rc = quantize_rows((const float*)x, ldx, codes, K, sx, M, K, counters, (int)(p.counters / 4), stream);
    if (rc) return rc;
    CUtensorMap mw, mx;
    rc = il_map(&mx, codes, M, K, K, p.bn ? p.bn : IL_BM);
    if (rc) return rc;
    rc = il_map(&mw, w, N, K, ldw, IL_BM);
    if (rc) return rc;
    const IlOut o{out, sx, sw, ldo, out_dtype == SSB_F32, add, M, N};
    switch (p.bn) {
        case 16: return il_stream<16, 11>(mw, mx, o, p, K, counters, pieces, error_word, stream);
        case 32: return il_stream<32, 10>(mw, mx, o, p, K, counters, pieces, error_word, stream);
        case 64: return il_stream<64, 8>(mw, mx, o, p, K, counters, pieces, error_word, stream);
        case 128: return il_stream<128, 6>(mw, mx, o, p, K, counters, pieces, error_word, stream);
    }
    static int max_pairs = 0;
    if (!max_pairs) {
        cudaError_t e = cudaFuncSetAttribute(int8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)IL_PAIR_SMEM);
        if (e != cudaSuccess) return (int)e;
        const int sms = ssb_sm_count();
        // how many pairs the device holds at once (a GPC with an odd SM left over holds one fewer)
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sms & ~1);
        cfg.blockDim = dim3(IL_THREADS);
        cfg.dynamicSmemBytes = IL_PAIR_SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, int8_pair_kernel, &cfg) != cudaSuccess || clusters <= 0) {
            cudaGetLastError();
            clusters = sms / 2;
        }
        max_pairs = std::min(clusters, sms / 2);
    }
    const int pairs = std::min(p.m_tiles * p.n_tiles, max_pairs);
    return ssb_launch(int8_pair_kernel, dim3(2 * pairs), dim3(IL_THREADS), IL_PAIR_SMEM, stream, true, mx, mw, o, p.m_tiles, p.n_tiles,
                      (K + IL_BK - 1) / IL_BK, std::min(16, p.m_tiles), error_word);
}

SSB_PACKED(ssb_int8_quantize_rows)
SSB_PACKED(ssb_int8_linear)
