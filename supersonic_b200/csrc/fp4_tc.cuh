// What the tcgen05 products in microscaled 4-bit floats share: descriptors, instructions, a tile's inner rows.
#pragma once
#include "fp4_codes.cuh"
#include "tc_helpers.cuh"

constexpr int FL_BM = 128;
constexpr int FL_THREADS = 192;           // warp 0: TMA, warp 1: MMA + tensor memory, warps 2-5: epilogue
constexpr int FL_ROW = 128;               // bytes of codes a row and k-block
constexpr uint32_t FL_CHUNK = F4_CHUNK;
enum { FL_STORE = 0, FL_GATED = 1, FL_ACT = 2 };

// D float32; A and B E2M1, both K-major; scales powers of two.  ``part``: which half of a scale word (blocks 0 1 or 2 3) A and B use.
__host__ __device__ constexpr uint32_t fl_idesc(int m, int n, int part) {
    return ((uint32_t)(2 * part) << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 4) << 24) |
           ((uint32_t)(2 * part) << 29);
}
// 32 lanes x 16 bytes of shared memory that lie together (8-row groups 128 bytes apart), no swizzle.
__device__ __forceinline__ uint64_t fl_scale_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (8ull << 16) | (8ull << 32) | (1ull << 46);
}
__device__ __forceinline__ void fl_copy_scales(uint32_t tmem, uint32_t addr) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(fl_scale_desc(addr)) : "memory");
}
// One lane of the warp, all of whose lanes call it together.  A warp issues its products from code that all its lanes run, under this
// lane's predicate.  (From a branch that one lane alone runs a k-block took 875 clocks with its waits, whatever the tile: 8 x 4,096 x 14,336
// 13.4 us for 10.9.)
__device__ __forceinline__ bool fl_elect() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.b32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
// A k-block: four instructions of 64 numbers (32 bytes along the swizzled row: 2 descriptor units); the first two use the scales at
// sa0 and sb0, the last two those at sa1 and sb1, each pair their first and their second halves (idesc0, idesc1).
#define FL_MMA_X4(group_)                                                                                                                 \
    asm volatile("{\n.reg .pred p, q;\n.reg .b64 a1, a2, a3, b1, b2, b3;\n"                                                               \
                 "setp.ne.b32 p, %9, 0;\nsetp.eq.b32 q, 0, 0;\n"                                                                          \
                 "add.u64 a1, %1, 2;\nadd.u64 a2, %1, 4;\nadd.u64 a3, %1, 6;\n"                                                           \
                 "add.u64 b1, %2, 2;\nadd.u64 b2, %2, 4;\nadd.u64 b3, %2, 6;\n"                                                           \
                 "tcgen05.mma.cta_group::" group_ ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n"              \
                 "tcgen05.mma.cta_group::" group_ ".kind::mxf4.block_scale.scale_vec::2X [%0], a1, b1, %4, [%5], [%6], q;\n"              \
                 "tcgen05.mma.cta_group::" group_ ".kind::mxf4.block_scale.scale_vec::2X [%0], a2, b2, %3, [%7], [%8], q;\n"              \
                 "tcgen05.mma.cta_group::" group_ ".kind::mxf4.block_scale.scale_vec::2X [%0], a3, b3, %4, [%7], [%8], q;\n}"             \
                 ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc0), "r"(idesc1), "r"(sa0), "r"(sb0), "r"(sa1), "r"(sb1),               \
                 "r"(accumulate) : "memory")
__device__ __forceinline__ void fl_mma_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc0, uint32_t idesc1, uint32_t sa0,
                                          uint32_t sb0, uint32_t sa1, uint32_t sb1, uint32_t accumulate) {
    FL_MMA_X4("1");
}
__device__ __forceinline__ void fl_mma_pair_x4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc0, uint32_t idesc1,
                                               uint32_t sa0, uint32_t sb0, uint32_t sa1, uint32_t sb1, uint32_t accumulate) {
    FL_MMA_X4("2");
}
__device__ __forceinline__ void fl_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fl_ld16(uint32_t taddr, float (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\ntcgen05.wait::ld.sync.aligned;"
                 : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]), "=f"(r[9]),
                   "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
                 : "r"(taddr) : "memory");
}
// An arrival at the pair's leader that orders tensor memory alone (by the tcgen05 fences around it): a release at cluster scope waits
// for whatever this thread has on its way to or from memory, 1,290 clocks where scales are being fetched ahead.
__device__ __forceinline__ void fl_arrive_leader(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// Whether any thread of the four epilogue warps says so; all of them meet here (barrier 1).
__device__ __forceinline__ bool fl_any_of_four(bool mine) {
    uint32_t any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.or.pred q, 1, 128, p;\nselp.b32 %0, 1, 0, q;\n}"
                 : "=r"(any) : "r"((uint32_t)mine) : "memory");
    return any != 0;
}
__device__ __forceinline__ void fl_meet_four() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }

constexpr int fl_power(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }
constexpr int FL_INNER_ROWS = 16;         // rows of an inner tile that meet in shared memory at a time
constexpr int FL_INNER_LD = 132;
// V (8 or 16) numbers of a block of 32 whose others the neighbouring lanes have: codes to ``dst`` (V / 2 bytes), the block's scale by the
// first of its lanes.
template <int V>
__device__ __forceinline__ void fl_put_inner(float (&v)[V], uint8_t* dst, uint8_t* scale, bool live) {
    constexpr int LANES = 32 / V;
    uint32_t most = f4_most(v);
    if (__any_sync(0xffffffffu, most >= F4_WILD)) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = f4_finite(v[i]);
        most = f4_most(v);
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
    const int byte = f4_scale_byte(most);
    const float inverse = f4_inverse(byte);
    uint32_t w[V / 8];
#pragma unroll
    for (int i = 0; i < V / 8; ++i) w[i] = f4_encode8(v + 8 * i, inverse);
    if (live) {
        if (V == 16) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[V / 8 - 1]);
        else *reinterpret_cast<uint32_t*>(dst) = w[0];
        if ((threadIdx.x & (LANES - 1)) == 0) *scale = (uint8_t)byte;
    }
}

// Up to 16 rows' sums of a tile of 128 channels (a thread of four warps one channel) become inner rows in 4 bits; all four warps call it.
// A gate's exponential is the fast one, good to some 1e-6 of the result, where a 4-bit step is 1/12 of it at least: a number in some hundred
// thousand is rounded to the other side of a border.
// Rows c0, ... of ``rows``; row m0 of the codes and row s0 of the scales are the tile's first.  A block of 32 channels is wanted in
// neighbouring lanes: they meet in ``inner``.
template <int MODE>
__device__ __forceinline__ void fl_inner_tile(const float (&sum)[FL_INNER_ROWS], float* inner, int quarter, int lane, int who, int c0, int m0, int s0,
                                              int rows, int nt, int n_tiles, int N, int kind, float limit, const float* row_scale,
                                              uint8_t* codes, long long ld, uint8_t* scales, int inner_blocks) {
    constexpr int CH = FL_INNER_ROWS, WIDE = MODE == FL_GATED ? 64 : 128, V = WIDE / 8, PER = WIDE / V;     // inner channels a tile, a thread, threads a row
    static_assert(CH * PER == 128, "");
    const int width = MODE == FL_GATED ? N / 2 : N, left = rows - c0;
    if (MODE == FL_GATED) {
        const bool up = lane >= 16;
        const int at_ch = quarter * 16 + (lane & 15);
#pragma unroll
        for (int j = 0; j < CH; j += 2) {
            if (j >= left) break;
            // lanes 0-15 finish row j, lanes 16-31 row j + 1
            const float own = up ? sum[j + 1] : sum[j], give = up ? sum[j] : sum[j + 1];
            const float got = __shfl_xor_sync(0xffffffffu, give, 16);
            float z = ssb_gate_fast(up ? got : own, up ? own : got, kind, limit);
            const int r = c0 + j + (up ? 1 : 0);
            if (row_scale && r < rows) z *= row_scale[m0 + r];
            inner[(j + (up ? 1 : 0)) * FL_INNER_LD + at_ch] = z;
        }
    } else {
#pragma unroll
        for (int j = 0; j < CH; ++j)
            if (j < left) inner[j * FL_INNER_LD + quarter * 32 + lane] = ssb_activate(sum[j], kind) * limit;
    }
    fl_meet_four();
    const int r = who / PER, piece = who % PER, k = nt * WIDE + piece * V;
    if ((who & ~31) / PER < left) {                  // some of this warp's rows are there
        float v[V];
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const float4 q = *reinterpret_cast<const float4*>(inner + r * FL_INNER_LD + piece * V + e);
            v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
        }
        fl_put_inner<V>(v, codes + (size_t)(m0 + c0 + r) * ld + k / 2, scales + f4_scale_at(s0 + c0 + r, k / F4_BLOCK, inner_blocks),
                        r < left && k < width);
        // behind the last channel: scales of zero up to a whole k-block
        if (nt == n_tiles - 1 && r < left && piece == 0)
            for (int b = width / F4_BLOCK; b < 8 * inner_blocks; ++b) scales[f4_scale_at(s0 + c0 + r, b, inner_blocks)] = 0;
    }
    fl_meet_four();
}

__device__ __forceinline__ void fl_st8(uint32_t taddr, const uint4& a, const uint4& b) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(taddr), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
}
// ---- host side --------------------------------------------------------------------------------------------------------
// codes: rows of ``row_bytes`` bytes, boxes of box_rows x 128 bytes
static int fl_map(CUtensorMap* map, const void* base, long long rows, int row_bytes, int box_rows) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return SSB_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)row_bytes, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    cuuint32_t box[2] = {FL_ROW, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : SSB_ERR_BAD_SIZE;
}
// scales: ``chunks`` of 1,024 bytes, a chunk a box
static int fl_scale_map(CUtensorMap* map, const void* base, long long chunks) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return SSB_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {F4_CHUNK / 4, (cuuint64_t)chunks};
    cuuint64_t strides[1] = {F4_CHUNK};
    cuuint32_t box[2] = {F4_CHUNK / 4, 1};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : SSB_ERR_BAD_SIZE;
}

