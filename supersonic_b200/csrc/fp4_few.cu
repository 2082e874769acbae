// Products of few rows in microscaled 4-bit floats (the format: fp4_codes.cuh): the weights are read once and that is what it takes, so
// the kernel is made for a short way from memory to the sums.  Weights go through shared memory by cp.async, every warp a ring of its
// own (16 channels x 256 numbers a step), and no warp waits for another until a tile's sums meet; rows lie in shared memory whole,
// quantised there by every block if they come as numbers.
//
// A block of 32 numbers is two mma.sync (m16n8k16) of float16: 16 channels x 8 rows.  Codes are exact in float16, and so are a block's
// products and their sum in float32 (multiples of 0.25 up to 1,152); then come the two scales, and the float32 sum.  (With e4m3 operands,
// half as many products, 36 million instructions were counted for what takes half of them so.)
// tcgen05 with its own scales needs a tile's 128 channels and their rows in tensor memory before the first product and a way back after
// the last, and rows that come as numbers a launch before it: one row x 2,048 x 2,048 takes 5.2 us so and 3.4 here.  Where each is
// taken: fl_few.
#include "fp4_codes.cuh"
#include "fp4_few.cuh"
#include "per_device.h"
#include <algorithm>

typedef __nv_bfloat16 bf16;

constexpr int FW_WARPS = 16;
constexpr int FW_THREADS = 32 * FW_WARPS;
constexpr int FW_SLOT = 16 * 128 + 16 * 8;                          // a step's codes and scales
constexpr int FW_MOST_SMEM = 227 * 1024;

// A word's eight codes as pairs of float16.
__device__ __forceinline__ void fw_halves(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n.reg .b8 a, b, c, d;\nmov.b32 {a, b, c, d}, %4;\ncvt.rn.f16x2.e2m1x2 %0, a;\ncvt.rn.f16x2.e2m1x2 %1, b;\n"
        "cvt.rn.f16x2.e2m1x2 %2, c;\ncvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// The scale in byte ``i`` of a word; i is a constant.
__device__ __forceinline__ float fw_scale(uint32_t w, int i) {
    const uint32_t bits = (i == 0 ? w << 23 : i == 1 ? w << 15 : i == 2 ? w << 7 : w >> 1) & 0x7f800000u;
    return __uint_as_float(max(bits, 0x00400000u));
}
// d = the products of a block: channels g and g + 8 (words lo, hi), rows' words x; which of a lane's numbers meet is the same on both sides.
__device__ __forceinline__ void fw_mma(float (&d)[4], const uint32_t (&lo)[4], const uint32_t (&hi)[4], const uint32_t (&x)[4]) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(lo[0]), "r"(hi[0]), "r"(lo[1]), "r"(hi[1]), "r"(x[0]), "r"(x[1]), "f"(0.f));
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(lo[2]), "r"(hi[2]), "r"(lo[3]), "r"(hi[3]), "r"(x[2]), "r"(x[3]));
}
__device__ __forceinline__ void fw_cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void fw_cp4(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}

// Sums are held times 2^-11, which a row's scales bring in and the tile's end takes out: a block's products (up to 1,152, multiples of 0.25)
// times its row's scale are exact then for every scale from 2^-127 to 2^127, and what is too large is so as a whole.  (A sum below 2^-115 has
// float32's smallest steps times 2^11.  The smaller of the two scales first, 1 x 4,096 x 4,096: 5.65 us for 5.12; a look at each step's
// scales 5.38.)
constexpr float FW_HELD = 4.8828125e-4f, FW_WHOLE = 2048.f;
// A row's codes in shared memory, 16 bytes more than whole k-blocks apart: eight rows' pieces meet no bank twice.
__host__ __device__ constexpr int fw_row_bytes(int k_blocks) { return k_blocks * 128 + 16; }

template <int NB, int MODE>
__global__ void __launch_bounds__(FW_THREADS, 1) fp4_few_kernel(const FwArgs a) {
    constexpr int ROWS = 8 * NB;
    extern __shared__ __align__(16) unsigned char fw_smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const int kw = warp % a.k_warps, cg = warp / a.k_warps, CH = 16 * (FW_WARPS / a.k_warps), LD = CH + 4;
    const int row_bytes = fw_row_bytes(a.k_blocks), all_blocks = a.k_blocks * 8;
    unsigned char* x_s = fw_smem;                                    // [ROWS][row_bytes]
    float* sx_s = (float*)(x_s + ROWS * row_bytes);                  // [all_blocks][ROWS]
    float* red = sx_s + all_blocks * ROWS;                           // [2][k_warps][ROWS][LD]
    unsigned char* ring = (unsigned char*)(red + 2 * a.k_warps * ROWS * LD) + warp * a.slots * FW_SLOT;
    const int items = (a.N + CH - 1) / CH;
    const int begin = (int)((long long)items * blockIdx.x / gridDim.x), end = (int)((long long)items * (blockIdx.x + 1) / gridDim.x);
    const int steps = kw < a.k_blocks ? (a.k_blocks - kw + a.k_warps - 1) / a.k_warps : 0;      // of this warp, a tile

    // ---- this warp's stream of weights ----
    int in_item = begin, in_step = 0, in_slot = 0;
    const uint8_t *src = nullptr, *src_scale = nullptr;
    bool live_row[4], live_scale = false;
    auto load = [&]() {
        if (in_item < end && steps > 0) {
            if (in_step == 0) {
                const int ch0 = in_item * CH + cg * 16, ch = ch0 + (lane >> 1);
                src = a.w + (size_t)min(ch0, a.N - 1) * (a.K / 2);                  // clamped where nothing is read
#pragma unroll
                for (int q = 0; q < 4; ++q) live_row[q] = ch0 + (lane >> 3) + 4 * q < a.N;
                live_scale = ch < a.N;
                const int c = live_scale ? ch : 0;
                src_scale = a.ws + f4_scale_at(c, (lane & 1) * 4, a.k_blocks);
            }
            const int kb = kw + in_step * a.k_warps, at = kb * 128 + (lane & 7) * 16;
            unsigned char* slot = ring + in_slot * FW_SLOT;
            const uint32_t dst = (uint32_t)__cvta_generic_to_shared(slot);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int row = (lane >> 3) + 4 * q;
                const bool live = live_row[q] && at < a.K / 2;
                fw_cp16(dst + row * 128 + (((lane & 7) ^ (row & 7)) << 4), live ? src + (size_t)row * (a.K / 2) + at : a.w, live);
            }
            fw_cp4(dst + 2048 + lane * 4, src_scale + (size_t)kb * F4_CHUNK, live_scale);
            if (++in_step == steps) { in_step = 0; ++in_item; }
        }
        if (++in_slot == a.slots) in_slot = 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // weights are nobody's output: the first of them come while whatever writes the rows still runs
    for (int i = 0; i + 1 < a.slots; ++i) load();
    ssb_pdl_wait();
    ssb_pdl_launch_dependents();

    int out_slot = 0;
    const int rows = a.M;
    for (int item = begin; item < end; ++item) {
        const int ch0 = item * CH;
        if (item == begin) {                                         // the rows, which stay
            if (a.dtype < 0) {
                // 16 bytes of codes a thread and turn, a word of four blocks' scales; behind K zeros
                const int per_row = a.k_blocks * 8, words = a.k_blocks * 2;
                for (int u0 = tid; u0 < rows * per_row; u0 += 4 * FW_THREADS) {
                    uint4 v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int u = u0 + j * FW_THREADS, r = u / per_row, at = (u - r * per_row) * 16;
                        v[j] = make_uint4(0, 0, 0, 0);
                        if (u < rows * per_row && at < a.K / 2)
                            v[j] = *reinterpret_cast<const uint4*>((const uint8_t*)a.x + (size_t)r * (a.K / 2) + at);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int u = u0 + j * FW_THREADS, r = u / per_row;
                        if (u < rows * per_row) *reinterpret_cast<uint4*>(x_s + r * row_bytes + (u - r * per_row) * 16) = v[j];
                    }
                }
                for (int u = tid; u < rows * words; u += FW_THREADS) {
                    const int r = u / words, i = u - r * words;
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(a.xs + f4_scale_at(r, 4 * i, a.k_blocks));
#pragma unroll
                    for (int j = 0; j < 4; ++j) sx_s[(4 * i + j) * ROWS + r] = f4_scale(w >> (8 * j) & 255) * FW_HELD;
                }
            } else {
                // eight numbers a thread and turn, four neighbouring threads a block of 32; behind K zeros
                const int per_row = all_blocks * 4, units = rows * per_row;
                for (int u0 = 0; u0 < units; u0 += 4 * FW_THREADS) {
                    float v[4][8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int u = u0 + j * FW_THREADS + tid, r = u / per_row, k = (u - r * per_row) * 8;
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
                        if (u < units && k < a.K) {
                            const size_t row = r;
                            if (a.dtype == SSB_BF16) f4_load8((const bf16*)a.x + row * a.ldx + k, v[j]);
                            else f4_load8((const float*)a.x + row * a.ldx + k, v[j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int u = u0 + j * FW_THREADS + tid, r = u / per_row, i = u - r * per_row;
                        uint32_t most = f4_most(v[j]);
                        if (__any_sync(0xffffffffu, most >= F4_WILD)) {
#pragma unroll
                            for (int q = 0; q < 8; ++q) v[j][q] = f4_finite(v[j][q]);
                            most = f4_most(v[j]);
                        }
                        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
                        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
                        const int byte = f4_scale_byte(most);
                        if (u < units) {
                            *reinterpret_cast<uint32_t*>(x_s + r * row_bytes + i * 4) = f4_encode8(v[j], f4_inverse(byte));
                            if ((i & 3) == 0) sx_s[(i >> 2) * ROWS + r] = f4_scale(byte) * FW_HELD;
                        }
                    }
                }
            }
            __syncthreads();
        }
        float sum[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[nb][i] = 0.f;
        for (int step = 0; step < steps; ++step) {
            load();                                                  // into the slot that was read last
            switch (a.slots) {                                       // this step's copies have landed
                case 2: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
                case 3: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
                case 4: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
                default: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
            }
            __syncwarp();
            const unsigned char* slot = ring + out_slot * FW_SLOT;
            if (++out_slot == a.slots) out_slot = 0;
            const uint2 s_lo = *reinterpret_cast<const uint2*>(slot + 2048 + g * 8), s_hi = *reinterpret_cast<const uint2*>(slot + 2048 + g * 8 + 64);
            const int blk0 = (kw + step * a.k_warps) * 8;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const unsigned char* at = slot + g * 128 + ((b ^ g) << 4) + t4 * 4;
                const uint32_t w_lo = *reinterpret_cast<const uint32_t*>(at), w_hi = *reinterpret_cast<const uint32_t*>(at + 1024);
                uint32_t lo[4], hi[4];
                fw_halves(w_lo, lo);
                fw_halves(w_hi, hi);
                const float c_lo = fw_scale(b < 4 ? s_lo.x : s_lo.y, b & 3), c_hi = fw_scale(b < 4 ? s_hi.x : s_hi.y, b & 3);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    uint32_t x[4];
                    fw_halves(*reinterpret_cast<const uint32_t*>(x_s + (g + 8 * nb) * row_bytes + (blk0 + b) * 16 + t4 * 4), x);
                    const float2 sx = *reinterpret_cast<const float2*>(sx_s + (blk0 + b) * ROWS + 8 * nb + 2 * t4);
                    float d[4];
                    fw_mma(d, lo, hi, x);
                    sum[nb][0] = fmaf(d[0] * sx.x, c_lo, sum[nb][0]);
                    sum[nb][1] = fmaf(d[1] * sx.y, c_lo, sum[nb][1]);
                    sum[nb][2] = fmaf(d[2] * sx.x, c_hi, sum[nb][2]);
                    sum[nb][3] = fmaf(d[3] * sx.y, c_hi, sum[nb][3]);
                }
            }
            __syncwarp();                                            // the slot has been read
        }
        // the k-warps' sums meet; two places in turn, so that one barrier a tile is enough
        float* mine = red + ((item & 1) * a.k_warps + kw) * ROWS * LD + cg * 16;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float* to = mine + (8 * nb + 2 * t4) * LD + g;
            to[0] = sum[nb][0];
            to[LD] = sum[nb][1];
            to[8] = sum[nb][2];
            to[LD + 8] = sum[nb][3];
        }
        __syncthreads();
        const float* parts = red + (item & 1) * a.k_warps * ROWS * LD;
        auto total = [&](int r, int ch) {
            float s = 0.f;
            for (int k = 0; k < a.k_warps; ++k) s += parts[(k * ROWS + r) * LD + ch];
            return s * FW_WHOLE;
        };
        if (MODE == FW_STORE) {
            for (int i = tid; i < rows * CH; i += FW_THREADS) {
                const int r = i / CH, ch = i - r * CH;
                if (ch0 + ch >= a.N) continue;
                const float s = total(r, ch);
                const size_t at = (size_t)r * a.ldo + ch0 + ch;
                if (a.is_f32) ((float*)a.out)[at] = a.add ? ((float*)a.out)[at] + s : s;
                else ((bf16*)a.out)[at] = __float2bfloat16_rn(s);
            }
        } else {
            // a warp a block of 32 inner channels of a row, a channel a lane
            constexpr int WIDE = MODE == FW_GATED ? 64 : 32;         // channels of W a block
            const int per = CH / WIDE, width = MODE == FW_GATED ? a.N / 2 : a.N;
            for (int i = warp; i < rows * per; i += FW_WARPS) {
                const int r = i / per, q = i - r * per, k = (ch0 / WIDE + q) * 32;
                float z;
                if (MODE == FW_GATED) {
                    const int ch = q * 64 + (lane >> 4) * 32 + (lane & 15);
                    z = ssb_gate_fast(total(r, ch), total(r, ch + 16), a.kind, a.limit);
                    if (a.row_scale) z *= a.row_scale[r];
                } else {
                    z = ssb_activate(total(r, q * 32 + lane), a.kind) * a.limit;
                }
                f4_put_block(z, (uint8_t*)a.out + (size_t)r * a.ldo, a.out_scales, r, k, width, a.inner_blocks);
                // behind the last channel: scales of zero up to a whole k-block
                if (q == 0 && ch0 + CH >= a.N && width / F4_BLOCK + lane < 8 * a.inner_blocks && lane < 8)
                    a.out_scales[f4_scale_at(r, width / F4_BLOCK + lane, a.inner_blocks)] = 0;
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- host side --------------------------------------------------------------------------------------------------------
static size_t fw_fixed(int rows, int k_blocks, int k_warps) {
    const int ch = 16 * (FW_WARPS / k_warps);
    return (size_t)rows * fw_row_bytes(k_blocks) + (size_t)k_blocks * 8 * rows * 4 + (size_t)2 * k_warps * rows * (ch + 4) * 4;
}

template <int NB, int MODE>
static int fw_launch(const FwArgs& a, int blocks, size_t smem, bool early, cudaStream_t stream) {
    auto kernel = fp4_few_kernel<NB, MODE>;
    static SsbPerDevice<bool> set;
    bool* configured = set.here();
    if (!configured) return SSB_ERR_UNSUPPORTED;
    if (!*configured) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FW_MOST_SMEM);
        if (e != cudaSuccess) return (int)e;
        *configured = true;
    }
    return ssb_launch(kernel, dim3(blocks), dim3(FW_THREADS), smem, stream, early, a);
}

// How a product of M rows by N x K weights runs; slots 0: not by this kernel, which takes up to 16 rows, where it makes inner rows up to 8.
struct FwPlan { int nb, k_warps, slots, blocks; size_t smem; };
static FwPlan fw_plan(int M, int N, int K, int mode) {
    FwPlan p{};
    const int k_blocks = f4_k_blocks(K), sms = ssb_sm_count();
    if (M > (mode == FW_STORE ? 16 : 8)) return p;
    p.nb = M <= 8 ? 1 : 2;
    // channels a tile and warps along k: as few steps of a warp as can be, one after another on the fullest SM; a gated tile is 64
    // channels (32 inner ones, a block) at least, an ungated one of inner channels 32
    long long least = 0, steps = 0;
    for (int k_warps = mode == FW_STORE ? 16 : mode == FW_GATED ? 4 : 8; k_warps >= 1; k_warps /= 2) {
        const int ch = 16 * (FW_WARPS / k_warps), items = (N + ch - 1) / ch, rounds = (items + sms - 1) / sms;
        const int deep = (k_blocks + k_warps - 1) / k_warps;
        const long long cost = (long long)rounds * (2 * deep + 1);            // a tile's end is half a step
        if (p.k_warps && cost >= least) continue;
        least = cost;
        steps = (long long)rounds * deep;
        p.k_warps = k_warps;
        p.blocks = std::min(items, sms);
    }
    const size_t fixed = fw_fixed(8 * p.nb, k_blocks, p.k_warps);
    if (fixed >= FW_MOST_SMEM) return p;
    // no more slots than a block's steps want: what is left lets the next launch's blocks begin beside these
    p.slots = (int)std::min<long long>(std::min<long long>(5, std::max<long long>(2, steps)), (FW_MOST_SMEM - fixed) / (FW_WARPS * FW_SLOT));
    if (p.slots < 2) p.slots = 0;
    p.smem = fixed + (size_t)p.slots * FW_WARPS * FW_SLOT;
    return p;
}
bool fw_takes(int M, int N, int K, int mode) { return fw_plan(M, N, K, mode).slots > 0; }

int fw_product(FwArgs a, int mode, bool early, cudaStream_t stream) {
    const FwPlan p = fw_plan(a.M, a.N, a.K, mode);
    if (p.slots == 0) return SSB_ERR_UNSUPPORTED;
    a.k_warps = p.k_warps;
    a.slots = p.slots;
    a.k_blocks = f4_k_blocks(a.K);
    if (p.nb == 2) return fw_launch<2, FW_STORE>(a, p.blocks, p.smem, early, stream);
    return mode == FW_STORE ? fw_launch<1, FW_STORE>(a, p.blocks, p.smem, early, stream)
           : mode == FW_GATED ? fw_launch<1, FW_GATED>(a, p.blocks, p.smem, early, stream) : fw_launch<1, FW_ACT>(a, p.blocks, p.smem, early, stream);
}
