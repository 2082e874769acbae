// Matrix products in 8-bit integers: out[m, n] (+)= (sum_k xc[m, k] wc[n, k]) * sx[m] * sw[n], with the rows of x quantised as they
// come (sx = max |x_row| * (1/127), xc = rint(x / sx)) and weights that lie in codes with a scale per output channel.  The sums are
// exact: 32-bit integers up to k = 133,136 (127 * 127 * k < 2^31), which is checked.
//
// The reference's 8-bit lane of this architecture multiplies int8 weights by activations of the model's type
// (crates/runner/src/llama31_engine.rs:289-430).
#include "common.cuh"

typedef __nv_bfloat16 bf16;

constexpr float IL_LEAST_SCALE = 7.888609052210118e-31f;        // 2^-100: a row of zeros has a scale too
constexpr float IL_MOST = 1.7014118346046923e38f;               // 2^127: what an infinity counts as

// ---- rows to codes ------------------------------------------------------------------------------------------------
// A block a row: its largest magnitude, then its codes; the second reading comes from the caches.
template <typename T>
__global__ void __launch_bounds__(256)
int8_quantize_rows_kernel(const T* __restrict__ x, int ldx, int8_t* __restrict__ codes, int ldc, float* __restrict__ scale, int K) {
    const int row = blockIdx.x;
    const T* src = x + (size_t)row * ldx;
    __shared__ float warp_max[8];
    float most = 0.f;
    for (int k = threadIdx.x; k < K; k += 256) {
        const float v = ssb_to_float(src[k]);
        most = fmaxf(most, v != v ? 0.f : fminf(fabsf(v), IL_MOST));
    }
    most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = fmaxf(most, warp_max[w]);
    const float s = fmaxf(__fmul_rn(most, 1.f / 127.f), IL_LEAST_SCALE);
    for (int k = threadIdx.x; k < K; k += 256) {
        const float v = ssb_to_float(src[k]);
        codes[(size_t)row * ldc + k] = v != v ? 0 : (int8_t)(int)fminf(fmaxf(rintf(__fdiv_rn(v, s)), -127.f), 127.f);
    }
    if (threadIdx.x == 0) scale[row] = s;
}

SSB_API int ssb_int8_quantize_rows(const void* x, int ldx, int dtype, void* codes, int ldc, float* scale, int rows, int K,
                                   cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (K <= 0) return SSB_ERR_BAD_SIZE;
    if (dtype == SSB_BF16) int8_quantize_rows_kernel<bf16><<<rows, 256, 0, stream>>>((const bf16*)x, ldx, (int8_t*)codes, ldc, scale, K);
    else if (dtype == SSB_F32) int8_quantize_rows_kernel<float><<<rows, 256, 0, stream>>>((const float*)x, ldx, (int8_t*)codes, ldc, scale, K);
    else return SSB_ERR_BAD_DTYPE;
    return ssb_launch_status();
}

// ---- the product ----------------------------------------------------------------------------------------------------
// 32 x 32 results a block, four products of codes an instruction (dp4a).
template <typename T, bool ADD>
__global__ void __launch_bounds__(256)
int8_product_kernel(const int8_t* __restrict__ x, int ldx, const float* __restrict__ sx, const int8_t* __restrict__ w, int ldw,
                    const float* __restrict__ sw, T* __restrict__ out, int ldo, int M, int N, int K) {
    __shared__ int xs[32][17], ws[32][17];
    const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 32, tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    int sum[4] = {0, 0, 0, 0};
    for (int k0 = 0; k0 < K; k0 += 64) {
        for (int e = threadIdx.x; e < 32 * 16; e += 256) {
            const int r = e / 16, c = e % 16;
            const bool in = k0 + 4 * c < K;
            xs[r][c] = in && m0 + r < M ? *reinterpret_cast<const int*>(x + (size_t)(m0 + r) * ldx + k0 + 4 * c) : 0;
            ws[r][c] = in && n0 + r < N ? *reinterpret_cast<const int*>(w + (size_t)(n0 + r) * ldw + k0 + 4 * c) : 0;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __dp4a(xs[ty + 8 * i][c], ws[tx][c], sum[i]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = m0 + ty + 8 * i, n = n0 + tx;
        if (m < M && n < N) {
            const float y = __fmul_rn(__fmul_rn((float)sum[i], sx[m]), sw[n]);
            T* dst = out + (size_t)m * ldo + n;
            *dst = ssb_from_float<T>(ADD ? ssb_to_float(*dst) + y : y);
        }
    }
}

SSB_API int ssb_int8_product(const void* x, int ldx, const float* sx, const void* w, int ldw, const float* sw, void* out, int ldo,
                             int out_dtype, int M, int N, int K, int add, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || K % 16 || K > 133136 || ldx % 16 || ldw % 16 || (add && out_dtype != SSB_F32)) return SSB_ERR_BAD_SIZE;
    if (((uintptr_t)x | (uintptr_t)w) & 15) return SSB_ERR_BAD_SIZE;
    const dim3 grid((N + 31) / 32, (M + 31) / 32);
    if (grid.y > 65535) return SSB_ERR_BAD_SIZE;
    const int8_t *xc = (const int8_t*)x, *wc = (const int8_t*)w;
    if (out_dtype == SSB_BF16) int8_product_kernel<bf16, false><<<grid, 256, 0, stream>>>(xc, ldx, sx, wc, ldw, sw, (bf16*)out, ldo, M, N, K);
    else if (out_dtype != SSB_F32) return SSB_ERR_BAD_DTYPE;
    else if (add) int8_product_kernel<float, true><<<grid, 256, 0, stream>>>(xc, ldx, sx, wc, ldw, sw, (float*)out, ldo, M, N, K);
    else int8_product_kernel<float, false><<<grid, 256, 0, stream>>>(xc, ldx, sx, wc, ldw, sw, (float*)out, ldo, M, N, K);
    return ssb_launch_status();
}
