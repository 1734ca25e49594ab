// Products of 8-bit integers: y[m, n] = a_scale[m] w_scale[n] sum_k A[m, k] W[n, k], rows of integers with a scale each (quantize.cu).
//
// The sum is a 32-bit integer, so it has no rounding and no order: a row's result is the same bits whatever batch it comes in.  |sum| <= 127^2 K stays
// below 2^31 for K up to 133,144.
#include "common.cuh"

GFB_DEFINE_LAST_ERROR()

enum { EPI_STORE = 0, EPI_ADD = 1, EPI_SWIGLU = 2, EPI_GELU = 4, EPI_GELU_TANH = 5, EPI_SILU = 6, EPI_RELU2 = 7 };

namespace {

constexpr int TILE = 64, TK = 64;

__device__ __forceinline__ float finish(int epi, float x) {
    if (epi == EPI_GELU) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752440f));
    if (epi == EPI_GELU_TANH) return x / (1.0f + expf(-1.5957691216057308f * (x + 0.044715f * x * x * x)));
    if (epi == EPI_SILU) return x / (1.0f + expf(-x));
    if (epi == EPI_RELU2) { const float r = fmaxf(x, 0.f); return r * r; }
    return x;
}

// 64 x 64 outputs per block of 256 threads, 4 x 4 each; four products per instruction (dp4a).
template <typename TO>
__global__ void __launch_bounds__(256)
gemm_int8_simple_kernel(const int8_t* __restrict__ A, const float* __restrict__ as, int lda, const int8_t* __restrict__ W, const float* __restrict__ ws,
                        int ldw, TO* __restrict__ out, int M, int N, int K, int epi) {
    __shared__ __align__(16) int sa[TILE][TK / 4 + 1], sw[TILE][TK / 4 + 1];
    gfb_pdl_launch();
    gfb_pdl_wait();
    const int m0 = blockIdx.x * TILE, n0 = blockIdx.y * TILE, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += TK) {
        const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;            // a row's 16 bytes
        int4 va = make_int4(0, 0, 0, 0), vw = va;
        if (m0 + r < M && k0 + c < lda) va = *reinterpret_cast<const int4*>(A + (size_t)(m0 + r) * lda + k0 + c);
        if (n0 + r < N && k0 + c < ldw) vw = *reinterpret_cast<const int4*>(W + (size_t)(n0 + r) * ldw + k0 + c);
        __syncthreads();
        int* da = &sa[r][c / 4];
        da[0] = va.x; da[1] = va.y; da[2] = va.z; da[3] = va.w;
        int* dw = &sw[r][c / 4];
        dw[0] = vw.x; dw[1] = vw.y; dw[2] = vw.z; dw[3] = vw.w;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TK / 4; k++) {
            int a[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) { a[i] = sa[ty * 4 + i][k]; w[i] = sw[tx * 4 + i][k]; }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __dp4a(a[i], w[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int m = m0 + ty * 4 + i;
        if (m >= M) continue;
        const float sm = as[m];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = n0 + tx * 4 + j;
            if (n >= N) continue;
            const float y = (float)acc[i][j] * sm * ws[n];
            if (epi == EPI_SWIGLU) {
                if (j & 1) continue;
                const float u = (float)acc[i][j + 1] * sm * ws[n + 1];
                out[(size_t)m * (N / 2) + n / 2] = gfb_from_f32<TO>(finish(EPI_SILU, y) * u);
            } else if (epi == EPI_ADD) {
                out[(size_t)m * N + n] = gfb_from_f32<TO>(gfb_to_f32(out[(size_t)m * N + n]) + y);
            } else {
                out[(size_t)m * N + n] = gfb_from_f32<TO>(finish(epi, y));
            }
        }
    }
}

}  // namespace

// A [M, lda] and W [N, ldw] of 8-bit integers (pitches multiples of 16, columns from K on zeros), a_scale [M], w_scale [N]; out [M, N] (SwiGLU: [M, N / 2])
// of type out_dt; epi EPI_ADD: float32 out += product.
GFB_API int gfb_gemm_int8(const void* A, const float* a_scale, int lda, const void* W, const float* w_scale, int ldw, void* out, int out_dt, int M, int N, int K,
                          int epi, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || K > 133144) return gfb_fail("gfb_gemm_int8: rows of %d numbers (1 to 133,144, beyond which a sum may leave 32 bits)", K);
    if (lda % 16 || ldw % 16 || lda < K || ldw < K) return gfb_fail("gfb_gemm_int8: pitches %d and %d of rows of %d numbers (multiples of 16)", lda, ldw, K);
    if (((uintptr_t)A | (uintptr_t)W) & 15) return gfb_fail("gfb_gemm_int8: operands must be 16-byte aligned");
    if (epi == EPI_SWIGLU && N % 2) return gfb_fail("gfb_gemm_int8: SwiGLU needs pairs of rows, got %d", N);
    dim3 grid((M + TILE - 1) / TILE, (N + TILE - 1) / TILE);
    if (grid.y > 65535) return gfb_fail("gfb_gemm_int8: %d rows of weights exceed the grid", N);
    cudaError_t e;
    if (out_dt == GFB_BF16) e = gfb_launch(gemm_int8_simple_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, (const int8_t*)A, a_scale, lda, (const int8_t*)W, w_scale, ldw, (__nv_bfloat16*)out, M, N, K, epi);
    else e = gfb_launch(gemm_int8_simple_kernel<float>, grid, dim3(256), 0, stream, (const int8_t*)A, a_scale, lda, (const int8_t*)W, w_scale, ldw, (float*)out, M, N, K, epi);
    return gfb_check(e, "gfb_gemm_int8");
}
