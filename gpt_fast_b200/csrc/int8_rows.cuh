// Rows of 8-bit integers with one scale each: what the 8-bit products multiply and the 8-bit cache holds.
//
// A row x becomes scale = m / 127, m = max |x_i|, and the integers q_i nearest to 127 x_i / m (ties to even), so that q_i scale is within
// scale / 2 of x_i and |q_i| <= 127.  The integer is the one exact arithmetic gives for the 32-bit numbers x_i: a 32-bit quotient is off by two roundings,
// at most 127 x 2^-23 < 2e-5, so it is right unless it lies that near to a tie; then 254 |x_i| is compared with the odd multiple of m, each product as a 32-bit
// number and its rest.  The two rounded products are next to each other, so that their difference is exact, and the rests are multiples of a 256th of their
// last place, so theirs is too.
// So the same numbers give the same integers in every kernel here, whatever order its code computes in.
// A row of zeros has scale 0.  A row that holds a NaN or an infinity has scale NaN (and integers 0): it stands for NaN as a whole.
#pragma once
#include "common.cuh"

namespace {

// How a row's numbers become integers; `bits`: the largest |x_i| as its 32-bit pattern, which orders like the number and puts infinity and NaN on top.
struct RowScale {
    float most, lift, inv, scale;                       // most, inv: of the row times lift
    bool live;                                          // finite and not all zeros
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        const float m = __uint_as_float(bits);
        live = bits != 0u && bits < 0x7f800000u;
        lift = m < 0x1p-60f ? 0x1p64f : m > 0x1p100f ? 0x1p-30f : 1.f;      // keeps 127 / m and 254 m finite and their parts exact
        most = __fmul_rn(m, lift);
        inv = live ? __fdiv_rn(127.f, most) : 0.f;
        scale = bits < 0x7f800000u ? __fdiv_rn(m, 127.f) : __uint_as_float(0x7fc00000u);
    }
    // x: times lift
    __device__ __forceinline__ float nearest(float x) const {
        const float r = __fmul_rn(x, inv);
        float k = rintf(r);
        if (fabsf(r - k) > 0.49998f) {
            // 254 |x| against (2 f + 1) most: both products as a rounded one and its rest, which has few bits
            const float f = floorf(fabsf(r)), odd = 2.f * f + 1.f;
            const float p = __fmul_rn(254.f, fabsf(x)), t = __fmul_rn(odd, most);
            const float over = (p - t) + (__fmaf_rn(254.f, fabsf(x), -p) - __fmaf_rn(odd, most, -t));
            k = copysignf(over > 0.f || (over == 0.f && ((int)f & 1)) ? f + 1.f : f, x);
        }
        return k;
    }
    __device__ __forceinline__ int of(float x) const { return live ? (int)nearest(__fmul_rn(x, lift)) : 0; }
    // Eight numbers of the row in the bytes of two words.  Adding 1.5 x 2^23 rounds to an integer, ties to even, and leaves it in the low bits.
    __device__ __forceinline__ uint2 of8(const float* x) const {
        uint32_t w[8];
        float far = lift != 1.f ? 1.f : 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r = __fmul_rn(x[i], inv), t = __fadd_rn(r, 12582912.f);
            w[i] = __float_as_uint(t);
            far = fmaxf(far, fabsf(__fsub_rn(r, __fsub_rn(t, 12582912.f))));
        }
        if (far > 0.49998f) {                           // one of them next to a tie, or a row out of the ordinary
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = (uint32_t)(int)nearest(__fmul_rn(x[i], lift));
        }
        return packed(w);
    }
    __device__ __forceinline__ uint2 packed(const uint32_t (&w)[8]) const {
        const uint32_t lo = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
        const uint32_t hi = __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410);
        return live ? make_uint2(lo, hi) : make_uint2(0u, 0u);
    }
    // The same for rows of bfloat16 numbers, where about one number in 300 is a tie, so half of all warps meet one.  With eight bits each, 127 x, k m and so what k
    // leaves of 127 x are exact, and the integer k moves by one where that is more than half of m, or half of it and k odd.
    __device__ __forceinline__ uint2 of8_short(const float* x) const {
        if (lift != 1.f) return of8(x);
        uint32_t w[8];
        float far = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r = __fmul_rn(x[i], inv), t = __fadd_rn(r, 12582912.f);
            w[i] = __float_as_uint(t);
            far = fmaxf(far, fabsf(__fsub_rn(r, __fsub_rn(t, 12582912.f))));
        }
        if (far > 0.49998f) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float k = __fsub_rn(__uint_as_float(w[i]), 12582912.f), e = __fmaf_rn(-k, most, __fmul_rn(127.f, x[i])), over = __fmaf_rn(2.f, fabsf(e), -most);
                if (over > 0.f || (over == 0.f && (w[i] & 1u))) w[i] += e < 0.f ? -1 : 1;
            }
        }
        return packed(w);
    }
};

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint32_t block_max_bits(uint32_t v, uint32_t* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = blockDim.x >> 5;
    v = warp_max_bits(v);
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    return warp_max_bits(lane < n ? scratch[lane] : 0u);
}

// eight neighbouring numbers from an address that is a multiple of 16 bytes
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}

constexpr int ROW_VECTORS = 4;               // vectors of eight numbers that a thread keeps

// eight numbers as they came, so that a row waits for its maximum in few registers
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };
__device__ __forceinline__ uint32_t max_bits(const Raw8<float>& r) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 2; i++) m = max(max(max(m, r.w[i].x & 0x7fffffffu), max(r.w[i].y & 0x7fffffffu, r.w[i].z & 0x7fffffffu)), r.w[i].w & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ uint32_t max_bits(const Raw8<__nv_bfloat16>& r) {
    const uint32_t m = __vmaxu2(__vmaxu2(r.w[0].x & 0x7fff7fffu, r.w[0].y & 0x7fff7fffu), __vmaxu2(r.w[0].z & 0x7fff7fffu, r.w[0].w & 0x7fff7fffu));
    return max(m << 16, m & 0xffff0000u);
}

// q [R, pitch] and scale [R] of x [R, K], the columns from K to the pitch zeros.  One block per row, K a multiple of 8, rows aligned: one pass, the row in
// registers.  8,192 rows of 4,096 bfloat16 numbers take 25.3 us, 4.0 TB/s: instructions take half of that (about ten a number), and a
// block waits for its row's maximum between its loads and its stores.  Where rows are few it is bound by latency, hence more threads to a row then.
template <typename T>
__global__ void __launch_bounds__(1024)
quantize_rows_vec_kernel(const T* x, int8_t* q, float* scale, int K, int pitch, int early) {
    __shared__ uint32_t scratch[32];
    if (early) gfb_pdl_launch();
    gfb_pdl_wait();
    const T* row = x + (size_t)blockIdx.x * K;
    const int n = K >> 3;
    Raw8<T> v[ROW_VECTORS];
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) {
        const int i = threadIdx.x + k * blockDim.x;
#pragma unroll
        for (int u = 0; u < (int)sizeof(T) / 2; u++)
            v[k].w[u] = i < n ? *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row) + (size_t)i * 8 * sizeof(T) + 16 * u) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) m = max(m, max_bits(v[k]));
    const RowScale rs(block_max_bits(m, scratch));
    int8_t* out = q + (size_t)blockIdx.x * pitch;
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i < n) {
            float f[8];
            load8(reinterpret_cast<const T*>(v[k].w), f);
            *reinterpret_cast<uint2*>(out + 8 * i) = sizeof(T) == 2 ? rs.of8_short(f) : rs.of8(f);
        }
    }
    if (threadIdx.x == 0) {
        scale[blockIdx.x] = rs.scale;
        if (pitch > K) *reinterpret_cast<uint2*>(out + K) = make_uint2(0u, 0u);      // (a pitch of whole 16 bytes is at most 8 more)
    }
}

// The same for any K and alignment, reading the row twice.
template <typename T>
__global__ void __launch_bounds__(512)
quantize_rows_kernel(const T* x, int8_t* q, float* scale, int K, int pitch, int early) {
    __shared__ uint32_t scratch[32];
    if (early) gfb_pdl_launch();
    gfb_pdl_wait();
    const T* row = x + (size_t)blockIdx.x * K;
    uint32_t m = 0;
    for (int i = threadIdx.x; i < K; i += blockDim.x) m = max(m, abs_bits(gfb_to_f32(row[i])));
    const RowScale rs(block_max_bits(m, scratch));
    int8_t* out = q + (size_t)blockIdx.x * pitch;
    for (int i = threadIdx.x; i < pitch; i += blockDim.x) out[i] = i < K ? (int8_t)rs.of(gfb_to_f32(row[i])) : (int8_t)0;
    if (threadIdx.x == 0) scale[blockIdx.x] = rs.scale;
}

// Threads of a block for rows of n vectors: as many as there can be where rows are few and wait for one another's launches, as many vectors as a thread holds otherwise.
inline int row_threads(int R, int n) {
    const int each = R <= 296 ? (n + 1023) / 1024 : ROW_VECTORS;
    const int t = ((n + each - 1) / each + 31) / 32 * 32;
    return t < 64 ? 64 : t > 1024 ? 1024 : t;
}

// early: the next kernel may start while this one runs and waits for it before it reads the rows.  A product asks for its weights ahead of that wait, so rows
// that may become weights are made with early = 0: nothing starts before they are complete.
template <typename T>
cudaError_t quantize_rows_launch(const T* x, int8_t* q, float* scale, int R, int K, int pitch, int early, cudaStream_t stream) {
    const int n = K / 8, t = row_threads(R, n);
    if (K % 8 == 0 && n <= ROW_VECTORS * t && pitch - K <= 8 && ((uintptr_t)x & 15) == 0 && ((uintptr_t)q & 15) == 0)
        return gfb_launch(quantize_rows_vec_kernel<T>, dim3(R), dim3(t), 0, stream, x, q, scale, K, pitch, early);
    return gfb_launch(quantize_rows_kernel<T>, dim3(R), dim3(K >= 2048 ? 512 : 256), 0, stream, x, q, scale, K, pitch, early);
}

}  // namespace
