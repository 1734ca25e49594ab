// Rows of 8-bit integers with one scale each: what the 8-bit products multiply and the 8-bit cache holds.
//
// A row x becomes scale = m / 127, m = max |x_i|, and the integers q_i nearest to 127 x_i / m (ties to even), so that q_i scale is within
// scale / 2 of x_i and |q_i| <= 127.  The integer is the one exact arithmetic gives for the 32-bit numbers x_i: a first 32-bit quotient is right unless it
// lies within 1e-4 of a tie, and those few are decided by comparing 254 |x_i| with an odd multiple of m in 64 bits, where both are exact.
// So the same numbers give the same integers in every kernel here, whatever order its code computes in.
// A row of zeros has scale 0.  A row that holds a NaN or an infinity has scale NaN (and integers 0): it stands for NaN as a whole.
#include "common.cuh"

GFB_DEFINE_LAST_ERROR()

namespace {

// How a row's numbers become integers; `bits`: the largest |x_i| as its 32-bit pattern, which orders like the number and puts infinity and NaN on top.
struct RowScale {
    float most, lift, inv, scale;
    bool live;                                          // finite and not all zeros
    __device__ __forceinline__ explicit RowScale(uint32_t bits) {
        most = __uint_as_float(bits);
        live = bits != 0u && bits < 0x7f800000u;
        lift = most < 0x1p-60f ? 0x1p64f : 1.f;         // keeps the reciprocal of a tiny maximum finite
        inv = live ? __fdiv_rn(127.f, most * lift) : 0.f;
        scale = bits < 0x7f800000u ? __fdiv_rn(most, 127.f) : __uint_as_float(0x7fc00000u);
    }
    __device__ __forceinline__ int of(float x) const {
        if (!live) return 0;
        const float r = __fmul_rn(__fmul_rn(x, lift), inv);
        float k = rintf(r);
        if (fabsf(r - k) > 0.4999f) {                   // next to a tie, about one number in 5,000
            const float a = fabsf(r), f = floorf(a);
            const double twice = 254.0 * (double)fabsf(x), tie = (2.0 * (double)f + 1.0) * (double)most;
            k = (twice > tie || (twice == tie && ((int)f & 1))) ? f + 1.f : f;
            k = copysignf(k, x);
        }
        return (int)k;
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

// q [R, pitch] and scale [R] of x [R, K]; the columns from K to the pitch are zeros.  One block per row.
template <typename T>
__global__ void __launch_bounds__(256)
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

// The same of h = x * rsqrt(mean(x^2) + eps) * w in 32 bits, x float32 [T, D] with pending partial sums and picked rows as in gfb_rmsnorm.
template <typename TW>
__global__ void __launch_bounds__(256)
rmsnorm_quantize_kernel(float* x, const float* pending, int S, size_t slice, const TW* w,
                        int8_t* q, float* scale, const int* rows, int D, int pitch, float eps) {
    __shared__ float fscratch[32];
    __shared__ uint32_t scratch[32];
    gfb_pdl_launch();
    gfb_pdl_wait();
    const int r = blockIdx.x;
    const size_t row = (size_t)(rows ? rows[r] : r) * D;
    float ss = 0.f;
    for (int i = threadIdx.x; i < D; i += blockDim.x) {
        float v = x[row + i];
        if (pending != nullptr) {
            for (int p = 0; p < S; p++) v += pending[(size_t)p * slice + row + i];
            x[row + i] = v;
        }
        ss = fmaf(v, v, ss);
    }
    const float rstd = rsqrtf(gfb_block_sum(ss, fscratch) / (float)D + eps);
    uint32_t m = 0;
    for (int i = threadIdx.x; i < D; i += blockDim.x) m = max(m, abs_bits(x[row + i] * rstd * gfb_to_f32(w[i])));
    const RowScale rs(block_max_bits(m, scratch));
    int8_t* out = q + (size_t)r * pitch;
    for (int i = threadIdx.x; i < pitch; i += blockDim.x) out[i] = i < D ? (int8_t)rs.of(x[row + i] * rstd * gfb_to_f32(w[i])) : (int8_t)0;
    if (threadIdx.x == 0) scale[r] = rs.scale;
}

// The cache in 8 bits: pools [n_pages][G][page][d] of integers, scales [n_pages][G][page].
struct Int8KV {
    int8_t *k_pool, *v_pool;
    float *k_scale, *v_scale;
    const int* page_table;
    int max_pages, page_size, n_pages;
};

// The page's first (head 0) row of position pos of a slot, counted in rows; -1: there is none.
__device__ __forceinline__ long long cache_row(const int* page_table, int max_pages, int page_size, int n_pages, int G, int slot, int pos) {
    const int pi = pos / page_size;
    const int page = pos >= 0 && pi < max_pages ? page_table[(size_t)slot * max_pages + pi] : -1;
    return page < 0 || page >= n_pages ? -1 : (long long)page * G * page_size + (pos - pi * page_size);
}

// Rotate q and k by the token's position, q to q_out, k and v quantised per (token, head) to the token's place in the cache.
// One warp per head of a token; the rotation rounds each product and sum by itself.
template <typename T>
__global__ void __launch_bounds__(128)
rope_append_int8_kernel(const T* qkv, T* q_out, Int8KV kv, GfbBatch b, const float* table, int table_len,
                        int H, int G, int d, int pairing, int append, int* status) {
    gfb_pdl_launch();
    gfb_pdl_wait();
    const int t = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= H + (append ? 2 * G : 0)) return;
    const int s = b.tok_seq[t], slot = b.slots[s], pos = b.lengths[slot] + (t - b.cu_seqlens[s]);
    const int half = d >> 1;
    long long row = 0;
    bool ok = pos >= 0 && pos < table_len;
    if (ok && append) {
        row = cache_row(kv.page_table, kv.max_pages, kv.page_size, kv.n_pages, G, slot, pos);
        ok = row >= 0;
    }
    if (!ok && head == 0 && lane == 0) gfb_report(status, GFB_ERR_CACHE_RANGE, t, pos);
    const T* src = qkv + ((size_t)t * (H + 2 * G) + head) * d;
    T* dst = q_out + ((size_t)t * H + head) * d;
    const bool rot = head < H + G;
    uint32_t m = 0;
    for (int pass = 0; pass < 2; pass++) {
        const RowScale rs(pass ? warp_max_bits(m) : 0u);
        int8_t* o8 = nullptr;
        if (ok && head >= H) {
            const int g = head < H + G ? head - H : head - H - G;
            const size_t at = (size_t)row + (size_t)g * kv.page_size;
            o8 = (head < H + G ? kv.k_pool : kv.v_pool) + at * d;
            if (pass && lane == 0) (head < H + G ? kv.k_scale : kv.v_scale)[at] = rs.scale;
        }
        for (int i = lane; i < half; i += 32) {
            const int i0 = rot && pairing == 1 ? i : 2 * i, i1 = rot && pairing == 1 ? i + half : 2 * i + 1;
            float x0 = gfb_to_f32(src[i0]), x1 = gfb_to_f32(src[i1]);
            if (rot && ok) {
                const float c = table[((size_t)pos * half + i) * 2], sn = table[((size_t)pos * half + i) * 2 + 1];
                const float y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, sn)), y1 = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, sn));
                x0 = y0;
                x1 = y1;
            }
            if (head < H) {
                if (pass) continue;
                dst[i0] = gfb_from_f32<T>(ok ? x0 : 0.f);       // q stays defined so that later kernels read no garbage
                dst[i1] = gfb_from_f32<T>(ok ? x1 : 0.f);
            } else if (!pass) {
                m = max(m, max(abs_bits(x0), abs_bits(x1)));
            } else if (o8 != nullptr) {
                o8[i0] = (int8_t)rs.of(x0);
                o8[i1] = (int8_t)rs.of(x1);
            }
        }
    }
}

// What the cache holds at the places of the step's tokens: k_out, v_out [T, G, d].  One block per token.
template <typename TO>
__global__ void __launch_bounds__(256)
read_cache_int8_kernel(Int8KV kv, GfbBatch b, TO* k_out, TO* v_out, int G, int d, int* status) {
    gfb_pdl_launch();
    gfb_pdl_wait();
    const int t = blockIdx.x;
    const int s = b.tok_seq[t], slot = b.slots[s], pos = b.lengths[slot] + (t - b.cu_seqlens[s]);
    const long long row = cache_row(kv.page_table, kv.max_pages, kv.page_size, kv.n_pages, G, slot, pos);
    if (row < 0 && threadIdx.x == 0) gfb_report(status, GFB_ERR_CACHE_RANGE, t, pos);
    for (int i = threadIdx.x; i < G * d; i += blockDim.x) {
        const int g = i / d;
        const size_t at = (size_t)max(row, 0ll) + (size_t)g * kv.page_size;
        const size_t e = at * d + (i - g * d);
        const size_t o = (size_t)t * G * d + i;
        k_out[o] = gfb_from_f32<TO>(row < 0 ? 0.f : __fmul_rn((float)kv.k_pool[e], kv.k_scale[at]));
        v_out[o] = gfb_from_f32<TO>(row < 0 ? 0.f : __fmul_rn((float)kv.v_pool[e], kv.v_scale[at]));
    }
}

}  // namespace

// early: the next kernel may start while this one runs and waits for it before it reads the rows.  A product asks for its weights ahead of that wait, so rows
// that may become weights are made with early = 0: nothing starts before they are complete.
GFB_API int gfb_quantize_rows(const void* x, int dt, void* q, float* scale, int R, int K, int pitch, int early, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (K <= 0 || pitch < K) return gfb_fail("gfb_quantize_rows: rows of %d numbers with a pitch of %d", K, pitch);
    cudaError_t e;
    if (dt == GFB_BF16) e = gfb_launch(quantize_rows_kernel<__nv_bfloat16>, dim3(R), dim3(256), 0, stream, (const __nv_bfloat16*)x, (int8_t*)q, scale, K, pitch, early);
    else if (dt == GFB_F32) e = gfb_launch(quantize_rows_kernel<float>, dim3(R), dim3(256), 0, stream, (const float*)x, (int8_t*)q, scale, K, pitch, early);
    else return gfb_fail("gfb_quantize_rows: unknown type %d", dt);
    return gfb_check(e, "gfb_quantize_rows");
}

GFB_API int gfb_rmsnorm_quantize(float* x, const float* pending, int S, long slice, const void* w, int w_dt, void* q, float* scale,
                                 const int* rows, int R, int D, int pitch, float eps, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (D <= 0 || pitch < D) return gfb_fail("gfb_rmsnorm_quantize: rows of %d numbers with a pitch of %d", D, pitch);
    if (pending != nullptr && rows != nullptr) return gfb_fail("gfb_rmsnorm_quantize: pending partial sums cannot be combined with a row gather");
    cudaError_t e;
    if (w_dt == GFB_BF16) e = gfb_launch(rmsnorm_quantize_kernel<__nv_bfloat16>, dim3(R), dim3(256), 0, stream, x, pending, S, (size_t)slice, (const __nv_bfloat16*)w, (int8_t*)q, scale, rows, D, pitch, eps);
    else if (w_dt == GFB_F32) e = gfb_launch(rmsnorm_quantize_kernel<float>, dim3(R), dim3(256), 0, stream, x, pending, S, (size_t)slice, (const float*)w, (int8_t*)q, scale, rows, D, pitch, eps);
    else return gfb_fail("gfb_rmsnorm_quantize: unknown type %d", w_dt);
    return gfb_check(e, "gfb_rmsnorm_quantize");
}

// qkv [T, (H + 2G) d] and q_out [T, H, d] of type dt; the rest as gfb_rope_append, with a scale per cached row.
GFB_API int gfb_rope_append_int8(const void* qkv, void* q_out, int dt, void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                                 const int* page_table, int max_pages, int page_size, int n_pages,
                                 const int* cu_seqlens, const int* tok_seq, const int* slots, const int* lengths, int n_seqs, int n_tokens,
                                 const float* table, int table_len, int H, int G, int d, int pairing, int append, int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (d % 2) return gfb_fail("gfb_rope_append_int8: head_dim %d is odd", d);
    Int8KV kv{(int8_t*)k_pool, (int8_t*)v_pool, k_scale, v_scale, page_table, max_pages, page_size, n_pages};
    GfbBatch b{cu_seqlens, tok_seq, slots, lengths, n_seqs, n_tokens};
    dim3 grid(n_tokens, (H + (append ? 2 * G : 0) + 3) / 4);
    if (grid.y > 65535) return gfb_fail("gfb_rope_append_int8: %d heads exceed the grid", H + 2 * G);
    cudaError_t e;
    if (dt == GFB_BF16) e = gfb_launch(rope_append_int8_kernel<__nv_bfloat16>, grid, dim3(128), 0, stream, (const __nv_bfloat16*)qkv, (__nv_bfloat16*)q_out, kv, b, table, table_len, H, G, d, pairing, append, status);
    else if (dt == GFB_F32) e = gfb_launch(rope_append_int8_kernel<float>, grid, dim3(128), 0, stream, (const float*)qkv, (float*)q_out, kv, b, table, table_len, H, G, d, pairing, append, status);
    else return gfb_fail("gfb_rope_append_int8: unknown type %d", dt);
    return gfb_check(e, "gfb_rope_append_int8");
}

// k_out, v_out [T, G, d] of type dt: the values that the cache holds at the places of the step's tokens; zeros (and a status) where it has no page.
GFB_API int gfb_read_cache_int8(void* k_pool, void* v_pool, float* k_scale, float* v_scale, const int* page_table, int max_pages, int page_size, int n_pages,
                                const int* cu_seqlens, const int* tok_seq, const int* slots, const int* lengths, int n_seqs, int n_tokens,
                                void* k_out, void* v_out, int dt, int G, int d, int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    Int8KV kv{(int8_t*)k_pool, (int8_t*)v_pool, k_scale, v_scale, page_table, max_pages, page_size, n_pages};
    GfbBatch b{cu_seqlens, tok_seq, slots, lengths, n_seqs, n_tokens};
    cudaError_t e;
    if (dt == GFB_BF16) e = gfb_launch(read_cache_int8_kernel<__nv_bfloat16>, dim3(n_tokens), dim3(256), 0, stream, kv, b, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, G, d, status);
    else if (dt == GFB_F32) e = gfb_launch(read_cache_int8_kernel<float>, dim3(n_tokens), dim3(256), 0, stream, kv, b, (float*)k_out, (float*)v_out, G, d, status);
    else return gfb_fail("gfb_read_cache_int8: unknown type %d", dt);
    return gfb_check(e, "gfb_read_cache_int8");
}
