// Making 8-bit integers (int8_rows.cuh says how): rows for the 8-bit products, the norm that quantises its output, and the cache of 8-bit integers, written and read
// back.  All of it is bound by memory, and by latency in a decode step.
#include "int8_rows.cuh"

GFB_DEFINE_LAST_ERROR()

namespace {

// Rows of h = x * rsqrt(mean(x^2) + eps) * w in 32 bits, x float32 [T, D] with pending partial sums and picked rows as in gfb_rmsnorm.  One block per row, the row
// in registers (D a multiple of 8, rows aligned); the weights are fetched ahead of the wait for the kernel before.
template <typename TW>
__global__ void __launch_bounds__(1024)
rmsnorm_quantize_vec_kernel(float* x, const float* pending, int S, size_t slice, const TW* w, int8_t* q, float* scale, const int* rows, int D, int pitch, float eps) {
    __shared__ float fscratch[32];
    __shared__ uint32_t scratch[32];
    gfb_pdl_launch();
    const int r = blockIdx.x, n = D >> 3;
    uint4 wk[ROW_VECTORS][sizeof(TW) / 2];
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) {
        const int i = threadIdx.x + k * blockDim.x;
#pragma unroll
        for (int u = 0; u < (int)sizeof(TW) / 2; u++)
            if (i < n) wk[k][u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(w) + (size_t)i * 8 * sizeof(TW) + 16 * u);
    }
    gfb_pdl_wait();
    float* row = x + (size_t)(rows ? rows[r] : r) * D;
    float v[ROW_VECTORS][8];
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i < n) load8(row + 8 * i, v[k]);
    }
    if (pending != nullptr) {
        const float* p = pending + (row - x);
        for (int s = 0; s < S; s++, p += slice) {
            float a[ROW_VECTORS][8];
#pragma unroll
            for (int k = 0; k < ROW_VECTORS; k++) {
                const int i = threadIdx.x + k * blockDim.x;
                if (i < n) load8(p + 8 * i, a[k]);
            }
#pragma unroll
            for (int k = 0; k < ROW_VECTORS; k++)
                if (threadIdx.x + k * blockDim.x < n) {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[k][e] += a[k][e];
                }
        }
    }
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i < n) {
            if (pending != nullptr) {
                *reinterpret_cast<float4*>(row + 8 * i) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
                *reinterpret_cast<float4*>(row + 8 * i + 4) = make_float4(v[k][4], v[k][5], v[k][6], v[k][7]);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) ss = fmaf(v[k][e], v[k][e], ss);
        }
    }
    const float rstd = rsqrtf(gfb_block_sum(ss, fscratch) / (float)D + eps);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++)
        if (threadIdx.x + k * blockDim.x < n) {
            float f[8];
            load8(reinterpret_cast<const TW*>(&wk[k][0]), f);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[k][e] = v[k][e] * rstd * f[e];
                m = max(m, abs_bits(v[k][e]));
            }
        }
    const RowScale rs(block_max_bits(m, scratch));
    int8_t* out = q + (size_t)r * pitch;
#pragma unroll
    for (int k = 0; k < ROW_VECTORS; k++) {
        const int i = threadIdx.x + k * blockDim.x;
        if (i < n) *reinterpret_cast<uint2*>(out + 8 * i) = rs.of8(v[k]);
    }
    if (threadIdx.x == 0) {
        scale[r] = rs.scale;
        if (pitch > D) *reinterpret_cast<uint2*>(out + D) = make_uint2(0u, 0u);
    }
}

// The same for any D and alignment.
template <typename TW>
__global__ void __launch_bounds__(256)
rmsnorm_quantize_kernel(float* x, const float* pending, int S, size_t slice, const TW* w, int8_t* q, float* scale, const int* rows, int D, int pitch, float eps) {
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

// (x0, x1) turned by the angle of (cos, sin), every product and sum rounded by itself
__device__ __forceinline__ void turn(float& x0, float& x1, float c, float s) {
    const float y0 = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s)), y1 = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s));
    x0 = y0;
    x1 = y1;
}

// Rotate q and k by the token's position, q to q_out, k and v quantised per (token, head) to the token's place in the cache.
// One warp per head of a token, any even d and alignment; the rotation rounds each product and sum by itself.
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
                turn(x0, x1, c, sn);
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

// The same for heads of 64 and 128, aligned.  A lane has sixteen numbers of a head, whose pairs it turns by itself: two runs of eight at the same place of either half;
// D / 16 lanes make a head.  What bounds it is memory, and what stood in its way was latency: a row's place in the cache is found
// by four loads that wait for one another, and a block per token had little else to do meanwhile (packed prompts of 8,441 tokens, 32 query and 8 key heads of 128,
// 192 MB: 54.5 us).  So four blocks per SM go through units of a token's heads, with the rows of the next units on their way to shared
// memory (every thread fetches what it works on itself, so nothing waits for a block), and each lane of a warp finds the place of another of the
// next 32 units: 39.7 us, 4.9 TB/s.
constexpr int APPEND_WARPS = 4, HEADS_AT_ONCE = 3;

template <typename T, int N> struct alignas((N * sizeof(T) < 16 ? N * sizeof(T) : 16)) Few { T v[N]; };

__device__ __forceinline__ void copy16(uint4* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

template <typename T, int D, bool HALVES>
__global__ void __launch_bounds__(32 * APPEND_WARPS, 4)
rope_append_int8_vec_kernel(const T* qkv, T* q_out, Int8KV kv, GfbBatch b, const float* table, int table_len, int H, int G, int append, int* status) {
    constexpr int LANES = D / 16, HEADS = 32 / LANES, HALF = D / 2;      // lanes of a head, heads of a warp
    constexpr int UNIT = APPEND_WARPS * HEADS * HEADS_AT_ONCE;           // heads of a unit
    constexpr int PIECES = sizeof(T), STAGES = sizeof(T) == 2 ? 3 : 2;   // sixteen numbers are this many pieces of 16 bytes
    __shared__ uint4 ring[STAGES][HEADS_AT_ONCE][PIECES][32 * APPEND_WARPS];
    gfb_pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, li = lane % LANES, mine = warp * HEADS + lane / LANES;
    // pair i of this lane is (x[i], x[i + 8]) with pairs of halves, the head's pair 8 li + i; with neighbours it is (x[2i], x[2i + 1]), the head's pair 4 li + i
    // for the first four and D / 4 + 4 li + i - 4 for the rest
    const int at0 = 8 * li, at1 = HALF + 8 * li;
    const int heads = H + (append ? 2 * G : 0), per = (heads + UNIT - 1) / UNIT;         // per: units of a token
    const int units = b.n_tokens * per, step = gridDim.x;
    auto fetch = [&](int unit, int st) {
        if (unit < units) {
            const int t = unit / per, h0 = (unit - t * per) * UNIT + mine;
#pragma unroll
            for (int u = 0; u < HEADS_AT_ONCE; u++) {
                const int head = h0 + u * APPEND_WARPS * HEADS;
                if (head >= heads) break;
                const T* p = qkv + ((size_t)t * (H + 2 * G) + head) * D;
#pragma unroll
                for (int k = 0; k < PIECES; k++)
                    copy16(&ring[st][u][k][threadIdx.x], p + (k < PIECES / 2 ? at0 + k * (16 / PIECES) : at1 + (k - PIECES / 2) * (16 / PIECES)));
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    gfb_pdl_wait();
#pragma unroll
    for (int i = 0; i < STAGES - 1; i++) fetch(blockIdx.x + i * step, i);
    int places = -1;                                                     // of unit blockIdx.x + (i / 32 * 32 + lane) step: its position; -1: none
    long long rows = -1;                                                 // and its row in the cache
    int st = 0;
#pragma unroll 1
    for (int i = 0, unit = blockIdx.x; unit < units; i++, unit += step) {
        if ((i & 31) == 0) {
            const long long other = unit + (long long)lane * step;
            if (other < units) {
                const int t = (int)other / per, s = b.tok_seq[t], slot = b.slots[s];
                places = b.lengths[slot] + (t - b.cu_seqlens[s]);
                if (places >= table_len) places = -1;
                rows = append ? cache_row(kv.page_table, kv.max_pages, kv.page_size, kv.n_pages, G, slot, places) : 0;
            }
            __syncwarp();
        }
        const int pos = __shfl_sync(0xffffffffu, places, i & 31), t = unit / per, h0 = (unit - t * per) * UNIT;
        float4 cs[4];                                                    // (cos, sin) of two pairs each
        const float4* angles = reinterpret_cast<const float4*>(table + (size_t)max(pos, 0) * D) + (HALVES ? 4 * li : 2 * li);
#pragma unroll
        for (int k = 0; k < 4; k++) cs[k] = angles[k + (!HALVES && k >= 2 ? D / 8 - 2 : 0)];
        const long long row = __shfl_sync(0xffffffffu, rows, i & 31);
        const bool ok = pos >= 0 && row >= 0;
        if (!ok && threadIdx.x == 0 && h0 == 0) gfb_report(status, GFB_ERR_CACHE_RANGE, t, b.lengths[b.slots[b.tok_seq[t]]] + (t - b.cu_seqlens[b.tok_seq[t]]));
        fetch(unit + (STAGES - 1) * step, st == 0 ? STAGES - 1 : st - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
#pragma unroll
        for (int u = 0; u < HEADS_AT_ONCE; u++) {
            const int first = h0 + u * APPEND_WARPS * HEADS + warp * HEADS, head = first + lane / LANES;
            if (first >= heads) break;                                   // (the warp's)
            Few<T, 16> raw;
#pragma unroll
            for (int k = 0; k < PIECES; k++) reinterpret_cast<uint4*>(&raw)[k] = ring[st][u][k][threadIdx.x];
            float x[16];
#pragma unroll
            for (int k = 0; k < 16; k++) x[k] = gfb_to_f32(raw.v[k]);
            if (head < H + G) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float c = k & 1 ? cs[k >> 1].z : cs[k >> 1].x, sn = k & 1 ? cs[k >> 1].w : cs[k >> 1].y;
                    if (HALVES) turn(x[k], x[k + 8], c, sn);
                    else turn(x[2 * k], x[2 * k + 1], c, sn);
                }
            }
            if (head < H) {
                T* dst = q_out + ((size_t)t * H + head) * D;
                Few<T, 8> o[2];
#pragma unroll
                for (int k = 0; k < 16; k++) o[k >> 3].v[k & 7] = gfb_from_f32<T>(x[k]);
                if (!ok) o[0] = o[1] = Few<T, 8>{};                      // q stays defined so that later kernels read no garbage
                *reinterpret_cast<Few<T, 8>*>(dst + at0) = o[0];
                *reinterpret_cast<Few<T, 8>*>(dst + at1) = o[1];
            }
            if (first + HEADS <= H) continue;                            // the warp's are all queries
            uint32_t m = 0;
#pragma unroll
            for (int k = 0; k < 16; k++) m = max(m, abs_bits(x[k]));
#pragma unroll
            for (int o = LANES / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (head >= H && head < heads && ok) {
                const RowScale rs(m);
                const bool key = head < H + G;
                const size_t place = (size_t)row + (size_t)(head - (key ? H : H + G)) * kv.page_size;
                if (li == 0) (key ? kv.k_scale : kv.v_scale)[place] = rs.scale;
                int8_t* dst = (key ? kv.k_pool : kv.v_pool) + place * D;
                *reinterpret_cast<uint2*>(dst + at0) = rs.of8(x);
                *reinterpret_cast<uint2*>(dst + at1) = rs.of8(x + 8);
            }
            __syncwarp();
        }
        st = st + 1 == STAGES ? 0 : st + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// What the cache holds at the places of the step's tokens: k_out, v_out [T, G, d].  A block per token; VEC (sixteen, eight or one) numbers per thread at a time.  8,441 tokens, 8 heads of
// 128: 14.8 us, 3.5 TB/s; 12 behind the kernel that has just written them.
template <typename TO, int VEC>
__global__ void __launch_bounds__(128)
read_cache_int8_kernel(Int8KV kv, GfbBatch b, TO* k_out, TO* v_out, int G, int d, int* status) {
    gfb_pdl_launch();
    const int t = blockIdx.x;
    const int s = b.tok_seq[t], slot = b.slots[s], q_off = t - b.cu_seqlens[s];
    gfb_pdl_wait();
    const int pos = b.lengths[slot] + q_off;
    const long long row = cache_row(kv.page_table, kv.max_pages, kv.page_size, kv.n_pages, G, slot, pos);
    if (row < 0 && threadIdx.x == 0) gfb_report(status, GFB_ERR_CACHE_RANGE, t, pos);
    const int n = G * d / VEC;
    for (int i = threadIdx.x; i < 2 * n; i += blockDim.x) {
        const bool key = i < n;
        const int j = (key ? i : i - n) * VEC, g = j / d;
        const size_t at = (size_t)row + (size_t)g * kv.page_size;
        Few<int8_t, VEC> q = {};
        float sc = 0.f;
        if (row >= 0) {                                     // (a pool can have no row at all)
            q = *reinterpret_cast<const Few<int8_t, VEC>*>((key ? kv.k_pool : kv.v_pool) + at * d + (j - g * d));
            sc = (key ? kv.k_scale : kv.v_scale)[at];
        }
        Few<TO, VEC> o;
#pragma unroll
        for (int u = 0; u < VEC; u++) o.v[u] = gfb_from_f32<TO>(__fmul_rn((float)q.v[u], sc));
        *reinterpret_cast<Few<TO, VEC>*>((key ? k_out : v_out) + (size_t)t * G * d + j) = o;
    }
}

}  // namespace

GFB_API int gfb_quantize_rows(const void* x, int dt, void* q, float* scale, int R, int K, int pitch, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (K <= 0 || pitch < K) return gfb_fail("gfb_quantize_rows: rows of %d numbers with a pitch of %d", K, pitch);
    cudaError_t e;
    if (dt == GFB_BF16) e = quantize_rows_launch((const __nv_bfloat16*)x, (int8_t*)q, scale, R, K, pitch, 0, stream);
    else if (dt == GFB_F32) e = quantize_rows_launch((const float*)x, (int8_t*)q, scale, R, K, pitch, 0, stream);
    else return gfb_fail("gfb_quantize_rows: unknown type %d", dt);
    return gfb_check(e, "gfb_quantize_rows");
}

GFB_API int gfb_rmsnorm_quantize(float* x, const float* pending, int S, long slice, const void* w, int w_dt, void* q, float* scale,
                                 const int* rows, int R, int D, int pitch, float eps, cudaStream_t stream) {
    if (R <= 0) return 0;
    if (D <= 0 || pitch < D) return gfb_fail("gfb_rmsnorm_quantize: rows of %d numbers with a pitch of %d", D, pitch);
    if (pending != nullptr && rows != nullptr) return gfb_fail("gfb_rmsnorm_quantize: pending partial sums cannot be combined with a row gather");
    cudaError_t e;
    const int n = D / 8, t = row_threads(R, n);
    const bool vec = D % 8 == 0 && n <= ROW_VECTORS * t && pitch - D <= 8 && (((uintptr_t)x | (uintptr_t)pending | (uintptr_t)w | (uintptr_t)q) & 15) == 0 && slice % 4 == 0;
#define GO(TW) e = vec ? gfb_launch(rmsnorm_quantize_vec_kernel<TW>, dim3(R), dim3(t), 0, stream, x, pending, S, (size_t)slice, (const TW*)w, (int8_t*)q, scale, rows, D, pitch, eps) \
                       : gfb_launch(rmsnorm_quantize_kernel<TW>, dim3(R), dim3(256), 0, stream, x, pending, S, (size_t)slice, (const TW*)w, (int8_t*)q, scale, rows, D, pitch, eps)
    if (w_dt == GFB_BF16) GO(__nv_bfloat16);
    else if (w_dt == GFB_F32) GO(float);
    else return gfb_fail("gfb_rmsnorm_quantize: unknown type %d", w_dt);
#undef GO
    return gfb_check(e, "gfb_rmsnorm_quantize");
}

// qkv [T, (H + 2G) d] and q_out [T, H, d] of type dt; the rest as gfb_rope_append, with a scale per cached row.
GFB_API int gfb_rope_append_int8(const void* qkv, void* q_out, int dt, void* k_pool, void* v_pool, float* k_scale, float* v_scale,
                                 const int* page_table, int max_pages, int page_size, int n_pages,
                                 const int* cu_seqlens, const int* tok_seq, const int* slots, const int* lengths, int n_seqs, int n_tokens,
                                 const float* table, int table_len, int H, int G, int d, int pairing, int append, int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (d % 2) return gfb_fail("gfb_rope_append_int8: head_dim %d is odd", d);
    if (table_len < 1) return gfb_fail("gfb_rope_append_int8: an empty rotary table");
    Int8KV kv{(int8_t*)k_pool, (int8_t*)v_pool, k_scale, v_scale, page_table, max_pages, page_size, n_pages};
    GfbBatch b{cu_seqlens, tok_seq, slots, lengths, n_seqs, n_tokens};
    if ((d == 64 || d == 128) && (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)table) & 15) == 0) {
        cudaError_t ve;
        const int units = n_tokens * ((H + (append ? 2 * G : 0) + APPEND_WARPS * HEADS_AT_ONCE * 512 / d - 1) / (APPEND_WARPS * HEADS_AT_ONCE * 512 / d));
        int dev = 0, sms = 148;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        const int grid = min(units, 4 * sms);
#define GO2(T, D, HALVES) gfb_launch(rope_append_int8_vec_kernel<T, D, HALVES>, dim3(grid), dim3(32 * APPEND_WARPS), 0, stream, (const T*)qkv, (T*)q_out, kv, b, table, table_len, H, G, append, status)
#define GO(T, D) ve = pairing == 1 ? GO2(T, D, true) : GO2(T, D, false)
        if (dt == GFB_BF16 && d == 128) GO(__nv_bfloat16, 128);
        else if (dt == GFB_BF16) GO(__nv_bfloat16, 64);
        else if (dt == GFB_F32 && d == 128) GO(float, 128);
        else if (dt == GFB_F32) GO(float, 64);
        else return gfb_fail("gfb_rope_append_int8: unknown type %d", dt);
#undef GO
#undef GO2
        return gfb_check(ve, "gfb_rope_append_int8");
    }
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
    const int vec = (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_out | (uintptr_t)v_out) & 15) != 0 ? 1 : d % 16 == 0 ? 16 : d % 8 == 0 ? 8 : 1;
    cudaError_t e;
#define GO(TO, V) e = gfb_launch(read_cache_int8_kernel<TO, V>, dim3(n_tokens), dim3(128), 0, stream, kv, b, (TO*)k_out, (TO*)v_out, G, d, status)
#define GO3(TO) do { if (vec == 16) GO(TO, 16); else if (vec == 8) GO(TO, 8); else GO(TO, 1); } while (0)
    if (dt == GFB_BF16) GO3(__nv_bfloat16);
    else if (dt == GFB_F32) GO3(float);
    else return gfb_fail("gfb_read_cache_int8: unknown type %d", dt);
#undef GO3
#undef GO
    return gfb_check(e, "gfb_read_cache_int8");
}
