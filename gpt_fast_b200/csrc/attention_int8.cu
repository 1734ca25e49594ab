// Causal grouped-query attention over a paged cache of 8-bit integers with a scale per cached row (quantize.cu).
//
// For a query q at position p, over the keys j it sees (j <= p, and p - j < window when there is one):
//     s_j = scale ks_j (q . K_j),   w_j = exp(s_j - max s),   out = sum_j (w_j vs_j) V_j / sum_j w_j
// with integers K_j, V_j and their scales ks_j, vs_j.  The scales stay out of the products: a key's joins its score, a value's its weight.
#include "common.cuh"

GFB_DEFINE_LAST_ERROR()

namespace {

struct Int8KV {
    const int8_t *k_pool, *v_pool;      // [n_pages][G][page][d]
    const float *k_scale, *v_scale;     // [n_pages][G][page]
    const int* page_table;              // [n_slots][max_pages]
    int max_pages, page_size, n_pages;
};

constexpr int CHUNK = 128;      // keys per step = threads per block
constexpr int MAX_DPT = 4;      // head_dim <= CHUNK * MAX_DPT

// Any head size, number of heads, page size and mix of lengths, both types.  One block per (token, query head); keys in chunks of 128 of the absolute
// position with an online softmax between them, so a query's result is the same bits in any batch.
template <typename T>
__global__ void __launch_bounds__(CHUNK)
attention_int8_generic_kernel(const T* __restrict__ q, T* __restrict__ out, Int8KV kv, GfbBatch b, int H, int G, int d, float scale, int window, int* status) {
    extern __shared__ __align__(16) float smem[];
    float* qs = smem;              // [d]
    __shared__ float ps[CHUNK];    // w_j vs_j
    __shared__ float scratch[32];
    __shared__ long long row_at[CHUNK];
    gfb_pdl_launch();
    gfb_pdl_wait();
    const int t = blockIdx.x, h = blockIdx.y, g = h / (H / G), tid = threadIdx.x;
    const int s = b.tok_seq[t], slot = b.slots[s], pos = b.lengths[slot] + (t - b.cu_seqlens[s]);
    const int lo = window > 0 ? max(0, pos - window + 1) : 0;
    const int* pt = kv.page_table + (size_t)slot * kv.max_pages;
    const T* qrow = q + ((size_t)t * H + h) * d;
    for (int i = tid; i < d; i += CHUNK) qs[i] = gfb_to_f32(qrow[i]) * scale;
    float m_run = -INFINITY, l_run = 0.f, acc[MAX_DPT] = {};
    for (int c0 = lo / CHUNK * CHUNK; c0 <= pos; c0 += CHUNK) {
        __syncthreads();           // qs ready (first pass); ps and row_at free (later passes)
        const int j = c0 + tid;
        bool live = j >= lo && j <= pos;
        long long row = -1;
        if (live) {
            const int pi = j / kv.page_size;
            const int page = pi < kv.max_pages ? pt[pi] : -1;
            if (page < 0 || page >= kv.n_pages) {
                gfb_report(status, GFB_ERR_PAGE_TABLE, slot, pi);
                live = false;
            } else row = ((long long)page * G + g) * kv.page_size + (j - pi * kv.page_size);
        }
        row_at[tid] = row;
        float sc = -INFINITY, vs = 0.f;
        if (live) {
            const int8_t* k = kv.k_pool + row * d;
            float dot = 0.f;
            for (int i = 0; i < d; i++) dot = fmaf(qs[i], (float)k[i], dot);
            sc = dot * kv.k_scale[row];
            vs = kv.v_scale[row];
        }
        const float m_new = fmaxf(m_run, gfb_block_max(sc, scratch));
        const float p = live ? expf(sc - m_new) : 0.f;
        ps[tid] = live ? p * vs : 0.f;
        const float l_chunk = gfb_block_sum(p, scratch);       // also orders the stores to ps and row_at
        const float corr = m_run == -INFINITY ? 0.f : expf(m_run - m_new);
        l_run = l_run * corr + l_chunk;
        m_run = m_new;
        const int nkeys = min(CHUNK, pos - c0 + 1);
#pragma unroll
        for (int r = 0; r < MAX_DPT; r++) {
            const int dim = tid + r * CHUNK;
            if (dim < d) {
                float a = acc[r] * corr;
                for (int u = 0; u < nkeys; u++)
                    if (row_at[u] >= 0) a = fmaf(ps[u], (float)kv.v_pool[row_at[u] * d + dim], a);
                acc[r] = a;
            }
        }
    }
#pragma unroll
    for (int r = 0; r < MAX_DPT; r++) {
        const int dim = tid + r * CHUNK;
        if (dim < d) out[((size_t)t * H + h) * d + dim] = gfb_from_f32<T>(l_run == 0.f ? 0.f : acc[r] / l_run);
    }
}

}  // namespace

// q [T, H, d] and out [T, H * d] of type dt.  Any d up to 512, any page size.
GFB_API int gfb_attention_int8_generic(const void* q, void* out, int dt, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                                       const int* page_table, int max_pages, int page_size, int n_pages,
                                       const int* cu_seqlens, const int* tok_seq, const int* slots, const int* lengths, int n_seqs, int n_tokens,
                                       int H, int G, int d, float scale, int window, int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (d <= 0 || d > CHUNK * MAX_DPT) return gfb_fail("gfb_attention_int8: head size %d (at most %d)", d, CHUNK * MAX_DPT);
    if (G <= 0 || H % G || H > 65535) return gfb_fail("gfb_attention_int8: %d heads over %d", H, G);
    Int8KV kv{(const int8_t*)k_pool, (const int8_t*)v_pool, k_scale, v_scale, page_table, max_pages, page_size, n_pages};
    GfbBatch b{cu_seqlens, tok_seq, slots, lengths, n_seqs, n_tokens};
    dim3 grid(n_tokens, H);
    cudaError_t e;
    if (dt == GFB_BF16) e = gfb_launch(attention_int8_generic_kernel<__nv_bfloat16>, grid, dim3(CHUNK), d * 4, stream, (const __nv_bfloat16*)q, (__nv_bfloat16*)out, kv, b, H, G, d, scale, window, status);
    else if (dt == GFB_F32) e = gfb_launch(attention_int8_generic_kernel<float>, grid, dim3(CHUNK), d * 4, stream, (const float*)q, (float*)out, kv, b, H, G, d, scale, window, status);
    else return gfb_fail("gfb_attention_int8: unknown type %d", dt);
    return gfb_check(e, "gfb_attention_int8");
}
