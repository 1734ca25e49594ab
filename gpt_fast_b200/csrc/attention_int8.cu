// Causal grouped-query attention over a paged cache of 8-bit integers with a scale per cached row (quantize.cu).
//
// For a query q at position p, over the keys j it sees (j <= p, and p - j < window when there is one):
//     s_j = scale ks_j (q . K_j),   w_j = exp(s_j - max s),   out = sum_j (w_j vs_j) V_j / sum_j w_j
// with integers K_j, V_j and their scales ks_j, vs_j.  The scales stay out of the products: a key's joins its score, a value's its weight.
#include <cuda.h>
#include <cuda_fp16.h>

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
attention_int8_generic_kernel(const T* q, T* out, Int8KV kv, GfbBatch b, int H, int G, int d, float scale, int window, int* status) {
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

// ---- single tokens on the tensor cores: head sizes 64 and 128, pages of 64, at most 8 heads per key head -------------------------------
// A block owns (token, key head, slice of the sequence's pages) and serves all query heads of the group from one pass over the integers, which are what it
// is bound by.  A producer thread brings pages by TMA, NS of them in flight; each of four warps takes 16 of a page's 64 keys and runs an online
// softmax of its own over them, without a block-wide step until the end.
//
// Both products are mma.sync m16n8k16 in float16 with the cached integers as the A operand and the heads as its 8 columns: S^T = K q^T (16 keys x 8 heads)
// and O^T += V^T (w vs)^T (16 dims x 8 heads per chunk of 16 dims).  Two 8-bit integers become two float16 numbers in two operations (`pair`), exactly.  They
// are taken as bytes 0, 2 and bytes 1, 3 of a word, so no byte is moved: the order of the dims within a product over 16 of them is free as long as q
// has it too, and of V's transposed words the two halves are the rows of dims 2g and 2g + 1.  (As bfloat16 numbers they cost twice the integer
// operations, and the pipe for those, 74 % busy, was the limit: two sequences of 100,000 tokens 96 us, NOW so.)
// float16 has few exponents.  A query row comes times the power of two that takes its largest number to 2^14 .. 2^15: bfloat16 numbers down to 2^-32 of that
// stay exact.  The weights times their value's scale, w vs, have a reference M of their own beside the scores' reference m: the
// largest lies between 2^9 and 2^15, one 2^-26 of it keeps eleven bits.  Rounding them there is the only rounding ahead of the result's (a bfloat16 weight
// would be eight times coarser).  The sum of weights is of the unrounded ones.  Both references follow their maximum in steps, so a rescale is rare.
constexpr int DEC_WARPS = 4, DEC_THREADS = 32 * (DEC_WARPS + 1);
constexpr int PAGE = 64;
constexpr int MERGE_SLICES = 8;              // the largest portable cluster
constexpr unsigned long long WAIT_LIMIT_NS = 1000000000ull;   // a page that has not come after a second is given up
constexpr float LAG = 8.f;                   // log2 by which a score may pass the reference
constexpr float LIFT = 12.f;                 // log2 of what a weight at its reference is worth; it may pass it by 2^3
constexpr float LEAST_LOG_SCALE = -100.f;    // a smaller scale of values counts as this for the reference, which keeps 2^(m - M + LIFT) finite

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long v;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(v));
    return v;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) { asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory"); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Wait for the phase with `parity` to complete; false when the block gives up or time runs out.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status, int which) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = global_ns();
    for (;;) {
        for (int i = 0; i < 128; i++)
            if (mbar_try_wait(bar, parity)) return true;
        if (*gave_up) return false;
        if (global_ns() - t0 > WAIT_LIMIT_NS) {
            *gave_up = 1;
            gfb_report(status, GFB_ERR_WAIT_TIMEOUT, which, (int)(blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z)));
            return false;
        }
    }
}
// The same for a whole warp: one answer for all its lanes, which meet again at the aligned instructions behind it.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status, int which) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, gave_up, status, which));
}
__device__ __forceinline__ uint64_t l2_evict_first_policy() {
    uint64_t pol;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}
__device__ __forceinline__ void tma_load_2d_hint(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar), "l"(pol) : "memory");
}
// `bytes` (a multiple of 16) from a 16-byte boundary of global memory to one of shared memory
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {        // an 8 x 8 matrix of 16-bit numbers over the warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes 0 and 2 of x, signed, as two float16 numbers: a byte with its sign bit turned is the number + 128, behind 0x64 it is 1024 + that, and 1152 is taken off.
__device__ __forceinline__ uint32_t pair(uint32_t x) {
    const uint32_t a = (x & 0x00ff00ffu) ^ 0x64806480u;
    uint32_t y;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(0xE480E480u));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2_f16(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
// Byte offset of the 16-byte chunk at column `col` (a multiple of 16) of row `row` in a tile of rows of D bytes that came as lines of 128 bytes with 128-byte swizzle.
template <int D>
__device__ __forceinline__ uint32_t swz(int row, int col) {
    const int f = row * D + col, line = f >> 7;
    return (uint32_t)(line * 128 + ((((f >> 4) & 7) ^ (line & 7)) << 4));
}

template <int D, int NS>
struct DecodeSmem {
    static constexpr int TILE = PAGE * D, STAGE = 2 * TILE;            // K and V of a page
    static constexpr int OP = D + 8;                                   // floats per row of the merge area, which lies where the pages were
    static constexpr int SCALES = NS * STAGE, BARS = SCALES + NS * 2 * PAGE * 4;
    static constexpr int BYTES = 1024 + BARS + 2 * NS * 8 + NS * 4 + 16;
    static_assert(4 * 8 * OP * 4 + 64 * 4 + 8 * D * 4 + 16 * 4 <= NS * STAGE, "the merge area fits where the pages were");
};

// 2^x, 0 below 2^-126
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a warp keeps of a (token, key head) while it walks over pages: of every lane the heads 2 t4 and 2 t4 + 1 (e = 0, 1), dims 16 c + 2 g4 and + 1.
template <int D>
struct WarpRows {
    static constexpr int CH = D / 16;
    float o[CH][4];              // sums of w vs V times 2^(LIFT - M)
    float m[2], M[2];            // references of scores and of weighted scales, log2
    float l[2];                  // sums of weights, this lane's keys
    float F[2];                  // 2^(m - M + LIFT)
    uint32_t qb[CH][2];          // q as the B operand: column g4 is a head, its k numbers are the dims 4 t4 and + 2, and 4 t4 + 1 and + 3, of every 16
    float unit[2];               // what a product of integers and lifted queries is worth, log2(e) in it

    // `row`: the first of the group's query rows, `rep` of them
    __device__ __forceinline__ void start(const __nv_bfloat16* row, int rep, float scale_log2e, int g4, int t4) {
#pragma unroll
        for (int c = 0; c < CH; c++) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
        m[0] = m[1] = M[0] = M[1] = -INFINITY;
        l[0] = l[1] = F[0] = F[1] = 0.f;
        const __nv_bfloat16* qr = row + min(g4, rep - 1) * D;
        uint2 v[CH];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            v[c] = g4 < rep ? *reinterpret_cast<const uint2*>(qr + c * 16 + 4 * t4) : make_uint2(0u, 0u);
            top = max(top, max(max(v[c].x & 0x7fffu, (v[c].x >> 16) & 0x7fffu), max(v[c].y & 0x7fffu, (v[c].y >> 16) & 0x7fffu)));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // exponent of the row's largest number (of zeros, tiny and huge ones as far as the factor stays within a float's exponents)
        const int e = min(max((int)(top >> 7) - 127, -100), 100);
        const float lift = exp2f((float)(14 - e));
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const float f0 = __uint_as_float(v[c].x << 16) * lift, f1 = __uint_as_float(v[c].x & 0xffff0000u) * lift;
            const float f2 = __uint_as_float(v[c].y << 16) * lift, f3 = __uint_as_float(v[c].y & 0xffff0000u) * lift;
            qb[c][0] = pack2_f16(f0, f2);
            qb[c][1] = pack2_f16(f1, f3);
        }
        const float mine = exp2f((float)(e - 14)) * scale_log2e;
        unit[0] = __shfl_sync(0xffffffffu, mine, 8 * t4);
        unit[1] = __shfl_sync(0xffffffffu, mine, 8 * t4 + 4);
    }

    // The warp's 16 keys of a page: tiles of K and V, scales of the warp's first key on (ks, and PAGE further the values'); off: where this lane's row of the
    // four matrices that one ldmatrix takes lies, chunks 2 i and 2 i + 1.  see0, see1: whether keys g4 and g4 + 8 are seen.
    __device__ __forceinline__ void page(uint32_t kt, uint32_t vt, const uint32_t (&off)[CH / 2], const float* ks, bool see0, bool see1) {
        float sc[4] = {0.f, 0.f, 0.f, 0.f};                                 // (key g4, heads 2 t4 and + 1), (key g4 + 8, the same)
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            uint32_t r[4];
            ldsm_x4(kt + off[c / 2], r);
            mma_f16(sc, pair(r[0]), pair(r[1]), pair(r[0] >> 8), pair(r[1] >> 8), qb[c][0], qb[c][1]);
            mma_f16(sc, pair(r[2]), pair(r[3]), pair(r[2] >> 8), pair(r[3] >> 8), qb[c + 1][0], qb[c + 1][1]);
        }
        const float k0 = ks[0], k1 = ks[8], v0 = ks[PAGE], v1 = ks[PAGE + 8];
        sc[0] = see0 ? sc[0] * (k0 * unit[0]) : -INFINITY;
        sc[1] = see0 ? sc[1] * (k0 * unit[1]) : -INFINITY;
        sc[2] = see1 ? sc[2] * (k1 * unit[0]) : -INFINITY;
        sc[3] = see1 ? sc[3] * (k1 * unit[1]) : -INFINITY;
        float p[4], w[4];
        auto weigh = [&]() {
            const float r0 = m[0] == -INFINITY ? 0.f : m[0], r1 = m[1] == -INFINITY ? 0.f : m[1];
            p[0] = power2(sc[0] - r0); p[1] = power2(sc[1] - r1); p[2] = power2(sc[2] - r0); p[3] = power2(sc[3] - r1);
            w[0] = see0 ? p[0] * (v0 * F[0]) : 0.f; w[1] = see0 ? p[1] * (v0 * F[1]) : 0.f;     // an unseen key's value scale can be anything
            w[2] = see1 ? p[2] * (v1 * F[0]) : 0.f; w[3] = see1 ? p[3] * (v1 * F[1]) : 0.f;
        };
        weigh();
        const bool far = fmaxf(sc[0], sc[2]) > m[0] + LAG || fmaxf(sc[1], sc[3]) > m[1] + LAG || fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])) > 32768.f;
        if (__any_sync(0xffffffffu, far)) {
            const float lv0 = fmaxf(log2f(v0), LEAST_LOG_SCALE), lv1 = fmaxf(log2f(v1), LEAST_LOG_SCALE);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float x = fmaxf(sc[e], sc[e + 2]);
                float y = fmaxf(see0 ? sc[e] + lv0 : -INFINITY, see1 ? sc[e + 2] + lv1 : -INFINITY);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
                }
                const float now = fmaxf(m[e], x), Now = fmaxf(M[e], y);
                l[e] *= m[e] == -INFINITY ? 0.f : power2(m[e] - now);
                const float corr = M[e] == -INFINITY ? 0.f : power2(M[e] - Now);
                m[e] = now;
                M[e] = Now;
                F[e] = now == -INFINITY ? 0.f : power2(now - Now + LIFT);
#pragma unroll
                for (int c = 0; c < CH; c++) { o[c][e] *= corr; o[c][e + 2] *= corr; }
            }
            weigh();
        }
        l[0] += p[0] + p[2];
        l[1] += p[1] + p[3];
        const uint32_t wa = transposed(pack2_f16(w[0], w[1])), wb = transposed(pack2_f16(w[2], w[3]));
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            uint32_t r[4];
            ldsm_x4_trans(vt + off[c / 2], r);
            mma_f16(o[c], pair(r[0]), pair(r[0] >> 8), pair(r[1]), pair(r[1] >> 8), wa, wb);
            mma_f16(o[c + 1], pair(r[2]), pair(r[2] >> 8), pair(r[3]), pair(r[3] >> 8), wa, wb);
        }
    }

    __device__ __forceinline__ void sum_lanes() {
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
    }
};

// What the four warps of a block made of a head, brought together: the common reference of the scores, the sum of weights under it, and the factor that
// brings a warp's own sums (references m, M) there.
struct Common { float top, sum, factor; };
__device__ __forceinline__ Common common_of(const float* mw, const float* lw, int h, float m, float M) {
    Common c;
    c.top = fmaxf(fmaxf(mw[h], mw[8 + h]), fmaxf(mw[16 + h], mw[24 + h]));
    c.sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++)
        if (mw[w * 8 + h] != -INFINITY) c.sum += lw[w * 8 + h] * exp2f(mw[w * 8 + h] - c.top);
    c.factor = m == -INFINITY ? 0.f : exp2f(M - LIFT - c.top);
    return c;
}

// A page's integers and scales into a stage of the ring; a page that the table does not have is reported, its stage marked and nothing asked for.
template <int D>
__device__ __forceinline__ void fetch_page(const CUtensorMap* map_k, const CUtensorMap* map_v, const Int8KV& kv, int G, int g, int page, int slot, int index,
                                           uint32_t tile, uint32_t scales, uint32_t full, int* dead, uint64_t pol, int* status) {
    if (page < 0 || page >= kv.n_pages) {
        gfb_report(status, GFB_ERR_PAGE_TABLE, slot, index);
        *dead = 1;
        mbar_arrive(full);
        return;
    }
    *dead = 0;
    const size_t row = ((size_t)page * G + g) * PAGE;               // the page's first row in the pools
    const int line = (int)(row * D / 128);
    mbar_expect_tx(full, 2 * PAGE * D + 2 * PAGE * 4);
    tma_load_2d_hint(tile, map_k, 0, line, full, pol);
    bulk_load(scales, kv.k_scale + row, PAGE * 4, full);
    tma_load_2d_hint(tile + PAGE * D, map_v, 0, line, full, pol);
    bulk_load(scales + PAGE * 4, kv.v_scale + row, PAGE * 4, full);
}

// Few pages altogether: a block per (token, key head, slice); the slices of a (token, key head) are a cluster and merge through its shared memory.
// q [T, H, D], out [T, H * D].
template <int D, int NS>
__global__ void __launch_bounds__(DEC_THREADS, 4)
attention_int8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __nv_bfloat16* q,
                             __nv_bfloat16* out, Int8KV kv, GfbBatch b, int H, int G, float scale_log2e, int window, int splits, int* status) {
    using S = DecodeSmem<D, NS>;
    constexpr int CH = D / 16;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;      // swizzled tiles start on 1024-byte boundaries
    uint8_t* smem = smem_raw + (tiles - smem_u32(smem_raw));
    const float* scales = reinterpret_cast<const float*>(smem + S::SCALES);      // per stage 64 of the keys, 64 of the values
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS);                // per stage: full, empty
    int* dead = reinterpret_cast<int*>(bars + 2 * NS);                           // per stage: its page does not exist
    int* gave_up = dead + NS;
    const uint32_t bar0 = smem_u32(bars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
    const int t = blockIdx.x, g = blockIdx.y, z = blockIdx.z, rep = H / G;
    if (threadIdx.x == 0) {
        prefetch_map(&map_k);
        prefetch_map(&map_v);
        for (int i = 0; i < NS; i++) { mbar_init(bar0 + 16 * i, 1); mbar_init(bar0 + 16 * i + 8, DEC_WARPS); }
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    gfb_pdl_launch();
    const int s = b.tok_seq[t], slot = b.slots[s], q_off = t - b.cu_seqlens[s];
    gfb_pdl_wait();
    const int pos = b.lengths[slot] + q_off, lo = window > 0 ? max(0, pos - window + 1) : 0;
    const int first = lo / PAGE, n_pages = pos / PAGE - first + 1, per = (n_pages + splits - 1) / splits;
    const int p0 = first + z * per, n = max(0, min(per, n_pages - z * per));

    WarpRows<D> rows;
    if (warp == DEC_WARPS) {
        if (lane == 0) {
            const int* pt = kv.page_table + (size_t)slot * kv.max_pages;
            const uint64_t pol = l2_evict_first_policy();
            int next = n > 0 && p0 < kv.max_pages ? pt[p0] : -1;
            for (int i = 0; i < n; i++) {
                const int st = i % NS, page = next;
                next = i + 1 < n && p0 + i + 1 < kv.max_pages ? pt[p0 + i + 1] : -1;
                if (i >= NS && !mbar_wait(bar0 + 16 * st + 8, ((i / NS) & 1) ^ 1, gave_up, status, 301)) break;
                fetch_page<D>(&map_k, &map_v, kv, G, g, page, slot, p0 + i, tiles + st * S::STAGE, tiles + S::SCALES + st * 2 * PAGE * 4, bar0 + 16 * st, dead + st,
                              pol, status);
            }
        }
    } else {
        rows.start(q + ((size_t)t * H + g * rep) * D, rep, scale_log2e, g4, t4);
        uint32_t off[CH / 2];
#pragma unroll
        for (int c = 0; c < CH / 2; c++) off[c] = swz<D>(warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c * 32 + (lane >> 4) * 16);
        for (int i = 0; i < n; i++) {
            const int st = i % NS;
            if (!mbar_wait_warp(bar0 + 16 * st, (i / NS) & 1, gave_up, status, 300)) break;
            const uint32_t kt = tiles + st * S::STAGE;
            const int j0 = (p0 + i) * PAGE, j = j0 + warp * 16 + g4;
            const bool here = !dead[st], all = here && j0 >= lo && j0 + PAGE - 1 <= pos;       // uniform: every key of the page is seen
            rows.page(kt, kt + S::TILE, off, scales + st * 2 * PAGE + warp * 16 + g4, all || (here && j >= lo && j <= pos), all || (here && j + 8 >= lo && j + 8 <= pos));
            __syncwarp();
            if (lane == 0) mbar_arrive(bar0 + 16 * st + 8);
        }
    }
    __syncthreads();                                               // every page has been read, or the block gave up
    if (*gave_up) {
        // copies that were issued may still be landing in this block's shared memory
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 50000ull) __nanosleep(1000);
        __syncthreads();
    }

    // Merge of the four warps: they exchange (reference, sum), each brings its sums to the common reference of the scores (and, with one slice, divides them).
    float* Ow = reinterpret_cast<float*>(smem);                    // [4][8][OP]
    float* mw = Ow + 4 * 8 * S::OP;                                // [4][8]
    float* lw = mw + 32;                                           // [4][8]
    float* mine = lw + 32;                                         // [8][D]
    float* ml = mine + 8 * D;                                      // [8][2]
    if (warp < DEC_WARPS) {
        rows.sum_lanes();
        if (g4 == 0) {
            mw[warp * 8 + 2 * t4] = rows.m[0]; mw[warp * 8 + 2 * t4 + 1] = rows.m[1];
            lw[warp * 8 + 2 * t4] = rows.l[0]; lw[warp * 8 + 2 * t4 + 1] = rows.l[1];
        }
    }
    __syncthreads();
    if (warp < DEC_WARPS) {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int h = 2 * t4 + e;
            const Common c = common_of(mw, lw, h, rows.m[e], rows.M[e]);
            const float f = splits > 1 ? c.factor : c.sum == 0.f ? 0.f : c.factor / c.sum;
            float* row = Ow + (warp * 8 + h) * S::OP + 2 * g4;
#pragma unroll
            for (int i = 0; i < CH; i++) *reinterpret_cast<float2*>(row + i * 16) = make_float2(rows.o[i][e] * f, rows.o[i][e + 2] * f);
            if (warp == 0 && g4 == 0) { ml[2 * h] = c.top; ml[2 * h + 1] = c.sum; }
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < rep * (D / 2); idx += DEC_THREADS) {
        const int h = idx / (D / 2), dim = 2 * (idx - h * (D / 2)), head = g * rep + h;
        float2 acc = *reinterpret_cast<const float2*>(Ow + h * S::OP + dim);
#pragma unroll
        for (int w = 1; w < 4; w++) {
            const float2 a = *reinterpret_cast<const float2*>(Ow + (w * 8 + h) * S::OP + dim);
            acc.x += a.x;
            acc.y += a.y;
        }
        if (splits == 1) *reinterpret_cast<uint32_t*>(out + ((size_t)t * H + head) * D + dim) = pack2(acc.x, acc.y);
        else *reinterpret_cast<float2*>(mine + h * D + dim) = acc;
    }
    if (splits == 1) return;
    // each slice finishes its part of the numbers over all of them, in ascending order
    gfb_cluster_sync();
    for (int idx = z * DEC_THREADS + threadIdx.x; idx < rep * (D / 2); idx += splits * DEC_THREADS) {
        const int h = idx / (D / 2), dim = 2 * (idx - h * (D / 2)), head = g * rep + h;
        float2 part[MERGE_SLICES], row[MERGE_SLICES];
#pragma unroll
        for (int k = 0; k < MERGE_SLICES; k++)
            if (k < splits) {
                part[k] = gfb_cluster_load2(ml + 2 * h, k);
                row[k] = gfb_cluster_load2(mine + h * D + dim, k);
            }
        float top = -INFINITY, sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int k = 0; k < MERGE_SLICES; k++)
            if (k < splits) top = fmaxf(top, part[k].x);
#pragma unroll
        for (int k = 0; k < MERGE_SLICES; k++)
            if (k < splits && part[k].x != -INFINITY) {
                const float e = exp2f(part[k].x - top);
                sum = fmaf(part[k].y, e, sum);
                o0 = fmaf(row[k].x, e, o0);
                o1 = fmaf(row[k].y, e, o1);
            }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint32_t*>(out + ((size_t)t * H + head) * D + dim) = pack2(o0 * inv, o1 * inv);
    }
    gfb_cluster_sync();                                            // no block leaves while another reads its shared memory
}

// ---- many pages: every block an equal share of them ---------------------------------------------------------------
// The pages of all (token, key head) pairs, one after the other, are one row of U units; block c of C walks over the units c U / C .. (c + 1) U / C, across
// pairs, whatever the sequences' lengths are, which only the device knows: it adds them up for itself.  A pair that one block has whole is finished there; of the others every
// block leaves its sums under the common reference in scratch, slot 2 c + 1 for a pair that it begins and does not end, slot 2 c for one that it does not
// begin, and a second kernel merges a pair's blocks in ascending order.  The producer runs ahead across pairs, so the stream never stops between them.
// (A block per (token, key head, equal slice) waits for the longest sequence: 64 of 501 to 8,190 tokens 168 us, EVEN so.)
constexpr int LEAST_UNITS = 4;               // pages that a block takes at least

template <int D, int NS>
struct ShareSmem {
    static constexpr int TILE = PAGE * D, STAGE = 2 * TILE;
    static constexpr int SCALES = NS * STAGE, REFS = SCALES + NS * 2 * PAGE * 4, BARS = REFS + 64 * 4;
    static constexpr int BYTES = 1024 + BARS + 2 * NS * 8 + (NS + 4) * 4;
    static_assert(4 * 8 * D * 4 == STAGE, "a stage holds the sums of four warps");
};

// The pages that the token's query sees: first one, how many, and the positions.
struct Seen {
    int slot, pos, lo, first, n;
    __device__ __forceinline__ Seen(const GfbBatch& b, int t, int window) {
        const int s = b.tok_seq[t];
        slot = b.slots[s];
        pos = b.lengths[slot] + (t - b.cu_seqlens[s]);
        lo = window > 0 ? max(0, pos - window + 1) : 0;
        first = lo / PAGE;
        n = max(1, pos / PAGE - first + 1);
    }
};

// How the units are shared out.
constexpr int MOST_TOKENS = 4096;            // whose pages are counted where the ring of stages will be

struct Shares {
    long long U;
    int C;
    __device__ __forceinline__ Shares(long long units, int blocks) : U(units), C((int)max(1ll, min((long long)blocks, units / LEAST_UNITS))) {}
    __device__ __forceinline__ long long begin(int c) const { return (long long)c * U / C; }
    __device__ __forceinline__ int owner(long long u) const { return (int)(((u + 1) * C - 1) / U); }
};

// before [T + 1]: pages of the tokens ahead of each, and of all; scratch_o [2 gridDim.x][rep][D], scratch_ml [2 gridDim.x][rep][2].
template <int D, int NS>
__global__ void __launch_bounds__(DEC_THREADS, 4)
attention_int8_shares_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __nv_bfloat16* q,
                             __nv_bfloat16* out, float* scratch_o, float* scratch_ml, int* before,
                             Int8KV kv, GfbBatch b, int H, int G, float scale_log2e, int window, int* status) {
    using S = ShareSmem<D, NS>;
    constexpr int CH = D / 16;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t tiles = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (tiles - smem_u32(smem_raw));
    const float* scales = reinterpret_cast<const float*>(smem + S::SCALES);
    float* mw = reinterpret_cast<float*>(smem + S::REFS);                        // [4][8]
    float* lw = mw + 32;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS);
    int* dead = reinterpret_cast<int*>(bars + 2 * NS);
    int* gave_up = dead + NS;
    int* begin = gave_up + 1;                                                    // token of the block's first unit, units of it that others have, units of this block
    const uint32_t bar0 = smem_u32(bars);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t4 = lane & 3;
    const int rep = H / G, T = b.n_tokens;
    if (threadIdx.x == 0) {
        prefetch_map(&map_k);
        prefetch_map(&map_v);
        for (int i = 0; i < NS; i++) { mbar_init(bar0 + 16 * i, 1); mbar_init(bar0 + 16 * i + 8, DEC_WARPS); }
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    gfb_pdl_launch();
    gfb_pdl_wait();
    int* pages_of = reinterpret_cast<int*>(smem);                                // [T], where the ring will be
    for (int t = threadIdx.x; t < T; t += DEC_THREADS) pages_of[t] = Seen(b, t, window).n;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                 // pages come by TMA where the counts are
    __syncthreads();
    if (warp == DEC_WARPS) {
        int total = 0;
        for (int t = lane; t < T; t += 32) total += pages_of[t];
        total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
        const Shares sh((long long)total * G, (int)gridDim.x);
        const bool idle = (int)blockIdx.x >= sh.C || total == 0;
        const long long u0 = idle ? 0 : sh.begin(blockIdx.x), u1 = idle ? 0 : sh.begin(blockIdx.x + 1);
        int ahead = 0, t = 0, skip = 0;                                          // the token of the block's first unit, and its units that other blocks have
        for (int t0 = 0; t0 < T; t0 += 32) {
            const int n = t0 + lane < T ? pages_of[t0 + lane] : 0;
            int sum = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += x;
            }
            const long long mine = (long long)(ahead + sum - n) * G;             // the token's first unit
            const unsigned found = __ballot_sync(0xffffffffu, u0 < u1 && mine <= u0 && u0 < mine + (long long)n * G);
            if (found) {
                t = t0 + __ffs(found) - 1;
                skip = __shfl_sync(0xffffffffu, (int)(u0 - mine), __ffs(found) - 1);
            }
            if (blockIdx.x == 0 && t0 + lane < T) before[t0 + lane] = ahead + sum - n;
            ahead += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (blockIdx.x == 0 && lane == 0) before[T] = ahead;
        if (lane == 0) { begin[0] = t; begin[1] = skip; begin[2] = (int)(u1 - u0); }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();

    // Every warp walks over the same shares; a wait that runs out voids the results (the status says so), and the warps go on to meet at the barriers.
    int t = begin[0], left = begin[2];
    if (left > 0) {
        Seen seen(b, t, window);
        int g = begin[1] / seen.n, p = begin[1] - g * seen.n, it = 0;            // it: pages so far
        uint32_t off[CH / 2];
#pragma unroll
        for (int c = 0; c < CH / 2; c++) off[c] = swz<D>((warp & 3) * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c * 32 + (lane >> 4) * 16);
        for (;;) {
            const int n = min(seen.n - p, left);
            if (warp == DEC_WARPS) {
                if (lane == 0) {
                    const uint64_t pol = l2_evict_first_policy();
                    const int* pt = kv.page_table + (size_t)seen.slot * kv.max_pages;
                    const int p0 = seen.first + p;
                    int next = p0 < kv.max_pages ? pt[p0] : -1;
                    for (int i = 0; i < n; i++) {
                        const int k = it + i, st = k % NS, page = next;
                        next = i + 1 < n && p0 + i + 1 < kv.max_pages ? pt[p0 + i + 1] : -1;
                        if (k >= NS && !mbar_wait(bar0 + 16 * st + 8, ((k / NS) & 1) ^ 1, gave_up, status, 303)) break;
                        fetch_page<D>(&map_k, &map_v, kv, G, g, page, seen.slot, p0 + i, tiles + st * S::STAGE, tiles + S::SCALES + st * 2 * PAGE * 4, bar0 + 16 * st,
                                      dead + st, pol, status);
                    }
                }
                __syncwarp();
            } else {
                WarpRows<D> rows;
                rows.start(q + ((size_t)t * H + g * rep) * D, rep, scale_log2e, g4, t4);
                const int j1 = (seen.first + p) * PAGE;
                for (int i = 0; i < n; i++) {
                    const int st = (it + i) % NS;
                    if (!mbar_wait_warp(bar0 + 16 * st, ((it + i) / NS) & 1, gave_up, status, 302)) continue;
                    const uint32_t kt = tiles + st * S::STAGE;
                    const int j0 = j1 + i * PAGE, j = j0 + warp * 16 + g4;
                    const bool here = !dead[st], all = here && j0 >= seen.lo && j0 + PAGE - 1 <= seen.pos;
                    rows.page(kt, kt + S::TILE, off, scales + st * 2 * PAGE + warp * 16 + g4, all || (here && j >= seen.lo && j <= seen.pos),
                              all || (here && j + 8 >= seen.lo && j + 8 <= seen.pos));
                    __syncwarp();
                    if (lane == 0 && i + 1 < n) mbar_arrive(bar0 + 16 * st + 8);
                }
                // The four warps' sums meet where the share's last page was: [4][8][D], the 16 numbers of a chunk exchanged by the head's lane group so
                // that a warp's rows fall on different banks.
                const int st = (it + n - 1) % NS;
                float* Ow = reinterpret_cast<float*>(smem + st * S::STAGE);
                rows.sum_lanes();
                if (g4 == 0) {
                    mw[warp * 8 + 2 * t4] = rows.m[0]; mw[warp * 8 + 2 * t4 + 1] = rows.m[1];
                    lw[warp * 8 + 2 * t4] = rows.l[0]; lw[warp * 8 + 2 * t4 + 1] = rows.l[1];
                }
                asm volatile("barrier.cta.sync.aligned 1, 128;" ::: "memory");
                const bool whole = n == seen.n;
                const size_t part = 2 * (size_t)blockIdx.x + (p == 0 ? 1 : 0);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int h = 2 * t4 + e;
                    const Common c = common_of(mw, lw, h, rows.m[e], rows.M[e]);
                    const float f = !whole ? c.factor : c.sum == 0.f ? 0.f : c.factor / c.sum;
                    if (!whole && warp == 0 && g4 == 0 && h < rep) *reinterpret_cast<float2*>(scratch_ml + (part * rep + h) * 2) = make_float2(c.top, c.sum);
                    float* row = Ow + (warp * 8 + h) * D + 2 * g4;
#pragma unroll
                    for (int i = 0; i < CH; i++) *reinterpret_cast<float2*>(row + (i ^ t4) * 16) = make_float2(rows.o[i][e] * f, rows.o[i][e + 2] * f);
                }
                asm volatile("barrier.cta.sync.aligned 1, 128;" ::: "memory");
                for (int idx = threadIdx.x; idx < rep * (D / 2); idx += 32 * DEC_WARPS) {
                    const int h = idx / (D / 2), dim = 2 * (idx - h * (D / 2));
                    const float* at = Ow + h * D + (((dim >> 4) ^ (h >> 1)) << 4) + (dim & 15);
                    float2 x = *reinterpret_cast<const float2*>(at);
#pragma unroll
                    for (int w = 1; w < DEC_WARPS; w++) {
                        const float2 y = *reinterpret_cast<const float2*>(at + w * 8 * D);
                        x.x += y.x;
                        x.y += y.y;
                    }
                    if (whole) *reinterpret_cast<uint32_t*>(out + ((size_t)t * H + g * rep + h) * D + dim) = pack2(x.x, x.y);
                    else *reinterpret_cast<float2*>(scratch_o + (part * rep + h) * D + dim) = x;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // the next page comes by TMA where these numbers are
                __syncwarp();
                if (lane == 0) mbar_arrive(bar0 + 16 * st + 8);
            }
            it += n;
            left -= n;
            if (left <= 0) break;
            p = 0;
            if (++g == G) {
                g = 0;
                seen = Seen(b, ++t, window);
            }
        }
    }
    __syncthreads();
    if (*gave_up) {
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 50000ull) __nanosleep(1000);
    }
}

// The pairs that several blocks share, merged over them.  One block per (token, head): its four warps take every fourth of a pair's parts, in ascending order with
// four of them in flight, and what they have is added in ascending order of the warps.  blocks: of the kernel ahead.
template <int D>
__global__ void __launch_bounds__(128)
attention_int8_merge_kernel(const float* scratch_o, const float* scratch_ml, const int* before, __nv_bfloat16* out,
                            int T, int H, int G, int blocks) {
    constexpr int V = D / 32;                                     // numbers per lane
    __shared__ float refs[4][2];
    __shared__ float sums[4][D];
    gfb_pdl_launch();
    gfb_pdl_wait();
    const int t = blockIdx.x, head = blockIdx.y, rep = H / G, g = head / rep, h = head - g * rep, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ahead = before[t], n = before[t + 1] - ahead;
    if (n <= 0) return;
    const Shares sh((long long)before[T] * G, blocks);
    const long long u = (long long)ahead * G + (long long)g * n;
    const int c0 = sh.owner(u), c1 = sh.owner(u + n - 1);
    if (c0 == c1) return;
    float top = -INFINITY, sum = 0.f, o[V] = {};
    for (int c = c0 + warp; c <= c1; c += 16) {
        float2 ml[4];
        float x[4][V];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int part = min(c + 4 * k, c1);                  // (past the end: the last one again, with no weight)
            const size_t at = (2 * (size_t)part + (part == c0)) * rep + h;
            ml[k] = *reinterpret_cast<const float2*>(scratch_ml + at * 2);
            if (c + 4 * k > c1) ml[k] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int v = 0; v < V; v++) x[k][v] = scratch_o[at * D + lane + 32 * v];
        }
        float now = top;
#pragma unroll
        for (int k = 0; k < 4; k++) now = fmaxf(now, ml[k].x);
        const float down = top == -INFINITY ? 0.f : exp2f(top - now);
        top = now;
        sum *= down;
#pragma unroll
        for (int v = 0; v < V; v++) o[v] *= down;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (ml[k].x == -INFINITY) continue;
            const float w = exp2f(ml[k].x - now);
            sum = fmaf(ml[k].y, w, sum);
#pragma unroll
            for (int v = 0; v < V; v++) o[v] = fmaf(x[k][v], w, o[v]);
        }
    }
    if (lane == 0) { refs[warp][0] = top; refs[warp][1] = sum; }
#pragma unroll
    for (int v = 0; v < V; v++) sums[warp][lane + 32 * v] = o[v];
    __syncthreads();
    const float all = fmaxf(fmaxf(refs[0][0], refs[1][0]), fmaxf(refs[2][0], refs[3][0]));
    float total = 0.f, w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        w[k] = refs[k][0] == -INFINITY ? 0.f : exp2f(refs[k][0] - all);
        total = fmaf(refs[k][1], w[k], total);
    }
    for (int dim = threadIdx.x; dim < D; dim += 128) {
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) y = fmaf(sums[k][dim], w[k], y);
        out[((size_t)t * H + head) * D + dim] = __float2bfloat16_rn(total == 0.f ? 0.f : y / total);
    }
}

// ---- host side ----------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (fn == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)p;
    }
    return fn;
}

// A pool as lines of 128 bytes; a box is the 64 rows of one head of a page.
int pool_map(CUtensorMap* map, const void* pool, int n_pages, int G, int d) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return gfb_fail("gfb_attention_int8: the driver does not export cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {128, (cuuint64_t)n_pages * G * PAGE * d / 128};
    cuuint64_t strides[1] = {128};
    cuuint32_t box[2] = {128, (cuuint32_t)(PAGE * d / 128)};
    cuuint32_t estr[2] = {1, 1};
    if (dims[1] > 0x7fffffffull) return gfb_fail("gfb_attention_int8: a pool of %d pages exceeds a tensor map's coordinates", n_pages);
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return gfb_fail("gfb_attention_int8: cuTensorMapEncodeTiled failed with %d (%d pages)", (int)r, n_pages);
    return 0;
}

constexpr int MAX_DEVICES = 64;

// Shared memory beyond 48 KB is granted per kernel and device; asked for once for each.
template <typename F>
int room(F kern, size_t smem, bool (&configured)[MAX_DEVICES]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= MAX_DEVICES) return gfb_fail("gfb_attention_int8: device %d", dev);
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return gfb_fail("gfb_attention_int8: %zu bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
        configured[dev] = true;
    }
    return 0;
}

// What the host hands to the decode kernels.
struct Decode {
    const void* q;
    void* out;
    Int8KV kv;
    GfbBatch b;
    int H, G;
    float scale;
    int window;
    int* status;
    cudaStream_t stream;
};

template <int D, int NS>
int launch_decode(const Decode& a, int splits) {
    auto kern = attention_int8_decode_kernel<D, NS>;
    const size_t smem = DecodeSmem<D, NS>::BYTES;
    static bool configured[MAX_DEVICES] = {};
    if (room(kern, smem, configured)) return 1;
    CUtensorMap mk, mv;
    if (pool_map(&mk, a.kv.k_pool, a.kv.n_pages, a.G, D) || pool_map(&mv, a.kv.v_pool, a.kv.n_pages, a.G, D)) return 1;
    return gfb_check(gfb_launch_clusters(kern, dim3(a.b.n_tokens, a.G, splits), dim3(DEC_THREADS), smem, a.stream, dim3(1, 1, splits), mk, mv,
                                         (const __nv_bfloat16*)a.q, (__nv_bfloat16*)a.out, a.kv, a.b, a.H, a.G, a.scale * 1.4426950408889634f, a.window, splits,
                                         a.status), "gfb_attention_int8_decode");
}

template <int D, int NS>
int launch_shares(const Decode& a, int blocks, float* scratch) {
    auto kern = attention_int8_shares_kernel<D, NS>;
    const size_t smem = ShareSmem<D, NS>::BYTES;
    static bool configured[MAX_DEVICES] = {};
    if (room(kern, smem, configured)) return 1;
    CUtensorMap mk, mv;
    if (pool_map(&mk, a.kv.k_pool, a.kv.n_pages, a.G, D) || pool_map(&mv, a.kv.v_pool, a.kv.n_pages, a.G, D)) return 1;
    const int rep = a.H / a.G;
    float* ml = scratch + (size_t)2 * blocks * rep * D;
    int* before = (int*)(ml + (size_t)2 * blocks * rep * 2);
    if (gfb_check(gfb_launch(kern, dim3(blocks), dim3(DEC_THREADS), smem, a.stream, mk, mv, (const __nv_bfloat16*)a.q, (__nv_bfloat16*)a.out, scratch, ml, before, a.kv,
                             a.b, a.H, a.G, a.scale * 1.4426950408889634f, a.window, a.status), "gfb_attention_int8_decode (shares)")) return 1;
    return gfb_check(gfb_launch(attention_int8_merge_kernel<D>, dim3(a.b.n_tokens, a.H), dim3(128), 0, a.stream, (const float*)scratch, (const float*)ml, (const int*)before,
                                (__nv_bfloat16*)a.out, a.b.n_tokens, a.H, a.G, blocks), "gfb_attention_int8_decode (merge)");
}

}  // namespace

// One new token per sequence, bfloat16, d 64 or 128, pages of 64, at most 8 heads per key head.  Without scratch each sequence in `splits` equal slices (1 to 8),
// which merge within a cluster of blocks.  With scratch (float32 [2 blocks (H / G) (d + 2) + n_tokens + 1]) all pages in equal shares for `blocks` blocks.
GFB_API int gfb_attention_int8_decode(const void* q, void* out, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                                      const int* page_table, int max_pages, int page_size, int n_pages,
                                      const int* cu_seqlens, const int* tok_seq, const int* slots, const int* lengths, int n_seqs, int n_tokens,
                                      int H, int G, int d, float scale, int window, int splits, int blocks, float* scratch, int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if ((d != 64 && d != 128) || page_size != PAGE) return gfb_fail("gfb_attention_int8_decode: heads of %d, pages of %d", d, page_size);
    if (G <= 0 || H % G || H / G > 8 || G > 65535) return gfb_fail("gfb_attention_int8_decode: %d heads over %d", H, G);
    if (scratch == nullptr ? splits < 1 || splits > MERGE_SLICES : blocks < 1 || n_tokens > MOST_TOKENS) return gfb_fail("gfb_attention_int8_decode: %d slices, %d blocks, %d tokens", splits, blocks, n_tokens);
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_scale | (uintptr_t)v_scale | (uintptr_t)scratch) & 15)
        return gfb_fail("gfb_attention_int8_decode: everything must be 16-byte aligned");
    const Decode a{q, out, {(const int8_t*)k_pool, (const int8_t*)v_pool, k_scale, v_scale, page_table, max_pages, page_size, n_pages},
                   {cu_seqlens, tok_seq, slots, lengths, n_seqs, n_tokens}, H, G, scale, window, status, stream};
    if (scratch != nullptr) return d == 128 ? launch_shares<128, 3>(a, blocks, scratch) : launch_shares<64, 6>(a, blocks, scratch);
    return d == 128 ? launch_decode<128, 3>(a, splits) : launch_decode<64, 6>(a, splits);
}

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
