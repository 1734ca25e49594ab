// Causal grouped-query attention over a paged cache of 8-bit integers with a scale per cached row (quantize.cu).
//
// For a query q at position p, over the keys j it sees (j <= p, and p - j < window when there is one):
//     s_j = scale ks_j (q . K_j),   w_j = exp(s_j - max s),   out = sum_j (w_j vs_j) V_j / sum_j w_j
// with integers K_j, V_j and their scales ks_j, vs_j.  For single tokens the scales stay out of the
// products: a key's joins its score, a value's its weight.  For runs of tokens they are multiplied in ahead of the products, once per key (below).
#include <cuda.h>
#include <cuda_fp16.h>
#include <float.h>

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
// operations, and the pipe for those, 74 % busy, was the limit: two sequences of 100,000 tokens 96 us, 77 so.)
// float16 has few exponents.  A query row comes times the power of two that takes its largest number to 2^14 .. 2^15: bfloat16 numbers down to 2^-32 of that
// stay exact.  The weights times their value's scale, w vs, have a reference M of their own beside the scores' reference m: the
// largest lies between 2^12 and 2^15, one 2^-26 of it keeps eleven bits.  Rounding them there is the only rounding ahead of the result's (a bfloat16 weight
// would be eight times coarser).  The sum of weights is of the unrounded ones.  Both references follow their maximum in steps, so a rescale is rare.
constexpr int DEC_WARPS = 4, DEC_THREADS = 32 * (DEC_WARPS + 1);
constexpr int PAGE = 64;
constexpr int MERGE_SLICES = 8;              // the largest portable cluster
constexpr unsigned long long WAIT_LIMIT_NS = 1000000000ull;   // a page that has not come after a second is given up
constexpr float LAG = 8.f;                   // log2 by which a score may pass the reference
constexpr float NONE = -1e30f;               // the reference ahead of the first key: below every score, and finite, so that no difference is infinity less infinity
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
__device__ __forceinline__ bool lane_waits(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status, int which) {
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
__device__ __forceinline__ bool warp_waits(uint32_t bar, uint32_t parity, volatile int* gave_up, int* status, int which) {
    return __all_sync(0xffffffffu, lane_waits(bar, parity, gave_up, status, which));
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
template <int AHEAD>                                                // AHEAD bytes behind addr
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4+%5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr), "n"(AHEAD));
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

// What a score of a query row, lifted by 2^(14 - e), is worth, log2(e) in it.  top: the bfloat16 pattern of its largest number; a row with an infinity or a NaN has no
// softmax (infinite scores of one sign would pass for keys that are not seen): NaN, which reaches every score.
__device__ __forceinline__ float unit_of(uint32_t top, int e, float scale_log2e) {
    return top >= 0x7f80u ? __uint_as_float(0x7fc00000u) : exp2f((float)(e - 14)) * scale_log2e;
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
        m[0] = m[1] = M[0] = M[1] = NONE;
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
        // exponent of the row's largest number (of zeros and tiny ones as far as the factor stays within a float's exponents)
        const int e = max((int)(top >> 7) - 127, -100);
        const float lift = exp2f((float)(14 - e));
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const float f0 = __uint_as_float(v[c].x << 16) * lift, f1 = __uint_as_float(v[c].x & 0xffff0000u) * lift;
            const float f2 = __uint_as_float(v[c].y << 16) * lift, f3 = __uint_as_float(v[c].y & 0xffff0000u) * lift;
            qb[c][0] = pack2_f16(f0, f2);
            qb[c][1] = pack2_f16(f1, f3);
        }
        const float mine = unit_of(top, e, scale_log2e);
        unit[0] = __shfl_sync(0xffffffffu, mine, 8 * t4);
        unit[1] = __shfl_sync(0xffffffffu, mine, 8 * t4 + 4);
    }

    // The warp's 16 keys of a page: the tile of K, with V's behind it, scales of the warp's first key on (ks, and PAGE further the values'); off: where this
    // lane's row of the four matrices that one ldmatrix takes lies, chunks 2 i and 2 i + 1.  ALL: every key is seen; else see0, see1: whether g4 and g4 + 8 are.
    template <bool ALL>
    __device__ __forceinline__ void page(uint32_t kt, const uint32_t (&off)[CH / 2], const float* ks, bool see0 = true, bool see1 = true) {
        float sc[4] = {0.f, 0.f, 0.f, 0.f};                                 // (key g4, heads 2 t4 and + 1), (key g4 + 8, the same)
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
            uint32_t r[4];
            ldsm_x4(kt + off[c / 2], r);
            mma_f16(sc, pair(r[0]), pair(r[1]), pair(r[0] >> 8), pair(r[1] >> 8), qb[c][0], qb[c][1]);
            mma_f16(sc, pair(r[2]), pair(r[3]), pair(r[2] >> 8), pair(r[3] >> 8), qb[c + 1][0], qb[c + 1][1]);
        }
        const float k0 = ks[0], k1 = ks[8], v0 = ks[PAGE], v1 = ks[PAGE + 8];
        sc[0] *= k0 * unit[0]; sc[1] *= k0 * unit[1]; sc[2] *= k1 * unit[0]; sc[3] *= k1 * unit[1];
        if (!ALL) {
            if (!see0) sc[0] = sc[1] = -INFINITY;
            if (!see1) sc[2] = sc[3] = -INFINITY;
        }
        float p[4], w[4];
        auto weigh = [&]() {
            p[0] = power2(sc[0] - m[0]); p[1] = power2(sc[1] - m[1]); p[2] = power2(sc[2] - m[0]); p[3] = power2(sc[3] - m[1]);
            w[0] = p[0] * (v0 * F[0]); w[1] = p[1] * (v0 * F[1]); w[2] = p[2] * (v1 * F[0]); w[3] = p[3] * (v1 * F[1]);
            if (!ALL) {                                                     // an unseen key's value scale can be anything
                if (!see0) w[0] = w[1] = 0.f;
                if (!see1) w[2] = w[3] = 0.f;
            }
        };
        weigh();
        const bool far = fmaxf(sc[0], sc[2]) > m[0] + LAG || fmaxf(sc[1], sc[3]) > m[1] + LAG || fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])) > 32768.f;
        if (__any_sync(0xffffffffu, far)) {
            const float lv0 = fmaxf(log2f(v0), LEAST_LOG_SCALE), lv1 = fmaxf(log2f(v1), LEAST_LOG_SCALE);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float x = fmaxf(sc[e], sc[e + 2]);
                float y = fmaxf(ALL || see0 ? sc[e] + lv0 : -INFINITY, ALL || see1 ? sc[e + 2] + lv1 : -INFINITY);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
                }
                const float now = fmaxf(m[e], x), Now = fmaxf(M[e], y), corr = power2(M[e] - Now);
                l[e] *= power2(m[e] - now);
                m[e] = now;
                M[e] = Now;
                F[e] = power2(now - Now + LIFT);
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
            ldsm_x4_trans<PAGE * D>(kt + off[c / 2], r);
            mma_f16(o[c], pair(r[0]), pair(r[0] >> 8), pair(r[1]), pair(r[1] >> 8), wa, wb);
            mma_f16(o[c + 1], pair(r[2]), pair(r[2] >> 8), pair(r[3]), pair(r[3] >> 8), wa, wb);
        }
    }

    // The same for a page whose first position is j0, of which [lo, pos] are seen; none of a dead one.
    __device__ __forceinline__ void page_at(uint32_t kt, const uint32_t (&off)[CH / 2], const float* ks, int j0, int j, int lo, int pos, bool dead) {
        if (!dead && j0 >= lo && j0 + PAGE - 1 <= pos) page<true>(kt, off, ks);
        else page<false>(kt, off, ks, !dead && j >= lo && j <= pos, !dead && j + 8 >= lo && j + 8 <= pos);
    }

    __device__ __forceinline__ void sum_lanes() {
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
    }
};

// What the four warps of a block made of a head, brought together: the common reference of the scores, the sum of weights under it, and the factor that
// brings a warp's own sums (reference M) there.
struct Common { float top, sum, factor; };
__device__ __forceinline__ Common common_of(const float* mw, const float* lw, int h, float M) {
    Common c;
    c.top = fmaxf(fmaxf(mw[h], mw[8 + h]), fmaxf(mw[16 + h], mw[24 + h]));
    c.sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) c.sum = fmaf(lw[w * 8 + h], power2(mw[w * 8 + h] - c.top), c.sum);
    c.factor = power2(M - LIFT - c.top);
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
                if (i >= NS && !lane_waits(bar0 + 16 * st + 8, ((i / NS) & 1) ^ 1, gave_up, status, 301)) break;
                fetch_page<D>(&map_k, &map_v, kv, G, g, page, slot, p0 + i, tiles + st * S::STAGE, tiles + S::SCALES + st * 2 * PAGE * 4, bar0 + 16 * st, dead + st,
                              pol, status);
            }
        }
    } else {
        rows.start(q + ((size_t)t * H + g * rep) * D, rep, scale_log2e, g4, t4);
        uint32_t off[CH / 2];
#pragma unroll
        for (int c = 0; c < CH / 2; c++) off[c] = swz<D>(warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c * 32 + (lane >> 4) * 16);
        int st = 0, j0 = p0 * PAGE;
        uint32_t ph = 0;
        for (int i = 0; i < n; i++, j0 += PAGE) {
            if (!warp_waits(bar0 + 16 * st, ph, gave_up, status, 300)) break;
            rows.page_at(tiles + st * S::STAGE, off, scales + st * 2 * PAGE + warp * 16 + g4, j0, j0 + warp * 16 + g4, lo, pos, dead[st] != 0);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar0 + 16 * st + 8);
            if (++st == NS) { st = 0; ph ^= 1u; }
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
            const Common c = common_of(mw, lw, h, rows.M[e]);
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
        float top = NONE, sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int k = 0; k < MERGE_SLICES; k++)
            if (k < splits) top = fmaxf(top, part[k].x);
#pragma unroll
        for (int k = 0; k < MERGE_SLICES; k++)
            if (k < splits) {
                const float e = power2(part[k].x - top);
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
// (A block per (token, key head, equal slice) waits for the longest sequence: 64 of 501 to 8,190 tokens take 119 to 153 us, by the
// number of slices, and 106 so, 5.5 TB/s.)
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
    __device__ __forceinline__ Shares(long long units, int blocks, int least = LEAST_UNITS) : U(units), C((int)max(1ll, min((long long)blocks, units / least))) {}
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
        int g = begin[1] / seen.n, p = begin[1] - g * seen.n, st = 0;            // st, ph: the next page's stage and the phase of its barriers
        uint32_t ph = 0;
        bool again = false;                                                      // the producer: the ring has been filled once
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
                        const int page = next;
                        next = i + 1 < n && p0 + i + 1 < kv.max_pages ? pt[p0 + i + 1] : -1;
                        if (again && !lane_waits(bar0 + 16 * st + 8, ph ^ 1u, gave_up, status, 303)) break;
                        fetch_page<D>(&map_k, &map_v, kv, G, g, page, seen.slot, p0 + i, tiles + st * S::STAGE, tiles + S::SCALES + st * 2 * PAGE * 4, bar0 + 16 * st,
                                      dead + st, pol, status);
                        if (++st == NS) { st = 0; ph ^= 1u; again = true; }
                    }
                }
                __syncwarp();
            } else {
                WarpRows<D> rows;
                rows.start(q + ((size_t)t * H + g * rep) * D, rep, scale_log2e, g4, t4);
                int j0 = (seen.first + p) * PAGE, last = st;
                for (int i = 0; i < n; i++, j0 += PAGE) {
                    last = st;
                    if (warp_waits(bar0 + 16 * st, ph, gave_up, status, 302)) {
                        rows.page_at(tiles + st * S::STAGE, off, scales + st * 2 * PAGE + warp * 16 + g4, j0, j0 + warp * 16 + g4, seen.lo, seen.pos, dead[st] != 0);
                        __syncwarp();
                        if (lane == 0 && i + 1 < n) mbar_arrive(bar0 + 16 * st + 8);
                    }
                    if (++st == NS) { st = 0; ph ^= 1u; }
                }
                // The four warps' sums meet where the share's last page was: [4][8][D], the 16 numbers of a chunk exchanged by the head's lane group so
                // that a warp's rows fall on different banks.
                float* Ow = reinterpret_cast<float*>(smem + last * S::STAGE);
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
                    const Common c = common_of(mw, lw, h, rows.M[e]);
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
                if (lane == 0) mbar_arrive(bar0 + 16 * last + 8);
            }
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
    float top = NONE, sum = 0.f, o[V] = {};
    for (int c = c0 + warp; c <= c1; c += 16) {
        float2 ml[4];
        float x[4][V];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int part = min(c + 4 * k, c1);                  // (past the end: the last one again, with no weight)
            const size_t at = (2 * (size_t)part + (part == c0)) * rep + h;
            ml[k] = *reinterpret_cast<const float2*>(scratch_ml + at * 2);
            if (c + 4 * k > c1) ml[k] = make_float2(NONE, 0.f);
#pragma unroll
            for (int v = 0; v < V; v++) x[k][v] = scratch_o[at * D + lane + 32 * v];
        }
        float now = top;
#pragma unroll
        for (int k = 0; k < 4; k++) now = fmaxf(now, ml[k].x);
        const float down = power2(top - now);
        top = now;
        sum *= down;
#pragma unroll
        for (int v = 0; v < V; v++) o[v] *= down;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float w = c + 4 * k <= c1 ? power2(ml[k].x - now) : 0.f;
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
        w[k] = power2(refs[k][0] - all);
        total = fmaf(refs[k][1], w[k], total);
    }
    for (int dim = threadIdx.x; dim < D; dim += 128) {
        float y = 0.f;
#pragma unroll
        for (int k = 0; k < 4; k++) y = fmaf(sums[k][dim], w[k], y);
        out[((size_t)t * H + head) * D + dim] = __float2bfloat16_rn(total == 0.f ? 0.f : y / total);
    }
}

// ---- runs of new tokens on tcgen05: head sizes 64 and 128, pages of 64 ----------------------------------------------------------------
// A work item is two tiles of 128 rows, a row being (token, head of the group): 2 TQ consecutive tokens of one sequence and key head, TQ = 128 / (heads per
// group), against all of its keys or a part of them (PromptPlan).  Blocks are persistent, one per SM.  Per 128 keys:
//
//   converters (7 warps)    K and V from the cache through registers into shared memory as float16, with the 128-byte swizzle the tensor cores read: integers
//                           (`pair`) times their row's scale over a power of two that the 128 rows share, k_ref and v_ref
//   MMA (one thread)        S = Q K^T (128 x 128, A and B from shared memory) and O += W V (W from tensor memory, V as it lies, [key][dim]); the pipe
//                           alternates between the two tiles, so one's softmax runs under the other's products
//   softmax (8 warps per tile, two threads per row, 64 keys each)   s = S unit k_ref;  W = 2^(s + log2 v_ref - M + LIFT) as float16, over the first half of the
//                           thread's own scores;  l += W / v_ref
//
// Here scales are multiplied in ahead of the products, where a key's is needed once and not once per query: the number an integer and its scale stand for
// is rounded to float16, half a step being 2^-11 of it, an eighth of what a bfloat16 cache has.  (With the scales applied to scores and weights, exactly, the
// softmax warps took 2.3 times the instructions, two thirds of their loads from shared memory among them, and the step 476 us.)  The scale itself
// enters as two float16 numbers, so its own rounding does not add up over a row.  Queries are float16 times a power of two per row, as in the single-token
// kernel; M, the reference of weights with v_ref, follows their maximum in steps of 2^3 or more, and a weight is off by half a step of its own and 2^-37 of the row's largest
// (2^-25 where v_ref is as far above the values that the row sees as V_SPREAD allows).
// float16 has five bits of exponent, so this holds while the scales of a block's keys are within 2^K_SPREAD of their largest and those of its values within 2^V_SPREAD, zeros
// aside.  Beyond, one key would decide what is left of another for rows that do not see it.  A block of threads that met such
// keys goes through its items once more with powers of two per key that the softmax warps multiply in, a word of shared memory for each (WIDE): the 512 tokens behind
// 32,001 then take 1.2 ms.
// A key whose key or value scale is not finite has NaN for K and zeros for V: rows that see it become NaN through their score, and no other row meets a NaN.
// The order of four neighbouring dims is 0, 2, 1, 3 in Q, K and O, as `pair` leaves them; rows of Q are written so, rows of O read back so.
//
// What bounds it: 512 new tokens behind 32,001 cached ones, 32 query and 8 key heads of 128, take 361 to 371 us, 730 to 750 TFLOP/s, 46 % of the rate of a plain product.
// 128 keys of both tiles take about 6,100 cycles: a tile's softmax chain of 3,100 (two fetches of the scores, 64 exponentials a thread, the weights
// back) next to its products of 2,000, which share shared memory's bandwidth with the converters' stores.  Twelve packed prompts of 17 to 901 tokens with 32 key
// heads, 900 items of 1 to 8 blocks of keys, take 169 us: there an item's start and end (its queries, the first block's conversion, its rows' output) weigh as
// much as its blocks.
constexpr int ROWS = 128, KEYS = 128, KV_STAGES = 2, SC_STAGES = 4;
constexpr int LISTED = 1024;                 // pairs of tiles that a block sorts by weight; more of them come in the order of the sequences
constexpr int HALF_BYTES = 128 * 128;        // 128 rows x 64 float16
constexpr int SOFT_WARPS = 16, CONV_WARPS = 7, CONV_UNITS = 8, MMA_WARP = SOFT_WARPS + CONV_WARPS, PROMPT_THREADS = 32 * (MMA_WARP + 1);     // six warps per quarter of an SM: 80 registers each
// k_ref and v_ref are 2^ROOM below the power of two above the largest scale, so that the largest numbers are just within float16.  As exponents in a float's bits they are 2 to
// 252, so that both they and their reciprocals are normal; v_ref 37 at least, so that weights over it stay finite.
constexpr int ROOM = 8, LEAST_K_EXPONENT = 2, LEAST_V_EXPONENT = 37, MOST_EXPONENT = 252;
constexpr int K_SPREAD = 18;                 // a scale over k_ref is 2^-11 at least: its integers are normal float16 numbers, and it keeps 14 bits itself
constexpr int V_SPREAD = 12;                 // less, since M counts values as if they had the largest scale

struct PromptBars {
    unsigned long long q_full[2], q_empty[2];
    unsigned long long k_full[KV_STAGES], k_empty[KV_STAGES], v_full[KV_STAGES], v_empty[KV_STAGES];
    unsigned long long sc_full[SC_STAGES];
    unsigned long long s_full[2], p_ready[2], pv_done[2];
    uint32_t tmem_base;
    int gave_up, n_listed, wide;             // wide: scales were met that are too far apart
};
// the reference's exponent for a largest scale, by its bits
__device__ __forceinline__ int ref_exponent(uint32_t bits, int least) { return min(max((int)(bits >> 23) + 1 - ROOM, least), MOST_EXPONENT); }
__device__ __forceinline__ float of_exponent(uint32_t e) { return __uint_as_float(e << 23); }
// What a raw score is worth: the smallest normal number at least (scores are 0 below it, but what is masked, at -infinity, has to stay there), and finite (for
// scores that are 0).
__device__ __forceinline__ float worth(float x) { return x < FLT_MIN ? FLT_MIN : x > FLT_MAX ? FLT_MAX : x; }
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
// two float16 numbers x times the number hi + lo
__device__ __forceinline__ uint32_t times(uint32_t x, uint32_t hi, uint32_t lo) {
    uint32_t y;
    asm("{\n\t.reg .b32 t;\n\tmul.rn.f16x2 t, %1, %3;\n\tfma.rn.f16x2 %0, %1, %2, t;\n\t}" : "=r"(y) : "r"(x), "r"(hi), "r"(lo));
    return y;
}
// What the softmax warps have to know of 128 keys.
struct Refs {
    float k_ref, log_v_ref, inv_v_ref, unused;
    int missing[4];                          // per 32 keys: the page table has no page for them
};
template <int D>
struct PromptSmem {
    static constexpr int TILE = (D / 64) * HALF_BYTES;
    static constexpr int K = 2 * TILE, V = K + KV_STAGES * TILE, SC = V + KV_STAGES * TILE, ROWS_AT = SC + SC_STAGES * (int)sizeof(Refs);
    static constexpr int WORDS = ROWS_AT + 2 * 2 * ROWS * 4, LIST = WORDS + SC_STAGES * KEYS * 4, BEFORE = LIST + LISTED * 16, BARS = BEFORE + (LISTED + 2) * 4;
    static constexpr int BYTES = 1024 + BARS + (int)sizeof(PromptBars);
};

// K-major operand tile with 128-byte swizzle (rows of 128 bytes, 8-row groups 1024 bytes apart)
__device__ __forceinline__ uint64_t desc_kmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// MN-major: rows are keys, 64 dims per 128-byte row; the next 64 dims one half tile further (leading offset)
__device__ __forceinline__ uint64_t desc_mnmajor(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(HALF_BYTES >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// float16 x float16 -> 32-bit
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N, int b_mn_major) {
    return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t db, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
// The same load without the wait, and the wait as a separate step that names the registers, so that the compiler
// keeps every use of them behind it: several loads can then be in flight before one wait.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
          "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
          "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
          "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
        :: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr),
          "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
          "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
          "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
          "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15])),
          "r"(__float_as_uint(v[16])), "r"(__float_as_uint(v[17])), "r"(__float_as_uint(v[18])), "r"(__float_as_uint(v[19])),
          "r"(__float_as_uint(v[20])), "r"(__float_as_uint(v[21])), "r"(__float_as_uint(v[22])), "r"(__float_as_uint(v[23])),
          "r"(__float_as_uint(v[24])), "r"(__float_as_uint(v[25])), "r"(__float_as_uint(v[26])), "r"(__float_as_uint(v[27])),
          "r"(__float_as_uint(v[28])), "r"(__float_as_uint(v[29])), "r"(__float_as_uint(v[30])), "r"(__float_as_uint(v[31]))
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// two 32-bit numbers per instruction
__device__ __forceinline__ uint64_t both(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void apart(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// A pair of tiles: its sequence, its first token and that one's position, the tokens from it to the sequence's end.
struct alignas(16) TilePair { int seq, t0, pos, left; };
__device__ __forceinline__ int pairs_of(int tokens, int TQ) { return (tokens + 2 * TQ - 1) / (2 * TQ); }

// What a block's items are made of.  Few pairs (even): the key blocks of all (pair, key head), one after the other and ITEM_UNITS ahead of each for what an item costs besides,
// are one row of units, of which each block has an equal share, [first, end) here; else whole (pair, key head)s in a snake.
constexpr int ITEM_UNITS = 3;
struct PromptPlan {
    GfbBatch b;
    const TilePair* list;                    // the pairs, those with most key blocks first
    const int* before;                       // units ahead of each, and all
    int n_listed, n_x, n_items, G, TQ, window, end;      // n_listed: -1 where there is no list
    bool even;
};
// The items are sorted by weight, so blocks take them in a snake: P ascending, P descending, ...
__device__ __forceinline__ int snake_item(int pass, int block, int P) { return pass * P + ((pass & 1) ? P - 1 - block : block); }

// One work item; the same for every warp of a block.
struct PromptItem {
    int g, seq, t0;                          // key head, sequence, the first tile's first token
    int nq[2], pos0[2], lo[2], hi[2];        // per tile: tokens, first position, key blocks [lo, hi)
    int blk0, n, last_pos;                   // the item's key blocks, the last position any row sees
    int units, to_end;                       // how far the next item is, and the next (pair, key head)
    int part;                                // -1: all of the rows' keys; else where their sums under a reference of their own go
    __device__ __forceinline__ int tiles(const TilePair& p, int TQ, int window) {
        seq = p.seq;
        t0 = p.t0;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            nq[x] = max(0, min(TQ, p.left - x * TQ));
            pos0[x] = p.pos + x * TQ;
            lo[x] = hi[x] = 0;
            if (nq[x] > 0) {
                lo[x] = (window > 0 ? max(0, pos0[x] - window + 1) : 0) / KEYS;
                hi[x] = (pos0[x] + nq[x] - 1) / KEYS + 1;
            }
        }
        last_pos = pos0[0] + nq[0] + nq[1] - 1;
        return max(hi[0], hi[1]) - lo[0];                                // (the second tile's keys begin no earlier)
    }
    // The block's item at `at`, a unit (even) or a pass; false: there is none left.  n == 0: none here.
    __device__ __forceinline__ bool take(const PromptPlan& p, int at) {
        if (p.even) {
            if (at >= p.end) return false;
            int i = 0;
            for (int k = p.n_listed; k - i > 1;) {                       // the last pair that does not begin behind `at`
                const int mid = (i + k) >> 1;
                if (p.before[mid] <= at) i = mid;
                else k = mid;
            }
            const int most = tiles(p.list[i], p.TQ, p.window), all = most + ITEM_UNITS, rest = at - p.before[i];
            g = rest / all;
            const int u = rest - g * all;
            to_end = all - u;
            units = min(to_end, p.end - at);
            const int k0 = max(0, u - ITEM_UNITS), k1 = max(0, u + units - ITEM_UNITS);
            n = k1 - k0;
            blk0 = lo[0] + k0;
            part = n == most ? -1 : 2 * (int)blockIdx.x + (k0 == 0);     // a block begins at most one item that it does not end, and ends at most one that it does not begin
            return true;
        }
        const int w = snake_item(at, blockIdx.x, gridDim.x);
        if (w >= p.n_items) return false;
        const int xi = w / p.G;
        g = w - xi * p.G;
        part = -1;
        units = 1;
        if (p.n_listed >= 0) {
            n = tiles(p.list[xi], p.TQ, p.window);
        } else {                                                         // too many to sort: from a sequence's last tiles to its first
            int left = p.n_x - 1 - xi, from = 0, qlen = 0, k = 0;
            for (; k < p.b.n_seqs; k++) {
                from = p.b.cu_seqlens[k];
                qlen = p.b.cu_seqlens[k + 1] - from;
                const int nt = pairs_of(qlen, p.TQ);
                if (left < nt) break;
                left -= nt;
            }
            const int tq0 = left * 2 * p.TQ;
            n = 0;
            if (k == p.b.n_seqs) return true;
            n = tiles({k, from + tq0, p.b.lengths[p.b.slots[k]] + tq0, qlen - tq0}, p.TQ, p.window);
        }
        blk0 = lo[0];
        return true;
    }
    __device__ __forceinline__ bool active(int x, int j) const { return blk0 + j >= lo[x] && blk0 + j < hi[x]; }
};

// All threads of a block: the batch's pairs of tiles into `list`, those with most key blocks first (each is ranked by comparing it with all others, no more
// than two per thread), and their units into `before`; `found`, `keys`: room for as many, count: 0 ahead of a barrier, their number behind this.
__device__ __forceinline__ void list_pairs(const GfbBatch& b, TilePair* list, int* before, TilePair* found, ulonglong2* keys, int* count, int G, int TQ, int window) {
    for (int k = threadIdx.x; k < b.n_seqs; k += blockDim.x) {
        const int at = b.cu_seqlens[k], qlen = b.cu_seqlens[k + 1] - at, nt = pairs_of(qlen, TQ), pos = b.lengths[b.slots[k]];
        const int first = nt > 0 ? atomicAdd(count, nt) : 0;             // any order: they are sorted by weight and token
        for (int i = 0; i < nt && first + i < LISTED; i++) {
            const int tq0 = i * 2 * TQ;
            const TilePair p = {k, at + tq0, pos + tq0, qlen - tq0};
            PromptItem it;
            const int n = it.tiles(p, TQ, window);
            found[first + i] = p;
            keys[first + i] = make_ulonglong2((unsigned long long)(it.hi[0] - it.lo[0] + it.hi[1] - it.lo[1]) << 32 | (uint32_t)~p.t0, n + ITEM_UNITS);
        }
    }
    __syncthreads();
    const int n = min(*count, LISTED);
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const ulonglong2 mine = keys[i];
        int rank = 0, ahead = 0;
        for (int k = 0; k < n; k++) {
            const ulonglong2 other = keys[k];
            if (other.x > mine.x) {
                rank++;
                ahead += (int)other.y;
            }
        }
        list[rank] = found[i];
        before[rank] = ahead * G;
        if (rank == n - 1) before[n] = (ahead + (int)mine.y) * G;
    }
    if (n == 0 && threadIdx.x == 0) before[0] = 0;
    __syncthreads();
}

// Half of a row's query (dims [half D / 2, ..)) into the tile at `tile` (shared memory) as float16 times a power of two, zeros where there is none.  Two threads share
// a row, in warps that `meet`; both get what S times a key's scale is worth, log2(e) in it.
template <int D, typename Meet>
__device__ __forceinline__ float put_query(uint8_t* tile, int r, const __nv_bfloat16* src, float scale_log2e, int half, float* mine_at, const float* other_at, Meet meet) {
    uint4 v[D / 16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        v[i] = src != nullptr ? *reinterpret_cast<const uint4*>(src + half * (D / 2) + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        top = max(top, max(max(v[i].x & 0x7fffu, (v[i].x >> 16) & 0x7fffu), max(v[i].y & 0x7fffu, (v[i].y >> 16) & 0x7fffu)));
        top = max(top, max(max(v[i].z & 0x7fffu, (v[i].z >> 16) & 0x7fffu), max(v[i].w & 0x7fffu, (v[i].w >> 16) & 0x7fffu)));
    }
    *mine_at = __uint_as_float(top);                                     // (every thread of the pair reads it ahead of its next write: the scores in between wait for both)
    meet();
    top = max(top, __float_as_uint(*other_at));
    const int e = max((int)(top >> 7) - 127, -100);
    const float lift = exp2f((float)(14 - e));
#pragma unroll
    for (int k = 0; k < D / 16; k++) {
        const int i = half * (D / 16) + k;
        const float f0 = __uint_as_float(v[k].x << 16) * lift, f1 = __uint_as_float(v[k].x & 0xffff0000u) * lift;
        const float f2 = __uint_as_float(v[k].y << 16) * lift, f3 = __uint_as_float(v[k].y & 0xffff0000u) * lift;
        const float f4 = __uint_as_float(v[k].z << 16) * lift, f5 = __uint_as_float(v[k].z & 0xffff0000u) * lift;
        const float f6 = __uint_as_float(v[k].w << 16) * lift, f7 = __uint_as_float(v[k].w & 0xffff0000u) * lift;
        *reinterpret_cast<uint4*>(tile + (i >> 3) * HALF_BYTES + r * 128 + (((i & 7) ^ (r & 7)) << 4)) =
            make_uint4(pack2_f16(f0, f2), pack2_f16(f1, f3), pack2_f16(f4, f6), pack2_f16(f5, f7));
    }
    return unit_of(top, e, scale_log2e);
}

// q [T, H, D], out [T, H * D].  scratch_o, not null: even shares; parts of rows go to scratch_o [2 gridDim.x][2][ROWS][D] and scratch_ml [..][2] (M, l), and
// shared [gridDim.x] says what they are parts of.
struct alignas(16) SharedRows { int t0, left, g, last; };        // the (pair, key head) that a block begins and others, up to `last`, go on with; last < 0: none
constexpr int LEAST_BLOCKS = 4;              // units that a share has at least
struct PromptArgs {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    float *scratch_o, *scratch_ml;
    SharedRows* shared;
    Int8KV kv;
    GfbBatch b;
    int H, G;
    float scale_log2e;
    int window, n_x;
    int* status;
};
// Where a warp's role is: key blocks ahead of the item, items with keys, its tile's blocks (softmax), products W V issued per tile (MMA).
struct Progress {
    int g0;
    uint32_t n_item, n_done, n_pv[2];
};

// A block's items, each warp in its role.
template <int D, bool WIDE>
__device__ __forceinline__ void prompt_roles(const PromptArgs& p, Progress& done) {
    using S = PromptSmem<D>;
    constexpr int TILE = S::TILE;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
    Refs* refs = reinterpret_cast<Refs*>(smem + S::SC);
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + S::WORDS);      // WIDE, per key of a block: the exponent of its own k_ref, and 256 times that of its v_ref
    PromptBars* bars = reinterpret_cast<PromptBars*>(smem + S::BARS);
    volatile int* gave_up = &bars->gave_up;
    const __nv_bfloat16* q = p.q;
    __nv_bfloat16* out = p.out;
    float *scratch_o = p.scratch_o, *scratch_ml = p.scratch_ml;
    const Int8KV& kv = p.kv;
    const GfbBatch& b = p.b;
    int* status = p.status;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, H = p.H, G = p.G, window = p.window, rep = H / G, TQ = ROWS / rep;
    const float scale_log2e = p.scale_log2e;
    const uint32_t tmem = bars->tmem_base;
    int& g0 = done.g0;
    uint32_t &n_item = done.n_item, &n_done = done.n_done, (&n_pv)[2] = done.n_pv;
    PromptPlan plan = {b, reinterpret_cast<const TilePair*>(smem + S::LIST), reinterpret_cast<const int*>(smem + S::BEFORE), -1, p.n_x, p.n_x * G, G, TQ, window, 0, scratch_o != nullptr};
    int first = 0;
    if (p.n_x <= LISTED) {
        plan.n_listed = min(bars->n_listed, LISTED);
        plan.n_items = plan.n_listed * G;
        if (plan.even) {
            const Shares shares(plan.before[plan.n_listed], gridDim.x, LEAST_BLOCKS);
            first = (int)min(shares.begin(blockIdx.x), shares.U);
            plan.end = (int)min(shares.begin(blockIdx.x + 1), shares.U);
        }
    }
    PromptItem it;

    if (warp >= SOFT_WARPS && warp < MMA_WARP) {
        // ---- converters.  A unit is 32 keys of a block's K, or of its V; the block's eight units, K first, go round the warps.  A lane has 16 bytes of a row.
        constexpr int CH = D / 16, RPI = 32 / CH, LOADS = 32 / RPI;      // 16-byte chunks of a row, rows per load of a warp, loads
        // which row of a load's and which chunk: every eight lanes have four chunks of the same 64 dims of two neighbouring rows, whose 16-byte pieces meet
        // eight bank groups
        const int sub = CH == 8 ? ((lane >> 2) & 1) | ((lane >> 4) << 1) : lane >> 2, c = CH == 8 ? (lane & 3) | ((lane >> 1) & 4) : lane & 3;
        bool ok = true;
        for (int at = first; ok && it.take(plan, at); at += it.units) {
            if (it.n == 0) continue;
            const int slot = b.slots[it.seq];
            const int* pt = kv.page_table + (size_t)slot * kv.max_pages;
            const int last_page = it.last_pos / PAGE, first_unit = CONV_UNITS * g0, end = first_unit + CONV_UNITS * it.n;
            int U = first_unit + (warp - SOFT_WARPS + CONV_WARPS - first_unit % CONV_WARPS) % CONV_WARPS;      // the warp's first unit of the item
            // the pages of a unit's block; -1: not needed or not there
            auto pages_of = [&](int u) -> int2 {
                const int pi = (it.blk0 + ((u - first_unit) >> 3)) * 2;
                int2 p = make_int2(-1, -1);
                if (u < end) {
                    if (pi <= last_page && pi < kv.max_pages) p.x = pt[pi];
                    if (pi + 1 <= last_page && pi + 1 < kv.max_pages) p.y = pt[pi + 1];
                    if (p.x >= kv.n_pages) p.x = -1;
                    if (p.y >= kv.n_pages) p.y = -1;
                }
                return p;
            };
            auto row_of = [&](int page) -> size_t { return ((size_t)max(page, 0) * G + it.g) * PAGE; };         // a page's first row in the pools
            auto fetch = [&](int u, int2 p, uint4 (&v)[LOADS]) {
                const int page = (u & 2) ? p.y : p.x;
                const int8_t* src = ((u & 4) ? kv.v_pool : kv.k_pool) + (row_of(page) + (u & 1) * 32 + sub) * D + c * 16;
#pragma unroll
                for (int i = 0; i < LOADS; i++) v[i] = page >= 0 ? *reinterpret_cast<const uint4*>(src + i * RPI * D) : make_uint4(0u, 0u, 0u, 0u);
            };
            // scales of the 128 keys, four per lane: keys lane, lane + 32, ...
            auto fetch_scales = [&](int2 p, float (&ks)[4], float (&vs)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int page = i < 2 ? p.x : p.y;
                    const size_t row = row_of(page) + (i & 1) * 32 + lane;
                    ks[i] = page >= 0 ? kv.k_scale[row] : 0.f;
                    vs[i] = page >= 0 ? kv.v_scale[row] : 0.f;
                }
            };
            int2 page = pages_of(U), next = pages_of(U + CONV_WARPS);
            uint4 v[LOADS];
            float ks[4], vs[4];
            fetch(U, page, v);
            fetch_scales(page, ks, vs);
#pragma unroll 1
            for (; U < end; U += CONV_WARPS) {
                const int gj = U >> 3, s = gj & (KV_STAGES - 1), sc = gj & (SC_STAGES - 1), group = U & 3;
                const bool is_v = U & 4;
                // the powers of two above the largest finite scales of the block's keys, and this lane's key's scale over its own
                const int key0 = (it.blk0 + gj - g0) * KEYS + lane;
                uint32_t kt = 0, vt = 0, km = 0, vm = 0;                 // km, vm: the lane's key's (0: not there or not finite)
                float mine = 0.f;
                bool odd = false;                                        // a scale that is not finite
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool here = key0 + 32 * i <= it.last_pos;
                    const uint32_t kb = __float_as_uint(ks[i]) & 0x7fffffffu, vb = __float_as_uint(vs[i]) & 0x7fffffffu;
                    if (here && kb < 0x7f800000u) kt = max(kt, kb);
                    if (here && vb < 0x7f800000u) vt = max(vt, vb);
                    if (i == group) {
                        mine = here ? (is_v ? vs[i] : ks[i]) : 0.f;
                        odd = here && (kb >= 0x7f800000u || vb >= 0x7f800000u);
                        if (WIDE && here && !odd) {
                            km = kb;
                            vm = vb;
                        }
                    }
                }
                int ke = ref_exponent(warp_max_bits(kt), LEAST_K_EXPONENT), ve = ref_exponent(warp_max_bits(vt), LEAST_V_EXPONENT);
                if constexpr (WIDE) {                                    // of the lane's own key
                    ke = ref_exponent(km, LEAST_K_EXPONENT);
                    ve = ref_exponent(vm, LEAST_V_EXPONENT);
                } else if (mine != 0.f && __float_as_int(mine) < ((is_v ? ve - V_SPREAD : ke - K_SPREAD) + ROOM - 1) << 23) bars->wide = 1;
                const float over = mine * of_exponent(254 - (is_v ? ve : ke));
                const __half hi = __float2half_rn(over), lo = __float2half_rn(over - __half2float(hi));
                uint32_t factor = (uint32_t)__half_as_ushort(hi) | (uint32_t)__half_as_ushort(lo) << 16;
                if (odd) factor = is_v ? 0u : 0x7fff7fffu;
                const int2 after = pages_of(U + 2 * CONV_WARPS);
                ok = warp_waits(smem_u32(is_v ? &bars->v_empty[s] : &bars->k_empty[s]), ((uint32_t)(gj / KV_STAGES) & 1u) ^ 1u, gave_up, status, 401);
                if (!ok) break;
                uint8_t* line = smem + (is_v ? S::V : S::K) + s * TILE + (c >> 2) * HALF_BYTES + (group * 32 + sub) * 128;
                const int even = ((2 * (c & 3)) ^ (sub & 7)) << 4, odd_row = RPI == 4 ? even ^ 64 : even;      // (rows 4 further exchange pieces 4 further)
#pragma unroll
                for (int i = 0; i < LOADS; i++) {
                    const int piece = (i & 1) ? odd_row : even;
                    const uint32_t f = __shfl_sync(0xffffffffu, factor, sub + i * RPI);
                    const uint32_t hi2 = __byte_perm(f, f, 0x1010), lo2 = __byte_perm(f, f, 0x3232);
                    *reinterpret_cast<uint4*>(line + i * RPI * 128 + piece) = make_uint4(times(pair(v[i].x), hi2, lo2), times(pair(v[i].x >> 8), hi2, lo2),
                                                                                         times(pair(v[i].y), hi2, lo2), times(pair(v[i].y >> 8), hi2, lo2));
                    *reinterpret_cast<uint4*>(line + i * RPI * 128 + (piece ^ 16)) = make_uint4(times(pair(v[i].z), hi2, lo2), times(pair(v[i].z >> 8), hi2, lo2),
                                                                                                times(pair(v[i].w), hi2, lo2), times(pair(v[i].w >> 8), hi2, lo2));
                }
                fetch(U + CONV_WARPS, next, v);                          // in flight during what is left of this unit and the wait for the next one's place
                fetch_scales(next, ks, vs);
                if (WIDE && !is_v) words[sc * KEYS + group * 32 + lane] = (uint32_t)(ke | ve << 8);
                if (!is_v && lane == 0) {
                    const int mine_page = (group & 2) ? page.y : page.x, index = (it.blk0 + gj - g0) * 2 + (group >> 1);
                    if (group == 0) {
                        refs[sc].k_ref = of_exponent(ke);
                        refs[sc].log_v_ref = (float)(ve - 127);
                        refs[sc].inv_v_ref = of_exponent(254 - ve);
                    }
                    refs[sc].missing[group] = mine_page < 0 && index <= last_page;
                    if (mine_page < 0 && index <= last_page) gfb_report(status, GFB_ERR_PAGE_TABLE, slot, index);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");          // the tensor cores read it
                __syncwarp();
                if (lane == 0) {
                    if (!is_v) mbar_arrive(smem_u32(&bars->sc_full[sc]));
                    mbar_arrive(smem_u32(is_v ? &bars->v_full[s] : &bars->k_full[s]));
                }
                page = next;
                next = after;
            }
            g0 += it.n;
        }
    } else if (warp == MMA_WARP) {
        if (lane == 0) {
            constexpr uint32_t idesc_s = idesc_f16(ROWS, KEYS, 0), idesc_o = idesc_f16(ROWS, D, 1);
            bool ok = true;
            SharedRows begun = {0, 0, 0, -1};
            for (int at = first; ok && it.take(plan, at); at += it.units) {
                if (it.n == 0) continue;
                if (it.part >= 0 && (it.part & 1)) begun = {it.t0, it.nq[0] + it.nq[1], it.g, Shares(plan.before[plan.n_listed], gridDim.x, LEAST_BLOCKS).owner(at + it.to_end - 1)};
                for (int x = 0; x < 2 && ok; x++) ok = lane_waits(smem_u32(&bars->q_full[x]), n_item & 1u, gave_up, status, 403);
                n_item++;
                uint32_t mine[2] = {0, 0};                               // of this item
                auto issue_s = [&](int x, int j) {
                    const uint32_t kt = base + S::K + ((g0 + j) % KV_STAGES) * TILE;
#pragma unroll
                    for (int k = 0; k < D / 16; k++) {
                        const uint32_t off = (k >> 2) * HALF_BYTES;
                        umma_ss(tmem + 128 * x, desc_kmajor(base + x * TILE + off) + 2 * (k & 3), desc_kmajor(kt + off) + 2 * (k & 3), idesc_s, k != 0);
                    }
                    umma_commit(smem_u32(&bars->s_full[x]));
                };
                auto k_ready = [&](int j) {
                    return lane_waits(smem_u32(&bars->k_full[(g0 + j) % KV_STAGES]), (uint32_t)((g0 + j) / KV_STAGES) & 1u, gave_up, status, 404);
                };
                auto scores_issued = [&](int j) {                        // K of block j is free when they are done, and behind the last block Q is
                    umma_commit(smem_u32(&bars->k_empty[(g0 + j) % KV_STAGES]));
                    if (j + 1 == it.n) {
                        umma_commit(smem_u32(&bars->q_empty[0]));
                        umma_commit(smem_u32(&bars->q_empty[1]));
                    }
                };
                if (ok) ok = k_ready(0);
                if (ok) {
                    tc_fence_after();
                    if (it.active(0, 0)) issue_s(0, 0);
                    if (it.active(1, 0)) issue_s(1, 0);
                    scores_issued(0);
                }
                for (int j = 0; j < it.n && ok; j++) {
                    const int s = (g0 + j) % KV_STAGES;
                    bool k_next = false;                                 // whether K of block j + 1 has been waited for
                    ok = lane_waits(smem_u32(&bars->v_full[s]), (uint32_t)((g0 + j) / KV_STAGES) & 1u, gave_up, status, 405);
#pragma unroll
                    for (int x = 0; x < 2 && ok; x++) {
                        if (it.active(x, j)) {
                            ok = lane_waits(smem_u32(&bars->p_ready[x]), n_pv[x] & 1u, gave_up, status, 406);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int kk = 0; kk < 8; kk++)               // 16 keys per MMA: 8 columns of W (of the second 64 keys over their own scores), 2 KB of V
                                umma_ts(tmem + 256 + 128 * x, tmem + 128 * x + (kk >> 2) * 64 + (kk & 3) * 8, desc_mnmajor(base + S::V + s * TILE + kk * 2048),
                                        idesc_o, (mine[x] | (uint32_t)kk) != 0);
                            umma_commit(smem_u32(&bars->pv_done[x]));
                            n_pv[x]++;
                            mine[x]++;
                        }
                        if (j + 1 < it.n && it.active(x, j + 1)) {       // the tile's next scores, behind its W V
                            if (!k_next) { ok = k_ready(j + 1); k_next = true; if (!ok) break; tc_fence_after(); }
                            issue_s(x, j + 1);
                        }
                    }
                    if (!ok) break;
                    umma_commit(smem_u32(&bars->v_empty[s]));
                    if (j + 1 < it.n) {
                        if (!k_next) { ok = k_ready(j + 1); if (!ok) break; }
                        scores_issued(j + 1);
                    }
                }
                g0 += it.n;
            }
            if (plan.even) p.shared[blockIdx.x] = begun;
        }
    } else {
        // ---- softmax.  A wait that runs out voids the results (the status says so); the warps go on to meet at the barriers of two.
        const int x = warp >> 3, half = (warp >> 2) & 1, w4 = warp & 3;  // tile, which 64 keys, which 32 lanes of tensor memory
        const int r = w4 * 32 + lane;                                    // the thread's row
        const uint32_t lanes = tmem + ((uint32_t)(w4 * 32) << 16), col_s = lanes + 128 * x + 64 * half, col_o = lanes + 256 + 128 * x + (D / 2) * half;
        float* mine_at = reinterpret_cast<float*>(smem + S::ROWS_AT) + (x * 2 + half) * ROWS + r;
        const float* other_at = reinterpret_cast<const float*>(smem + S::ROWS_AT) + (x * 2 + (half ^ 1)) * ROWS + r;
        auto meet = [&]() { asm volatile("barrier.cta.sync.aligned %0, 64;" ::"r"(1 + x * 4 + w4) : "memory"); };     // the two warps of 32 rows
        bool ok = true;
        for (int at = first; it.take(plan, at); at += it.units) {
            if (it.n == 0) continue;
            float unit;
            {
                const int tq = r / rep;
                const size_t row = (size_t)(it.t0 + x * TQ + tq) * H + it.g * rep + (r - tq * rep);
                ok = ok && warp_waits(smem_u32(&bars->q_empty[x]), (n_item & 1u) ^ 1u, gave_up, status, 411);
                n_item++;
                unit = put_query<D>(smem + x * TILE, r, tq < it.nq[x] ? q + row * D : nullptr, scale_log2e, half, mine_at, other_at, meet);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&bars->q_full[x]));
            }
            // the tile's blocks [j, end) of the item's; of those [.., plain0) and [plain1, ..) have keys that some row does not see.  top, low: the last and the
            // first key the row sees, counted from the thread's first key of block j
            int j = max(0, it.lo[x] - it.blk0), top, low, plain0 = 0, plain1;
            const int end = min(it.n, it.hi[x] - it.blk0), was = (int)n_done;
            {
                const int row_pos = it.pos0[x] + r / rep, key0 = (it.blk0 + j) * KEYS + 64 * half;
                top = row_pos - key0;
                low = (window > 0 ? max(0, row_pos - window + 1) : 0) - key0;
                if (window > 0) plain0 = (max(0, it.pos0[x] + max(it.nq[x], 1) - window) + KEYS - 1) / KEYS - it.blk0;
                plain1 = (it.pos0[x] + 1) / KEYS - it.blk0;
            }
            const int item_n = it.n;
            float M = NONE, l = 0.f;
#pragma unroll 1
            for (; j < end; j++, top -= KEYS, low -= KEYS) {
                const Refs& ref = refs[(g0 + j) & (SC_STAGES - 1)];
                ok = ok && warp_waits(smem_u32(&bars->sc_full[(g0 + j) & (SC_STAGES - 1)]), (uint32_t)((g0 + j) / SC_STAGES) & 1u, gave_up, status, 407)
                     && warp_waits(smem_u32(&bars->s_full[x]), n_done & 1u, gave_up, status, 408);
                if (!ok) { meet(); continue; }
                tc_fence_after();
                const int gone = ref.missing[2 * half] | (ref.missing[2 * half + 1] << 1);       // 32 keys without a page: rare
                const bool need_mask = j < plain0 || j >= plain1 || gone;
                const float by = worth(unit * ref.k_ref);
                // 32 of the thread's scores, what the row does not see at -infinity.  They are fetched for the maximum and once more for the weights, since 64 of
                // them do not stay in registers.
                auto scores = [&](int c, uint32_t (&v)[32]) {
                    tmem_ld32_issue(col_s + 32 * c, v);
                    tmem_ld_wait32(v);
                    if (need_mask) {
                        const int t = (gone >> c & 1) ? -1 : top - 32 * c, f = low - 32 * c;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if (i > t || i < f) v[i] = 0xff800000u;
                    }
                };
                const uint32_t* word = words + ((g0 + j) & (SC_STAGES - 1)) * KEYS + 64 * half;
                float y;
                if constexpr (WIDE) {
                    y = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
                        uint32_t v[32];
                        scores(c, v);
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const uint32_t w = word[32 * c + i];
                            y = fmaxf(y, fmaf(__uint_as_float(v[i]), worth(unit * of_exponent(w & 255)), (float)((int)(w >> 8) - 127)));
                        }
                    }
                } else {
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
                        uint32_t v[32];
                        scores(c, v);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                    }
                    y = fmaf(fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), by, ref.log_v_ref);
                }
                *mine_at = y;
                meet();
                y = fmaxf(y, *other_at);
                const float M_new = y > M + (15.f - LIFT) ? y : M, corr = power2(M - M_new), off = (WIDE ? 0.f : ref.log_v_ref) + LIFT - M_new;
                M = M_new;
                if constexpr (WIDE) {
                    l *= corr;
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
                        uint32_t v[32], pk[16];
                        scores(c, v);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const uint32_t wa = word[32 * c + i], wb = word[32 * c + i + 1];
                            const float e0 = power2(fmaf(__uint_as_float(v[i]), worth(unit * of_exponent(wa & 255)), off));
                            const float e1 = power2(fmaf(__uint_as_float(v[i + 1]), worth(unit * of_exponent(wb & 255)), off));
                            l += e0 + e1;
                            pk[i >> 1] = pack2_f16(e0 * of_exponent(wa >> 8), e1 * of_exponent(wb >> 8));
                        }
                        tmem_st16(col_s + c * 16, pk);
                    }
                } else {
                    const uint64_t by2 = both(by, by), off2 = both(off, off);
                    uint64_t sums[2] = {0ull, 0ull};
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
                        uint32_t v[32], pk[16];
                        scores(c, v);
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float t0, t1;
                            apart(fma2(both(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), by2, off2), t0, t1);
                            const float w0 = power2(t0), w1 = power2(t1);
                            sums[(i >> 1) & 1] = add2(sums[(i >> 1) & 1], both(w0, w1));
                            pk[i >> 1] = pack2_f16(w0, w1);
                        }
                        tmem_st16(col_s + c * 16, pk);
                    }
                    float s0, s1, s2, s3;
                    apart(sums[0], s0, s1);
                    apart(sums[1], s2, s3);
                    l = fmaf(l, corr, ((s0 + s1) + (s2 + s3)) * ref.inv_v_ref);
                }
                // O follows the reference, rarely (S of this block was issued behind the tile's previous W V, so that phase is over)
                if (was != (int)n_done && __any_sync(0xffffffffu, corr != 1.f)) {
                    ok = warp_waits(smem_u32(&bars->pv_done[x]), (n_done - 1u) & 1u, gave_up, status, 409);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 64; c++) {
                        float o[32];
                        tmem_ld32(col_o + c * 32, o);
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] *= corr;
                        tmem_st32(col_o + c * 32, o);
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(smem_u32(&bars->p_ready[x]));
                n_done++;
            }
            const bool some = was != (int)n_done;                        // the part has keys of this tile
            meet();                                                      // the other half has read this one's last maximum
            *mine_at = l;
            meet();
            l = half ? *other_at + l : l + *other_at;
            meet();
            if (some) ok = ok && warp_waits(smem_u32(&bars->pv_done[x]), (n_done - 1u) & 1u, gave_up, status, 410);
            if (ok) {
                tc_fence_after();
                it.take(plan, at);                                       // once more: it did not stay in registers
                const int tq = r / rep;
                const bool row_ok = tq < it.nq[x];
                const size_t row = (size_t)(it.t0 + x * TQ + tq) * H + it.g * rep + (r - tq * rep), place = (size_t)(it.part * 2 + x) * ROWS + r;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                if (it.part >= 0 && row_ok && half == 0) *reinterpret_cast<float2*>(scratch_ml + place * 2) = make_float2(some ? M : NONE, some ? l : 0.f);
#pragma unroll 1
                for (int c = 0; c < D / 64; c++) {
                    if (!some && it.part >= 0) break;                    // nothing of this row in this part: its (M, l) say so
                    float o[32];
                    if (some) tmem_ld32(col_o + c * 32, o);
                    else {
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = 0.f;
                    }
                    if (!row_ok) continue;
                    const int dim = half * (D / 2) + c * 32;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {                    // dims 0, 2, 1, 3 of every four
                        if (it.part >= 0) {
                            float* dst = scratch_o + place * D + dim + i;
                            *reinterpret_cast<float4*>(dst) = make_float4(o[i], o[i + 2], o[i + 1], o[i + 3]);
                            *reinterpret_cast<float4*>(dst + 4) = make_float4(o[i + 4], o[i + 6], o[i + 5], o[i + 7]);
                        } else {
                            *reinterpret_cast<uint4*>(out + row * D + dim + i) =
                                make_uint4(pack2(o[i] * inv, o[i + 2] * inv), pack2(o[i + 1] * inv, o[i + 3] * inv),
                                           pack2(o[i + 4] * inv, o[i + 6] * inv), pack2(o[i + 5] * inv, o[i + 7] * inv));
                        }
                    }
                }
                tc_fence_before();
            }
            g0 += item_n;
        }
    }
}

// The same once more for scales that are far apart: a function of its own, so that the common one keeps its registers.
template <int D>
__device__ __noinline__ void prompt_again(const PromptArgs& p, Progress done) { prompt_roles<D, true>(p, done); }

template <int D>
__global__ void __launch_bounds__(PROMPT_THREADS, 1)
attention_int8_prompt_kernel(const __grid_constant__ PromptArgs p) {
    using S = PromptSmem<D>;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
    PromptBars* bars = reinterpret_cast<PromptBars*>(smem + S::BARS);
    volatile int* gave_up = &bars->gave_up;
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int x = 0; x < 2; x++) {
            mbar_init(smem_u32(&bars->q_full[x]), SOFT_WARPS / 2);
            mbar_init(smem_u32(&bars->q_empty[x]), 1);
            mbar_init(smem_u32(&bars->s_full[x]), 1);
            mbar_init(smem_u32(&bars->p_ready[x]), SOFT_WARPS / 2);
            mbar_init(smem_u32(&bars->pv_done[x]), 1);
        }
        for (int s = 0; s < KV_STAGES; s++) {
            mbar_init(smem_u32(&bars->k_full[s]), 4);
            mbar_init(smem_u32(&bars->k_empty[s]), 1);
            mbar_init(smem_u32(&bars->v_full[s]), 4);
            mbar_init(smem_u32(&bars->v_empty[s]), 1);
        }
        for (int s = 0; s < SC_STAGES; s++) mbar_init(smem_u32(&bars->sc_full[s]), 4);
        bars->gave_up = bars->n_listed = bars->wide = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    gfb_pdl_launch();
    gfb_pdl_wait();

    if (p.n_x <= LISTED)                                                 // (the tiles' shared memory is free yet)
        list_pairs(p.b, reinterpret_cast<TilePair*>(smem + S::LIST), reinterpret_cast<int*>(smem + S::BEFORE), reinterpret_cast<TilePair*>(smem),
                   reinterpret_cast<ulonglong2*>(smem + LISTED * 16), &bars->n_listed, p.G, ROWS / (p.H / p.G), p.window);

    Progress done = {0, 0, 0, {0, 0}};
    prompt_roles<D, false>(p, done);
    __syncthreads();
    if (bars->wide && !*gave_up) prompt_again<D>(p, done);

    tc_fence_before();
    __syncthreads();
    if (*gave_up) {
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 50000ull) __nanosleep(1000);
    }
    if (warp == MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// The rows of the (pair, key head) that block x of the kernel ahead began and others went on with, merged over them in ascending order; y: eight rows of either tile.
// A warp per row, four parts in flight.
template <int D>
__global__ void __launch_bounds__(256)
attention_int8_parts_kernel(const float* scratch_o, const float* scratch_ml, const SharedRows* shared, __nv_bfloat16* out, int H, int G) {
    constexpr int V = D / 32;
    gfb_pdl_launch();
    gfb_pdl_wait();
    const SharedRows p = shared[blockIdx.x];
    const int c0 = blockIdx.x, x = blockIdx.y >> 4, rep = H / G, TQ = ROWS / rep, lane = threadIdx.x & 31, r = (blockIdx.y & 15) * 8 + (threadIdx.x >> 5);
    if (p.last < 0 || r >= max(0, min(TQ, p.left - x * TQ)) * rep) return;
    float top = NONE, sum = 0.f, o[V] = {};
    for (int c = c0; c <= p.last; c += 4) {
        float2 ml[4];
        float from[4][V];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int cc = min(c + k, p.last);
            const size_t place = (size_t)((2 * cc + (cc == c0)) * 2 + x) * ROWS + r;
            ml[k] = *reinterpret_cast<const float2*>(scratch_ml + place * 2);
#pragma unroll
            for (int v = 0; v < V; v++) from[k][v] = scratch_o[place * D + lane * V + v];
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (c + k > p.last || ml[k].y == 0.f) continue;              // a part without a key of the row has written nothing (NaN scores make a NaN sum, which stays)
            const float now = fmaxf(top, ml[k].x), down = power2(top - now), w = power2(ml[k].x - now);
            top = now;
            sum = sum * down + ml[k].y * w;
#pragma unroll
            for (int v = 0; v < V; v++) o[v] = fmaf(from[k][v], w, o[v] * down);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int tq = r / rep;
    const size_t row = (size_t)(p.t0 + x * TQ + tq) * H + p.g * rep + (r - tq * rep);
#pragma unroll
    for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(out + row * D + lane * V + v) = pack2(o[v] * inv, o[v + 1] * inv);
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

template <int D>
int launch_prompt(const Decode& a, int n_x, int blocks, float* scratch) {
    auto kern = attention_int8_prompt_kernel<D>;
    const size_t smem = PromptSmem<D>::BYTES;
    static bool configured[MAX_DEVICES] = {};
    if (room(kern, smem, configured)) return 1;
    const long items = (long)n_x * a.G;
    if (items > 0x3fffffffL) return gfb_fail("gfb_attention_int8_prompt: %ld work items", items);
    const size_t rows = (size_t)4 * blocks * ROWS;
    float* ml = scratch ? scratch + rows * D : nullptr;
    SharedRows* shared = scratch ? (SharedRows*)(ml + rows * 2) : nullptr;
    const PromptArgs args{(const __nv_bfloat16*)a.q, (__nv_bfloat16*)a.out, scratch, ml, shared, a.kv, a.b, a.H, a.G, a.scale * 1.4426950408889634f, a.window, n_x, a.status};
    const unsigned grid = scratch ? blocks : (unsigned)(items < blocks ? items : blocks);
    if (gfb_check(gfb_launch(kern, dim3(grid), dim3(PROMPT_THREADS), smem, a.stream, args), "gfb_attention_int8_prompt")) return 1;
    if (scratch == nullptr) return 0;
    return gfb_check(gfb_launch(attention_int8_parts_kernel<D>, dim3(blocks, 32), dim3(256), 0, a.stream, (const float*)scratch, (const float*)ml, (const SharedRows*)shared,
                                (__nv_bfloat16*)a.out, a.H, a.G), "gfb_attention_int8_prompt (parts)");
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

// Any number of new tokens per sequence, bfloat16, d 64 or 128, pages of 64, at most 128 heads per key head, scale > 0.  n_x: at least the tile pairs there are,
// sum over sequences of ceil(new tokens / (2 floor(128 / (H / G)))).  blocks: one per SM.  With scratch (at most 1,024 pairs; float32 [512 blocks (d + 2) + 4 blocks]) every
// block has an equal share of all pairs' keys, without it whole pairs.
GFB_API int gfb_attention_int8_prompt(const void* q, void* out, const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
                                      const int* page_table, int max_pages, int page_size, int n_pages,
                                      const int* cu_seqlens, const int* tok_seq, const int* slots, const int* lengths, int n_seqs, int n_tokens,
                                      int H, int G, int d, float scale, int window, int n_x, int blocks, float* scratch, int* status, cudaStream_t stream) {
    if (n_tokens <= 0 || n_seqs <= 0) return 0;
    if ((d != 64 && d != 128) || page_size != PAGE) return gfb_fail("gfb_attention_int8_prompt: heads of %d, pages of %d", d, page_size);
    if (G <= 0 || H % G || H / G > ROWS) return gfb_fail("gfb_attention_int8_prompt: %d heads over %d", H, G);
    if (!(scale > 0.f)) return gfb_fail("gfb_attention_int8_prompt: a scale of %g (the maximum is taken of unscaled scores)", (double)scale);
    if (blocks < 1 || n_x < 1 || (scratch && n_x > LISTED)) return gfb_fail("gfb_attention_int8_prompt: %d blocks, %d pairs of tiles", blocks, n_x);
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)scratch) & 15)
        return gfb_fail("gfb_attention_int8_prompt: everything must be 16-byte aligned");
    const Decode a{q, out, {(const int8_t*)k_pool, (const int8_t*)v_pool, k_scale, v_scale, page_table, max_pages, page_size, n_pages},
                   {cu_seqlens, tok_seq, slots, lengths, n_seqs, n_tokens}, H, G, scale, window, status, stream};
    return d == 128 ? launch_prompt<128>(a, n_x, blocks, scratch) : launch_prompt<64>(a, n_x, blocks, scratch);
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
