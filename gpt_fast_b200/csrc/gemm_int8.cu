// Products of 8-bit integers on the 5th-generation tensor cores: y[m, n] = a_scale[m] w_scale[n] sum_k A[m, k] W[n, k] for rows of integers
// with a scale each (int8_rows.cuh).
//
// The sum is a 32-bit integer in tensor memory (tcgen05.mma kind::i8), so it has no rounding and no order: however K is split and whatever batch a row
// comes in, its result is the same bits.  |sum| <= 127^2 K stays below 2^31 for K up to 133,144.  Behind it everything is 32-bit floating point: the integer
// (rounded once if it has more than 24 bits) times the row's scale, times the column's, then the mode's function; one rounding to the output's type.
//
// Both operands lie K-major, a byte per number, and arrive by TMA as tiles of 128 bytes of K with 128-byte swizzle (zeros beyond K and beyond the last row).
//   few tokens   (gemm_int8_few_kernel): 128 weight rows are the rows of the MMA, the tokens, padded to 16, 32, 64 or 128, its columns.  A step streams every
//                weight once; what bounds it is that stream.  The K axis is split over a cluster of up to 8 blocks, as far as all blocks are on the
//                chip at once, and the blocks add up their integers through shared memory.  8 tokens, 28,672 x 4,096: 21.4 us, 5.5 TB/s; one token, 6,144 x
//                4,096: 7.4 us, 3.4 TB/s, where the kernel's start and its merge weigh as much as the stream.
//   many tokens  (gemm_int8_pair_kernel): 256 x 256 tiles on pairs of SMs (cta_group::2), persistent, two accumulators in tensor memory, so that a tile's
//                epilogue runs under the next one's products.  What bounds it is the tensor pipe, 90 % busy, and the power it takes: 8,192 tokens, 28,672 x
//                4,096: 562 us, 3.4 POP/s, as a single launch.
// Roles in a block of 192 threads: warp 0 = TMA producer (one lane), warp 1 = tensor-memory allocation and MMA issue (one lane), warps 2..5 = epilogue.
// Waits on barriers are bounded by wall-clock time, as in gemm_tc.cu; those for the preceding kernel, for tensor memory and for the other blocks of a
// cluster end for the reasons given there.
//
// Weights are taken to be complete before the kernel ahead of this one starts: the ring is filled with them ahead of the wait for it.  quantize_rows, which
// makes them, lets no kernel start before it has ended.
#include "int8_rows.cuh"

#include <cuda.h>

GFB_DEFINE_LAST_ERROR()

enum { EPI_STORE = 0, EPI_ADD = 1, EPI_SWIGLU = 2, EPI_GELU = 4, EPI_GELU_TANH = 5, EPI_SILU = 6, EPI_RELU2 = 7 };

namespace {

constexpr int BM = 128;              // MMA rows per tile
constexpr int BK = 128;              // k per stage: 128 bytes = one swizzle span
constexpr int UMMA_K = 32;           // k of one tcgen05.mma for 8-bit inputs
constexpr int MAX_STAGES = 12;
constexpr int X_TILE_BYTES = BM * BK;
constexpr unsigned long long WAIT_LIMIT_NS = 2000000000ull;    // 2 s: far beyond any healthy wait

// The first TMA copy through a tensor map fetches the 128-byte map; asking for it at once hides that behind the
// block's set-up.
__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ unsigned long long global_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok;
}
// Wait for the phase with `parity` to complete; false when the block aborts or time runs out.
__device__ __forceinline__ bool lane_waits(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int which) {
    if (mbar_try_wait(bar, parity)) return true;
    unsigned long long t0 = global_ns();
    for (;;) {
        for (int i = 0; i < 128; i++)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag) return false;
        if (global_ns() - t0 > WAIT_LIMIT_NS) {
            *abort_flag = 1;
            gfb_report(status, GFB_ERR_WAIT_TIMEOUT, which, (int)(blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z)));
            return false;
        }
        __nanosleep(64);
    }
}
// The same for a whole warp: one answer for all its lanes.  Where a wait runs out lanes can differ (one sees the abort flag, another its barrier), and
// a warp that parted there would never meet again at the aligned instructions behind it.
__device__ __forceinline__ bool warp_waits(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int which) {
    return __all_sync(0xffffffffu, lane_waits(bar, parity, abort_flag, status, which));
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

// The same with an L2 policy: weights of a decode step are read once per step and are far larger than L2, so they
// are marked to be evicted first and leave the cache to what is read again soon (activations, partial sums, the
// key/value pages).
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

// Shared-memory matrix descriptor of a K-major tile with 128-byte swizzle: rows of
// 128 bytes, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t umma_smem_desc(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFFu) >> 4);      // start address, 16-byte units
    d |= (uint64_t)1 << 16;                        // leading byte offset (unused with swizzle): 1
    d |= (uint64_t)(1024 >> 4) << 32;              // stride byte offset between 8-row groups
    d |= (uint64_t)1 << 46;                        // descriptor version of sm_100
    d |= (uint64_t)2 << 61;                        // layout: 128-byte swizzle
    return d;
}

// Instruction descriptor: signed 8-bit x signed 8-bit -> 32-bit integers, both operands K-major, M x N.
__host__ __device__ constexpr uint32_t umma_idesc(int M, int N) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16_raw(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32_raw(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
template <int N> __device__ __forceinline__ void tmem_ld_group(uint32_t taddr, uint32_t (&r)[N]);
template <> __device__ __forceinline__ void tmem_ld_group<16>(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16_raw(taddr, r); }
template <> __device__ __forceinline__ void tmem_ld_group<32>(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32_raw(taddr, r); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

// ---- what becomes of a sum ----------------------------------------------------------------------------------
// The same expressions in both kernels, with every product rounded by itself where a sum follows (a compiler that may draw the two together does so in one place and not
// in another): a row's bits do not depend on which of them made it.
__device__ __forceinline__ float scaled(uint32_t sum, float row_scale) { return __fmul_rn(__int2float_rn((int)sum), row_scale); }
// x / (1 + e^t), which SiLU (t = -x) and the tanh form of GELU are.  Outputs of 16 bits take the short exponential and quotient, off by up to 2 + 1.2 |t| steps of 32 bits, 2^-17 of
// the result where it counts; 32-bit outputs take the full ones, off by a few.
template <typename TO>
__device__ __forceinline__ float over_one_plus_exp(float x, float t) {
    return sizeof(TO) == 4 ? __fdiv_rn(x, __fadd_rn(1.f, expf(t))) : __fdividef(x, 1.f + __expf(t));
}
template <typename TO> __device__ __forceinline__ float gated(float g, float u) { return over_one_plus_exp<TO>(g, -g) * u; }
template <typename TO>
__device__ __forceinline__ float unary(int epi, float x) {
    if (epi == EPI_GELU) return 0.5f * x * __fadd_rn(1.0f, erff(x * 0.70710678118654752440f));
    if (epi == EPI_GELU_TANH)           // 0.5 x (1 + tanh(z)) = x / (1 + e^(-2z)), z = sqrt(2 / pi) (x + 0.044715 x^3)
        return over_one_plus_exp<TO>(x, -1.5957691216057308f * __fmaf_rn(0.044715f * x * x, x, x));
    if (epi == EPI_SILU) return over_one_plus_exp<TO>(x, -x);
    if (epi == EPI_RELU2) { const float r = x < 0.f ? 0.f : x; return r * r; }      // (a maximum would make 0 of NaN)
    return x;
}

// kinds of epilogue that are kernels of their own; UNARY's function is an argument
enum { KIND_STORE = 0, KIND_ADD = 1, KIND_SWIGLU = 2, KIND_UNARY = 3 };
template <int KIND, typename TO>
__device__ __forceinline__ float fin(int epi, float x) { return KIND == KIND_UNARY ? unary<TO>(epi, x) : x; }

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put2(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void put2(__nv_bfloat16* p, float a, float b) { *reinterpret_cast<uint32_t*>(p) = pack_bf16(a, b); }
__device__ __forceinline__ void put4(float* p, float a, float b, float c, float d) { *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d); }
__device__ __forceinline__ void put4(__nv_bfloat16* p, float a, float b, float c, float d) { *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(a, b), pack_bf16(c, d)); }

// Products e[0..3] of token m with the weight rows n .. n + 3 (n a multiple of four, N of them altogether) to the output.  vec: all four exist and a
// store of them is aligned, for every m and n.
template <int KIND, typename TO>
__device__ __forceinline__ void finish4(TO* out, const float (&e)[4], size_t m, int n, int N, int ldo, bool vec, int epi) {
    TO* row = out + m * ldo;
    if (KIND == KIND_SWIGLU) {
        const float a = gated<TO>(e[0], e[1]), b = gated<TO>(e[2], e[3]);
        if (vec) put2(row + (n >> 1), a, b);
        else {
            if (n < N) put(row + (n >> 1), a);
            if (n + 2 < N) put(row + (n >> 1) + 1, b);
        }
    } else if (KIND == KIND_ADD) {
        if (vec) {
            float4 x = *reinterpret_cast<const float4*>((float*)row + n);
            x.x += e[0]; x.y += e[1]; x.z += e[2]; x.w += e[3];
            *reinterpret_cast<float4*>((float*)row + n) = x;
        } else {
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (n + u < N) ((float*)row)[n + u] += e[u];
        }
    } else {
        if (vec) put4(row + n, fin<KIND, TO>(epi, e[0]), fin<KIND, TO>(epi, e[1]), fin<KIND, TO>(epi, e[2]), fin<KIND, TO>(epi, e[3]));
        else {
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (n + u < N) put(row + n + u, fin<KIND, TO>(epi, e[u]));
        }
    }
}

// ---- few tokens ----------------------------------------------------------------------------------------------
struct Barriers {
    unsigned long long full[MAX_STAGES];
    unsigned long long empty[MAX_STAGES];
    unsigned long long accum;
    uint32_t tmem_base;
    int abort_flag;
};

// map_w: W [N, K], map_a: A [M, K].  Block (x, y, z): weight rows 128 x .., tokens BN y .., part z of K; the parts of a tile are one cluster.
template <int BN, int KIND, typename TO>
__global__ void __launch_bounds__(192)
gemm_int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const float* a_scale,
                     const float* w_scale, TO* out, int M, int N, int K, int ldo, int kb_per_split, int stages, int vec, int epi, int* status) {
    constexpr int Y_TILE_BYTES = BN * BK;
    constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
    constexpr int GROUP = BN < 32 ? BN : 32;
    extern __shared__ uint8_t smem_raw[];
    if (threadIdx.x == 32) { prefetch_map(&map_w); prefetch_map(&map_a); }
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;          // swizzled tiles need 1024-byte alignment
    uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t xs = base;
    const uint32_t ys = base + (uint32_t)stages * X_TILE_BYTES;
    Barriers* bars = reinterpret_cast<Barriers*>(aligned + (size_t)stages * (X_TILE_BYTES + Y_TILE_BYTES));
    volatile int* abort_flag = &bars->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * BM, col0 = blockIdx.y * BN;
    const int total_kb = (K + BK - 1) / BK;
    const int kb0 = blockIdx.z * kb_per_split;
    const int nkb = min(kb_per_split, total_kb - kb0);
    const int n_pre = min(stages, nkb);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) {
            mbar_init(smem_u32(&bars->full[s]), 1);
            mbar_init(smem_u32(&bars->empty[s]), 1);
        }
        mbar_init(smem_u32(&bars->accum), 1);
        bars->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        // the ring is filled with weights at once (no other thread touches the barriers before the block's barrier below)
        for (int i = 0; i < n_pre; i++) {                   // fresh barriers: every stage is free
            const uint32_t full = smem_u32(&bars->full[i]);
            mbar_expect_tx(full, X_TILE_BYTES + Y_TILE_BYTES);
            tma_load_2d_hint(xs + i * X_TILE_BYTES, &map_w, (kb0 + i) * BK, row0, full, l2_evict_first_policy());
        }
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&bars->tmem_base)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    gfb_pdl_launch();
    gfb_pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pol = l2_evict_first_policy();
            for (int i = 0; i < n_pre; i++) tma_load_2d(ys + i * Y_TILE_BYTES, &map_a, (kb0 + i) * BK, col0, smem_u32(&bars->full[i]));
            for (int i = n_pre; i < nkb; i++) {
                const int s = i % stages;
                const uint32_t ph = (uint32_t)(i / stages) & 1u;
                if (!lane_waits(smem_u32(&bars->empty[s]), ph ^ 1u, abort_flag, status, 1)) break;
                const uint32_t full = smem_u32(&bars->full[s]);
                mbar_expect_tx(full, X_TILE_BYTES + Y_TILE_BYTES);
                tma_load_2d_hint(xs + s * X_TILE_BYTES, &map_w, (kb0 + i) * BK, row0, full, pol);
                tma_load_2d(ys + s * Y_TILE_BYTES, &map_a, (kb0 + i) * BK, col0, full);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = umma_idesc(BM, BN);
            bool ok = true;
            for (int i = 0; i < nkb && ok; i++) {
                const int s = i % stages;
                const uint32_t ph = (uint32_t)(i / stages) & 1u;
                ok = lane_waits(smem_u32(&bars->full[s]), ph, abort_flag, status, 2);
                if (!ok) break;
                tc_fence_after();
                const uint64_t da = umma_smem_desc(xs + s * X_TILE_BYTES);
                const uint64_t db = umma_smem_desc(ys + s * Y_TILE_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; k++)       // 32 bytes further along K: +2 in 16-byte units
                    umma_i8(tmem, da + 2 * k, db + 2 * k, idesc, (i | k) != 0);
                umma_commit(smem_u32(&bars->empty[s]));    // the stage is free once these MMAs have read it
            }
            if (ok) umma_commit(smem_u32(&bars->accum));
        }
    } else {
        // The tile goes through shared memory (the ring is free by then): [tokens][128 rows], so that a warp finishes a token's 128 rows side by side.
        const int q = warp & 3;                             // tensor-memory lanes 32q .. 32q+31 belong to this warp
        const bool ok = warp_waits(smem_u32(&bars->accum), 0, abort_flag, status, 3);
        tc_fence_after();
        uint32_t* tile = reinterpret_cast<uint32_t*>(aligned);
        if (ok) {
            const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
#pragma unroll 1
            for (int c = 0; c < BN; c += GROUP) {
                if (col0 + c >= M) break;                   // uniform: nothing left in this tile
                uint32_t raw[GROUP];
                tmem_ld_group<GROUP>(taddr + c, raw);
#pragma unroll
                for (int j = 0; j < GROUP; j++) tile[(c + j) * BM + q * 32 + lane] = raw[j];
            }
        }
    }
    __syncwarp();
    gfb_cluster_sync();                                     // (of one block where K is not split)
    if (warp >= 2 && !*abort_flag) {
        const uint32_t* tile = reinterpret_cast<const uint32_t*>(aligned);
        const int n_tok = min(BN, M - col0), splits = (int)gridDim.z, n = row0 + 4 * lane;
        float ws[4];
#pragma unroll
        for (int u = 0; u < 4; u++) ws[u] = n + u < N ? w_scale[n + u] : 0.f;
        for (int j = (int)blockIdx.z + splits * (warp - 2); j < n_tok; j += 4 * splits) {
            uint4 v = make_uint4(0, 0, 0, 0);
            const float sm = a_scale[col0 + j];
            for (int k = 0; k < splits; k++) {
                const float4 p = gfb_cluster_load4(tile + j * BM + 4 * lane, k);
                v.x += __float_as_uint(p.x); v.y += __float_as_uint(p.y); v.z += __float_as_uint(p.z); v.w += __float_as_uint(p.w);
            }
            const float e[4] = {__fmul_rn(scaled(v.x, sm), ws[0]), __fmul_rn(scaled(v.y, sm), ws[1]), __fmul_rn(scaled(v.z, sm), ws[2]), __fmul_rn(scaled(v.w, sm), ws[3])};
            finish4<KIND, TO>(out, e, (size_t)(col0 + j), n, N, ldo, vec && n + 3 < N, epi);
        }
    }
    __syncwarp();
    gfb_cluster_sync();                       // no block leaves while another reads its shared memory
    if (*abort_flag) {
        // copies that were issued may still be landing in this block's shared memory
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 50000ull) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM_COLS) : "memory");
    }
}

// ---- many tokens: pairs of SMs ----------------------------------------------------------------------------------
// Two blocks of a cluster work as one 256 x 256 tile: each loads its own 128 rows of A and half of the weight tile (128 of the 256 weight rows); one
// tcgen05.mma issued by the leader multiplies with operands from both blocks' shared memory and writes 128 accumulator rows into each block's tensor
// memory.  Barriers: `full` lives in the leader and counts the bytes of both blocks' loads; the MMA's commit goes to both blocks' `empty` and
// `acc_full`; both blocks' epilogue warps arrive on the leader's `acc_empty`.  No TMA multicast.
struct PBarriers {
    unsigned long long full[MAX_STAGES];
    unsigned long long empty[MAX_STAGES];
    unsigned long long acc_full[2];
    unsigned long long acc_empty[2];
    uint32_t tmem_base;
    int abort_flag;
};
constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;          // clears the bit that tells the two blocks of a pair apart
constexpr int PAIR_STAGE_BYTES = 2 * X_TILE_BYTES;   // 128 token rows + 128 weight rows, 128 k each
constexpr int PCW = 32;                              // columns staged at a time
constexpr int PSP = PCW + 4;                         // staging row pitch in floats
constexpr int P_STAGING_BYTES = 4 * 32 * PSP * 4;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t leader_bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(leader_bar) : "memory");
}
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {      // arrives on `bar` in both blocks
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A warp's 32 rows x PCW columns [c0, c0 + PCW) of a tile: tensor memory -> 32-bit numbers times the row's scale in shared memory -> whole lines of the
// output.  sm: the scale of row `lane`.  ldo, N: of the output's weight rows; vec: N is a multiple of 8 (SwiGLU: 16).
template <int KIND, typename TO>
__device__ __forceinline__ void drain_chunk(float* stage, uint32_t taddr, int c0, int lane, float sm, const float* w_scale, TO* out, size_t grow0, int gcol0,
                                            int rows, int N, int ldo, bool vec, int epi) {
    const int gc = gcol0 + c0;
    if (!vec) {
        // sizes that fill no vector: a column per lane
        uint32_t raw[32];
        tmem_ld32_raw(taddr + c0, raw);
#pragma unroll
        for (int j = 0; j < 32; j++) stage[lane * PSP + j] = scaled(raw[j], sm);
        __syncwarp();
        const int n = gc + lane;
        const float w = n < N ? w_scale[n] : 0.f, w1 = n + 1 < N ? w_scale[n + 1] : 0.f;
        for (int r = 0; r < rows; r++) {
            const float y = __fmul_rn(stage[r * PSP + lane], w);
            if (KIND == KIND_SWIGLU) {
                if (n < N && !(lane & 1)) put(out + (grow0 + r) * ldo + (n >> 1), gated<TO>(y, __fmul_rn(stage[r * PSP + lane + 1], w1)));
            } else if (n < N) {
                TO* o = out + (grow0 + r) * ldo + n;
                if (KIND == KIND_ADD) *(float*)o += y;
                else put(o, fin<KIND, TO>(epi, y));
            }
        }
        __syncwarp();
        return;
    }
    constexpr bool WIDE = KIND == KIND_ADD || (sizeof(TO) == 4 && KIND != KIND_SWIGLU);      // four columns per lane, else eight
    constexpr int COLS = WIDE ? 4 : 8, LPR = PCW / COLS, RPI = 32 / LPR;
    const int sub = lane / LPR, col = (lane % LPR) * COLS;
    float w[COLS];
    const bool live = gc + col < N;
#pragma unroll
    for (int u = 0; u < COLS; u += 4) {
        const float4 t = live ? *reinterpret_cast<const float4*>(w_scale + gc + col + u) : make_float4(0.f, 0.f, 0.f, 0.f);
        w[u] = t.x; w[u + 1] = t.y; w[u + 2] = t.z; w[u + 3] = t.w;
    }
    {
        uint32_t raw[32];
        tmem_ld32_raw(taddr + c0, raw);
#pragma unroll
        for (int j = 0; j < 32; j += 4)
            *reinterpret_cast<float4*>(stage + lane * PSP + j) = make_float4(scaled(raw[j], sm), scaled(raw[j + 1], sm), scaled(raw[j + 2], sm), scaled(raw[j + 3], sm));
    }
    __syncwarp();
#pragma unroll 2
    for (int rr = 0; rr < rows; rr += RPI) {
        const int r = rr + sub;
        if (r < rows && live) {
            float y[COLS];
#pragma unroll
            for (int u = 0; u < COLS; u += 4) {
                const float4 t = *reinterpret_cast<const float4*>(stage + r * PSP + col + u);
                y[u] = __fmul_rn(t.x, w[u]); y[u + 1] = __fmul_rn(t.y, w[u + 1]); y[u + 2] = __fmul_rn(t.z, w[u + 2]); y[u + 3] = __fmul_rn(t.w, w[u + 3]);
            }
            TO* o = out + (grow0 + r) * ldo;
            if constexpr (KIND == KIND_SWIGLU) {
                put4(o + ((gc + col) >> 1), gated<TO>(y[0], y[1]), gated<TO>(y[2], y[3]), gated<TO>(y[4], y[5]), gated<TO>(y[6], y[7]));
            } else if constexpr (KIND == KIND_ADD) {
                float4 x = *reinterpret_cast<const float4*>((float*)o + gc + col);
                x.x += y[0]; x.y += y[1]; x.z += y[2]; x.w += y[3];
                *reinterpret_cast<float4*>((float*)o + gc + col) = x;
            } else if constexpr (WIDE) {
                put4(o + gc + col, fin<KIND, TO>(epi, y[0]), fin<KIND, TO>(epi, y[1]), fin<KIND, TO>(epi, y[2]), fin<KIND, TO>(epi, y[3]));
            } else {
                uint4 pk;
                pk.x = pack_bf16(fin<KIND, TO>(epi, y[0]), fin<KIND, TO>(epi, y[1])); pk.y = pack_bf16(fin<KIND, TO>(epi, y[2]), fin<KIND, TO>(epi, y[3]));
                pk.z = pack_bf16(fin<KIND, TO>(epi, y[4]), fin<KIND, TO>(epi, y[5])); pk.w = pack_bf16(fin<KIND, TO>(epi, y[6]), fin<KIND, TO>(epi, y[7]));
                *reinterpret_cast<uint4*>(o + gc + col) = pk;
            }
        }
    }
    __syncwarp();                      // the staging rows are rewritten by the next chunk
}

template <int KIND, typename TO>
__global__ void __launch_bounds__(192)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const float* a_scale,
                      const float* w_scale, TO* out, int M, int N, int K, int ldo, int stages, int vec, int epi, int* status) {
    extern __shared__ uint8_t smem_raw[];
    if (threadIdx.x == 32) { prefetch_map(&map_a); prefetch_map(&map_w); }
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* aligned = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t xs = base;
    const uint32_t ys = base + (uint32_t)stages * X_TILE_BYTES;
    float* staging = reinterpret_cast<float*>(aligned + (size_t)stages * PAIR_STAGE_BYTES);
    PBarriers* bars = reinterpret_cast<PBarriers*>(aligned + (size_t)stages * PAIR_STAGE_BYTES + P_STAGING_BYTES);
    volatile int* abort_flag = &bars->abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int pair = (int)blockIdx.x >> 1, n_pairs = (int)gridDim.x >> 1;
    const int row_tiles = (M + 255) / 256, n_tiles = row_tiles * ((N + 255) / 256);
    const int nkb = (K + BK - 1) / BK;
    const int my_tiles = pair < n_tiles ? (n_tiles - 1 - pair) / n_pairs + 1 : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; s++) {
            mbar_init(smem_u32(&bars->full[s]), 1);
            mbar_init(smem_u32(&bars->empty[s]), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(smem_u32(&bars->acc_full[a]), 1);
            mbar_init(smem_u32(&bars->acc_empty[a]), 8);       // four epilogue warps in each of the two blocks
        }
        bars->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    gfb_cluster_sync();                          // both blocks' barriers exist before anything signals them
    tc_fence_after();
    const uint32_t tmem = bars->tmem_base;
    gfb_pdl_launch();
    if (!(warp == 0 && lane == 0)) gfb_pdl_wait();

    if (warp == 0) {
        if (lane == 0) {
            const int total = my_tiles * nkb;
            // the weight halves of the first round of the ring ahead of the wait for the preceding kernel, the rows of A behind it
            const int n_pre = min(stages, total);
            {
                int kb = 0, tile = pair;
                for (int it = 0; it < n_pre; it++) {
                    const uint32_t full = smem_u32(&bars->full[it]) & PEER_MASK;
                    if (leader) mbar_expect_tx(smem_u32(&bars->full[it]), 2 * PAIR_STAGE_BYTES);
                    tma_load_2d_pair(ys + it * X_TILE_BYTES, &map_w, kb * BK, (tile / row_tiles) * 256 + (int)rank * 128, full);
                    if (++kb == nkb) { kb = 0; tile += n_pairs; }
                }
            }
            gfb_pdl_wait();
            int kb = 0, tile = pair, s = 0;
            uint32_t ph = 0;
            int row0 = (tile % row_tiles) * 256 + (int)rank * 128, wrow0 = (tile / row_tiles) * 256 + (int)rank * 128;
            for (int it = 0; it < total; it++) {
                const uint32_t full = smem_u32(&bars->full[s]) & PEER_MASK;        // the leader's barrier
                if (it >= n_pre) {
                    if (!lane_waits(smem_u32(&bars->empty[s]), ph ^ 1u, abort_flag, status, 1)) break;
                    if (leader) mbar_expect_tx(smem_u32(&bars->full[s]), 2 * PAIR_STAGE_BYTES);
                    tma_load_2d_pair(ys + s * X_TILE_BYTES, &map_w, kb * BK, wrow0, full);
                }
                tma_load_2d_pair(xs + s * X_TILE_BYTES, &map_a, kb * BK, row0, full);
                if (++s == stages) { s = 0; ph ^= 1u; }
                if (++kb == nkb) {
                    kb = 0;
                    tile += n_pairs;
                    row0 = (tile % row_tiles) * 256 + (int)rank * 128;
                    wrow0 = (tile / row_tiles) * 256 + (int)rank * 128;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && leader) {
            constexpr uint32_t idesc = umma_idesc(256, 256);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int ti = 0; ti < my_tiles && ok; ti++) {
                const int ab = ti & 1;
                ok = lane_waits(smem_u32(&bars->acc_empty[ab]), ((uint32_t)(ti >> 1) & 1u) ^ 1u, abort_flag, status, 4);
                if (!ok) break;
                tc_fence_after();
                const uint32_t acc = tmem + (uint32_t)(ab * 256);
                for (int kb = 0; kb < nkb; kb++) {
                    ok = lane_waits(smem_u32(&bars->full[s]), ph, abort_flag, status, 2);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t da = umma_smem_desc(xs + s * X_TILE_BYTES);
                    const uint64_t db = umma_smem_desc(ys + s * X_TILE_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; k++) umma_i8_pair(acc, da + 2 * k, db + 2 * k, idesc, (kb | k) != 0);
                    umma_commit_pair(smem_u32(&bars->empty[s]));
                    if (++s == stages) { s = 0; ph ^= 1u; }
                }
                if (ok) umma_commit_pair(smem_u32(&bars->acc_full[ab]));
            }
        }
    } else {
        const int q = warp & 3;
        float* stage = staging + q * 32 * PSP;
        for (int ti = 0; ti < my_tiles; ti++) {
            const int ab = ti & 1;
            const int tile = pair + ti * n_pairs;
            const int row0 = (tile % row_tiles) * 256 + (int)rank * 128 + q * 32, col0 = (tile / row_tiles) * 256;
            const int rows = min(32, M - row0);
            const float sm = lane < rows ? a_scale[row0 + lane] : 0.f;
            if (!warp_waits(smem_u32(&bars->acc_full[ab]), (uint32_t)(ti >> 1) & 1u, abort_flag, status, 3)) break;
            tc_fence_after();
            const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(ab * 256);
#pragma unroll 1
            for (int c0 = 0; c0 < 256; c0 += PCW) {
                if (col0 + c0 >= N || rows <= 0) break;
                drain_chunk<KIND, TO>(stage, taddr, c0, lane, sm, w_scale, out, (size_t)row0, col0, rows, N, ldo, vec != 0, epi);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(smem_u32(&bars->acc_empty[ab]) & PEER_MASK);
        }
    }

    if (*abort_flag) {
        const unsigned long long t0 = global_ns();
        while (global_ns() - t0 < 50000ull) __nanosleep(1000);
    }
    tc_fence_before();
    __syncthreads();
    gfb_cluster_sync();                          // neither block leaves while the other may still signal it
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
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

// 2-D map over rows of K bytes, `pitch` apart: box = 128 k x box_rows rows, 128-byte swizzle, zeros outside.
int make_map(CUtensorMap* map, const void* base, int rows, int K, int pitch, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return gfb_fail("gfb_gemm_int8: the driver does not export cuTensorMapEncodeTiled");
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)pitch};
    cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return gfb_fail("gfb_gemm_int8: cuTensorMapEncodeTiled failed with %d (rows %d, K %d)", (int)r, rows, K);
    return 0;
}

constexpr int MAX_DEVICES = 64;

// Shared memory beyond 48 KB is granted per kernel and device; asked for once for each.
template <typename F>
int room(F kern, size_t smem, size_t (&configured)[MAX_DEVICES]) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= MAX_DEVICES) return gfb_fail("gfb_gemm_int8: device %d", dev);
    if (smem > configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return gfb_fail("gfb_gemm_int8: %zu bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
        configured[dev] = smem;
    }
    return 0;
}

struct Product {
    const void *A, *W;
    const float *a_scale, *w_scale;
    void* out;
    int lda, ldw, M, N, K, ldo, epi;
    int* status;
    cudaStream_t stream;
};

size_t few_smem(int bn, int stages) { return 1024 + (size_t)stages * (X_TILE_BYTES + bn * BK) + sizeof(Barriers); }
size_t pair_smem(int stages) { return 1024 + (size_t)stages * PAIR_STAGE_BYTES + P_STAGING_BYTES + sizeof(PBarriers); }

template <int BN, int KIND, typename TO>
int launch_few(const Product& p, int splits, int kbps, int stages) {
    auto kern = gemm_int8_few_kernel<BN, KIND, TO>;
    const size_t smem = few_smem(BN, stages);
    static size_t configured[MAX_DEVICES] = {};
    if (room(kern, smem, configured)) return 1;
    CUtensorMap mw, ma;
    if (make_map(&mw, p.W, p.N, p.K, p.ldw, BM) || make_map(&ma, p.A, p.M, p.K, p.lda, BN)) return 1;
    const dim3 grid((p.N + BM - 1) / BM, (p.M + BN - 1) / BN, splits);
    const int vec = KIND == KIND_SWIGLU ? p.ldo % 2 == 0 : p.ldo % 4 == 0;
    return gfb_check(gfb_launch_clusters(kern, grid, dim3(192), smem, p.stream, dim3(1, 1, splits), mw, ma, p.a_scale, p.w_scale, (TO*)p.out, p.M, p.N, p.K, p.ldo,
                                         kbps, stages, vec, p.epi, p.status), "gfb_gemm_int8");
}

template <int KIND, typename TO>
int launch_pair(const Product& p) {
    auto kern = gemm_int8_pair_kernel<KIND, TO>;
    const int stages = 6;
    const size_t smem = pair_smem(stages);
    static size_t configured[MAX_DEVICES] = {};
    if (room(kern, smem, configured)) return 1;
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    CUtensorMap ma, mw;
    if (make_map(&ma, p.A, p.M, p.K, p.lda, BM) || make_map(&mw, p.W, p.N, p.K, p.ldw, 128)) return 1;
    const long tiles = (long)((p.M + 255) / 256) * ((p.N + 255) / 256);
    const int pairs = tiles < sms / 2 ? (int)tiles : sms / 2;
    const int vec = p.N % (KIND == KIND_SWIGLU ? 16 : 8) == 0;
    return gfb_check(gfb_launch_cluster(kern, dim3(2 * pairs), dim3(192), smem, p.stream, 2u, ma, mw, p.a_scale, p.w_scale, (TO*)p.out, p.M, p.N, p.K, p.ldo,
                                        stages, vec, p.epi, p.status), "gfb_gemm_int8 (pairs)");
}

template <int KIND, typename TO>
int launch(const Product& p, int bn, int splits, int stages) {
    if (bn == 256) return launch_pair<KIND, TO>(p);
    const int total_kb = (p.K + BK - 1) / BK;
    splits = splits < 1 ? 1 : splits > 8 ? 8 : splits;             // 8: the largest portable cluster
    if (splits > total_kb) splits = total_kb;
    const int kbps = (total_kb + splits - 1) / splits;
    splits = (total_kb + kbps - 1) / kbps;                          // no empty part
    if (bn == 16) return launch_few<16, KIND, TO>(p, splits, kbps, stages);
    if (bn == 32) return launch_few<32, KIND, TO>(p, splits, kbps, stages);
    if (bn == 64) return launch_few<64, KIND, TO>(p, splits, kbps, stages);
    return launch_few<128, KIND, TO>(p, splits, kbps, stages);
}

}  // namespace

// A [M, lda] and W [N, ldw] of 8-bit integers between -127 and 127 (pitches multiples of 16), a_scale [M], w_scale [N]; out [M, N] (SwiGLU: [M, N / 2], W's
// rows alternate gate, up) of type out_dt; EPI_ADD: float32 out += product.  bn 16, 32, 64 or 128: tiles of 128 weight rows x bn tokens, K in up to
// `splits` parts of a cluster, a ring of `stages` stages per block; bn 256: tiles of 256 x 256 on pairs of SMs.
GFB_API int gfb_gemm_int8(const void* A, const float* a_scale, int lda, const void* W, const float* w_scale, int ldw, void* out, int out_dt, int M, int N, int K,
                          int epi, int bn, int splits, int stages, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || K > 133144) return gfb_fail("gfb_gemm_int8: rows of %d numbers (1 to 133,144, beyond which a sum may leave 32 bits)", K);
    if (lda % 16 || ldw % 16 || lda < K || ldw < K) return gfb_fail("gfb_gemm_int8: pitches %d and %d of rows of %d numbers (multiples of 16)", lda, ldw, K);
    if (((uintptr_t)A | (uintptr_t)W) & 15) return gfb_fail("gfb_gemm_int8: operands must be 16-byte aligned");
    if (((uintptr_t)out | (uintptr_t)w_scale) & 15) return gfb_fail("gfb_gemm_int8: the output and the weights' scales must be 16-byte aligned");
    if (epi == EPI_SWIGLU && N % 2) return gfb_fail("gfb_gemm_int8: SwiGLU needs pairs of rows, got %d", N);
    if (epi == EPI_ADD && out_dt != GFB_F32) return gfb_fail("gfb_gemm_int8: the residual sum is float32");
    if (bn != 16 && bn != 32 && bn != 64 && bn != 128 && bn != 256) return gfb_fail("gfb_gemm_int8: tiles of %d tokens", bn);
    if (bn != 256) {
        // the ring also holds the finished tile of 128 x bn sums
        if (stages < 2 || stages > MAX_STAGES || few_smem(bn, stages) > 227 * 1024 || stages * (X_TILE_BYTES + bn * BK) < BM * bn * 4)
            return gfb_fail("gfb_gemm_int8: %d stages of tiles of %d tokens", stages, bn);
        if ((M + bn - 1) / bn > 65535) return gfb_fail("gfb_gemm_int8: %d tokens exceed the grid", M);
    }
    const Product p{A, W, a_scale, w_scale, out, lda, ldw, M, N, K, epi == EPI_SWIGLU ? N / 2 : N, epi, status, stream};
    if (epi == EPI_ADD) return launch<KIND_ADD, float>(p, bn, splits, stages);
#define GO(KIND) return out_dt == GFB_BF16 ? launch<KIND, __nv_bfloat16>(p, bn, splits, stages) : launch<KIND, float>(p, bn, splits, stages)
    if (epi == EPI_SWIGLU) GO(KIND_SWIGLU);
    if (epi == EPI_STORE) GO(KIND_STORE);
    if (epi == EPI_GELU || epi == EPI_GELU_TANH || epi == EPI_SILU || epi == EPI_RELU2) GO(KIND_UNARY);
#undef GO
    return gfb_fail("gfb_gemm_int8: unknown epilogue %d", epi);
}

// The same with a [M, K] of bfloat16 or float32 (a_dt) that is quantised on the way: scratch of M (pitch + 4) bytes, pitch = K rounded up to 16.
GFB_API int gfb_linear_int8(const void* a, int a_dt, void* scratch, const void* W, const float* w_scale, int ldw, void* out, int out_dt, int M, int N, int K, int epi,
                            int bn, int splits, int stages, int* status, cudaStream_t stream) {
    if (M <= 0 || N <= 0) return 0;
    if (K <= 0 || K > 133144) return gfb_fail("gfb_linear_int8: rows of %d numbers (1 to 133,144, beyond which a sum may leave 32 bits)", K);
    const int pitch = (K + 15) / 16 * 16;
    int8_t* q = (int8_t*)scratch;
    float* scale = (float*)(q + (size_t)M * pitch);
    cudaError_t e;
    if (a_dt == GFB_BF16) e = quantize_rows_launch((const __nv_bfloat16*)a, q, scale, M, K, pitch, 1, stream);
    else if (a_dt == GFB_F32) e = quantize_rows_launch((const float*)a, q, scale, M, K, pitch, 1, stream);
    else return gfb_fail("gfb_linear_int8: unknown type %d", a_dt);
    if (gfb_check(e, "gfb_linear_int8")) return 1;
    return gfb_gemm_int8(q, scale, pitch, W, w_scale, ldw, out, out_dt, M, N, K, epi, bn, splits, stages, status, stream);
}
