// Tree attention on the tensor cores (fp16, bf16): tcgen05 products with the accumulators in TMEM, operands by TMA.
//
// A CTA owns a tile of up to 128 query rows of one (batch, head) -- all drafted tokens of all query heads that share the
// cache head -- and a run of key tiles of 64 rows.  Per tile
//     S = Q K^T  [128 x 64]   fp32 in TMEM; Q and K are K-major operands in 128-byte-swizzled shared memory
//     P = exp2(c S - m)       one thread per query row: TMEM -> registers -> 16-bit P back into S's columns
//     O += P V   [128 x Dh]   A = P from TMEM, B = V as it lies in the cache (MN-major)
// so a cache row is read from HBM once for all query rows.  A tile of 64 keys x 128 is 32 KB, 1400 cycles of an SM's share of HBM, and about 650
// of products, although half of each and more is padding or copies (256 pairs x 4096, 64 query rows: tensor pipe active 40 % of the time, DRAM at 71 %
// of its peak with starts and ends): what bounds a long cache is HBM.
//
// Warps: 0 issues the TMA loads, 1 allocates TMEM and issues the products, 2..5 do the softmax (a warp can only reach the 32 TMEM
// lanes of its rank modulo 4).  S has two buffers, so that S of the next tile is computed while the softmax of this one runs.
// Few query rows are copied: up to 32 rows stand in the product's 128 four times, up to 64 twice (REP), and each copy weighs its
// share of the tile's keys, with zeros for the others -- the copies' results are added at the end.  All four warps then work on any
// tree, and the chain of waits and instructions per tile, not a throughput, is what a softmax warp spends its time on.
// The running maximum is raised lazily: weights are taken relative to a reference that follows the true maximum only when that
// is more than 8 (in powers of two) ahead, so O is rarely rescaled and weights stay below 256, exact in either type's range.
// The sum is taken of the weights in fp32; what meets V is 16-bit.  With up to 32 query rows (a one-token step and most trees) a weight goes into the
// product as the sum of two numbers of the type, what it rounds to and the rest, and the result is as close to the exact one as its own
// rounding allows, like the one-token step's, whose weights are fp32: 2.1e-4 in the 2-norm for fp16, 1.7e-3 for bf16.  That costs a second
// product per 16 keys, 6 % there (fp16, 320 pairs x 1237 x 64, 27 rows: 40.2 -> 42.7 us), where the chain of a tile's waits bounds.  With more rows the
// products and, in a long loop, their power bound: 65.6 -> 77 us (128 pairs x 1920 x 256, 100 rows), 98 -> 120 (16 pairs x 32705 x 128, two tiles of 66)
// and 745 -> 850 to 950 (bf16, 1024 pairs x 8128 x 128, 64 rows).  There a weight is rounded once, and the result is 1.4 times as far off: 2.9e-4 and
// 2.3e-3.  (The rests in copies of the query rows of their own instead of a second product, 64 rows: 864 us where a second product takes 770 and
// neither 700; each thread then has twice the exponentials.)
#pragma once
#include <cuda.h>

#include "ffa_tree_kernel.cuh"

namespace ffa_dev {

constexpr int kUmmaRows = 128;     // query rows per CTA
constexpr int kUmmaKeys = 64;      // keys per tile
constexpr int kUmmaThreads = 192;
constexpr int kUmmaSoftmaxThreads = 128;
constexpr int kUmmaMaxStages = 12;
constexpr int kQBoxRows = 32;      // Q arrives in boxes of 32 rows
// copies of the query rows in a tile of the product
constexpr int umma_rep(int tile_rows) { return tile_rows <= 32 ? 4 : tile_rows <= 64 ? 2 : 1; }
constexpr bool umma_rests(int rep) { return rep == 4; }   // whether the weights' rests meet V too, see above
constexpr float kLazyRescale = 8.f;
constexpr int kFmaPairs = 3;       // of 8 pairs of exponentials, those that the FMA units take
// fp16 weights are held 2^7 times as large (2^15 at most, the type ends at 65504): parts of a weight vanish below 2^-32 of the largest one
template <typename T>
__device__ __forceinline__ constexpr float weight_shift() { return std::is_same<T, __half>::value ? 7.f : 0.f; }

// padded head dimension, as whole 128-byte (64-element) boxes; what lies behind Dh is zero-filled by the TMA unit
constexpr int umma_dp(int dh) { return (dh + 63) / 64 * 64; }
constexpr int umma_tile_bytes(int dh) { return umma_dp(dh) * 2 * kUmmaKeys; }
constexpr int umma_q_bytes(int dh) { return umma_dp(dh) * 2 * kUmmaRows; }
constexpr int umma_ctas_per_sm(int dh) { return umma_dp(dh) <= 128 ? 2 : 1; }   // TMEM: Dh + 128 columns of 512
constexpr int umma_tmem_cols(int dh) { return umma_dp(dh) <= 128 ? 256 : 512; }
// ring buffers of one K or V tile each: what is left of an SM's shared memory
constexpr int umma_stages(int dh) { return umma_dp(dh) == 64 ? 12 : 5; }
// behind Q and the ring
struct UmmaTail {
    uint64_t bars[2 * kUmmaMaxStages + 8];
    uint32_t bad[kTreeMaxRows / 32];   // drafted tokens with an infinity or NaN in V
    uint32_t tmem_base;
    uint32_t pos[8], neg[8];           // columns with +infinity, -infinity (NaN: both) in a cached V row of this CTA's tiles
    uint32_t poisoned;                 // groups of 16 columns of O that hold one
    int flags[1];                      // a wait ran out
    int any_bad;
};
constexpr int umma_smem(int dh) { return umma_q_bytes(dh) + umma_stages(dh) * umma_tile_bytes(dh) + (int)sizeof(UmmaTail); }

struct FfaTreeUmmaParams {
    CUtensorMap q, k_new, v_new, k_cache, v_cache;
    FfaTreeParams p;
};

// ---- PTX wrappers ----
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t smem_result, uint32_t cols)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_result), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcgen05_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// arrives on the barrier when every product issued so far by this thread has completed
__device__ __forceinline__ void umma_commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// true in one lane of the (whole) warp, always the same
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// Consecutive columns of this warp's 32 TMEM lanes: r[OFF + i] = column i of the thread's lane
template <int OFF, int N>
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[N])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15}, [%16];"
                 : "=r"(r[OFF + 0]), "=r"(r[OFF + 1]), "=r"(r[OFF + 2]), "=r"(r[OFF + 3]), "=r"(r[OFF + 4]),
                   "=r"(r[OFF + 5]), "=r"(r[OFF + 6]), "=r"(r[OFF + 7]), "=r"(r[OFF + 8]), "=r"(r[OFF + 9]),
                   "=r"(r[OFF + 10]), "=r"(r[OFF + 11]), "=r"(r[OFF + 12]), "=r"(r[OFF + 13]), "=r"(r[OFF + 14]),
                   "=r"(r[OFF + 15])
                 : "r"(addr));
}
template <int OFF, int N>
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[N])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[OFF + 0]), "=r"(r[OFF + 1]), "=r"(r[OFF + 2]), "=r"(r[OFF + 3]), "=r"(r[OFF + 4]),
                   "=r"(r[OFF + 5]), "=r"(r[OFF + 6]), "=r"(r[OFF + 7]), "=r"(r[OFF + 8]), "=r"(r[OFF + 9]),
                   "=r"(r[OFF + 10]), "=r"(r[OFF + 11]), "=r"(r[OFF + 12]), "=r"(r[OFF + 13]), "=r"(r[OFF + 14]),
                   "=r"(r[OFF + 15]), "=r"(r[OFF + 16]), "=r"(r[OFF + 17]), "=r"(r[OFF + 18]), "=r"(r[OFF + 19]),
                   "=r"(r[OFF + 20]), "=r"(r[OFF + 21]), "=r"(r[OFF + 22]), "=r"(r[OFF + 23]), "=r"(r[OFF + 24]),
                   "=r"(r[OFF + 25]), "=r"(r[OFF + 26]), "=r"(r[OFF + 27]), "=r"(r[OFF + 28]), "=r"(r[OFF + 29]),
                   "=r"(r[OFF + 30]), "=r"(r[OFF + 31])
                 : "r"(addr));
}
template <int OFF, int N>
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[N])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15};" ::"r"(r[OFF + 0]), "r"(r[OFF + 1]), "r"(r[OFF + 2]), "r"(r[OFF + 3]),
                   "r"(r[OFF + 4]), "r"(r[OFF + 5]), "r"(r[OFF + 6]), "r"(r[OFF + 7]), "r"(r[OFF + 8]),
                   "r"(r[OFF + 9]), "r"(r[OFF + 10]), "r"(r[OFF + 11]), "r"(r[OFF + 12]), "r"(r[OFF + 13]),
                   "r"(r[OFF + 14]), "r"(r[OFF + 15]), "r"(addr) : "memory");
}
template <int OFF, int N>
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[N])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, "
                 "%31};" ::"r"(r[OFF + 0]), "r"(r[OFF + 1]), "r"(r[OFF + 2]), "r"(r[OFF + 3]), "r"(r[OFF + 4]),
                   "r"(r[OFF + 5]), "r"(r[OFF + 6]), "r"(r[OFF + 7]), "r"(r[OFF + 8]), "r"(r[OFF + 9]),
                   "r"(r[OFF + 10]), "r"(r[OFF + 11]), "r"(r[OFF + 12]), "r"(r[OFF + 13]), "r"(r[OFF + 14]),
                   "r"(r[OFF + 15]), "r"(r[OFF + 16]), "r"(r[OFF + 17]), "r"(r[OFF + 18]), "r"(r[OFF + 19]),
                   "r"(r[OFF + 20]), "r"(r[OFF + 21]), "r"(r[OFF + 22]), "r"(r[OFF + 23]), "r"(r[OFF + 24]),
                   "r"(r[OFF + 25]), "r"(r[OFF + 26]), "r"(r[OFF + 27]), "r"(r[OFF + 28]), "r"(r[OFF + 29]),
                   "r"(r[OFF + 30]), "r"(r[OFF + 31]), "r"(addr) : "memory");
}
// The registers of a load may be read behind this; naming them keeps the compiler from reading them earlier
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[N])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand with the 128-byte swizzle: atoms of 8 rows of 128 bytes.  K-major (Q, K): `stride` is the distance of
// the atoms along the rows.  MN-major (V): `stride` is the distance of the atoms along the keys, `leading` along the columns.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t leading, uint32_t stride)
{
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
template <typename T>
constexpr uint32_t umma_idesc(int n, bool b_mn_major)
{
    const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (type << 7) | (type << 10) | (b_mn_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kUmmaRows >> 4) << 24);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w)
{
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// the 16-bit elements of a word whose exponent is all ones (infinity or NaN), as a mask of their bits
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w)
{
    constexpr uint32_t E = std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    uint32_t m = 0;
    if ((w & E) == E) m |= 0xffffu;
    if (((w >> 16) & E) == E) m |= 0xffff0000u;
    return m;
}

// Notes the columns of those groups of 16 that hold an infinity or NaN in V's cached rows [lo, hi) of the pair: thread `rank` of
// `threads`.  A product with a weight of 0 (another copy's key, a weight that vanished) has turned such a value into NaN in O.
template <typename T, int DH>
__device__ __noinline__ void find_nonfinite(const FfaTreeParams& P, int bh, int lo, int hi, uint32_t groups, uint32_t* pos, uint32_t* neg, int rank, int threads)
{
    for (int r = lo + rank; r < hi; r += threads) {
        const uint4* row = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(P.v_cache) + cache_row_offset(P, bh, r, DH * 2));
        for (uint32_t g = groups; g != 0; g &= g - 1) {
            const int first = __ffs(g) - 1;
            for (int i = 2 * first; i < 2 * first + 2; ++i) {
                const uint4 x = row[i];
                if (!(nonfinite_mask<T>(x.x) | nonfinite_mask<T>(x.y) | nonfinite_mask<T>(x.z) | nonfinite_mask<T>(x.w))) continue;
                float y[8];
                Elem<T>::unpack(x, y);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (isfinite(y[e])) continue;
                    if (!(y[e] < 0.f)) atomicOr(&pos[i >> 2], 1u << (8 * (i & 3) + e));
                    if (!(y[e] > 0.f)) atomicOr(&neg[i >> 2], 1u << (8 * (i & 3) + e));
                }
            }
        }
    }
}

// the largest of three; NaN if one of them is
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 2^y for a pair of arguments on the FMA units: y = n + f with n the nearest integer, 2^f on [-1/2, 1/2] by the polynomial of degree 4
// whose largest relative error is smallest (Remez exchange; 2.7e-6 in fp32, a hundredth of a 16-bit weight's rounding), n added
// to the exponent.  For finite arguments; below -126 the result is 2^-126: next to a largest weight of 1 that is nothing.  The
// MUFU unit takes 8 cycles per warp and exponential and would otherwise bound the softmax.
__device__ __forceinline__ float2 exp2_fma(float2 y)
{
    const float magic = 12582912.f;   // 1.5 * 2^23: the sum's low bits are n
    y = make_float2(fmaxf(y.x, -126.f), fmaxf(y.y, -126.f));
    const float2 t = __fadd2_rn(y, make_float2(magic, magic));
    const float2 n = __fadd2_rn(t, make_float2(-magic, -magic));
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), y);
    float2 p = make_float2(0.009570102207362652f, 0.009570102207362652f);
    p = __ffma2_rn(p, f, make_float2(0.05591785907745361f, 0.05591785907745361f));
    p = __ffma2_rn(p, f, make_float2(0.240247443318367f, 0.240247443318367f));
    p = __ffma2_rn(p, f, make_float2(0.6931217908859253f, 0.6931217908859253f));
    p = __ffma2_rn(p, f, make_float2(0.9999992847442627f, 0.9999992847442627f));
    return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(t.x) << 23)),
                       __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(t.y) << 23)));
}

template <typename T, int DH, int REP>
__global__ void __launch_bounds__(kUmmaThreads, umma_ctas_per_sm(DH)) ffa_tree_umma_kernel(const __grid_constant__ FfaTreeUmmaParams U)
{
    constexpr int DP = umma_dp(DH), NB = DP / 64, TILE = umma_tile_bytes(DH), STAGES = umma_stages(DH), ROWB = DH * 2;
    constexpr int BOX = 64 * 128;   // bytes of a tile's box: 64 rows of 128 bytes
    constexpr uint32_t S_COL = DP;  // TMEM columns: O at 0, the two S / P buffers behind it
    constexpr int QUADS = 4 / REP, COLS = kUmmaKeys / REP;   // warps per copy of the query rows; keys of a tile that a copy weighs
    constexpr bool RESTS = umma_rests(REP);
    constexpr int WORDS = RESTS ? 16 : 8;   // columns of P for 16 keys
    const FfaTreeParams& P = U.p;
    // No static shared memory: the dynamic part then starts on the 1024-byte boundary that swizzled operands need, without
    // slack (two CTAs with 112 KB of operands leave 1.5 KB of an SM)
    extern __shared__ __align__(1024) unsigned char raw[];
    UmmaTail& tail = *reinterpret_cast<UmmaTail*>(raw + umma_q_bytes(DH) + STAGES * TILE);
    int* flags = tail.flags;
    uint32_t* bad = tail.bad;
    const uint32_t q_smem = smem_u32(raw), ring = q_smem + umma_q_bytes(DH);
    const uint32_t full = smem_u32(tail.bars), empty = full + 8 * STAGES, q_full = empty + 8 * STAGES, s_full = q_full + 8, p_ready = s_full + 16,
                   pv_done = p_ready + 16, drained = pv_done + 16;
    volatile int* dead = flags;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int R = P.groups * P.tokens;
    if (tid == 0) {
        flags[0] = 0, tail.any_bad = 0, tail.poisoned = 0;
        tma_prefetch_map(&U.q), tma_prefetch_map(&U.k_cache), tma_prefetch_map(&U.v_cache), tma_prefetch_map(&U.k_new), tma_prefetch_map(&U.v_new);
    }
    if (tid >= 64 && tid < 64 + kTreeMaxRows / 32) bad[tid - 64] = 0;
    if (tid >= 96 && tid < 104) tail.pos[tid - 96] = tail.neg[tid - 96] = 0;
    pdl_wait();
    const TreeCut<kUmmaKeys> cut(P);
    const int row0 = cut.rt * P.tile_rows, rows = min(P.tile_rows, R - row0);
    const bool whole = P.splits == 1;
    T* out = static_cast<T*>(P.out) + ((size_t)cut.bh * R + row0) * DH;
    float* part = whole ? nullptr : tree_partial(P, cut.bh, cut.rt, cut.split, DH);
    const bool missing = tree_page_missing(P, cut.b, cut.sr);
    if ((!cut.sr.ok || missing) && tid == 0) atomicOr(P.status, missing ? kStatusBadIndex : kStatusBadLength);   // refused: zeros, nothing appended
    if (!cut.sr.ok || missing || cut.split >= cut.splits) {
        if (!whole) tree_empty_partial(part, rows, DH, tid, kUmmaThreads);
        else for (int i = tid; i < rows * DH; i += kUmmaThreads) Elem<T>::store(out + i, 0.f);
        return;
    }
    const int copy_warps = min(QUADS, (rows + 31) / 32), softmax_warps = copy_warps * REP;   // warps whose rows exist
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1);
        mbar_init(q_full, 1);
        for (int i = 0; i < 2; ++i) mbar_init(s_full + 8 * i, 1), mbar_init(p_ready + 8 * i, 32 * softmax_warps), mbar_init(pv_done + 8 * i, 1);
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // TMEM after pdl_wait: a CTA that held some while it waits for the previous grid could keep that grid from ever finishing; and
    // the next grid may start only when this one has its own
    if (warp == 1) tmem_alloc(smem_u32(&tail.tmem_base), umma_tmem_cols(DH)), tmem_relinquish();
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    pdl_release();
    const uint32_t tmem = tail.tmem_base;
    const int n_tiles = cut.u1 - cut.u0;
    uint32_t issued = 0;   // K and V loads of the issuing thread

    if (warp == 0) {
        // ---------------- TMA ----------------
        if (lane == 0) {
            mbar_expect_tx(q_full, (uint32_t)(softmax_warps * kQBoxRows * 128 * NB));
            for (int x = 0; x < NB; ++x)
                for (int i = 0; i < REP; ++i)
                    for (int w = 0; w < copy_warps; ++w)
                        tma_load_2d(q_smem + x * (kUmmaRows * 128) + (i * QUADS + w) * (kQBoxRows * 128), &U.q, 64 * x,
                                    cut.bh * R + row0 + w * kQBoxRows, q_full);
            uint32_t stage = 0, use = 0;
            // loads in the order the products take them: K0, K1, V0, K2, V1, ..., V(last)
            auto load = [&](int j, bool is_v) -> bool {
                const int u = cut.u0 + j;
                if (use > 0 && !mbar_wait_bounded(empty + 8 * stage, (use - 1) & 1, dead)) return false;
                const bool cached = u < cut.cache_tiles;
                const int first = (cached ? cut.c0 + u : u - cut.cache_tiles) * kUmmaKeys;
                const CUtensorMap* map = cached ? (is_v ? &U.v_cache : &U.k_cache) : (is_v ? &U.v_new : &U.k_new);
                int y;
                if (!cached) y = cut.bh * P.tokens + first;
                else if (P.page_table == nullptr) y = cut.bh * P.Lmax + first;
                else {
                    const int h = cut.bh - cut.b * P.H;
                    y = (P.page_table[(size_t)cut.b * P.max_pages + first / P.page_rows] * P.H + h) * P.page_rows + first % P.page_rows;
                }
                mbar_expect_tx(full + 8 * stage, TILE);
                for (int x = 0; x < NB; ++x) tma_load_2d(ring + stage * TILE + x * BOX, map, 64 * x, y, full + 8 * stage);
                ++issued;
                if (++stage == STAGES) stage = 0, ++use;
                return true;
            };
            bool ok = load(0, false);
            for (int j = 1; ok && j < n_tiles; ++j) ok = load(j, false) && load(j - 1, true);
            if (ok) load(n_tiles - 1, true);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---------------- products ----------------
        // The whole warp walks the loop and one elected lane issues: addresses and descriptors are then the same for the warp and
        // stay in uniform registers, which is where the instructions take them from (a loop of one lane spends 100 cycles on each).
        constexpr uint32_t S_DESC = umma_idesc<T>(kUmmaKeys, false), O_DESC = umma_idesc<T>(DP, true);
        const uint64_t q_desc = umma_desc(q_smem, 0, 1024), k_desc = umma_desc(ring, 0, 1024), v_desc = umma_desc(ring, BOX, 1024);
        auto together = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
        uint32_t stage = 0, phase = 0;
        auto next = [&]() {
            if (++stage == STAGES) stage = 0, phase ^= 1;
        };
        auto values = [&](int j) -> bool {   // O += P_j V_j
            if (!together(mbar_wait_bounded(p_ready + 8 * (j & 1), (j >> 1) & 1, dead))) return false;
            if (!together(mbar_wait_bounded(full + 8 * stage, phase, dead))) return false;
            tcgen05_after_sync();
            const uint64_t v = v_desc + stage * (TILE / 16);
            const uint32_t p = tmem + S_COL + kUmmaKeys * (j & 1);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < kUmmaKeys / 16; ++k) {   // 16 keys: 8 columns of packed P (and 8 of the weights' rests), two atoms of V
                    umma_ts(tmem, p + WORDS * k, v + (2048 / 16) * k, O_DESC, j > 0 || k > 0);
                    if (RESTS) umma_ts(tmem, p + WORDS * k + 8, v + (2048 / 16) * k, O_DESC, true);
                }
                umma_commit(empty + 8 * stage);
                umma_commit(pv_done + 8 * (j & 1));
            }
            __syncwarp();
            next();
            return true;
        };
        bool ok = together(mbar_wait_bounded(q_full, 0, dead));
        for (int j = 0; ok && j < n_tiles; ++j) {
            // S_j goes where P_(j-2) was: that product has to be through
            ok = together(mbar_wait_bounded(full + 8 * stage, phase, dead) &&
                          (j < 2 || mbar_wait_bounded(pv_done + 8 * (j & 1), ((j >> 1) - 1) & 1, dead)));
            if (!ok) break;
            tcgen05_after_sync();
            const uint64_t k = k_desc + stage * (TILE / 16);
            const uint32_t s = tmem + S_COL + kUmmaKeys * (j & 1);
            if (elect_one()) {
#pragma unroll
                for (int x = 0; x < DP / 16; ++x)
                    umma_ss(s, q_desc + ((x / 4) * (kUmmaRows * 128) + (x % 4) * 32) / 16, k + ((x / 4) * BOX + (x % 4) * 32) / 16, S_DESC, x > 0);
                umma_commit(empty + 8 * stage);
                umma_commit(s_full + 8 * (j & 1));
            }
            __syncwarp();
            next();
            if (j > 0) ok = values(j - 1);
        }
        if (ok) values(n_tiles - 1);
        // products in flight end before their operands and TMEM go away, also when a wait ran out
        if (elect_one()) {
            umma_commit(drained);
            for (uint32_t n = 0; n < kDrainPolls && !mbar_try_wait(drained, 0); ++n) __nanosleep(64);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: one thread per query row (of a copy) ----------------
        const int quad = warp & 3, rep = quad / QUADS;   // the TMEM lanes this warp can reach: 32 * quad ..
        const int r = (quad % QUADS) * 32 + lane;
        if (quad % QUADS < copy_warps) {
            const int st = (rep * copy_warps + quad % QUADS) * 32 + lane, threads = 32 * softmax_warps;   // rank among the working threads
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
            const bool real = r < rows;
            const unsigned char* tree = P.tree + (size_t)(P.tree_per_sample ? cut.b : 0) * P.tokens * P.tokens;
            // c > 0: a negative scale flips the scores' sign instead, and a zero one becomes too small to matter (0 * -inf is NaN)
            const bool flip = P.scale < 0.f;
            const float c = fmaxf(fabsf(P.scale) * 1.4426950408889634f, 1e-30f);
            // tiles of the cache's inside are visible as a whole; the first and last ones and the drafted tokens' need masks
            const int whole_from = cut.sr.first % kUmmaKeys != 0 ? 1 : 0, whole_to = cut.cache_tiles - (cut.sr.row % kUmmaKeys != 0 ? 1 : 0);
            // The drafted tokens' k and v go to the cache two 16-byte vectors a tile and thread, loaded before the wait for S and
            // stored after the softmax: in one go they would cost a row of memory latencies (100 tokens of 512 bytes: 13 us).
            constexpr int VPR = ROWB / 16;
            const int news = cut.owns_new_tokens() ? 2 * P.tokens * VPR : 0;
            int sent = st;
            auto fetch = [&](int i) {
                const int kv = i >= P.tokens * VPR ? 1 : 0;
                const uint4* from = static_cast<const uint4*>(kv ? P.v : P.k) + (size_t)cut.bh * P.tokens * VPR;
                return from[i - kv * P.tokens * VPR];
            };
            auto append = [&](int i, uint4 x) {
                const int kv = i >= P.tokens * VPR ? 1 : 0;
                i -= kv * P.tokens * VPR;
                unsigned char* to = static_cast<unsigned char*>(kv ? P.v_cache : P.k_cache);
                *reinterpret_cast<uint4*>(to + cache_row_offset(P, cut.bh, cut.sr.row + i / VPR, ROWB) + (i % VPR) * 16) = x;
            };
            float m = -CUDART_INF_F, l = 0.f;
            // TMEM instructions are taken by whole warps: a wait that ran out for one lane ran out for all
            auto together = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
            bool ok = true;
            for (int j = 0; j < n_tiles; ++j) {
                const int u = cut.u0 + j;
                const bool cached = u < cut.cache_tiles, masked = u < whole_from || u >= whole_to;
                uint4 new0, new1;
                if (sent < news) new0 = fetch(sent);
                if (sent + threads < news) new1 = fetch(sent + threads);
                ok = together(mbar_wait_bounded(s_full + 8 * (j & 1), (j >> 1) & 1, dead));
                if (!ok) break;
                tcgen05_after_sync();
                const uint32_t s_addr = lanes + S_COL + kUmmaKeys * (j & 1);
                uint32_t s[COLS];
                if constexpr (COLS == 64) tmem_ld32<0>(s_addr, s), tmem_ld32<32>(s_addr + 32, s);
                else if constexpr (COLS == 32) tmem_ld32<0>(s_addr + 32 * rep, s);
                else tmem_ld16<0>(s_addr + 16 * rep, s);
                tmem_wait_ld(s);
                if (flip) {
#pragma unroll
                    for (int i = 0; i < COLS; ++i) s[i] ^= 0x80000000u;
                }
                int first = 0, lo = 0, hi = kUmmaKeys;   // valid keys of the tile
                if (masked) {
                    first = (cached ? cut.c0 + u : u - cut.cache_tiles) * kUmmaKeys;
                    if (cached) lo = max(0, cut.sr.first - first), hi = min(kUmmaKeys, cut.sr.row - first);
                    else hi = min(kUmmaKeys, P.tokens - first);
                    unsigned long long visible = (hi >= 64 ? ~0ull : (1ull << hi) - 1ull) & ~((1ull << lo) - 1ull);
                    if (!cached) {
                        unsigned long long see = 0;
                        if (real) {
                            const unsigned char* sees = tree + (size_t)((row0 + r) % P.tokens) * P.tokens + first;
                            for (int i = rep * COLS; i < min(hi, (rep + 1) * COLS); ++i) see |= (unsigned long long)(sees[i] != 0) << i;
                        }
                        visible &= see;
                    }
                    visible >>= rep * COLS;
#pragma unroll
                    for (int i = 0; i < COLS; ++i)
                        if (!((visible >> i) & 1)) s[i] = 0xff800000u;
                }
                float top = -CUDART_INF_F, top2 = -CUDART_INF_F;
#pragma unroll
                for (int i = 0; i < COLS; i += 4) {
                    top = max3_nan(top, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
                    top2 = max3_nan(top2, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                }
                top = real ? max3_nan(top, top2, top2) * c : -CUDART_INF_F;
                if (!(top < CUDART_INF_F)) l = CUDART_NAN_F;   // a visible NaN or infinite score: the row is NaN whatever its other weights
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, top > m + kLazyRescale)) {
                    const float raised = fmaxf(m, top);
                    const float f = m == -CUDART_INF_F ? 0.f : fast_exp2(m - raised);
                    m = raised, l *= f;
                    ok = together(mbar_wait_bounded(pv_done + 8 * ((j - 1) & 1), ((j - 1) >> 1) & 1, dead));   // O holds the tiles before this one
                    if (!ok) break;
                    tcgen05_after_sync();
#pragma unroll
                    for (int x = 0; x < DP; x += 16) {
                        uint32_t o[16];
                        tmem_ld16<0>(lanes + x, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16<0>(lanes + x, o);
                    }
                    tmem_wait_st();
                }
                const float minus = m == -CUDART_INF_F ? 0.f : -m;
                const float2 cc = make_float2(c, c), mm = make_float2(minus + weight_shift<T>(), minus + weight_shift<T>());
                float2 la = make_float2(0.f, 0.f), lb = make_float2(0.f, 0.f);
                constexpr int OWN = COLS / 16 * WORDS;
                uint32_t p[OWN];   // per 16 keys 8 words of weights and then, if there are any, 8 of their rests
                auto weigh = [&](auto fma_tag) {
#pragma unroll
                    for (int i = 0; i < COLS / 2; ++i) {
                        const float2 y = __ffma2_rn(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), cc, mm);
                        const float2 x = decltype(fma_tag)::value && i % 8 < kFmaPairs ? exp2_fma(y) : make_float2(fast_exp2(y.x), fast_exp2(y.y));
                        if (i & 1) lb = __fadd2_rn(lb, x);
                        else la = __fadd2_rn(la, x);
                        const uint32_t w = pack2<T>(x.x, x.y);
                        p[i / 8 * WORDS + i % 8] = w;
                        if constexpr (RESTS) {
                            const float2 rest = __ffma2_rn(unpack2<T>(w), make_float2(-1.f, -1.f), x);
                            p[i / 8 * WORDS + i % 8 + 8] = pack2<T>(rest.x, rest.y);
                        }
                    }
                };
                // where a score may be -inf its weight has to be 0, so that a row which sees nothing adds up to 0
                if (masked) weigh(std::false_type{});
                else weigh(std::true_type{});
                l += (la.x + la.y) + (lb.x + lb.y);
                if constexpr (REP == 1) {
                    tmem_st32<0>(s_addr, p);
                } else {   // the other copies' keys get weight 0 in this one
                    static_assert(OWN == 16, "a share of the keys is 16 columns of P");
                    uint32_t none[OWN];
#pragma unroll
                    for (int i = 0; i < OWN; ++i) none[i] = 0;
#pragma unroll
                    for (int i = 1; i < REP; ++i) tmem_st16<0>(s_addr + ((rep + i) % REP) * OWN, none);
                    tmem_st16<0>(s_addr + rep * OWN, p);
                }
                if (masked) {
                    // What V holds outside the valid rows, and infinities and NaN of drafted tokens, must not meet a weight of 0:
                    // cleared in shared memory (the latter remembered for the end).
                    const uint32_t at = j < n_tiles - 1 ? 2 * j + 2 : 2 * n_tiles - 1;   // V_j's place in the order of loads
                    const uint32_t slot = at % STAGES;
                    ok = together(mbar_wait_bounded(full + 8 * slot, (at / STAGES) & 1, dead));
                    if (!ok) break;
                    unsigned char* vt = raw + umma_q_bytes(DH) + slot * TILE;
                    for (int i = st; i < kUmmaKeys * NB * 8; i += threads) {
                        const int key = (i >> 3) % kUmmaKeys;
                        uint4* vec = reinterpret_cast<uint4*>(vt + (size_t)i * 16);   // box, key, 16 bytes: any order within a row does
                        if (key < lo || key >= hi) {
                            *vec = make_uint4(0, 0, 0, 0);
                        } else if (!cached) {
                            uint4 x = *vec;
                            const uint4 mk = make_uint4(nonfinite_mask<T>(x.x), nonfinite_mask<T>(x.y), nonfinite_mask<T>(x.z), nonfinite_mask<T>(x.w));
                            if (mk.x | mk.y | mk.z | mk.w) {
                                x.x &= ~mk.x, x.y &= ~mk.y, x.z &= ~mk.z, x.w &= ~mk.w;
                                *vec = x;
                                atomicOr(&bad[(first + key) >> 5], 1u << ((first + key) & 31));
                                tail.any_bad = 1;
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                tmem_wait_st();
                tcgen05_before_sync();
                mbar_arrive(p_ready + 8 * (j & 1));
                if (sent < news) append(sent, new0);
                if (sent + threads < news) append(sent + threads, new1);
                sent += 2 * threads;
            }
            for (; sent < news; sent += 4 * threads) {   // more tokens than the tiles had room for
                uint4 x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (sent + i * threads < news) x[i] = fetch(sent + i * threads);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (sent + i * threads < news) append(sent + i * threads, x[i]);
            }
            // (A barrier per parity of the tile: this thread may come here long after the last product, and one barrier for all of
            // them would by then have passed the phase before it, which a wait by parity takes for one still to come.)
            if (ok) ok = together(mbar_wait_bounded(pv_done + 8 * ((n_tiles - 1) & 1), ((n_tiles - 1) >> 1) & 1, dead));
            // every product and copy is through: O goes through the operands' shared memory, where the copies of a row meet
            float* const o_smem = reinterpret_cast<float*>(raw);
            constexpr int STRIDE = ffa_tree_part_stride(DH);
            if (ok) {
                tcgen05_after_sync();
                float* mine = o_smem + (size_t)(rep * rows + r) * STRIDE;
                uint32_t poisoned = 0;
#pragma unroll 1
                for (int x = 0; x < DH; x += 16) {
                    uint32_t o[16];
                    tmem_ld16<0>(lanes + x, o);
                    tmem_wait_ld(o);
                    if (real) {
                        float zero = 0.f;   // NaN once one of them is not finite
#pragma unroll
                        for (int i = 0; i < 16; ++i) zero = fmaf(0.f, __uint_as_float(o[i]), zero);
                        if (zero != 0.f) poisoned |= 1u << (x / 16);
#pragma unroll
                        for (int i = 0; i < 16; i += 4) *reinterpret_cast<uint4*>(mine + x + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    }
                    __syncwarp();
                }
                if (real) mine[DH] = m, mine[DH + 1] = l;
                if (poisoned) atomicOr(&tail.poisoned, poisoned);
            }
            named_bar_sync(1, threads);   // (every warp comes here, also after a wait that ran out)
            const uint32_t poisoned = tail.poisoned;
            if (poisoned) {   // (the same for all of them)
                find_nonfinite<T, DH>(P, cut.bh, max(cut.sr.first, (cut.c0 + cut.u0) * kUmmaKeys),
                                      min(cut.sr.row, (cut.c0 + min(cut.u1, cut.cache_tiles)) * kUmmaKeys), poisoned, tail.pos, tail.neg, st, threads);
                named_bar_sync(1, threads);
            }
            if (ok) {
                constexpr int OCT = DH / 8;   // eight columns at a time
                for (int i = st; i < rows * OCT; i += threads) {
                    const int row = i / OCT, x = (i - row * OCT) * 8;
                    float w[REP], M = -CUDART_INF_F, L = 0.f;
#pragma unroll
                    for (int q = 0; q < REP; ++q) M = fmaxf(M, o_smem[(size_t)(q * rows + row) * STRIDE + DH]);
#pragma unroll
                    for (int q = 0; q < REP; ++q) {
                        const float mq = o_smem[(size_t)(q * rows + row) * STRIDE + DH];
                        w[q] = mq == -CUDART_INF_F ? 0.f : fast_exp2(mq - M);
                        L = fmaf(w[q], o_smem[(size_t)(q * rows + row) * STRIDE + DH + 1], L);
                    }
                    float o[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = 0.f;
#pragma unroll
                    for (int q = 0; q < REP; ++q) {
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const float4 y = *reinterpret_cast<const float4*>(o_smem + (size_t)(q * rows + row) * STRIDE + x + e);
                            o[e] = fmaf(w[q], y.x, o[e]), o[e + 1] = fmaf(w[q], y.y, o[e + 1]);
                            o[e + 2] = fmaf(w[q], y.z, o[e + 2]), o[e + 3] = fmaf(w[q], y.w, o[e + 3]);
                        }
                    }
                    if (poisoned) {   // an infinity or NaN in a cached row decides its column, whatever its weight
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const bool up = (tail.pos[x >> 5] >> ((x & 31) + e)) & 1, down = (tail.neg[x >> 5] >> ((x & 31) + e)) & 1;
                            if (up || down) o[e] = up && down ? CUDART_NAN_F : up ? CUDART_INF_F : -CUDART_INF_F;
                        }
                    }
                    if (tail.any_bad) {   // and so does one in a drafted token that the row sees
                        const T* v = static_cast<const T*>(P.v) + (size_t)cut.bh * P.tokens * DH + x;
                        const unsigned char* sees = tree + (size_t)((row0 + row) % P.tokens) * P.tokens;
                        for (int k = 0; k < P.tokens; ++k) {
                            if (!((bad[k >> 5] >> (k & 31)) & 1) || sees[k] == 0) continue;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float y = Elem<T>::to_float(v[(size_t)k * DH + e]);
                                if (!isfinite(y)) o[e] += y;
                            }
                        }
                    }
                    if (whole) {
                        const float inv = L == 0.f ? 0.f : 1.f / L;
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = pack2<T>(o[2 * e] * inv, o[2 * e + 1] * inv);
                        *reinterpret_cast<uint4*>(out + (size_t)row * DH + x) = make_uint4(y[0], y[1], y[2], y[3]);
                    } else {
                        float* to = part + (size_t)row * STRIDE;
                        *reinterpret_cast<float4*>(to + x) = make_float4(o[0], o[1], o[2], o[3]);
                        *reinterpret_cast<float4*>(to + x + 4) = make_float4(o[4], o[5], o[6], o[7]);
                        if (x == 0) to[DH] = M, to[DH + 1] = L;
                    }
                }
            }
        }
    }
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    if (warp == 1) tmem_dealloc(tmem, umma_tmem_cols(DH));
    if (tid == 0 && flags[0]) {
        atomicOr(P.status, kStatusWaitTimeout);
        // a wait ran out: let the copies already issued land before the CTA releases its shared memory (bounded again)
        const uint32_t pending = issued < STAGES ? issued : STAGES;
        for (uint32_t k = 0; k < pending; ++k) {
            const uint32_t id = issued - 1 - k;
            for (uint32_t n = 0; n < kDrainPolls && !mbar_try_wait(full + 8 * (id % STAGES), (id / STAGES) & 1); ++n) __nanosleep(256);
        }
        for (uint32_t n = 0; n < kDrainPolls && !mbar_try_wait(q_full, 0); ++n) __nanosleep(256);
    }
}

}  // namespace ffa_dev
