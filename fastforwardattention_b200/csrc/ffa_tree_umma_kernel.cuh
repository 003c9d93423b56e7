// Tree attention on the tensor cores (fp16, bf16): tcgen05 products with the accumulators in TMEM, operands by TMA.
//
// A CTA owns a tile of up to 128 query rows of one (batch, head) -- all drafted tokens of all query heads that share the
// cache head -- and a run of key tiles of 64 rows.  Per tile
//     S = Q K^T  [128 x 64]   fp32 in TMEM; Q and K are K-major operands in 128-byte-swizzled shared memory
//     P = exp2(c S - m)       one thread per query row: TMEM -> registers -> 16-bit P back into S's columns
//     O += P V   [128 x Dh]   A = P from TMEM, B = V as it lies in the cache (MN-major)
// so a cache row is read from HBM once for all query rows.  The matrix units idle most of the time even with every product
// padded to 128 rows (64 KB of K and V take 2.8 us of an SM's share of HBM, the products 0.5 us): what bounds a long cache is HBM.
//
// Warps: 0 issues the TMA loads, 1 allocates TMEM and issues the products, 2..5 do the softmax (a warp can only reach the 32 TMEM
// lanes of its rank modulo 4).  S has two buffers, so that S of the next tile is computed while the softmax of this one runs.
// The running maximum is raised lazily: weights are taken relative to a reference that follows the true maximum only when that
// is more than 8 (in powers of two) ahead, so O is rarely rescaled and weights stay below 256, exact in either type's range.
// P is rounded to the tensors' type, the sum is taken of the unrounded weights in fp32.
#pragma once
#include <cuda.h>

#include "ffa_tree_kernel.cuh"

namespace ffa_dev {

constexpr int kUmmaRows = 128;     // query rows per CTA
constexpr int kUmmaKeys = 64;      // keys per tile
constexpr int kUmmaThreads = 192;
constexpr int kUmmaSoftmaxThreads = 128;
constexpr int kUmmaMaxStages = 12;
constexpr int kQBoxRows = 32;      // Q arrives in boxes of 32 rows: a short tree loads one
constexpr float kLazyRescale = 8.f;

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
    int flags[2];                      // [0] a wait ran out, [1] last arriver
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
// 32 consecutive columns of this warp's 32 lanes: register i = column i of the thread's lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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

template <typename T, int DH>
__global__ void __launch_bounds__(kUmmaThreads, umma_ctas_per_sm(DH)) ffa_tree_umma_kernel(const __grid_constant__ FfaTreeUmmaParams U)
{
    constexpr int DP = umma_dp(DH), NB = DP / 64, TILE = umma_tile_bytes(DH), STAGES = umma_stages(DH), ROWB = DH * 2;
    constexpr int BOX = 64 * 128;   // bytes of a tile's box: 64 rows of 128 bytes
    constexpr uint32_t S_COL = DP;  // TMEM columns: O at 0, the two S / P buffers behind it
    const FfaTreeParams& P = U.p;
    // No static shared memory: the dynamic part then starts on the 1024-byte boundary that swizzled operands need, without
    // slack (two CTAs with 112 KB of operands leave 1.5 KB of an SM)
    extern __shared__ __align__(1024) unsigned char raw[];
    UmmaTail& tail = *reinterpret_cast<UmmaTail*>(raw + umma_q_bytes(DH) + STAGES * TILE);
    int* flags = tail.flags;
    uint32_t* bad = tail.bad;
    const uint32_t q_smem = smem_u32(raw), ring = q_smem + umma_q_bytes(DH);
    const uint32_t full = smem_u32(tail.bars), empty = full + 8 * STAGES, q_full = empty + 8 * STAGES, s_full = q_full + 8, p_ready = s_full + 16,
                   pv_done = p_ready + 16, drained = pv_done + 8;
    volatile int* dead = flags;

    pdl_release();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int R = P.groups * P.tokens;
    if (tid == 0) {
        flags[0] = 0, flags[1] = 0, tail.any_bad = 0;
        tma_prefetch_map(&U.q), tma_prefetch_map(&U.k_cache), tma_prefetch_map(&U.v_cache), tma_prefetch_map(&U.k_new), tma_prefetch_map(&U.v_new);
    }
    if (tid >= 64 && tid < 64 + kTreeMaxRows / 32) bad[tid - 64] = 0;
    pdl_wait();
    const TreeCut<kUmmaKeys> cut(P);
    if (cut.split >= cut.splits) return;
    const int row0 = cut.rt * kUmmaRows, rows = min(kUmmaRows, R - row0);
    T* out = static_cast<T*>(P.out) + ((size_t)cut.bh * R + row0) * DH;
    if (!cut.sr.ok) {   // refused: zeros, nothing appended
        if (cut.split == 0) {
            for (int i = tid; i < rows * DH; i += kUmmaThreads) Elem<T>::store(out + i, 0.f);
            if (tid == 0) atomicOr(P.status, kStatusBadLength);
        }
        return;
    }
    const int softmax_warps = (rows + 31) / 32;   // warps whose rows exist
    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1);
        mbar_init(q_full, 1);
        for (int i = 0; i < 2; ++i) mbar_init(s_full + 8 * i, 1), mbar_init(p_ready + 8 * i, 32 * softmax_warps);
        mbar_init(pv_done, 1), mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // after pdl_wait: a CTA that held TMEM while it waits for the previous grid could keep that grid from ever finishing
    if (warp == 1) tmem_alloc(smem_u32(&tail.tmem_base), umma_tmem_cols(DH)), tmem_relinquish();
    tcgen05_before_sync();
    __syncthreads();
    tcgen05_after_sync();
    const uint32_t tmem = tail.tmem_base;
    const int n_tiles = cut.u1 - cut.u0;
    uint32_t issued = 0;   // K and V loads of the issuing thread

    if (warp == 0) {
        // ---------------- TMA ----------------
        if (lane == 0) {
            mbar_expect_tx(q_full, (uint32_t)(softmax_warps * kQBoxRows * 128 * NB));
            for (int x = 0; x < NB; ++x)
                for (int i = 0; i < softmax_warps; ++i)
                    tma_load_2d(q_smem + x * (kUmmaRows * 128) + i * (kQBoxRows * 128), &U.q, 64 * x, cut.bh * R + row0 + i * kQBoxRows, q_full);
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
        if (lane == 0) {
            constexpr uint32_t S_DESC = umma_idesc<T>(kUmmaKeys, false), O_DESC = umma_idesc<T>(DP, true);
            uint32_t stage = 0, phase = 0;
            auto next = [&]() {
                if (++stage == STAGES) stage = 0, phase ^= 1;
            };
            auto values = [&](int j) -> bool {   // O += P_j V_j
                if (!mbar_wait_bounded(p_ready + 8 * (j & 1), (j >> 1) & 1, dead)) return false;
                if (!mbar_wait_bounded(full + 8 * stage, phase, dead)) return false;
                tcgen05_after_sync();
                const uint32_t v = ring + stage * TILE, p = tmem + S_COL + kUmmaKeys * (j & 1);
#pragma unroll
                for (int k = 0; k < kUmmaKeys / 16; ++k)   // 16 keys: 8 columns of packed P, two atoms of V
                    umma_ts(tmem, p + 8 * k, umma_desc(v + 2048 * k, BOX, 1024), O_DESC, j > 0 || k > 0);
                umma_commit(empty + 8 * stage);
                umma_commit(pv_done);
                next();
                return true;
            };
            bool ok = mbar_wait_bounded(q_full, 0, dead);
            for (int j = 0; ok && j < n_tiles; ++j) {
                // S_j goes where P_(j-2) was: that product has to be through
                ok = mbar_wait_bounded(full + 8 * stage, phase, dead) && (j < 2 || mbar_wait_bounded(pv_done, j & 1, dead));
                if (!ok) break;
                tcgen05_after_sync();
                const uint32_t k = ring + stage * TILE, s = tmem + S_COL + kUmmaKeys * (j & 1);
#pragma unroll
                for (int x = 0; x < DP / 16; ++x)
                    umma_ss(s, umma_desc(q_smem + (x / 4) * (kUmmaRows * 128) + (x % 4) * 32, 0, 1024),
                            umma_desc(k + (x / 4) * BOX + (x % 4) * 32, 0, 1024), S_DESC, x > 0);
                umma_commit(empty + 8 * stage);
                umma_commit(s_full + 8 * (j & 1));
                next();
                if (j > 0) ok = values(j - 1);
            }
            if (ok) values(n_tiles - 1);
            // products in flight end before their operands and TMEM go away, also when a wait ran out
            umma_commit(drained);
            for (uint32_t n = 0; n < kDrainPolls && !mbar_try_wait(drained, 0); ++n) __nanosleep(64);
        }
        __syncwarp();
    } else {
        // ---------------- softmax: one thread per query row ----------------
        const int quad = warp & 3;            // the TMEM lanes this warp can reach: rows 32 * quad ..
        const int r = quad * 32 + lane;
        const int st = tid - 64;              // 0..127
        if (cut.owns_new_tokens()) tree_append(P, cut.bh, cut.sr.row, ROWB, st, kUmmaSoftmaxThreads);
        if (quad < softmax_warps) {
            const int ft = r, fixers = 32 * softmax_warps;   // threads that repair a tile of V between them
            const uint32_t lanes = (uint32_t)(quad * 32) << 16;
            const bool real = r < rows;
            const int t = (row0 + r) % P.tokens;
            const unsigned char* sees = P.tree + ((size_t)(P.tree_per_sample ? cut.b : 0) * P.tokens + t) * P.tokens;
            // c > 0: a negative scale flips the scores' sign instead, and a zero one becomes too small to matter (0 * -inf is NaN)
            const bool flip = P.scale < 0.f;
            const float c = fmaxf(fabsf(P.scale) * 1.4426950408889634f, 1e-30f);
            float m = -CUDART_INF_F, l = 0.f;
            // TMEM instructions are taken by whole warps: a wait that ran out for one lane ran out for all
            auto together = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
            bool ok = true;
            for (int j = 0; j < n_tiles; ++j) {
                const int u = cut.u0 + j;
                const bool cached = u < cut.cache_tiles;
                const int first = (cached ? cut.c0 + u : u - cut.cache_tiles) * kUmmaKeys;
                const int lo = cached ? max(0, cut.sr.first - first) : 0;
                const int hi = cached ? min(kUmmaKeys, cut.sr.row - first) : min(kUmmaKeys, P.tokens - first);
                unsigned long long visible = ~0ull;
                if (lo > 0 || hi < kUmmaKeys) visible = (hi >= 64 ? ~0ull : (1ull << hi) - 1ull) & ~((1ull << lo) - 1ull);
                if (!cached) {
                    unsigned long long see = 0;
                    if (real)
                        for (int i = 0; i < hi; ++i) see |= (unsigned long long)(sees[first + i] != 0) << i;
                    visible &= see;
                }
                ok = together(mbar_wait_bounded(s_full + 8 * (j & 1), (j >> 1) & 1, dead));
                if (!ok) break;
                tcgen05_after_sync();
                const uint32_t s_addr = tmem + lanes + S_COL + kUmmaKeys * (j & 1);
                uint32_t a[32], b[32];
                tmem_ld32(s_addr, a);
                tmem_ld32(s_addr + 32, b);
                tmem_wait_ld();
                if (flip) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) a[i] ^= 0x80000000u, b[i] ^= 0x80000000u;
                }
                if (__any_sync(0xffffffffu, visible != ~0ull)) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        if (!((visible >> i) & 1)) a[i] = 0xff800000u;
                        if (!((visible >> (32 + i)) & 1)) b[i] = 0xff800000u;
                    }
                }
                float top = -CUDART_INF_F, top2 = -CUDART_INF_F;
#pragma unroll
                for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(a[i])), top2 = fmaxf(top2, __uint_as_float(b[i]));
                top = real ? fmaxf(top, top2) * c : -CUDART_INF_F;
                if (j == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, top > m + kLazyRescale)) {
                    const float raised = fmaxf(m, top);
                    const float f = m == -CUDART_INF_F ? 0.f : fast_exp2(m - raised);
                    m = raised, l *= f;
                    ok = together(mbar_wait_bounded(pv_done, (j - 1) & 1, dead));   // O holds the tiles before this one
                    if (!ok) break;
                    tcgen05_after_sync();
#pragma unroll
                    for (int x = 0; x < DP; x += 32) {
                        uint32_t o[32];
                        tmem_ld32(tmem + lanes + x, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st32(tmem + lanes + x, o);
                    }
                    tmem_wait_st();
                }
                const float minus = m == -CUDART_INF_F ? 0.f : -m;
                float l0 = 0.f, l1 = 0.f, l2 = 0.f, l3 = 0.f;
                uint32_t p[32];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x0 = fast_exp2(fmaf(__uint_as_float(a[2 * i]), c, minus)), x1 = fast_exp2(fmaf(__uint_as_float(a[2 * i + 1]), c, minus));
                    const float y0 = fast_exp2(fmaf(__uint_as_float(b[2 * i]), c, minus)), y1 = fast_exp2(fmaf(__uint_as_float(b[2 * i + 1]), c, minus));
                    l0 += x0, l1 += x1, l2 += y0, l3 += y1;
                    p[i] = pack2<T>(x0, x1), p[16 + i] = pack2<T>(y0, y1);
                }
                l += (l0 + l1) + (l2 + l3);
                tmem_st32(s_addr, p);
                if (lo > 0 || hi < kUmmaKeys || !cached) {
                    // What V holds outside the valid rows, and infinities and NaN of drafted tokens, must not meet a weight of 0:
                    // cleared in shared memory (the latter remembered for the end).
                    const uint32_t at = j < n_tiles - 1 ? 2 * j + 2 : 2 * n_tiles - 1;   // V_j's place in the order of loads
                    const uint32_t slot = at % STAGES;
                    ok = together(mbar_wait_bounded(full + 8 * slot, (at / STAGES) & 1, dead));
                    if (!ok) break;
                    unsigned char* vt = raw + umma_q_bytes(DH) + slot * TILE;
                    for (int i = ft; i < kUmmaKeys * NB * 8; i += fixers) {
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
            }
            // one phase after the other: the barrier tells phases apart by their parity only
            if (ok && n_tiles > 1) ok = together(mbar_wait_bounded(pv_done, n_tiles & 1, dead));
            if (ok) ok = together(mbar_wait_bounded(pv_done, (n_tiles - 1) & 1, dead));
            named_bar_sync(1, 32 * softmax_warps);   // `bad` is complete (every warp comes here, also after a wait that ran out)
            if (ok) {
                tcgen05_after_sync();
                const bool whole = cut.splits == 1, fix = tail.any_bad != 0;
                const float inv = whole ? (l > 0.f ? 1.f / l : 0.f) : 1.f;
                const size_t tile_index = (size_t)cut.bh * P.row_tiles + cut.rt;
                float* part = whole ? nullptr : P.partials + ((tile_index * P.splits + cut.split) * P.part_rows + r) * ffa_tree_part_stride(DH);
#pragma unroll 1
                for (int x = 0; x < DH; x += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem + lanes + x, o);
                    tmem_wait_ld();
                    if (real) {
                        if (fix) {   // a visible infinity or NaN decides its column
                            const T* v = static_cast<const T*>(P.v) + (size_t)cut.bh * P.tokens * DH;
                            for (int k = 0; k < P.tokens; ++k) {
                                if (!((bad[k >> 5] >> (k & 31)) & 1) || sees[k] == 0) continue;
    #pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    if (x + i < DH) {
                                        const float y = Elem<T>::to_float(v[(size_t)k * DH + x + i]);
                                        if (!isfinite(y)) o[i] = __float_as_uint(__uint_as_float(o[i]) + y);
                                    }
                                }
                            }
                        }
    #pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (x + i < DH) {
                                if (whole) {
                                    uint32_t w[4];
    #pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        w[e] = pack2<T>(__uint_as_float(o[i + 2 * e]) * inv, __uint_as_float(o[i + 2 * e + 1]) * inv);
                                    *reinterpret_cast<uint4*>(out + (size_t)r * DH + x + i) = make_uint4(w[0], w[1], w[2], w[3]);
                                } else {
                                    *reinterpret_cast<uint4*>(part + x + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                                    *reinterpret_cast<uint4*>(part + x + i + 4) = make_uint4(o[i + 4], o[i + 5], o[i + 6], o[i + 7]);
                                }
                            }
                        }
                    }
                    __syncwarp();
                }
                if (!whole && real) part[DH] = m, part[DH + 1] = l;
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
    if (cut.splits == 1) return;
    // whoever arrives last merges; nobody waits (the fences are those of the decode kernels' merge)
    int* ticket = P.tickets + cut.bh * kTreeTicketsPerPair + cut.rt;
    if (tid == 0) {
        __threadfence();
        flags[1] = atomicAdd(ticket, 1) == cut.splits - 1;
        __threadfence();
    }
    __syncthreads();
    if (flags[1]) {
        const size_t tile_index = (size_t)cut.bh * P.row_tiles + cut.rt;
        tree_merge<T, DH, true>(P.partials + tile_index * P.splits * P.part_rows * ffa_tree_part_stride(DH), cut.splits, P.part_rows, rows, out, tid, kUmmaThreads);
        if (tid == 0) *ticket = 0;
    }
}

}  // namespace ffa_dev
