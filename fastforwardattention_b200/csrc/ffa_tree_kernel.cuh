// Attention of a tree of drafted tokens over a cache, and the acceptance of a verified path.
//
//   S[r, j] = scale * q_r . k_j     j over the cache rows first..n-1 (visible to every row) and the drafted tokens
//                                   (visible where tree[t(r), j]); r = (query head of the group, drafted token)
//   O[r]    = sum_j exp(S[r, j] - m_r) v_j / sum_j exp(S[r, j] - m_r);  a row that sees nothing is 0
//
// The drafted tokens are read from the call's k and v and appended to the cache by one CTA of the pair, so no CTA ever
// waits for another one's append.
#pragma once
#include "ffa_device_common.cuh"

namespace ffa_dev {

constexpr int kTreeThreads = 256;
constexpr int kTreeWarps = kTreeThreads / 32;
constexpr int kTreeKeys = 32;   // keys per tile of the CUDA-core kernel: one per lane

// What one CTA of a tree attention works on: a pair, a tile of its query rows, a run of its key tiles.  Key tiles are
// whole tiles of the cache (KEYS rows, aligned to KEYS) followed by tiles of drafted tokens; a sample with fewer tiles
// than splits uses one split per tile.
template <int KEYS>
struct TreeCut {
    int bh, b, rt, split, splits;   // splits that own at least one tile
    int c0, cache_tiles, u0, u1;    // first cache tile, number of them, this split's run of tiles
    SampleRange sr;
    __device__ __forceinline__ explicit TreeCut(const FfaTreeParams& P)
    {
        int i = blockIdx.x;
        rt = i % P.row_tiles, i /= P.row_tiles;
        split = i % P.splits, bh = i / P.splits;
        b = bh / P.H;
        sr = sample_range(P, b);
        if (sr.ok && sr.row > P.Lmax - P.tokens) sr.ok = false;
        c0 = sr.first / KEYS;
        cache_tiles = sr.ok && sr.row > sr.first ? (sr.row + KEYS - 1) / KEYS - c0 : 0;
        const int tiles = cache_tiles + (P.tokens + KEYS - 1) / KEYS;
        splits = min(P.splits, tiles);
        u0 = split < splits ? (int)((long long)tiles * split / splits) : 0;
        u1 = split < splits ? (int)((long long)tiles * (split + 1) / splits) : 0;
    }
    __device__ __forceinline__ bool owns_new_tokens() const { return split == splits - 1 && rt == 0; }
};

// k and v of the drafted tokens -> rows n..n+tokens-1 of the cache, by `threads` threads
__device__ __forceinline__ void tree_append(const FfaTreeParams& P, int bh, int row, int rowb, int tid, int threads)
{
    const int vpr = rowb / 16;
    const unsigned char* ks = static_cast<const unsigned char*>(P.k) + (size_t)bh * P.tokens * rowb;
    const unsigned char* vs = static_cast<const unsigned char*>(P.v) + (size_t)bh * P.tokens * rowb;
    for (int i = tid; i < P.tokens * vpr; i += threads) {
        const int j = i / vpr, c = i - j * vpr;
        const size_t to = cache_row_offset(P, bh, row + j, rowb) + c * 16;
        *reinterpret_cast<uint4*>(static_cast<unsigned char*>(P.k_cache) + to) = *reinterpret_cast<const uint4*>(ks + (size_t)i * 16);
        *reinterpret_cast<uint4*>(static_cast<unsigned char*>(P.v_cache) + to) = *reinterpret_cast<const uint4*>(vs + (size_t)i * 16);
    }
}

// A split that has no key tiles (a sample shorter than the bound, or refused) leaves an empty partial result: the merge reads
// nothing else of it.
__device__ __forceinline__ float* tree_partial(const FfaTreeParams& P, int bh, int rt, int split, int dh)
{
    return P.partials + (((size_t)bh * P.row_tiles + rt) * P.splits + split) * P.part_rows * ffa_tree_part_stride(dh);
}
__device__ __forceinline__ void tree_empty_partial(float* part, int rows, int dh, int tid, int threads)
{
    for (int r = tid; r < rows; r += threads) {
        part[(size_t)r * ffa_tree_part_stride(dh) + dh] = -CUDART_INF_F;
        part[(size_t)r * ffa_tree_part_stride(dh) + dh + 1] = 0.f;
    }
}

// Combines the splits' partial results in split order.  A warp per query row: the lanes find the row's maximum and sum (a split
// each), then take the columns (16 bytes of every partial at a time, eight partials in flight).  A kernel of its own rather than
// the work of the CTA that arrives last: 128 rows of nine splits are 600 KB, which one CTA takes 20 us and more to read and the
// whole device a few; launched with programmatic overlap it costs about what the arrival counter and its fences did.
constexpr int kMergeWarps = 4;
template <typename T, int DH, bool kLog2>
__global__ void __launch_bounds__(32 * kMergeWarps) ffa_tree_merge_kernel(const FfaTreeParams P)
{
    constexpr int STRIDE = ffa_tree_part_stride(DH), VECS = DH / 4, VPL = (VECS + 31) / 32;
    __shared__ float weight[kMergeWarps][kTreeMaxSplits];
    pdl_release();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int R = P.groups * P.tokens;
    const long long row = (long long)blockIdx.x * kMergeWarps + warp;
    if (row >= (long long)P.B * P.H * R) return;
    const int bh = (int)(row / R), r = (int)(row - (long long)bh * R), rt = r / P.tile_rows;
    const float* part = tree_partial(P, bh, rt, 0, DH) + (size_t)(r - rt * P.tile_rows) * STRIDE;
    const size_t step = (size_t)P.part_rows * STRIDE;
    auto expo = [](float x) { return kLog2 ? fast_exp2(x) : expf(x); };
    float M = -CUDART_INF_F;
    for (int s = lane; s < P.splits; s += 32) M = fmaxf(M, part[s * step + DH]);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    float L = 0.f;
    for (int s = lane; s < P.splits; s += 32) {
        const float m = part[s * step + DH];
        const float w = m == -CUDART_INF_F ? 0.f : expo(m - M);
        // an empty split has no maximum: its columns are not read (a weight of -1); one whose weight vanished still is
        weight[warp][s] = m == -CUDART_INF_F ? -1.f : w;
        L = fmaf(w, part[s * step + DH + 1], L);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    __syncwarp();
    T* out = static_cast<T*>(P.out) + (size_t)row * DH;
#pragma unroll
    for (int x = 0; x < VPL; ++x) {
        const int c = lane + 32 * x;
        if (c >= VECS) break;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < P.splits; s0 += 8) {
            float4 a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (s0 + i < P.splits && weight[warp][s0 + i] >= 0.f) a[i] = *reinterpret_cast<const float4*>(part + (s0 + i) * step + 4 * c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (s0 + i >= P.splits) continue;
                const float w = weight[warp][s0 + i];
                if (!(w >= 0.f)) continue;   // empty, or NaN: then the sum is NaN too
                // a split's infinity stays one however small its share is
                acc.x = isfinite(a[i].x) ? fmaf(w, a[i].x, acc.x) : acc.x + a[i].x;
                acc.y = isfinite(a[i].y) ? fmaf(w, a[i].y, acc.y) : acc.y + a[i].y;
                acc.z = isfinite(a[i].z) ? fmaf(w, a[i].z, acc.z) : acc.z + a[i].z;
                acc.w = isfinite(a[i].w) ? fmaf(w, a[i].w, acc.w) : acc.w + a[i].w;
            }
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        Elem<T>::store(out + 4 * c, acc.x * inv), Elem<T>::store(out + 4 * c + 1, acc.y * inv);
        Elem<T>::store(out + 4 * c + 2, acc.z * inv), Elem<T>::store(out + 4 * c + 3, acc.w * inv);
    }
}

// CUDA-core kernel.  8 warps; a warp owns RPW query rows, a lane one key of the tile: the scores of a row live in one warp, so
// the softmax needs shuffles only.  K and V tiles (32 keys) come through a two-stage cp.async ring with 16 bytes of padding per
// row (a quarter warp's 16-byte reads of 8 different rows then hit different banks).  Rows outside the valid range are
// zero-filled, never read, so that what a cache holds behind its last row cannot reach the result.
template <typename T, int DH, int RPW>
__global__ void __launch_bounds__(kTreeThreads) ffa_tree_simt_kernel(const FfaTreeParams P)
{
    constexpr int BM = kTreeWarps * RPW, BN = kTreeKeys, ROWB = DH * (int)sizeof(T), PITCH = ROWB + 16, VPR = ROWB / 16;
    constexpr int EPV = Elem<T>::EPV, DPL = (DH + 31) / 32;
    extern __shared__ __align__(128) unsigned char smem[];
    float* qs = reinterpret_cast<float*>(smem);                       // [BM][DH], scaled
    unsigned char* ring = smem + (size_t)BM * DH * 4;                  // [2 stages][K | V][BN][PITCH]

    pdl_release();
    pdl_wait();
    const TreeCut<BN> cut(P);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int R = P.groups * P.tokens, row0 = cut.rt * BM, rows = min(BM, R - row0);
    const bool whole = P.splits == 1;
    T* out = static_cast<T*>(P.out) + ((size_t)cut.bh * R + row0) * DH;
    float* part = whole ? nullptr : tree_partial(P, cut.bh, cut.rt, cut.split, DH);
    if (!cut.sr.ok && tid == 0) atomicOr(P.status, kStatusBadLength);   // refused: zeros, nothing appended
    if (!cut.sr.ok || cut.split >= cut.splits) {
        if (!whole) tree_empty_partial(part, rows, DH, tid, kTreeThreads);
        else for (int i = tid; i < rows * DH; i += kTreeThreads) Elem<T>::store(out + i, 0.f);
        return;
    }

    auto load_tile = [&](int u, int stage) {
        const bool cached = u < cut.cache_tiles;
        const int base = (cached ? cut.c0 + u : u - cut.cache_tiles) * BN;
        const int lo = cached ? cut.sr.first : 0, hi = cached ? cut.sr.row : P.tokens;
        const size_t off = cached ? cache_row_offset(P, cut.bh, base, ROWB) : ((size_t)cut.bh * P.tokens + base) * ROWB;
        const unsigned char* ks = static_cast<const unsigned char*>(cached ? P.k_cache : P.k) + off;
        const unsigned char* vs = static_cast<const unsigned char*>(cached ? P.v_cache : P.v) + off;
        const uint32_t dst = smem_u32(ring) + stage * 2 * BN * PITCH;
        for (int i = tid; i < BN * VPR; i += kTreeThreads) {
            const int r = i / VPR, c = i - r * VPR;
            const bool in = base + r >= lo && base + r < hi;
            const size_t from = in ? (size_t)i * 16 : 0;
            cp_async_16_or_zero(dst + r * PITCH + c * 16, in ? ks + from : static_cast<const unsigned char*>(P.k), in ? 16u : 0u);
            cp_async_16_or_zero(dst + (BN + r) * PITCH + c * 16, in ? vs + from : static_cast<const unsigned char*>(P.v), in ? 16u : 0u);
        }
        cp_async_commit();
    };

    load_tile(cut.u0, 0);
    {
        const T* q = static_cast<const T*>(P.q) + ((size_t)cut.bh * R + row0) * DH;
        for (int i = tid; i < BM * DH; i += kTreeThreads) qs[i] = i < rows * DH ? Elem<T>::to_float(q[i]) * P.scale : 0.f;
    }
    if (cut.owns_new_tokens()) tree_append(P, cut.bh, cut.sr.row, ROWB, tid, kTreeThreads);

    float m[RPW], l[RPW], acc[RPW][DPL];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        m[i] = -CUDART_INF_F, l[i] = 0.f;
#pragma unroll
        for (int x = 0; x < DPL; ++x) acc[i][x] = 0.f;
    }
    const bool busy = warp * RPW < rows;   // this warp has query rows
    for (int u = cut.u0; u < cut.u1; ++u) {
        const int stage = (u - cut.u0) & 1;
        if (u + 1 < cut.u1) {
            load_tile(u + 1, stage ^ 1);
            cp_async_wait<1>();
        } else {
            cp_async_wait<0>();
        }
        __syncthreads();
        if (busy) {
            const unsigned char* kt = ring + (size_t)stage * 2 * BN * PITCH;
            const unsigned char* vt = kt + BN * PITCH;
            const bool cached = u < cut.cache_tiles;
            const int key = (cached ? cut.c0 + u : u - cut.cache_tiles) * BN + lane;
            float s[RPW];
#pragma unroll
            for (int i = 0; i < RPW; ++i) s[i] = 0.f;
#pragma unroll 4
            for (int c = 0; c < VPR; ++c) {
                float kf[EPV];
                Elem<T>::unpack(*reinterpret_cast<const uint4*>(kt + lane * PITCH + c * 16), kf);
#pragma unroll
                for (int i = 0; i < RPW; ++i) {
                    const float* qr = qs + (warp * RPW + i) * DH + c * EPV;
#pragma unroll
                    for (int e = 0; e < EPV; e += 4) {
                        const float4 q4 = *reinterpret_cast<const float4*>(qr + e);
                        s[i] = fmaf(q4.x, kf[e], s[i]), s[i] = fmaf(q4.y, kf[e + 1], s[i]);
                        s[i] = fmaf(q4.z, kf[e + 2], s[i]), s[i] = fmaf(q4.w, kf[e + 3], s[i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < RPW; ++i) {
                const int r = row0 + warp * RPW + i;
                bool see = r < R;
                if (cached) {
                    see = see && key >= cut.sr.first && key < cut.sr.row;
                } else {
                    const int t = r % P.tokens;
                    see = see && key < P.tokens &&
                          P.tree[((size_t)(P.tree_per_sample ? cut.b : 0) * P.tokens + t) * P.tokens + key] != 0;
                }
                s[i] = see ? s[i] : -CUDART_INF_F;
                float mx = s[i];
#pragma unroll
                for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                mx = fmaxf(m[i], mx);
                const float base = mx == -CUDART_INF_F ? 0.f : mx;   // nothing seen so far: every weight is 0, not NaN
                const float corr = expf(m[i] - base);
                m[i] = mx;
                s[i] = see ? expf(s[i] - base) : 0.f;
                l[i] = l[i] * corr + s[i];   // this lane's keys; the lanes are added at the end
#pragma unroll
                for (int x = 0; x < DPL; ++x) acc[i][x] *= corr;
            }
#pragma unroll 4
            for (int j = 0; j < BN; ++j) {
                const T* vr = reinterpret_cast<const T*>(vt + j * PITCH);
                float vf[DPL];
#pragma unroll
                for (int x = 0; x < DPL; ++x) vf[x] = (DH % 32 == 0 || lane + 32 * x < DH) ? Elem<T>::to_float(vr[lane + 32 * x]) : 0.f;
#pragma unroll
                for (int i = 0; i < RPW; ++i) {
                    const float pj = __shfl_sync(0xffffffffu, s[i], j);
                    if (pj != 0.f) {   // a hidden token has no part in the row, whatever its values
#pragma unroll
                        for (int x = 0; x < DPL; ++x) acc[i][x] = fmaf(pj, vf[x], acc[i][x]);
                    }
                }
            }
        }
        __syncthreads();   // the stage may be filled again
    }

#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        const int r = warp * RPW + i;
        if (r >= rows) break;
        float L = l[i];
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
#pragma unroll
        for (int x = 0; x < DPL; ++x) {
            const int d = lane + 32 * x;
            if (DH % 32 != 0 && d >= DH) break;
            if (whole) Elem<T>::store(out + r * DH + d, L == 0.f ? 0.f : acc[i][x] / L);
            else part[r * ffa_tree_part_stride(DH) + d] = acc[i][x];
        }
        if (!whole && lane == 0) part[r * ffa_tree_part_stride(DH) + DH] = m[i], part[r * ffa_tree_part_stride(DH) + DH + 1] = L;
    }
}

// Rows n + path[i] -> n + i of every pair, in place.  A thread owns one 16-byte column of K or V and walks the path: indices
// increase, so path[i] >= i and a row is read before anything is written to it (eight rows are read, then eight written).
__global__ void __launch_bounds__(256) ffa_tree_accept_kernel(const FfaAcceptParams P)
{
    const int bh = blockIdx.x, b = bh / P.H;
    const int vpr = P.row_bytes / 16;
    const int* path = P.path + (size_t)b * P.path_len;
    const int n = P.seq_lengths != nullptr ? P.seq_lengths[b] : P.t;
    if (n < 0 || n >= P.Lmax) {
        if (threadIdx.x == 0) atomicOr(P.status, kStatusBadLength);
        return;
    }
    int count = 0, prev = -1;
    for (; count < P.path_len; ++count) {
        const int j = path[count];
        if (j < 0) break;
        if (j <= prev || j >= P.Lmax - n) {
            if (threadIdx.x == 0) atomicOr(P.status, kStatusBadIndex);
            return;
        }
        prev = j;
    }
    if ((int)threadIdx.x >= 2 * vpr) return;
    const int c = threadIdx.x % vpr;
    unsigned char* cache = static_cast<unsigned char*>((int)threadIdx.x < vpr ? P.k_cache : P.v_cache) + c * 16;
    for (int i0 = 0; i0 < count; i0 += 8) {
        uint4 x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < count) x[i] = *reinterpret_cast<const uint4*>(cache + cache_row_offset(P, bh, n + path[i0 + i], P.row_bytes));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i0 + i < count && path[i0 + i] != i0 + i)
                *reinterpret_cast<uint4*>(cache + cache_row_offset(P, bh, n + i0 + i, P.row_bytes)) = x[i];
    }
}

}  // namespace ffa_dev
