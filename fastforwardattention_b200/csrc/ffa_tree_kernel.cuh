// Attention of a tree of drafted tokens over a cache, and the acceptance of a verified path.
//
//   S[r, j] = scale * q_r . k_j     j over the cache rows first..n-1 (visible to every row) and the drafted tokens
//                                   (visible where tree[t(r), j]); r = (query head of the group, drafted token)
//   O[r]    = sum_j exp(S[r, j] - m_r) v_j / sum_j exp(S[r, j] - m_r);  a row that sees nothing is 0
//
// The drafted tokens are read from the call's k and v; the pair's CTAs append them to the cache (fp16, bf16: one of them does), so no CTA ever
// waits for another one's append.
#pragma once
#include "ffa_device_common.cuh"

namespace ffa_dev {

constexpr int kTreeThreads = 256;
constexpr int kTreeKeys = 64;   // keys per tile of the CUDA-core kernel

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

// Whether a page that the sample's rows 0..row+tokens-1 need is missing from its table; the same for all threads of the CTA.
__device__ __forceinline__ bool tree_page_missing(const FfaTreeParams& P, int b, const SampleRange& sr)
{
    bool missing = false;
    if (P.page_table != nullptr && sr.ok) {
        const int pages = (sr.row + P.tokens + P.page_rows - 1) / P.page_rows;
        for (int i = threadIdx.x; i < pages; i += blockDim.x) {
            const int page = P.page_table[(size_t)b * P.max_pages + i];
            missing = missing || page < 0 || page >= P.pool_pages;
        }
    }
    return P.page_table != nullptr && __syncthreads_or(missing);
}

// k and v of the drafted tokens -> rows n..n+tokens-1 of the cache: vectors first, first + step, ... of the tokens' 16-byte vectors
__device__ __forceinline__ void tree_append(const FfaTreeParams& P, int bh, int row, int rowb, int first, int step)
{
    const int vpr = rowb / 16, total = P.tokens * vpr;
    const uint4* ks = static_cast<const uint4*>(P.k) + (size_t)bh * total;
    const uint4* vs = static_cast<const uint4*>(P.v) + (size_t)bh * total;
    for (int i0 = first; i0 < total; i0 += 4 * step) {
        uint4 x[4], y[4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (i0 + n * step < total) x[n] = ks[i0 + n * step], y[n] = vs[i0 + n * step];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int i = i0 + n * step;
            if (i >= total) break;
            const size_t to = cache_row_offset(P, bh, row + i / vpr, rowb) + (i % vpr) * 16;
            *reinterpret_cast<uint4*>(static_cast<unsigned char*>(P.k_cache) + to) = x[n];
            *reinterpret_cast<uint4*>(static_cast<unsigned char*>(P.v_cache) + to) = y[n];
        }
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

// CUDA-core kernel (fp32).  A CTA of 16 x 16 threads takes 16 * RT query rows and tiles of 64 keys.
//   S   a thread computes RT rows x 4 keys: per 16 bytes of the head dimension RT + 4 shared-memory reads feed 8 * RT packed FMAs
//       (rows of K are padded by 16 bytes: 8 lanes' 16-byte reads of 8 rows then hit different banks; a warp reads two rows of Q)
//   P   through shared memory, transposed, the groups of rows XORed with the key so that neither side has bank conflicts
//   O   a thread keeps RT rows x DH / 16 columns
// K and V have one buffer each: V of a tile arrives while S is computed, K of the next one while O is.  Rows outside the valid range
// are zero-filled, never read, so that what a cache holds behind its last row cannot reach the result.  What bounds it: fp32 FMAs and the
// reads from shared memory that feed them.
template <int DH, int RT>
__global__ void __launch_bounds__(kTreeThreads) ffa_tree_simt_kernel(const FfaTreeParams P)
{
    constexpr int BM = 16 * RT, BN = kTreeKeys, VPR = DH / 4, KP = DH + 4, XV = (VPR + 15) / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    float* qs = reinterpret_cast<float*>(smem);   // [BM][DH], scaled
    float* ks = qs + BM * DH;                      // [BN][KP]
    float* vs = ks + BN * KP;                      // [BN][DH]
    float* ps = vs + BN * DH;                      // [BN][16 groups of RT]

    pdl_release();
    pdl_wait();
    const TreeCut<BN> cut(P);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int R = P.groups * P.tokens, row0 = cut.rt * BM, rows = min(BM, R - row0);
    const bool whole = P.splits == 1;
    float* out = static_cast<float*>(P.out) + ((size_t)cut.bh * R + row0) * DH;
    float* part = whole ? nullptr : tree_partial(P, cut.bh, cut.rt, cut.split, DH);
    const bool missing = tree_page_missing(P, cut.b, cut.sr);
    if ((!cut.sr.ok || missing) && tid == 0) atomicOr(P.status, missing ? kStatusBadIndex : kStatusBadLength);   // refused: zeros, nothing appended
    if (!cut.sr.ok || missing || cut.split >= cut.splits) {
        if (!whole) tree_empty_partial(part, rows, DH, tid, kTreeThreads);
        else for (int i = tid; i < rows * DH; i += kTreeThreads) out[i] = 0.f;
        return;
    }

    auto load = [&](int u, bool is_v) {
        const bool cached = u < cut.cache_tiles;
        const int base = (cached ? cut.c0 + u : u - cut.cache_tiles) * BN;
        const int lo = cached ? cut.sr.first : 0, hi = cached ? cut.sr.row : P.tokens;
        const size_t off = cached ? cache_row_offset(P, cut.bh, base, DH * 4) : ((size_t)cut.bh * P.tokens + base) * (DH * 4);
        const unsigned char* src = static_cast<const unsigned char*>(is_v ? (cached ? P.v_cache : P.v) : (cached ? P.k_cache : P.k));
        const uint32_t dst = smem_u32(is_v ? vs : ks);
        const int pitch = (is_v ? DH : KP) * 4;
        for (int i = tid; i < BN * VPR; i += kTreeThreads) {
            const int r = i / VPR, c = i - r * VPR;
            const bool in = base + r >= lo && base + r < hi;
            cp_async_16_or_zero(dst + r * pitch + c * 16, in ? src + off + (size_t)i * 16 : static_cast<const unsigned char*>(P.k), in ? 16u : 0u);
        }
        cp_async_commit();
    };

    load(cut.u0, false);
    load(cut.u0, true);
    {
        const float* q = static_cast<const float*>(P.q) + ((size_t)cut.bh * R + row0) * DH;
        for (int i = tid; i < BM * DH; i += kTreeThreads) qs[i] = i < rows * DH ? q[i] * P.scale : 0.f;
    }

    float m[RT], l[RT];
    float2 o[RT][XV][2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        m[i] = -CUDART_INF_F, l[i] = 0.f;
#pragma unroll
        for (int x = 0; x < XV; ++x) o[i][x][0] = o[i][x][1] = make_float2(0.f, 0.f);
    }
    const bool busy = (ty & ~1) * RT < rows;   // this warp has query rows
    for (int u = cut.u0; u < cut.u1; ++u) {
        const bool cached = u < cut.cache_tiles;
        const int base = (cached ? cut.c0 + u : u - cut.cache_tiles) * BN;
        cp_async_wait<1>();   // K is here, V may be on its way
        __syncthreads();
        if (busy) {
            float2 acc[RT][4];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int n = 0; n < 4; ++n) acc[i][n] = make_float2(0.f, 0.f);
#pragma unroll 4
            for (int c = 0; c < VPR; ++c) {
                float4 q4[RT], k4[4];
#pragma unroll
                for (int i = 0; i < RT; ++i) q4[i] = *reinterpret_cast<const float4*>(qs + (ty * RT + i) * DH + 4 * c);
#pragma unroll
                for (int n = 0; n < 4; ++n) k4[n] = *reinterpret_cast<const float4*>(ks + (tx + 16 * n) * KP + 4 * c);
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        acc[i][n] = __ffma2_rn(make_float2(q4[i].x, q4[i].y), make_float2(k4[n].x, k4[n].y), acc[i][n]);
                        acc[i][n] = __ffma2_rn(make_float2(q4[i].z, q4[i].w), make_float2(k4[n].z, k4[n].w), acc[i][n]);
                    }
            }
            float p[4][RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const int r = row0 + ty * RT + i;
                const unsigned char* sees = P.tree + ((size_t)(P.tree_per_sample ? cut.b : 0) * P.tokens + r % P.tokens) * P.tokens;
                float s[4], top = -CUDART_INF_F;
                bool see[4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int key = base + tx + 16 * n;
                    see[n] = r < R && (cached ? key >= cut.sr.first && key < cut.sr.row : key < P.tokens && sees[key] != 0);
                    s[n] = see[n] ? acc[i][n].x + acc[i][n].y : -CUDART_INF_F;
                    top = fmaxf(top, s[n]);
                }
#pragma unroll
                for (int off = 8; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                top = fmaxf(m[i], top);
                const float ref = top == -CUDART_INF_F ? 0.f : top;   // nothing seen so far: every weight is 0, not NaN
                const float corr = expf(m[i] - ref);
                m[i] = top;
                l[i] *= corr;   // this thread's keys; the threads are added at the end
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    p[n][i] = see[n] ? expf(s[n] - ref) : 0.f;
                    l[i] += p[n][i];
                }
#pragma unroll
                for (int x = 0; x < XV; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) o[i][x][h] = __fmul2_rn(o[i][x][h], make_float2(corr, corr));
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const int key = tx + 16 * n;
                float* to = ps + key * BM + (ty ^ (key & 15)) * RT;
#pragma unroll
                for (int i = 0; i < RT; ++i) to[i] = p[n][i];
            }
        }
        cp_async_wait<0>();
        __syncthreads();   // P is written, V is here, K's buffer is free
        if (u + 1 < cut.u1) load(u + 1, false);
        if (busy) {
            auto values = [&](auto guard_tag) {
                constexpr bool kGuard = decltype(guard_tag)::value;
#pragma unroll 4
                for (int key = 0; key < BN; ++key) {
                    float pr[RT];
#pragma unroll
                    for (int i = 0; i < RT; ++i) pr[i] = ps[key * BM + (ty ^ (key & 15)) * RT + i];
#pragma unroll
                    for (int x = 0; x < XV; ++x) {
                        const int c = tx + 16 * x;
                        if (VPR % 16 != 0 && c >= VPR) break;
                        const float4 v4 = *reinterpret_cast<const float4*>(vs + key * DH + 4 * c);
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            if (kGuard && pr[i] == 0.f) continue;   // a hidden token has no part in the row, whatever its values
                            o[i][x][0] = __ffma2_rn(make_float2(pr[i], pr[i]), make_float2(v4.x, v4.y), o[i][x][0]);
                            o[i][x][1] = __ffma2_rn(make_float2(pr[i], pr[i]), make_float2(v4.z, v4.w), o[i][x][1]);
                        }
                    }
                }
            };
            if (cached) values(std::false_type{});
            else values(std::true_type{});
        }
        __syncthreads();   // V's buffer and P are free
        if (u + 1 < cut.u1) load(u + 1, true);
    }

#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = ty * RT + i;
        float L = l[i];
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
        if (r >= rows) continue;
        const float inv = whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f;
        float* to = whole ? out + (size_t)r * DH : part + (size_t)r * ffa_tree_part_stride(DH);
#pragma unroll
        for (int x = 0; x < XV; ++x) {
            const int c = tx + 16 * x;
            if (VPR % 16 != 0 && c >= VPR) break;
            *reinterpret_cast<float4*>(to + 4 * c) = make_float4(o[i][x][0].x * inv, o[i][x][0].y * inv, o[i][x][1].x * inv, o[i][x][1].y * inv);
        }
        if (!whole && tx == 0) to[DH] = m[i], to[DH + 1] = L;
    }
    // the drafted tokens go to the cache behind the last read of this CTA, a share from each of the pair's CTAs
    const int ctas = cut.splits * P.row_tiles, mine = cut.split * P.row_tiles + cut.rt;
    tree_append(P, cut.bh, cut.sr.row, DH * 4, mine * kTreeThreads + tid, ctas * kTreeThreads);
}

// The same for few query rows (RG * 8 of them; fp32).  With 16 x 16 threads every warp would read the whole tile from shared memory for
// two rows of its own; here a warp owns 16 keys of a tile, for all rows: what a warp loads only it reads, so the loop has no CTA
// barrier, and K and V pass through shared memory once.
//   S   lane = (one of 4 groups of keys, one of 8 slices of the columns): 8 rows x 4 keys a pass, 32 products to 12 reads of 16 bytes,
//       then added over the slices so that a lane is left with one row.  (With whole columns and 2 rows x 2 keys to a lane, 4 products
//       to 4 reads, the kernel waits for shared memory.)
//   O   lane = columns: all rows x DH / 32 columns, the weights broadcast from shared memory (Dh 64: half a warp each takes every other key)
// Each warp has its own running maximum and sum; the warps meet once, at the end.  With head_dim 128, many pairs and at most 8 rows HBM bounds,
// otherwise latency and shared memory (256 pairs x 2000 x 64, 6 drafted: 83 us at a floor of 40).  This kernel and the one above, each at its number of
// splits: 256 pairs x 2000 tokens x 128, 6 drafted 100 / 178 us (floor 81), 16 drafted 175 / 350; 16 pairs x 8000 x 80, 5 drafted 31 / 41;
// 32 pairs x 995 x 64, 5 drafted and accepted 14.9 / 15.0, 12 drafted 17.3 / 17.0.
constexpr int kFewWarps = 4, kFewKeys = 16;   // keys a warp and tile
constexpr int few_kv_floats(int dh) { return 2 * kFewKeys * dh; }   // K and V of a warp
constexpr int few_stages(int dh) { return dh <= 64 ? 2 : 1; }   // as many as leave room for three CTAs to an SM (by registers two, with 16 rows)
constexpr int few_smem(int dh, int rg)
{
    const int ring = kFewWarps * (few_stages(dh) * few_kv_floats(dh) + kFewKeys * 8 * rg), merge = kFewWarps * 8 * rg * ffa_tree_part_stride(dh);
    return 4 * (8 * rg * dh + (ring > merge ? ring : merge));
}
template <int DH, int RG>
__global__ void __launch_bounds__(32 * kFewWarps, RG == 1 ? 3 : 2) ffa_tree_few_kernel(const FfaTreeParams P)
{
    constexpr int ROWS = 8 * RG, VPR = DH / 4, XV = (VPR + 31) / 32, KEYS_AT_ONCE = VPR <= 16 ? 2 : 1, KV = few_kv_floats(DH), STAGES = few_stages(DH), STRIDE = ffa_tree_part_stride(DH);
    extern __shared__ __align__(128) unsigned char smem[];
    float* qs = reinterpret_cast<float*>(smem);     // [ROWS][DH], scaled
    float* area = qs + ROWS * DH;                 // K and V, then weights; at the end the warps' results

    pdl_release();
    pdl_wait();
    const TreeCut<kTreeKeys> cut(P);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = P.groups * P.tokens;   // all of the pair's
    const bool whole = P.splits == 1;
    float* out = static_cast<float*>(P.out) + (size_t)cut.bh * rows * DH;
    float* part = whole ? nullptr : tree_partial(P, cut.bh, 0, cut.split, DH);
    const bool missing = tree_page_missing(P, cut.b, cut.sr);
    if ((!cut.sr.ok || missing) && tid == 0) atomicOr(P.status, missing ? kStatusBadIndex : kStatusBadLength);   // refused: zeros, nothing appended
    if (!cut.sr.ok || missing || cut.split >= cut.splits) {
        if (!whole) tree_empty_partial(part, rows, DH, tid, 32 * kFewWarps);
        else for (int i = tid; i < rows * DH; i += 32 * kFewWarps) out[i] = 0.f;
        return;
    }

    float* ring = area + warp * STAGES * KV;                                // K, V of every stage
    float* ps = area + kFewWarps * STAGES * KV + warp * kFewKeys * ROWS;   // [key][row]
    // this warp's 16 keys of tile u; those outside the valid range are zero-filled, never read
    auto load = [&](int u, bool is_v, int stage) {
        const bool cached = u < cut.cache_tiles;
        const int base = (cached ? cut.c0 + u : u - cut.cache_tiles) * kTreeKeys + warp * kFewKeys;
        const int lo = cached ? cut.sr.first : 0, hi = cached ? cut.sr.row : P.tokens;
        if (u < cut.u1 && base + kFewKeys > lo && base < hi) {
            const size_t off = cached ? cache_row_offset(P, cut.bh, base, DH * 4) : ((size_t)cut.bh * P.tokens + base) * (DH * 4);
            const unsigned char* src = static_cast<const unsigned char*>(is_v ? (cached ? P.v_cache : P.v) : (cached ? P.k_cache : P.k)) + off;
            const uint32_t dst = smem_u32(ring + stage * KV + (is_v ? kFewKeys * DH : 0));
#pragma unroll
            for (int i0 = 0; i0 < kFewKeys * VPR; i0 += 32) {
                const int i = i0 + lane, r = i / VPR;
                const bool in = base + r >= lo && base + r < hi;
                cp_async_16_or_zero(dst + i * 16, in ? src + (size_t)i * 16 : static_cast<const unsigned char*>(P.k), in ? 16u : 0u);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i) load(cut.u0 + i, false, i), load(cut.u0 + i, true, i);
    {
        const float* q = static_cast<const float*>(P.q) + (size_t)cut.bh * rows * DH;
        for (int i = tid; i < ROWS * DH; i += 32 * kFewWarps) qs[i] = i < rows * DH ? q[i] * P.scale : 0.f;
    }
    __syncthreads();

    const int kg = lane >> 3, ds = lane & 7;   // this lane's keys are kg, kg + 4, ..., its chunks of 4 columns ds, ds + 8, ..., its rows ds, ds + 8
    float m[RG], l[RG];
    float4 o[ROWS][XV];
#pragma unroll
    for (int i = 0; i < RG; ++i) m[i] = -CUDART_INF_F, l[i] = 0.f;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int x = 0; x < XV; ++x) o[r][x] = make_float4(0.f, 0.f, 0.f, 0.f);

    for (int u = cut.u0, stage = 0; u < cut.u1; ++u, stage = stage + 1 == STAGES ? 0 : stage + 1) {
        const float* ks = ring + stage * KV;
        const float* vs = ks + kFewKeys * DH;
        cp_async_wait<2 * STAGES - 1>();   // K is here, V and later tiles may be on their way
        __syncwarp();
        const bool cached = u < cut.cache_tiles;
        const int base = (cached ? cut.c0 + u : u - cut.cache_tiles) * kTreeKeys + warp * kFewKeys;
        const int lo = cached ? cut.sr.first : 0, hi = cached ? cut.sr.row : P.tokens;
        const bool any = base + kFewKeys > lo && base < hi;   // some of the warp's keys are valid
        if (any) {
            float sum[RG][4];   // of this lane's rows and keys
#pragma unroll
            for (int h = 0; h < RG; ++h) {
                float2 acc[8][4];
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[r][j] = make_float2(0.f, 0.f);
#pragma unroll (RG == 1 ? 1 : 2)   // (registers)
                for (int i = 0; i < (VPR + 7) / 8; ++i) {
                    const int c = ds + 8 * i;
                    if (VPR % 8 != 0 && c >= VPR) break;
                    float4 k4[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const float4*>(ks + (kg + 4 * j) * DH + 4 * c);
#pragma unroll
                    for (int r = 0; r < 8; ++r) {
                        const float4 q4 = *reinterpret_cast<const float4*>(qs + (8 * h + r) * DH + 4 * c);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            acc[r][j] = __ffma2_rn(make_float2(q4.x, q4.y), make_float2(k4[j].x, k4[j].y), acc[r][j]);
                            acc[r][j] = __ffma2_rn(make_float2(q4.z, q4.w), make_float2(k4[j].z, k4[j].w), acc[r][j]);
                        }
                    }
                }
                // over the 8 lanes of a key: each step halves the rows that a lane holds, until its own is left
                float a[8][4];
#pragma unroll
                for (int r = 0; r < 8; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[r][j] = acc[r][j].x + acc[r][j].y;
#pragma unroll
                for (int n = 4; n >= 1; n >>= 1)
#pragma unroll
                    for (int r = 0; r < n; ++r)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const bool upper = (ds & n) != 0;
                            const float other = __shfl_xor_sync(0xffffffffu, upper ? a[r][j] : a[r + n][j], n);
                            a[r][j] = (upper ? a[r + n][j] : a[r][j]) + other;
                        }
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[h][j] = a[0][j];
            }
            __syncwarp();
            load(u + STAGES, false, stage);
            float corr[RG];
            bool moved = false;
#pragma unroll
            for (int h = 0; h < RG; ++h) {
                const int r = 8 * h + ds;
                float top = m[h];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = base + kg + 4 * j;
                    bool see = r < rows && key >= lo && key < hi;
                    if (!cached && see) see = P.tree[((size_t)(P.tree_per_sample ? cut.b : 0) * P.tokens + r % P.tokens) * P.tokens + key] != 0;
                    if (!see) sum[h][j] = -CUDART_INF_F;
                    top = fmaxf(top, sum[h][j]);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));   // over the row's lanes
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float ref = top == -CUDART_INF_F ? 0.f : top;   // nothing seen so far: every weight is 0, not NaN
                corr[h] = expf(m[h] - ref);
                moved = moved || top != m[h];
                m[h] = top;
                float w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) ps[(kg + 4 * j) * ROWS + r] = w[j] = expf(sum[h][j] - ref);
                l[h] = fmaf(l[h], corr[h], (w[0] + w[1]) + (w[2] + w[3]));   // this lane's keys; the lanes are added at the end
            }
            cp_async_wait<2 * STAGES - 1>();   // V is here
            __syncwarp();
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    const float f = __shfl_sync(0xffffffffu, corr[r >> 3], r & 7);
#pragma unroll
                    for (int x = 0; x < XV; ++x) o[r][x].x *= f, o[r][x].y *= f, o[r][x].z *= f, o[r][x].w *= f;
                }
            }
            auto values = [&](auto guard_tag) {
                constexpr bool kGuard = decltype(guard_tag)::value;
#pragma unroll
                for (int k0 = 0; k0 < kFewKeys; k0 += KEYS_AT_ONCE) {
                    const int k = KEYS_AT_ONCE == 2 ? k0 + (lane >> 4) : k0;
#pragma unroll
                    for (int x = 0; x < XV; ++x) {
                        const int c = (KEYS_AT_ONCE == 2 ? lane & 15 : lane) + 32 * x;
                        if (c >= VPR) break;
                        const float4 v4 = *reinterpret_cast<const float4*>(vs + k * DH + 4 * c);
#pragma unroll
                        for (int r0 = 0; r0 < ROWS; r0 += 4) {
                            const float4 p4 = *reinterpret_cast<const float4*>(ps + k * ROWS + r0);
                            const float pr[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (kGuard && pr[i] == 0.f) continue;   // a hidden token has no part in the row, whatever its values
                                const float2 pp = make_float2(pr[i], pr[i]);
                                const float2 a = __ffma2_rn(pp, make_float2(v4.x, v4.y), make_float2(o[r0 + i][x].x, o[r0 + i][x].y));
                                const float2 b = __ffma2_rn(pp, make_float2(v4.z, v4.w), make_float2(o[r0 + i][x].z, o[r0 + i][x].w));
                                o[r0 + i][x] = make_float4(a.x, a.y, b.x, b.y);
                            }
                        }
                    }
                }
            };
            if (cached) values(std::false_type{});
            else values(std::true_type{});
        }
        __syncwarp();   // V and the weights may be overwritten
        if (!any) load(u + STAGES, false, stage);
        load(u + STAGES, true, stage);
    }
    cp_async_wait<0>();

    // the warps' results: [warp][row][columns, maximum, sum]
    __syncthreads();
#pragma unroll
    for (int h = 0; h < RG; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8), l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
        float* to = area + (size_t)(warp * ROWS + 8 * h + ds) * STRIDE;
        if (kg == 0) to[DH] = m[h], to[DH + 1] = l[h];
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int x = 0; x < XV; ++x) {
            if (KEYS_AT_ONCE == 2) {   // the half-warps' keys
                o[r][x].x += __shfl_xor_sync(0xffffffffu, o[r][x].x, 16), o[r][x].y += __shfl_xor_sync(0xffffffffu, o[r][x].y, 16);
                o[r][x].z += __shfl_xor_sync(0xffffffffu, o[r][x].z, 16), o[r][x].w += __shfl_xor_sync(0xffffffffu, o[r][x].w, 16);
            }
            const int c = lane + 32 * x;
            if (c >= VPR) break;
            *reinterpret_cast<float4*>(area + (size_t)(warp * ROWS + r) * STRIDE + 4 * c) = o[r][x];
        }
    __syncthreads();
    for (int i = tid; i < rows * VPR; i += 32 * kFewWarps) {
        const int r = i / VPR, c = i - r * VPR;
        float M = -CUDART_INF_F, L = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) M = fmaxf(M, area[(size_t)(w * ROWS + r) * STRIDE + DH]);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) {
            const float* from = area + (size_t)(w * ROWS + r) * STRIDE;
            const float f = from[DH] == -CUDART_INF_F && from[DH + 1] == 0.f ? 0.f : expf(from[DH] - M);   // 0: saw nothing
            const float4 y = *reinterpret_cast<const float4*>(from + 4 * c);
            L = fmaf(f, from[DH + 1], L);
            sum.x = isfinite(y.x) ? fmaf(f, y.x, sum.x) : sum.x + y.x, sum.y = isfinite(y.y) ? fmaf(f, y.y, sum.y) : sum.y + y.y;
            sum.z = isfinite(y.z) ? fmaf(f, y.z, sum.z) : sum.z + y.z, sum.w = isfinite(y.w) ? fmaf(f, y.w, sum.w) : sum.w + y.w;
        }
        const float inv = whole ? (L == 0.f ? 0.f : 1.f / L) : 1.f;
        float* to = whole ? out + (size_t)r * DH : part + (size_t)r * STRIDE;
        *reinterpret_cast<float4*>(to + 4 * c) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        if (!whole && c == 0) to[DH] = M, to[DH + 1] = L;
    }
    tree_append(P, cut.bh, cut.sr.row, DH * 4, cut.split * 32 * kFewWarps + tid, cut.splits * 32 * kFewWarps);
}

// Rows n + path[i] -> n + i of every pair, in place.  A thread owns one 16-byte column of K or V and walks the path: indices
// increase, so path[i] >= i and a row is read before anything is written to it (eight rows are read, then eight written).
__global__ void __launch_bounds__(256) ffa_tree_accept_kernel(const FfaAcceptParams P)
{
    pdl_release();
    pdl_wait();
    const int bh = blockIdx.x, b = bh / P.H;
    const int vpr = P.row_bytes / 16;
    const int* path = P.path + (size_t)b * P.path_len;
    const int n = P.seq_lengths != nullptr ? P.seq_lengths[b] : P.t;
    if (n < 0 || n > P.Lmax) {   // (a full cache has an empty path)
        if (threadIdx.x == 0) atomicOr(P.status, kStatusBadLength);
        return;
    }
    int count = 0, prev = -1;
    for (; count < P.path_len; ++count) {
        const int j = path[count];
        if (j < 0) break;
        bool refused = j <= prev || j >= P.Lmax - n;
        if (!refused && P.page_table != nullptr) {   // the row itself and the one it moves to: an increasing path has count <= j, so both lie in the table
            const int from = P.page_table[(size_t)b * P.max_pages + (n + j) / P.page_rows], to = P.page_table[(size_t)b * P.max_pages + (n + count) / P.page_rows];
            refused = from < 0 || from >= P.pool_pages || to < 0 || to >= P.pool_pages;
        }
        if (refused) {
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
