// Eviction by accumulated attention weight: of a pair's n cached rows the `keep` heaviest stay, ties going to the lower row.
// Rows whose position is among the `recent` newest or below `first` always stay.  The rows that stay and lie at `keep` or
// behind move into the freed rows in front (k-th survivor to k-th freed row, both ascending), so that a pair which drops one
// row moves one row whatever its length; the order of a pair's rows means nothing to attention, and `positions` keeps the
// tokens' order.
//
// One CTA per pair.  (1) The newest position.  (2) The keep-th largest key by radix selection, 8 bits a pass: a key is the
// weight's bits made monotonic, or all ones for a protected row.  (3) A bit per row that stays.  (4) Ranks of freed and
// surviving rows by a scan over the bits.  (5) The moves, a warp per word of 32 rows.
#include <climits>

#include "ffa_device_common.cuh"
#include "ffa_internal.h"

using namespace ffa_dev;

namespace {

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;

// fp32 bits in the order of the values; -0 like 0, NaN below everything
__device__ __forceinline__ uint32_t ordered_key(float w)
{
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of one value per thread over the CTA; returns the total in *total.  `warp_sums`: [kEvictWarps + 1].
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int* total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = x;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, off);
        if (lane >= off) inc += y;
    }
    __syncthreads();   // warp_sums may still be read from the previous call
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const int s = lane < kEvictWarps ? warp_sums[lane] : 0;
        int t = s;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, t, off);
            if (lane >= off) t += y;
        }
        if (lane < kEvictWarps) warp_sums[lane] = t - s;
        if (lane == kEvictWarps - 1) warp_sums[kEvictWarps] = t;
    }
    __syncthreads();
    *total = warp_sums[kEvictWarps];
    return warp_sums[warp] + inc - x;
}

// position of the n-th (from 0) set bit of w
__device__ __forceinline__ int nth_bit(uint32_t w, int n)
{
    for (int i = 0; i < n; ++i) w &= w - 1;
    return __ffs(w) - 1;
}

__global__ void __launch_bounds__(kEvictThreads) ffa_evict_kernel(const FfaEvictParams P)
{
    extern __shared__ __align__(16) uint32_t bits[];   // [words] rows that stay
    __shared__ int warp_sums[kEvictWarps + 1];
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left, s_newest;
    __shared__ int2 moves[kEvictWarps][32];

    pdl_release();
    pdl_wait();
    const int bh = blockIdx.x, b = bh / P.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = P.rows[b], keep = P.keep;
    int* kept = P.kept + (size_t)bh * keep;
    if (n < 0 || n > P.max_rows) {
        for (int r = tid; r < keep; r += kEvictThreads) kept[r] = -1;
        if (tid == 0) atomicOr(P.status, kStatusBadLength);
        return;
    }
    if (n <= keep) {
        for (int r = tid; r < keep; r += kEvictThreads) kept[r] = r < n ? r : -1;
        return;
    }
    float* w = P.weights + (size_t)bh * P.Lmax;
    int* pos = P.positions + (size_t)bh * P.Lmax;
    const int words = (n + 31) / 32;
    int* before = reinterpret_cast<int*>(bits + words);   // [words + 1] ranks, see below

    if (tid == 0) s_newest = INT_MIN, s_prefix = 0, s_left = keep;
    __syncthreads();
    {
        int newest = INT_MIN;
        for (int r = tid; r < n; r += kEvictThreads) newest = max(newest, pos[r]);
        newest = __reduce_max_sync(0xffffffffu, newest);
        if (lane == 0) atomicMax(&s_newest, newest);
    }
    __syncthreads();
    const long long oldest_recent = (long long)s_newest - P.recent;   // positions above it are recent
    auto key = [&](int r) -> uint32_t {
        const int p = pos[r];
        return p < P.first || p > oldest_recent ? 0xffffffffu : ordered_key(w[r]);
    };
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int r = tid; r < n; r += kEvictThreads) {
            const uint32_t u = key(r);
            if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1);
        }
        __syncthreads();
        if (warp == 0) {   // the digit at which the count from above reaches what is left to keep: 8 digits a lane, from the top
            int mine[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine[i] = hist[255 - (lane * 8 + i)], sum += mine[i];
            int inc = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc, off);
                if (lane >= off) inc += y;
            }
            const int left = s_left;
            int above = inc - sum;
            __syncwarp();
            if (above < left && inc >= left) {
                int digit = 255 - lane * 8;
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (above + mine[i] < left) above += mine[i], --digit;
                    else break;
                s_prefix = prefix | ((uint32_t)digit << shift);
                s_left = left - above;
            }
        }
        __syncthreads();
    }
    const uint32_t border = s_prefix;   // the keep-th largest key; s_left rows that have it stay, the lowest ones
    const int left = s_left;
    // rows above the border, and per word how many lie on it
    for (int x = warp; x < words; x += kEvictWarps) {
        const int r = x * 32 + lane;
        const uint32_t u = r < n ? key(r) : 0u;
        const uint32_t above = __ballot_sync(0xffffffffu, r < n && u > border);
        const uint32_t on = __ballot_sync(0xffffffffu, r < n && u == border);
        if (lane == 0) bits[x] = above, before[x] = (int)on;
    }
    __syncthreads();
    const int per = (words + kEvictThreads - 1) / kEvictThreads, x0 = min(words, tid * per), x1 = min(words, x0 + per);
    int total = 0;
    {
        int count = 0;
        for (int x = x0; x < x1; ++x) count += __popc((uint32_t)before[x]);
        int rank = block_scan(count, warp_sums, &total);
        for (int x = x0; x < x1; ++x) {
            uint32_t on = (uint32_t)before[x];
            const int c = __popc(on);
            if (rank + c > left) {   // only the lowest of them
                uint32_t some = 0;
                for (int i = max(0, left - rank); i > 0; --i) some |= on & (~on + 1), on &= on - 1;
                on = some;
            }
            bits[x] |= on;
            rank += c;
        }
    }
    __syncthreads();
    // ranks: before[x] = freed rows in front of word x (words with rows < keep), before[x + 1] = survivors at `keep` or behind in
    // front of word x (words with rows >= keep); the word that has both kinds is the last of the first and the first of the second
    const int last_front = (keep - 1) / 32, first_back = keep / 32;
    auto freed_of = [&](int x) -> uint32_t {
        const uint32_t in = x < first_back ? 0xffffffffu : x == first_back ? (1u << (keep & 31)) - 1u : 0u;
        return ~bits[x] & in;
    };
    auto back_of = [&](int x) -> uint32_t {
        const uint32_t in = x > first_back ? 0xffffffffu : x == first_back ? ~((1u << (keep & 31)) - 1u) : 0u;
        return bits[x] & in;
    };
    int freed_total = 0;
    {
        int count = 0, back = 0;
        for (int x = x0; x < x1; ++x) count += __popc(freed_of(x)), back += __popc(back_of(x));
        int rank = block_scan(count, warp_sums, &freed_total);
        int rank_back = block_scan(back, warp_sums, &total);
        for (int x = x0; x < x1; ++x) {
            if (x <= last_front) before[x] = rank;
            rank += __popc(freed_of(x));
        }
        for (int x = x0; x < x1; ++x) {
            if (x >= first_back) before[x + 1] = rank_back;
            rank_back += __popc(back_of(x));
        }
    }
    __syncthreads();
    const int vpr = P.row_bytes / 16, per_row = 2 * vpr;
    uint4* kc = static_cast<uint4*>(P.k_cache) + (size_t)bh * P.Lmax * vpr;
    uint4* vc = static_cast<uint4*>(P.v_cache) + (size_t)bh * P.Lmax * vpr;
    for (int x = warp; x <= last_front; x += kEvictWarps) {
        const int r = x * 32 + lane;
        const uint32_t freed = freed_of(x);
        const bool free_row = (freed >> lane) & 1u;
        int src = r;
        if (free_row) {
            const int rank = before[x] + __popc(freed & ((1u << lane) - 1u));
            int lo = first_back, hi = words - 1;   // the last word with at most `rank` survivors in front of it
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (before[mid + 1] <= rank) lo = mid;
                else hi = mid - 1;
            }
            src = lo * 32 + nth_bit(back_of(lo), rank - before[lo + 1]);
            w[r] = w[src];
            pos[r] = pos[src];
            moves[warp][__popc(freed & ((1u << lane) - 1u))] = make_int2(r, src);
        }
        if (r < keep) kept[r] = src;
        __syncwarp();
        const int total_vecs = __popc(freed) * per_row;
        for (int i = lane; i < total_vecs; i += 32) {
            const int2 mv = moves[warp][i / per_row];
            const int c = i % per_row;
            uint4* cache = c < vpr ? kc : vc;
            const int col = c < vpr ? c : c - vpr;
            cache[(size_t)mv.x * vpr + col] = cache[(size_t)mv.y * vpr + col];
        }
        __syncwarp();
    }
}

}  // namespace

int ffa_k_evict_smem(int max_rows)
{
    const int words = (max_rows + 31) / 32;
    return (2 * words + 1) * 4;
}

int ffa_k_evict_prepare(int max_smem)
{
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, ffa_evict_kernel);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(ffa_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem - (int)a.sharedSizeBytes);
    return (int)e;
}

int ffa_k_evict(const FfaEvictParams& P, int smem, cudaStream_t stream)
{
    ffa_evict_kernel<<<(unsigned)(P.B * P.H), kEvictThreads, (size_t)smem, stream>>>(P);
    return (int)cudaGetLastError();
}
