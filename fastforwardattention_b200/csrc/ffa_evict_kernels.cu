// Eviction by accumulated attention weight: of a pair's n cached rows the `keep` heaviest stay, ties going to the lower row.
// Rows whose position is among the `recent` newest or below `first` always stay.  The rows that stay and lie at `keep` or
// behind move into the freed rows in front (k-th survivor to k-th freed row, both ascending), so that a pair which drops one
// row moves one row whatever its length; the order of a pair's rows means nothing to attention, and `positions` keeps the
// tokens' order.
//
// One CTA per pair decides.  It reads positions and weights once into 32-bit keys in shared memory (a weight's bits made
// monotonic, all ones for a protected row).  One row too many, the steady state of a loop that evicts every token: the smallest key
// is found by one reduction and its row takes the last one's place.  Otherwise: the keep-th largest key by radix selection, 8 bits a pass;
// a bit per row that stays; ranks of freed and surviving rows by a scan over the bits; kept[] says which row moves where.  The rows
// of K and V then move in a kernel of their own over the whole device (a CTA moves some 100 GB/s, so that a prompt's thousands of
// rows must not be left to one CTA per pair).  Bound by latency for short pairs (a dozen passes with a barrier each), by HBM for the moves.
#include <climits>

#include "ffa_device_common.cuh"
#include "ffa_internal.h"
#include "ffa_launch.cuh"

using namespace ffa_dev;

namespace {

constexpr int kEvictMaxWarps = 32;
// keys fit into shared memory beside the bits and ranks up to here; longer pairs recompute them from positions and weights in every pass
constexpr int kKeysInSmem = 48 * 1024;

// fp32 bits in the order of the values; -0 like 0, NaN below everything
__device__ __forceinline__ uint32_t ordered_key(float w)
{
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum of one value per thread over the CTA; returns the total in *total.  `warp_sums`: [kEvictMaxWarps + 1].
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int* total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
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
        const int s = lane < warps ? warp_sums[lane] : 0;
        int t = s;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, t, off);
            if (lane >= off) t += y;
        }
        __syncwarp();
        if (lane < warps) warp_sums[lane] = t - s;
        if (lane == 31) warp_sums[kEvictMaxWarps] = t;
    }
    __syncthreads();
    *total = warp_sums[kEvictMaxWarps];
    return warp_sums[warp] + inc - x;
}

// position of the n-th (from 0) set bit of w
__device__ __forceinline__ int nth_bit(uint32_t w, int n)
{
    for (int i = 0; i < n; ++i) w &= w - 1;
    return __ffs(w) - 1;
}

// kept[] alone says what moves; weights and positions move here, K and V rows in ffa_evict_move_kernel unless one row moves
template <bool kSmemKeys>
__global__ void __launch_bounds__(1024) ffa_evict_kernel(const FfaEvictParams P)
{
    extern __shared__ __align__(16) uint32_t keys[];   // [max_rows] keys (kSmemKeys), then bits and ranks
    __shared__ int warp_sums[kEvictMaxWarps + 1];
    __shared__ unsigned long long warp_min[kEvictMaxWarps];
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left, s_newest;

    pdl_release();
    pdl_wait();
    const int bh = blockIdx.x, b = bh / P.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, T = blockDim.x, warps = T >> 5;
    const int n = P.rows[b], keep = P.keep;
    int* kept = P.kept + (size_t)bh * keep;
    if (n < 0 || n > P.max_rows) {
        for (int r = tid; r < keep; r += T) kept[r] = -1;
        if (tid == 0) atomicOr(P.status, kStatusBadLength);
        return;
    }
    if (n <= keep) {
        for (int r = tid; r < keep; r += T) kept[r] = r < n ? r : -1;
        return;
    }
    float* w = P.weights + (size_t)bh * P.Lmax;
    int* pos = P.positions + (size_t)bh * P.Lmax;
    const int words = (n + 31) / 32;
    uint32_t* bits = keys + (kSmemKeys ? n : 0);            // [words] rows that stay
    int* before = reinterpret_cast<int*>(bits + words);     // [words + 1] ranks, see below

    if (tid == 0) s_newest = INT_MIN, s_prefix = 0, s_left = keep;
    __syncthreads();
    {
        int newest = INT_MIN;
        for (int r0 = tid; r0 < n; r0 += 8 * T) {
            int p[8];
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = r0 + i * T;
                p[i] = r < n ? pos[r] : INT_MIN;
                if (kSmemKeys) x[i] = r < n ? w[r] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = r0 + i * T;
                newest = max(newest, p[i]);
                if (kSmemKeys && r < n) keys[r] = p[i] < P.first ? 0xffffffffu : ordered_key(x[i]);
            }
        }
        newest = __reduce_max_sync(0xffffffffu, newest);
        if (lane == 0) atomicMax(&s_newest, newest);
    }
    __syncthreads();
    const long long oldest_recent = (long long)s_newest - P.recent;   // positions above it are recent
    if (kSmemKeys && P.recent > 0) {
        for (int r0 = tid; r0 < n; r0 += 8 * T) {
            int p[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = r0 + i * T < n ? pos[r0 + i * T] : INT_MIN;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (r0 + i * T < n && p[i] > oldest_recent) keys[r0 + i * T] = 0xffffffffu;
        }
        // (no barrier: a thread reads back its own keys only, until the one below)
    }
    auto key = [&](int r) -> uint32_t {
        if (kSmemKeys) return keys[r];
        const int p = pos[r];
        return p < P.first || p > oldest_recent ? 0xffffffffu : ordered_key(w[r]);
    };
    if (n == keep + 1) {
        // the smallest key's row goes, of equal ones the highest; the last row takes its place
        unsigned long long least = ~0ull;
        for (int r = tid; r < n; r += T) least = min(least, ((unsigned long long)key(r) << 32) | (uint32_t)~r);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, off));
        if (lane == 0) warp_min[warp] = least;
        __syncthreads();
        least = lane < warps ? warp_min[lane] : ~0ull;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) least = min(least, __shfl_xor_sync(0xffffffffu, least, off));
        const int gone = (int)~(uint32_t)least;
        for (int r = tid; r < keep; r += T) kept[r] = r == gone ? keep : r;
        if (gone == keep) return;
        if (tid == 0) w[gone] = w[keep], pos[gone] = pos[keep];
        const int vpr = P.row_bytes / 16;
        for (int i = tid; i < 2 * vpr; i += T) {
            uint4* cache = static_cast<uint4*>(i < vpr ? P.k_cache : P.v_cache) + (size_t)bh * P.Lmax * vpr + (i < vpr ? i : i - vpr);
            cache[(size_t)gone * vpr] = cache[(size_t)keep * vpr];
        }
        return;
    }
    __syncthreads();
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int r = tid; r < n; r += T) {
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
    for (int x = warp; x < words; x += warps) {
        const int r = x * 32 + lane;
        const uint32_t u = r < n ? key(r) : 0u;
        const uint32_t above = __ballot_sync(0xffffffffu, r < n && u > border);
        const uint32_t on = __ballot_sync(0xffffffffu, r < n && u == border);
        if (lane == 0) bits[x] = above, before[x] = (int)on;
    }
    __syncthreads();
    const int per = (words + T - 1) / T, x0 = min(words, tid * per), x1 = min(words, x0 + per);
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
    for (int x = warp; x <= last_front; x += warps) {
        const int r = x * 32 + lane;
        const uint32_t freed = freed_of(x);
        int src = r;
        if ((freed >> lane) & 1u) {
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
        }
        if (r < keep) kept[r] = src;
    }
}

// Rows r <- kept[r] of K and V wherever they differ.  Sources lie at `keep` or behind and destinations before it, so nothing is read that
// another warp writes.  A warp takes 32 rows of kept[]; four vectors of a lane are read before they are written.
constexpr int kMoveWarps = 8;
__global__ void __launch_bounds__(32 * kMoveWarps) ffa_evict_move_kernel(const FfaEvictParams P)
{
    __shared__ int2 moves[kMoveWarps][32];
    pdl_release();
    pdl_wait();
    const int words = (P.keep + 31) / 32, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long item = (long long)blockIdx.x * kMoveWarps + warp;
    if (item >= (long long)P.B * P.H * words) return;
    const int bh = (int)(item / words), r = (int)(item - (long long)bh * words) * 32 + lane, n = P.rows[bh / P.H];
    if (n <= P.keep + 1 || n > P.max_rows) return;   // nothing moves, or the one row has moved
    const int src = r < P.keep ? P.kept[(size_t)bh * P.keep + r] : r;
    const uint32_t moving = __ballot_sync(0xffffffffu, src != r);
    if (moving == 0) return;
    if (src != r) moves[warp][__popc(moving & ((1u << lane) - 1u))] = make_int2(r, src);
    __syncwarp();
    const int vpr = P.row_bytes / 16, total = __popc(moving) * 2 * vpr;
    uint4* kc = static_cast<uint4*>(P.k_cache) + (size_t)bh * P.Lmax * vpr;
    uint4* vc = static_cast<uint4*>(P.v_cache) + (size_t)bh * P.Lmax * vpr;
    for (int i0 = lane; i0 < total; i0 += 128) {
        uint4 x[4];
        uint4* to[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + 32 * k;
            if (i < total) {
                const int2 mv = moves[warp][i / (2 * vpr)];
                const int c = i % (2 * vpr);
                uint4* cache = c < vpr ? kc + c : vc + (c - vpr);
                x[k] = cache[(size_t)mv.y * vpr];
                to[k] = cache + (size_t)mv.x * vpr;
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i0 + 32 * k < total) *to[k] = x[k];
    }
}

}  // namespace

namespace {

int select_smem(int max_rows)
{
    const int words = (max_rows + 31) / 32;
    return ((max_rows <= kKeysInSmem ? max_rows : 0) + 2 * words + 1) * 4;
}

}  // namespace

int ffa_k_evict_prepare(int max_smem)
{
    auto raise = [&](auto kernel) -> cudaError_t {
        cudaFuncAttributes a;
        const cudaError_t e = cudaFuncGetAttributes(&a, kernel);
        return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, max_smem - (int)a.sharedSizeBytes);
    };
    const cudaError_t e = raise(ffa_evict_kernel<true>);
    return (int)(e != cudaSuccess ? e : raise(ffa_evict_kernel<false>));
}

int ffa_k_evict(const FfaEvictParams& P, cudaStream_t stream)
{
    // eight small CTAs to an SM while a thread has at most 16 rows; large ones for long pairs, of which there are few
    const int threads = P.max_rows <= 4096 ? 256 : 1024;
    const auto kernel = P.max_rows <= kKeysInSmem ? ffa_evict_kernel<true> : ffa_evict_kernel<false>;
    int e = (int)launch_pdl(kernel, P.B * P.H, threads, select_smem(P.max_rows), 0, true, stream, P);
    if (e != 0 || P.max_rows <= P.keep + 1) return e;
    const long long items = (long long)P.B * P.H * ((P.keep + 31) / 32);
    return (int)launch_pdl(ffa_evict_move_kernel, (int)((items + kMoveWarps - 1) / kMoveWarps), 32 * kMoveWarps, 0, 0, true, stream, P);
}
