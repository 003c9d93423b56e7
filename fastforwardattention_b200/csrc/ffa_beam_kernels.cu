// Beam search: selection over beams and vocabulary, and the reordering of the caches by parent beam.
#include <climits>

#include "ffa_device_common.cuh"
#include "ffa_internal.h"
#include "ffa_launch.cuh"

using namespace ffa_dev;

namespace {

// ------------------------------------------------------------------------------------------
// Selection
// ------------------------------------------------------------------------------------------
//   score(i, v) = s_i + (x_iv - logsumexp(x_i))     the num best over (i, v) of a sample, ties to the lowest i * vocab + v
//
// A thread-block cluster of 8 CTAs per sample; each of its 128 warps owns a segment of one beam's logits (every SEG-th block of
// 32 vectors, so that the best tokens of a sorted vocabulary do not sit in one segment).
//   pass 1   running maximum and sum of exponentials per lane; every warp stores its maximum, the maxima of its four quarters
//            and its sum into every CTA of the cluster;                                              -- cluster barrier --
//            every CTA now has all beams' logsumexp and 128 scores that exist: the num-th largest of them is a lower bound of
//            the num-th best score (the quarters' maxima serve when too few warps have one, as in a first step with one live beam)
//   pass 2   (L1 / L2) the lanes whose maximum reaches the bound look at their part again; every element at or above it goes into
//            the leader CTA's list, about num of them;                                                -- cluster barrier --
//            the leader ranks the list and writes the result.
// Where more elements reach the bound than the list holds (a vocabulary of ties), the cluster finds the exact border instead: a
// radix selection, 8 bits a pass, over the 64-bit score and then the index.
// The sums of exponentials are fp32 per lane (a few dozen terms) and double across lanes and warps; scores are compared as
// doubles, so that two beams' candidates a rounding of fp32 apart still come in the right order.
constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelCluster = 8;
constexpr int kSelSegments = kSelWarps * kSelCluster;   // 128
constexpr int kSelList = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct SelRecord {       // one segment
    float m;             // largest logit, -inf: none
    float quarter[4];    // largest logit of lanes 0-7, 8-15, 16-23, 24-31
    float pad;
    double l;            // sum of exp(x - m)
};
struct SelCandidate {
    double score;
    unsigned flat;       // beam * vocab + token
    unsigned pad;
};

__device__ __forceinline__ uint32_t map_peer(const void* own_smem_ptr, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(own_smem_ptr)), "r"(rank));
    return a;
}
__device__ __forceinline__ void st_peer_v4(uint32_t addr, uint4 v)
{
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ unsigned add_peer_u32(uint32_t addr, unsigned x)
{
    unsigned old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(x) : "memory");
    return old;
}
__device__ __forceinline__ unsigned ld_peer_u32(uint32_t addr)
{
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

// doubles in the order of their values (no NaN)
__device__ __forceinline__ unsigned long long ordered64(double x)
{
    const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// 16 bytes that start `skew` bytes into the 32 at `p` (16-byte aligned); skew is a multiple of 2 below 16, the same for the warp
__device__ __forceinline__ uint4 load_skewed(const uint4* p, unsigned skew)
{
    const uint4 a = p[0];
    if (skew == 0) return a;
    const uint4 b = p[1];
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (skew & 8u) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (skew & 4u) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (skew & 2u) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Visits this warp's part of a row of logits: f(x, token) with the logits of EPV tokens and the first of them; elements behind the
// row are -inf.  Which lane takes which token does not depend on where the row starts in memory, so that equal rows give equal
// sums: an unaligned row is read through pairs of aligned vectors, and element by element where those would leave it.
template <typename T, typename F>
__device__ __forceinline__ void visit_segment(const T* row, int vocab, int seg, int segs, int lane, F&& f)
{
    constexpr int EPV = Elem<T>::EPV, AT_ONCE = 4;   // vectors whose loads are in flight together
    const unsigned skew = (unsigned)(reinterpret_cast<uintptr_t>(row) & 15u);
    const int ahead = (int)(skew / sizeof(T));
    const int vecs = (vocab + EPV - 1) / EPV, step = segs * 32;
    auto inside = [&](int t0) { return t0 >= ahead && t0 - ahead + (skew != 0 ? 2 * EPV : EPV) <= vocab; };
    for (int v0 = seg * 32 + lane; v0 < vecs; v0 += AT_ONCE * step) {
        uint4 raw[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int t0 = (v0 + i * step) * EPV;
            if (v0 + i * step < vecs && inside(t0)) raw[i] = load_skewed(reinterpret_cast<const uint4*>(row + t0 - ahead), skew);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (v0 + i * step >= vecs) break;
            const int t0 = (v0 + i * step) * EPV;
            float x[EPV];
            if (inside(t0)) {
                Elem<T>::unpack(raw[i], x);
            } else {
#pragma unroll
                for (int e = 0; e < EPV; ++e) x[e] = t0 + e < vocab ? Elem<T>::to_float(row[t0 + e]) : -CUDART_INF_F;
            }
            f(x, t0);
        }
    }
}

template <typename T>
__global__ void __cluster_dims__(kSelCluster, 1, 1) __launch_bounds__(kSelThreads) ffa_beam_select_kernel(const FfaBeamParams P)
{
    constexpr int EPV = Elem<T>::EPV;
    __shared__ __align__(16) SelRecord records[kSelSegments];
    __shared__ __align__(16) SelCandidate list[kSelList];
    __shared__ double lse[kMaxBeams];
    __shared__ __align__(16) float bound_of[4 * kSelSegments];
    __shared__ unsigned hist[256];
    __shared__ unsigned count;
    __shared__ float s_bound;
    __shared__ unsigned long long s_prefix;
    __shared__ unsigned s_left;

    const int b = blockIdx.x / kSelCluster;
    const uint32_t rank = cluster_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int beams = P.beams, segs = kSelSegments / beams, vocab = P.vocab;
    const int mine = (int)rank + kSelCluster * warp;   // this warp's segment: neighbouring segments in different CTAs
    const int beam = mine / segs, seg = mine - beam * segs;
    const bool works = beam < beams;
    const T* row = static_cast<const T*>(P.logits) + ((size_t)b * beams + (works ? beam : 0)) * P.row_stride;

    pdl_release();
    if (tid == 0) count = 0, s_bound = -CUDART_INF_F;
    cluster_arrive();   // this CTA runs and its counter is clear: the peers wait for that before they store into it
    pdl_wait();
    const bool done = works && P.finished != nullptr && P.finished[(size_t)b * beams + beam] != 0;
    const float s0 = works ? P.scores[(size_t)b * beams + beam] : -CUDART_INF_F;
    const bool alive = works && s0 > -CUDART_INF_F;   // a beam without a score has no candidates

    float m = -CUDART_INF_F, l = 0.f;
    if (alive && !done) {
        visit_segment(row, vocab, seg, segs, lane, [&](const float (&x)[EPV], int) {
            float top = x[0];
#pragma unroll
            for (int e = 1; e < EPV; ++e) top = fmaxf(top, x[e]);
            if (top > m) l *= fast_exp2((m - top) * kLog2e), m = top;
            if (m == -CUDART_INF_F) {   // nothing yet, unless NaN hides among the -inf
#pragma unroll
                for (int e = 0; e < EPV; ++e) l += x[e] != x[e] ? CUDART_NAN_F : 0.f;
                return;
            }
#pragma unroll
            for (int e = 0; e < EPV; ++e) l += fast_exp2((x[e] - m) * kLog2e);
        });
    } else if (alive && done && seg == 0) {
        m = 0.f, l = lane == 0 ? 1.f : 0.f;   // a finished beam offers one candidate: its score as it is
    }
    SelRecord rec;
    {
        float t = m;
#pragma unroll
        for (int off = 4; off >= 1; off >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, off));
#pragma unroll
        for (int i = 0; i < 4; ++i) rec.quarter[i] = __shfl_sync(0xffffffffu, t, 8 * i);
        rec.m = fmaxf(fmaxf(rec.quarter[0], rec.quarter[1]), fmaxf(rec.quarter[2], rec.quarter[3]));
        if (done) rec.quarter[1] = rec.quarter[2] = rec.quarter[3] = -CUDART_INF_F;
        rec.pad = 0.f;
        // a lane without a finite logit adds its l (0, or NaN)
        double sum = m == -CUDART_INF_F ? (double)l : (double)l * exp((double)m - (double)rec.m);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        rec.l = sum;
    }
    cluster_wait();
    if (lane < kSelCluster) {
        const uint32_t to = map_peer(&records[mine], (uint32_t)lane);
        const uint4* from = reinterpret_cast<const uint4*>(&rec);
        st_peer_v4(to, from[0]);
        st_peer_v4(to + 16, from[1]);
    }
    cluster_sync_all();

    for (int i = warp; i < beams; i += kSelWarps) {
        float top = -CUDART_INF_F;
        for (int s = lane; s < segs; s += 32) top = fmaxf(top, records[i * segs + s].m);
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        double sum = 0.0;
        for (int s = lane; s < segs; s += 32) {
            const SelRecord& r = records[i * segs + s];
            sum += r.m == -CUDART_INF_F ? r.l : r.l * exp((double)r.m - (double)top);
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        // NaN or -inf when the row holds NaN or +inf, or nothing above -inf: then it has no candidates
        if (lane == 0) lse[i] = (double)top + log(sum);
    }
    __syncthreads();
    // lower bound of the num-th best score: the num-th largest of scores that exist, rounded down to fp32.  Each of n scores is ranked
    // by kSelThreads / n threads, which compare it with a share of the others and add up (n is a power of two).
    auto find_bound = [&](auto n_tag) {
        constexpr int n = decltype(n_tag)::value, SHARE = kSelThreads / n;
        __syncthreads();
        const int i = tid / SHARE, part = tid % SHARE;
        const float me = bound_of[i];
        int above = 0;
#pragma unroll 8
        for (int k = part * (n / SHARE); k < (part + 1) * (n / SHARE); k += 4) {
            const float4 x = *reinterpret_cast<const float4*>(bound_of + k);
            above += x.x > me || (x.x == me && k < i);
            above += x.y > me || (x.y == me && k + 1 < i);
            above += x.z > me || (x.z == me && k + 2 < i);
            above += x.w > me || (x.w == me && k + 3 < i);
        }
#pragma unroll
        for (int off = SHARE / 2; off >= 1; off >>= 1) above += __shfl_xor_sync(0xffffffffu, above, off);
        if (part == 0 && above == P.num - 1) s_bound = me;
        __syncthreads();
    };
    auto record_score = [&](int s, float x) -> float {
        const int i = s / segs;
        if (i >= beams || x == -CUDART_INF_F) return -CUDART_INF_F;
        const double v = (double)P.scores[(size_t)b * beams + i] + ((double)x - lse[i]);
        return v > -CUDART_INF ? __double2float_rd(v) : -CUDART_INF_F;   // also where v is NaN
    };
    if (tid < kSelSegments) bound_of[tid] = record_score(tid, records[tid].m);
    find_bound(std::integral_constant<int, kSelSegments>{});
    if (s_bound == -CUDART_INF_F) {
        bound_of[tid] = record_score(tid >> 2, records[tid >> 2].quarter[tid & 3]);
        find_bound(std::integral_constant<int, 4 * kSelSegments>{});
    }
    const double bound = (double)s_bound;

    // visits this warp's candidates: f(score, flat) for every element whose score is above -inf and at least `least`
    auto candidates = [&](double least, auto&& f) {
        if (!alive) return;
        const double base = lse[beam];
        if (done) {
            if (seg == 0 && lane == 0 && (double)s0 >= least) f((double)s0, (unsigned)(beam * vocab + P.pad_token));
            return;
        }
        if (!(base > -CUDART_INF)) return;
        // the smallest logit that can reach `least`, a little lower than it is so that rounding cannot lose one
        const double need = least - (double)s0 + base;
        const float low = __double2float_rd(need - 1e-6 * (1.0 + fabs(least) + fabs((double)s0) + fabs(base)));
        if (m < low) return;   // this lane's largest logit, from pass 1: hardly a lane in a hundred looks at its part again
        visit_segment(row, vocab, seg, segs, lane, [&](const float (&x)[EPV], int t0) {
            float top = x[0];
#pragma unroll
            for (int e = 1; e < EPV; ++e) top = fmaxf(top, x[e]);
            if (top < low || top == -CUDART_INF_F) return;
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
                if (x[e] >= low && x[e] > -CUDART_INF_F) {
                    const double score = (double)s0 + ((double)x[e] - base);
                    if (score >= least && score > -CUDART_INF) f(score, (unsigned)(beam * vocab + t0 + e));
                }
            }
        });
    };
    const uint32_t leader_count = map_peer(&count, 0), leader_list = map_peer(&list[0], 0);
    auto offer = [&](double score, unsigned flat) {
        const unsigned at = add_peer_u32(leader_count, 1u);
        if (at < kSelList) {
            const unsigned long long u = (unsigned long long)__double_as_longlong(score);
            st_peer_v4(leader_list + at * (uint32_t)sizeof(SelCandidate), make_uint4((unsigned)u, (unsigned)(u >> 32), flat, 0u));
        }
    };
    candidates(bound, offer);
    cluster_sync_all();

    if (ld_peer_u32(leader_count) > kSelList) {
        // exact border: 8 passes over the score, then 4 over the index of those that tie with it (lowest index first)
        cluster_sync_all();   // everyone has read the count
        if (tid == 0) count = 0, s_prefix = 0, s_left = (unsigned)P.num;
        unsigned long long border = 0;   // score key of the num-th best
        unsigned last = UINT_MAX;        // largest index that still belongs to the result among the ties
        for (int pass = 0; pass < 12; ++pass) {
            const bool by_index = pass >= 8;
            const int shift = by_index ? 24 - 8 * (pass - 8) : 56 - 8 * pass;
            if (pass == 8) {
                __syncthreads();
                border = s_prefix;
                __syncthreads();
                if (tid == 0) s_prefix = 0;
            }
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const unsigned long long prefix = s_prefix;
            candidates(-CUDART_INF, [&](double score, unsigned flat) {
                const unsigned long long s = ordered64(score);
                if (by_index && s != border) return;
                // indices are counted from the lowest: their complement, so that "larger first" serves both
                const unsigned long long u = by_index ? (unsigned long long)(~flat) : s;
                const int top = by_index ? 24 : 56;
                if (shift == top || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(u >> shift) & 255], 1u);
            });
            cluster_sync_all();
            if (tid == 0) {
                unsigned left = s_left;
                int digit = 255;
                for (; digit > 0; --digit) {
                    unsigned n = 0;
                    for (uint32_t r = 0; r < kSelCluster; ++r) n += ld_peer_u32(map_peer(&hist[digit], r));
                    if (n >= left) break;
                    left -= n;
                }
                s_prefix = prefix | ((unsigned long long)digit << shift);
                s_left = left;
            }
            cluster_sync_all();   // the histograms have been read
        }
        last = ~(unsigned)s_prefix;
        candidates(-CUDART_INF, [&](double score, unsigned flat) {
            const unsigned long long s = ordered64(score);
            if (s > border || (s == border && flat <= last)) offer(score, flat);
        });
        cluster_sync_all();
    }
    if (rank == 0) {
        const int n = min((int)count, kSelList);
        for (int i = tid; i < n; i += kSelThreads) {
            const SelCandidate c = list[i];
            int above = 0;
#pragma unroll 4
            for (int k = 0; k < n; ++k) above += list[k].score > c.score || (list[k].score == c.score && list[k].flat < c.flat);
            if (above < P.num) {
                const size_t o = (size_t)b * P.num + above;
                P.out_scores[o] = (float)c.score;
                P.out_parents[o] = (int)(c.flat / (unsigned)vocab);
                P.out_tokens[o] = (int)(c.flat % (unsigned)vocab);
            }
        }
        for (int i = n + tid; i < P.num; i += kSelThreads) {   // fewer candidates than asked for
            const size_t o = (size_t)b * P.num + i;
            P.out_scores[o] = -CUDART_INF_F, P.out_parents[o] = 0, P.out_tokens[o] = P.pad_token;
        }
    }
    cluster_sync_all();   // the leader's counter is read by the others: it stays until all are here
}

// ------------------------------------------------------------------------------------------
// Reordering
// ------------------------------------------------------------------------------------------
// Rows [first, rows) of beam j <- beam parent[j], in place, for every group of beams and every head.  Beams exchange whole
// columns: a thread takes one 16-byte vector of a row from every beam it needs before it stores any, so no copy of the cache and
// no order among beams is needed; beams that stay are neither read (unless they are a parent) nor written.
template <int NB>
__global__ void __launch_bounds__(256) ffa_reorder_kernel(const FfaReorderParams P)
{
    const int chunk = blockIdx.x % P.chunks, pair = blockIdx.x / P.chunks, h = pair % P.H, g = pair / P.H;
    __shared__ int parent[NB];
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    if ((int)threadIdx.x < P.beams) {
        const int p = P.parents[(size_t)g * P.beams + threadIdx.x];
        parent[threadIdx.x] = p;
        if (p < 0 || p >= P.beams) bad = 1;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) atomicOr(P.status, kStatusBadIndex);
        return;
    }
    const int vpr = P.row_bytes / 16;
    const long long vecs = (long long)(P.rows - P.first) * vpr, slab = (long long)P.Lmax * vpr;
    uint4* cache = static_cast<uint4*>(blockIdx.y == 0 ? P.k_cache : P.v_cache) + (long long)P.first * vpr;
    auto at = [&](int j) { return (((long long)g * P.beams + j) * P.H + h) * slab; };
    for (long long i = (long long)chunk * blockDim.x + threadIdx.x; i < vecs; i += (long long)P.chunks * blockDim.x) {
        uint4 x[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (j < P.beams && parent[j] != j) x[j] = cache[at(parent[j]) + i];
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (j < P.beams && parent[j] != j) cache[at(j) + i] = x[j];
    }
}

}  // namespace

int ffa_k_beam_select(int dtype, const FfaBeamParams& P, cudaStream_t stream)
{
    const auto kernel = dtype == 0 ? ffa_beam_select_kernel<float> : dtype == 1 ? ffa_beam_select_kernel<__half> : ffa_beam_select_kernel<__nv_bfloat16>;
    return (int)launch_pdl(kernel, P.batch * kSelCluster, kSelThreads, 0, 0, true, stream, P);
}

int ffa_k_reorder(FfaReorderParams P, int sms, cudaStream_t stream)
{
    const long long vecs = (long long)(P.rows - P.first) * (P.row_bytes / 16);
    const long long pairs = (long long)P.groups * P.H;
    const long long most = (16LL * sms + 2 * pairs - 1) / (2 * pairs);   // about 16 blocks per SM over both tensors and all heads
    long long chunks = (vecs + 255) / 256;
    if (chunks > most) chunks = most;
    P.chunks = (int)chunks;
    const dim3 grid((unsigned)(chunks * pairs), 2);
    if (P.beams <= 4) ffa_reorder_kernel<4><<<grid, 256, 0, stream>>>(P);
    else if (P.beams <= 8) ffa_reorder_kernel<8><<<grid, 256, 0, stream>>>(P);
    else if (P.beams <= 16) ffa_reorder_kernel<16><<<grid, 256, 0, stream>>>(P);
    else ffa_reorder_kernel<32><<<grid, 256, 0, stream>>>(P);
    return (int)cudaGetLastError();
}
