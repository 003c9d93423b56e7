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
// A thread-block cluster of C CTAs per sample (8, fewer where a batch fills the device anyway); each of its 16 C warps owns a segment
// of one beam's logits (every SEG-th block of 32 vectors, so that the best tokens of a sorted vocabulary do not sit in one segment).
//   pass 1   running maximum and sum of exponentials per lane; every warp stores its maximum, the maxima of its four quarters
//            and its sum into every CTA of the cluster;                                              -- cluster barrier --
//            every CTA now has all beams' logsumexp and 16 C scores that exist: the num-th largest of them is a lower bound of
//            the num-th best score (the quarters' maxima serve where a beam has fewer warps than candidates may come from it: when one beam
//            is far ahead, or the only live one, all of them do)
//   pass 2   (L1 / L2) the lanes whose maximum reaches the bound look at their part again and note what does, about num elements
//            of the sample in all; the notes are weighed and go into the CTA's part of the leader's list; -- cluster barrier --
//            the leader ranks the list and writes the result.
// A CTA that notes more than its part of the list holds (a vocabulary of ties) finds its own num best by radix selection, 8 bits a
// pass, over the 64-bit score and then the index: more than those cannot be in the result.
// Exponentials are fp32; a lane adds 32 or 64 of them in fp32 and these sums, like those of lanes and warps, as doubles.  A log-sum is then off by
// 3e-6 at most: 2^-22 for an exponential, (2^-24 + 1.5 2^-24) |x - reference| for its argument, whose mean under the softmax is at most about 11,
// 11 2^-24 for the fp32 sums, 2^-22 for joining lanes and segments.  Scores are compared as doubles: tokens of one beam come in the exact order,
// two beams' candidates whose scores lie closer than their log-sums' errors may come in either.
constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelShare = 128;   // candidates that the leader's list holds of each CTA
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.f;    // a lane's sum is rescaled when a logit is this far above its reference: what it held is then a small part of
                                 // the sum, and the errors of many rescalings (an ascending vocabulary) cannot add up
constexpr int kFlush = 8;        // vectors that a lane adds in fp32

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
__device__ __forceinline__ void st_peer_u32(uint32_t addr, unsigned v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// floats in the order of their values (no NaN), and back
__device__ __forceinline__ uint32_t ordered32(float x)
{
    const uint32_t u = __float_as_uint(x + 0.f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered32(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u); }
// doubles in the order of their values (no NaN)
__device__ __forceinline__ unsigned long long ordered64(double x)
{
    const unsigned long long u = (unsigned long long)__double_as_longlong(x + 0.0);
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

// 16 bytes that start `skew` bytes into the 32 of a and b; skew is a multiple of 2 from 2 to 14, the same for the warp
__device__ __forceinline__ uint4 shift_window(uint4 a, uint4 b, unsigned skew)
{
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

// Visits vectors first, first + step, ... of a row of logits: f(x, token) with the logits of EPV tokens and the first of them;
// elements behind the row are -inf.  Which lane takes which token does not depend on where the row starts in memory, so that equal rows give equal
// sums: an unaligned row (kSkewed) is read through pairs of aligned vectors, and element by element where those would leave it.
template <bool kSkewed, typename T, typename F>
__device__ __forceinline__ void visit_vectors(const T* row, int vocab, int first, int step, F&& f)
{
    constexpr int EPV = Elem<T>::EPV, AT_ONCE = kSkewed ? 2 : 4;   // vectors whose loads are in flight together
    const unsigned skew = (unsigned)(reinterpret_cast<uintptr_t>(row) & 15u);
    const int ahead = kSkewed ? (int)(skew / sizeof(T)) : 0;
    const int vecs = (vocab + EPV - 1) / EPV;
    auto inside = [&](int t0) { return t0 >= ahead && t0 - ahead + (kSkewed ? 2 * EPV : EPV) <= vocab; };
#pragma unroll 1
    for (int v0 = first; v0 < vecs; v0 += AT_ONCE * step) {
        uint4 raw[AT_ONCE], next[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {   // loads only: nothing here waits for one of them
            const int t0 = (v0 + i * step) * EPV;
            const bool ok = v0 + i * step < vecs && inside(t0);
            const uint4* p = reinterpret_cast<const uint4*>(row + t0 - ahead);
            raw[i] = next[i] = make_uint4(0, 0, 0, 0);
            if (ok) raw[i] = p[0];
            if (kSkewed && ok) next[i] = p[1];
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (v0 + i * step >= vecs) break;
            const int t0 = (v0 + i * step) * EPV;
            float x[EPV];
            if (inside(t0)) {
                Elem<T>::unpack(kSkewed ? shift_window(raw[i], next[i], skew) : raw[i], x);
            } else {
#pragma unroll
                for (int e = 0; e < EPV; ++e) x[e] = t0 + e < vocab ? Elem<T>::to_float(row[t0 + e]) : -CUDART_INF_F;
            }
            f(x, t0);
        }
    }
}
template <typename T, typename F>
__device__ __forceinline__ void visit(const T* row, int vocab, int first, int step, F&& f)
{
    if ((reinterpret_cast<uintptr_t>(row) & 15u) == 0) visit_vectors<false>(row, vocab, first, step, f);
    else visit_vectors<true>(row, vocab, first, step, f);
}

// Calls f(x, token) for every element of those vectors that is at least `low` and above -inf.  Few are: the vectors are
// only compared, and what to do with an element stands once in the code (unrolled over a vector's elements it would be tens of
// kilobytes that a warp walks through once, fetching every line of it: 5 us).
template <typename T, typename F>
__device__ __forceinline__ void visit_from(const T* row, int vocab, int first, int step, float low, F&& f)
{
    constexpr int EPV = Elem<T>::EPV;
    visit(row, vocab, first, step, [&](const float (&x)[EPV], int t0) {
        uint32_t some = 0;
#pragma unroll
        for (int e = 0; e < EPV; ++e) some |= (x[e] >= low && x[e] > -CUDART_INF_F ? 1u : 0u) << e;
#pragma unroll 1
        for (; some != 0; some &= some - 1) {
            const int t = t0 + __ffs(some) - 1;
            f(Elem<T>::to_float(row[t]), t);
        }
    });
}

template <typename T, int C>
__global__ void __launch_bounds__(kSelThreads) ffa_beam_select_kernel(const FfaBeamParams P)
{
    constexpr int kSelCluster = C, kSelSegments = kSelWarps * C, kSelList = kSelShare * C;
    constexpr int EPV = Elem<T>::EPV;
    __shared__ __align__(16) SelRecord records[kSelSegments];
    __shared__ __align__(16) SelCandidate list[kSelList];
    __shared__ double lse[kMaxBeams];
    __shared__ __align__(16) uint32_t bound_of[4 * kSelSegments];
    __shared__ __align__(16) uint32_t lane_best[kSelThreads];
    __shared__ uint2 found[kSelShare];          // elements of this CTA that may reach the bound: index, logit
    __shared__ float beam_score[kMaxBeams];
    __shared__ unsigned hist[256];
    __shared__ unsigned found_count, count;     // of them, and candidates of this CTA
    __shared__ unsigned counts[kSelCluster];    // of every CTA
    __shared__ uint32_t s_bound;
    __shared__ unsigned s_digit, s_left, s_here;

    const int b = blockIdx.x / kSelCluster;
    const uint32_t rank = cluster_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int beams = P.beams, segs = kSelSegments / beams, vocab = P.vocab;
    const int mine = (int)rank + kSelCluster * warp;   // this warp's segment: neighbouring segments in different CTAs
    const int beam = mine / segs, seg = mine - beam * segs;
    const bool works = beam < beams;
    const T* row = static_cast<const T*>(P.logits) + ((size_t)b * beams + (works ? beam : 0)) * P.row_stride;

    pdl_release();
    if (tid == 0) count = 0, found_count = 0, s_bound = 0;
    cluster_arrive();   // this CTA runs: the peers wait for that before they store into it
    pdl_wait();
    // the first vectors of the lane's part, so that they are on their way while the beam's score is
    if (works) {
        constexpr int EPL = 16 / (int)sizeof(T);
        for (int i = 0; i < 4; ++i) {
            const int t = ((seg + i * segs) * 32 + lane) * EPL;
            if (t < vocab) prefetch_l1(row + t);
        }
    }
    if (tid < beams) beam_score[tid] = P.scores[(size_t)b * beams + tid];
    const bool done = works && P.finished != nullptr && P.finished[(size_t)b * beams + beam] != 0;
    const float s0 = works ? P.scores[(size_t)b * beams + beam] : -CUDART_INF_F;
    const bool alive = works && s0 > -CUDART_INF_F;   // a beam without a score has no candidates

    float m = -CUDART_INF_F, ref = -CUDART_INF_F, l = 0.f;   // the lane's largest logit, what its terms are relative to, their newest ones' sum
    double total = 0.0;                                       // and the others'
    int adds = 0;
    if (alive && !done) {
        visit(row, vocab, seg * 32 + lane, segs * 32, [&](const float (&x)[EPV], int) {
            float top = x[0];
#pragma unroll
            for (int e = 1; e < EPV; ++e) top = fmaxf(top, x[e]);
            m = fmaxf(m, top);
            if (top > ref + kRaise) {
                const float f = fast_exp2((ref - top) * kLog2e);
                l *= f, total *= (double)f, ref = top;
            }
            if (ref == -CUDART_INF_F) {   // nothing yet, unless NaN hides among the -inf
#pragma unroll
                for (int e = 0; e < EPV; ++e) l += x[e] != x[e] ? CUDART_NAN_F : 0.f;
                return;
            }
            float t[EPV];
#pragma unroll
            for (int e = 0; e < EPV; ++e) t[e] = fast_exp2((x[e] - ref) * kLog2e);
#pragma unroll
            for (int n = EPV / 2; n >= 1; n /= 2)
#pragma unroll
                for (int e = 0; e < n; ++e) t[e] += t[e + n];
            l += t[0];
            if (++adds == kFlush) total += (double)l, l = 0.f, adds = 0;
        });
    } else if (alive && done && seg == 0) {
        m = ref = 0.f, l = lane == 0 ? 1.f : 0.f;   // a finished beam offers one candidate: its score as it is
    }
    total += (double)l;
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
        // a lane without a finite logit adds its total (0, or NaN)
        double sum = ref == -CUDART_INF_F ? total : total * (double)expf(ref - rec.m);
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
            sum += r.m == -CUDART_INF_F ? r.l : r.l * (double)expf(r.m - top);
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        // NaN or -inf when the row holds NaN or +inf, or nothing above -inf: then it has no candidates
        if (lane == 0) lse[i] = (double)top + log(sum);
    }
    __syncthreads();
    // Lower bound of the num-th best score: the num-th largest of scores that exist.  Scores are rounded down to fp32, and as integers in
    // the order of the floats their lowest bits give way to their index: all are different, and a rank is one comparison each.
    auto find_bound = [&](const uint32_t* of, int n) {
        __syncthreads();
        if (tid < n) {
            const uint32_t me = of[tid];
            int above = 0;
#pragma unroll 4
            for (int k = 0; k < n; k += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(of + k);
                above += x.x > me, above += x.y > me, above += x.z > me, above += x.w > me;
            }
            if (above == P.num - 1) s_bound = me;
        }
        __syncthreads();
    };
    constexpr uint32_t kIndexBits = 4 * kSelSegments - 1, kMinusInf = 0x007fffffu;   // ordered32(-inf)
    auto record_score = [&](int s, float x, int index) -> uint32_t {
        const int i = s / segs;
        const double v = i < beams && x > -CUDART_INF_F ? (double)beam_score[i] + ((double)x - lse[i]) : -CUDART_INF;
        const float f = v > -CUDART_INF ? __double2float_rd(v) : -CUDART_INF_F;   // also where v is NaN
        return f > -CUDART_INF_F ? (ordered32(f) & ~kIndexBits) | (uint32_t)index : (uint32_t)index;
    };
    if (segs >= P.num) {
        if (tid < kSelSegments) bound_of[tid] = record_score(tid, records[tid].m, tid);
        find_bound(bound_of, kSelSegments);
    }
    if (s_bound <= kMinusInf) {
        if (tid < 4 * kSelSegments) bound_of[tid] = record_score(tid >> 2, records[tid >> 2].quarter[tid & 3], tid);
        find_bound(bound_of, 4 * kSelSegments);
    }
    const bool candidates_here = alive && (done ? seg == 0 : lse[beam] > -CUDART_INF);
    if (s_bound <= kMinusInf) {
        // a vocabulary so short, or so few live beams, that less than num quarters hold anything: the maxima of this CTA's lanes bound what
        // it can contribute (500 tokens of one beam, num 16: without this all of them are candidates: 33 us instead of 18)
        const double v = candidates_here && m > -CUDART_INF_F && (!done || lane == 0) ? (double)beam_score[beam] + ((double)m - lse[beam]) : -CUDART_INF;
        const float f = v > -CUDART_INF ? __double2float_rd(v) : -CUDART_INF_F;
        lane_best[tid] = f > -CUDART_INF_F ? (ordered32(f) & ~(kSelThreads - 1u)) | (uint32_t)tid : (uint32_t)tid;
        find_bound(lane_best, kSelThreads);
    }
    const double bound = s_bound > kMinusInf ? (double)from_ordered32(s_bound & ~(kSelThreads - 1u)) : -CUDART_INF;

    // the smallest logit of a beam that can reach the bound, a little lower than it is so that rounding cannot lose one
    auto lowest = [&](int i) -> float {
        const double base = lse[i], s = (double)beam_score[i], need = bound - s + base;
        if (s == CUDART_INF) return -CUDART_INF_F;       // every token of such a beam is as good as can be
        if (bound == CUDART_INF) return CUDART_INF_F;    // and next to enough of them nothing else is
        return __double2float_rd(need - 1e-6 * (1.0 + fabs(bound) + fabs(s) + fabs(base)));
    };
    auto score_of = [&](int i, float x) -> double { return (double)beam_score[i] + ((double)x - lse[i]); };
    const uint32_t share = map_peer(&list[rank * kSelShare], 0);   // this CTA's part of the leader's list
    auto offer = [&](double score, unsigned flat) {
        const unsigned at = atomicAdd(&count, 1u);
        if (at < kSelShare) {
            const unsigned long long u = (unsigned long long)__double_as_longlong(score);
            st_peer_v4(share + at * (uint32_t)sizeof(SelCandidate), make_uint4((unsigned)u, (unsigned)(u >> 32), flat, 0u));
        }
    };
    auto publish = [&]() {   // this CTA's count to everyone
        __syncthreads();
        if (tid < kSelCluster) st_peer_u32(map_peer(&counts[rank], (uint32_t)tid), count);
        cluster_sync_all();
    };
    // pass 2: lanes only note what may reach the bound; the few notes are then weighed side by side, a thread each
    auto note = [&](float x, int t) {
        const unsigned at = atomicAdd(&found_count, 1u);
        if (at < kSelShare) found[at] = make_uint2((unsigned)(beam * vocab + t), __float_as_uint(x));
    };
    if (candidates_here) {
        if (done) {
            if (lane == 0) note(0.f, P.pad_token);   // its logsumexp is 0
        } else {
            const float low = lowest(beam);
            if (m >= low) visit_from(row, vocab, seg * 32 + lane, segs * 32, low, note);   // m: this lane's largest logit, from pass 1
        }
    }
    __syncthreads();
    if (found_count <= kSelShare) {
        if (tid < (int)found_count) {
            const uint2 c = found[tid];
            const double score = score_of((int)(c.x / (unsigned)vocab), __uint_as_float(c.y));
            if (score >= bound && score > -CUDART_INF) offer(score, c.x);
        }
    } else {
        // every element of this CTA that may reach the bound; all warps share each segment, since the elements may all be in one
        auto candidates = [&](auto&& f) {
#pragma unroll 1
            for (int w = 0; w < kSelWarps; ++w) {
                const int at = (int)rank + kSelCluster * w, i = at / segs, sg = at - i * segs;
                if (i >= beams || records[at].m == -CUDART_INF_F || !(lse[i] > -CUDART_INF)) continue;
                if (P.finished != nullptr && P.finished[(size_t)b * beams + i] != 0) {
                    if (tid == 0) f((double)beam_score[i], (unsigned)(i * vocab + P.pad_token));   // (its record is in segment 0)
                    continue;
                }
                const float low = lowest(i);
                if (records[at].m < low) continue;
                visit_from(static_cast<const T*>(P.logits) + ((size_t)b * beams + i) * P.row_stride, vocab, sg * 32 + lane + warp * segs * 32,
                           kSelWarps * segs * 32, low, [&](float x, int t) {
                               const double score = score_of(i, x);
                               if (score > -CUDART_INF) f(score, (unsigned)(i * vocab + t));
                           });
            }
        };
        // Larger first, in both: scores as ordered integers, and among equal scores the complement of the index.  `border` holds the
        // bits that are settled, those from `shift` up; everything that agrees with them or is larger belongs to the num best as
        // soon as as many elements agree as are left to find.
        unsigned long long border = 0, tie = 0;
        int left = P.num, shift = 64;
        bool exact = false, by_index = false;
        for (int pass = 0; pass < 12 && !exact; ++pass) {
            by_index = pass >= 8;
            if (pass == 8) tie = border, border = 0, shift = 32;
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            candidates([&](double score, unsigned flat) {
                const unsigned long long s = ordered64(score);
                if (by_index && s != tie) return;
                const unsigned long long u = by_index ? (unsigned long long)(~flat) : s;
                if (shift == 64 || (u >> shift) == (border >> shift)) atomicAdd(&hist[(u >> (shift - 8)) & 255], 1u);
            });
            __syncthreads();
            if (warp == 0) {   // the digit at which the count from above reaches what is left: 8 digits a lane, from the top
                unsigned mine[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) mine[i] = hist[255 - (lane * 8 + i)], sum += mine[i];
                unsigned inc = sum;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const unsigned y = __shfl_up_sync(0xffffffffu, inc, off);
                    if (lane >= off) inc += y;
                }
                unsigned above = inc - sum;
                if (above < (unsigned)left && inc >= (unsigned)left) {
                    int i = 0;
#pragma unroll
                    for (int k = 0; k < 7; ++k)
                        if (i == k && above + mine[k] < (unsigned)left) above += mine[k], i = k + 1;
                    unsigned here = 0;
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (i == k) here = mine[k];
                    s_digit = 255u - (unsigned)(lane * 8 + i), s_left = (unsigned)left - above, s_here = here;
                }
            }
            __syncthreads();
            shift -= 8;
            border |= (unsigned long long)s_digit << shift;
            left = (int)s_left;
            exact = s_here == s_left;
        }
        candidates([&](double score, unsigned flat) {
            const unsigned long long s = ordered64(score);
            if (by_index ? s > tie || (s == tie && ((unsigned long long)(~flat) >> shift) >= (border >> shift)) : (s >> shift) >= (border >> shift))
                offer(score, flat);
        });
    }
    publish();
    if (rank != 0) return;   // nothing in this CTA's shared memory is needed any more
    {
        // C threads rank a candidate, each among one CTA's part of the list
        int n = 0;
#pragma unroll
        for (int c = 0; c < kSelCluster; ++c) n += (int)counts[c];
        const int q = tid % kSelCluster, others = (int)counts[q];
        const SelCandidate* other = list + q * kSelShare;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += kSelThreads / kSelCluster) {
            const int i = min(i0 + tid / kSelCluster, n - 1);
            int part = 0, at = i;   // the i-th candidate: place `at` of a CTA's part
#pragma unroll 1
            for (; at >= (int)counts[part]; ++part) at -= (int)counts[part];
            const SelCandidate c = list[part * kSelShare + at];
            int above = 0;
#pragma unroll 1
            for (int k = 0; k < others; ++k) above += other[k].score > c.score || (other[k].score == c.score && other[k].flat < c.flat);
#pragma unroll
            for (int off = kSelCluster / 2; off >= 1; off >>= 1) above += __shfl_xor_sync(0xffffffffu, above, off);
            if (q == 0 && i == i0 + tid / kSelCluster && above < P.num) {
                const size_t o = (size_t)b * P.num + above;
                const unsigned parent = c.flat / (unsigned)vocab;
                P.out_scores[o] = (float)c.score;
                P.out_parents[o] = (int)parent;
                P.out_tokens[o] = (int)(c.flat - parent * (unsigned)vocab);
            }
        }
        for (int i = n + tid; i < P.num; i += kSelThreads) {   // fewer candidates than asked for
            const size_t o = (size_t)b * P.num + i;
            P.out_scores[o] = -CUDART_INF_F, P.out_parents[o] = 0, P.out_tokens[o] = P.pad_token;
        }
    }
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

int ffa_k_beam_select(int dtype, const FfaBeamParams& P, int sms, cudaStream_t stream)
{
    // As many CTAs to a sample as the device holds for the whole batch (two to an SM): a second wave costs the chain of phases again
    // (bf16, 64 samples x 50257: 18.2 us with 8, 9.1 us with 4).  A beam needs a warp, and the bound 4 scores a warp.
    int cluster = 8;
    while (cluster > 1 && (long long)P.batch * cluster > 2LL * sms && P.beams <= kSelWarps * (cluster / 2) && P.num <= 2 * kSelWarps * cluster) cluster /= 2;
    auto launch = [&](auto kernel) { return (int)launch_pdl(kernel, P.batch * cluster, kSelThreads, 0, cluster, true, stream, P); };
    auto of_type = [&](auto t) {
        using T = decltype(t);
        switch (cluster) {
            case 1: return launch(ffa_beam_select_kernel<T, 1>);
            case 2: return launch(ffa_beam_select_kernel<T, 2>);
            case 4: return launch(ffa_beam_select_kernel<T, 4>);
            default: return launch(ffa_beam_select_kernel<T, 8>);
        }
    };
    return dtype == 0 ? of_type(float{}) : dtype == 1 ? of_type(__half{}) : of_type(__nv_bfloat16{});
}

int ffa_k_reorder(FfaReorderParams P, int sms, cudaStream_t stream)
{
    const long long vecs = (long long)(P.rows - P.first) * (P.row_bytes / 16);
    const long long pairs = (long long)P.groups * P.H;
    const long long most = (16LL * sms + 2 * pairs - 1) / (2 * pairs);   // about 16 blocks per SM over both tensors and all heads
    long long chunks = (vecs + 255) / 256;
    if (chunks > most) chunks = most;
    P.chunks = (int)chunks;
    // launched without programmatic overlap: blocks that wait for the previous kernel hold the SMs it would use (158 -> 177 us for 1 GB)
    const dim3 grid((unsigned)(chunks * pairs), 2);
    if (P.beams <= 4) ffa_reorder_kernel<4><<<grid, 256, 0, stream>>>(P);
    else if (P.beams <= 8) ffa_reorder_kernel<8><<<grid, 256, 0, stream>>>(P);
    else if (P.beams <= 16) ffa_reorder_kernel<16><<<grid, 256, 0, stream>>>(P);
    else ffa_reorder_kernel<32><<<grid, 256, 0, stream>>>(P);
    return (int)cudaGetLastError();
}
