// C entries of the tree attention (include/ffa_c_api.h): argument checks, the cut over CTAs and the parameter fill.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>

#include "../../include/ffa_c_api.h"
#include "ffa_internal.h"
#include "ffa_plan.h"

namespace {

// A CTA's time is its key tiles plus a fixed part (start, first tile, epilogue), and more when a pair is split (partial results and
// their merge).  The CTAs of a wave share HBM, and a tile takes each of them a certain time however few they are.  The number of
// splits is the one with the smallest sum over the waves.  Measured with 1 / 2 / 4 / 7 / 9 / 10 / 18 splits: bf16 x 128, 32 pairs, 16000
// tokens, 8 drafted: 190 / 102 / 56 / 47 / 50 / 64 / 54 us (7 is taken); 16 pairs, 32 K tokens, 132 query rows (9 is taken): 447 / 235 / 129 / 95 /
// 83 / 116 / 96 us.
FfaTreeShape tree_shape(const ffa_plan* p, int groups, int tokens, int t)
{
    FfaTreeShape s;
    ffa_k_tree_shape(p->dtype, p->Dh, groups * tokens, &s);
    const long long items = (long long)p->B * p->H * s.row_tiles, slots = (long long)p->sms * s.ctas_per_sm;
    const long long tiles = (t + s.tile_keys - 1) / s.tile_keys + (tokens + s.tile_keys - 1) / s.tile_keys;
    const double share_us = 2.0 * s.tile_keys * p->Dh * ffa_elem_size(p->dtype) / 6.0e6;   // a tile at the whole device's bandwidth
    double best = 0;
    s.splits = 1;
    for (long long splits = 1; splits <= tiles && splits <= kTreeMaxSplits; ++splits) {
        const long long ctas = items * splits, full = ctas / slots, rest = ctas % slots;
        const double run = (double)((tiles + splits - 1) / splits);
        const double fixed = 5.0 + (splits > 1 ? 2.0 + 0.05 * splits : 0.0);
        auto wave = [&](long long n) {
            // CTAs that share an SM slow one another down by about half of what they would without overlap
            const double crowd = s.tile_us * (n > p->sms ? 0.5 + 0.5 * n / p->sms : 1.0), shared = n * share_us;
            return n == 0 ? 0.0 : run * (crowd > shared ? crowd : shared) + fixed;
        };
        const double us = full * wave(slots) + wave(rest);
        if (splits == 1 || us < best) best = us, s.splits = (int)splits;
    }
    return s;
}

size_t tree_partials_bytes(const ffa_plan* p, const FfaTreeShape& s)
{
    if (s.splits <= 1) return 0;
    return (size_t)p->B * p->H * s.row_tiles * s.splits * s.part_rows * ffa_tree_part_stride(p->Dh) * sizeof(float);
}

int check_sizes(const ffa_plan* plan, int groups, int tokens, int t)
{
    if (plan == nullptr) return ffa_fail(FFA_ERR_ARG, "null plan");
    if (groups <= 0 || tokens <= 0) return ffa_fail(FFA_ERR_RANGE, "groups (%d) and tokens (%d) must be positive", groups, tokens);
    if (tokens > kTreeMaxRows || groups > kTreeMaxRows || groups * tokens > kTreeMaxRows)
        return ffa_fail(FFA_ERR_RANGE, "groups * tokens (%d * %d) exceeds %d query rows per cache head", groups, tokens, kTreeMaxRows);
    if (t < 0 || t >= plan->Lmax) return ffa_fail(FFA_ERR_RANGE, "t = %d outside [0, %d)", t, plan->Lmax);
    if ((long long)plan->B * plan->H * groups * tokens >= (1LL << 31)) return ffa_fail(FFA_ERR_RANGE, "sizes exceed int range");
    return FFA_OK;
}

int check_pages(const ffa_plan* plan, const int* page_table, int max_pages, int page_rows, int pool_pages)
{
    if (page_table == nullptr) return FFA_OK;
    if (pool_pages <= 0 || (long long)pool_pages * plan->H * (page_rows > 0 ? page_rows : 1) >= (1LL << 31))
        return ffa_fail(FFA_ERR_RANGE, "pool_pages = %d: must be positive, and the pool's rows below 2^31", pool_pages);
    if (page_rows <= 0 || page_rows % 128 != 0)
        return ffa_fail(FFA_ERR_RANGE, "page_rows (%d) must be a positive multiple of 128", page_rows);
    if (max_pages <= 0 || (long long)max_pages * page_rows != plan->Lmax)
        return ffa_fail(FFA_ERR_RANGE, "max_pages * page_rows (%d * %d) must equal the plan's max_len (%d)", max_pages, page_rows, plan->Lmax);
    return FFA_OK;
}

}  // namespace

extern "C" {

int ffa_tree_scratch_bytes(const ffa_plan_t* plan, int groups, int tokens, int t, size_t* bytes)
{
    const int r = check_sizes(plan, groups, tokens, t);
    if (r != FFA_OK) return r;
    if (bytes == nullptr) return ffa_fail(FFA_ERR_ARG, "null output pointer");
    *bytes = tree_partials_bytes(plan, tree_shape(plan, groups, tokens, t));
    return FFA_OK;
}

int ffa_tree_attention(ffa_plan_t* plan, const void* q, const void* k, const void* v, void* k_cache, void* v_cache,
                       const unsigned char* tree, int tree_per_sample, int groups, int tokens, void* out, float softmax_scale, int t,
                       const int* seq_lengths, int right_or_no_padding, const int* page_table, int max_pages, int page_rows, int pool_pages,
                       void* scratch, size_t scratch_bytes, void* stream)
{
    int r = check_sizes(plan, groups, tokens, t);
    if (r != FFA_OK) return r;
    if (!q || !k || !v || !k_cache || !v_cache || !tree || !out) return ffa_fail(FFA_ERR_ARG, "null tensor pointer");
    if (!ffa_aligned16(q) || !ffa_aligned16(k) || !ffa_aligned16(v) || !ffa_aligned16(k_cache) || !ffa_aligned16(v_cache) || !ffa_aligned16(out))
        return ffa_fail(FFA_ERR_ARG, "tensor pointers must be 16-byte aligned");
    if (!std::isfinite(softmax_scale)) return ffa_fail(FFA_ERR_RANGE, "softmax_scale is not finite");
    if (seq_lengths == nullptr && !right_or_no_padding)
        return ffa_fail(FFA_ERR_ARG, "left padding (right_or_no_padding = 0) needs seq_lengths");
    if ((seq_lengths == nullptr || !right_or_no_padding) && tokens > plan->Lmax - t)
        return ffa_fail(FFA_ERR_RANGE, "t + tokens (%d + %d) exceeds the cache length %d", t, tokens, plan->Lmax);
    r = check_pages(plan, page_table, max_pages, page_rows, pool_pages);
    if (r != FFA_OK) return r;
    if (plan->offline) return ffa_fail(FFA_ERR_ARG, "this plan was created offline (planning only) and cannot launch");
    if (plan->ws == nullptr) return ffa_fail(FFA_ERR_WORKSPACE, "no workspace bound (ffa_workspace_bind)");
    const FfaTreeShape s = tree_shape(plan, groups, tokens, t);
    const size_t need = tree_partials_bytes(plan, s);
    if (need > 0 && (scratch == nullptr || scratch_bytes < need))
        return ffa_fail(FFA_ERR_WORKSPACE, "scratch of %zu bytes, need %zu (ffa_tree_scratch_bytes)", scratch ? scratch_bytes : (size_t)0, need);
    if (need > 0 && !ffa_aligned16(scratch)) return ffa_fail(FFA_ERR_ARG, "scratch must be 16-byte aligned");
    if ((long long)plan->B * plan->H * s.row_tiles * s.splits >= (1LL << 31)) return ffa_fail(FFA_ERR_RANGE, "sizes exceed int range");
    FfaTreeParams P;
    std::memset(&P, 0, sizeof(P));
    P.q = q, P.k = k, P.v = v, P.k_cache = k_cache, P.v_cache = v_cache, P.out = out;
    P.tree = tree, P.tree_per_sample = tree_per_sample != 0;
    P.seq_lengths = seq_lengths, P.right_or_no_padding = right_or_no_padding != 0;
    P.B = plan->B, P.H = plan->H, P.Lmax = plan->Lmax, P.t = t, P.groups = groups, P.tokens = tokens;
    P.scale = softmax_scale;
    P.splits = s.splits, P.row_tiles = s.row_tiles, P.part_rows = s.part_rows, P.tile_rows = s.tile_rows;
    P.partials = static_cast<float*>(scratch), P.status = plan->status;
    P.page_table = page_table, P.max_pages = max_pages, P.page_rows = page_rows, P.pool_pages = pool_pages;
    r = ffa_k_tree_attention(plan->dtype, plan->Dh, P, static_cast<cudaStream_t>(stream));
    if (r != 0) return ffa_cuda_fail(r, "tree attention launch");
    ffa_count_launches(s.splits > 1 ? 2 : 1);
    return FFA_OK;
}

int ffa_tree_accept(ffa_plan_t* plan, void* k_cache, void* v_cache, const int* path, int path_len, int t, const int* seq_lengths,
                    const int* page_table, int max_pages, int page_rows, int pool_pages, void* stream)
{
    if (plan == nullptr) return ffa_fail(FFA_ERR_ARG, "null plan");
    if (path_len < 0 || path_len > kTreeMaxRows) return ffa_fail(FFA_ERR_RANGE, "path length %d outside [0, %d]", path_len, kTreeMaxRows);
    if (t < 0 || t >= plan->Lmax) return ffa_fail(FFA_ERR_RANGE, "t = %d outside [0, %d)", t, plan->Lmax);
    if (!k_cache || !v_cache || (path_len > 0 && !path)) return ffa_fail(FFA_ERR_ARG, "null tensor pointer");
    if (!ffa_aligned16(k_cache) || !ffa_aligned16(v_cache)) return ffa_fail(FFA_ERR_ARG, "tensor pointers must be 16-byte aligned");
    int r = check_pages(plan, page_table, max_pages, page_rows, pool_pages);
    if (r != FFA_OK) return r;
    if (plan->offline) return ffa_fail(FFA_ERR_ARG, "this plan was created offline (planning only) and cannot launch");
    if (plan->ws == nullptr) return ffa_fail(FFA_ERR_WORKSPACE, "no workspace bound (ffa_workspace_bind)");
    if (path_len == 0) return FFA_OK;
    FfaAcceptParams P;
    std::memset(&P, 0, sizeof(P));
    P.k_cache = k_cache, P.v_cache = v_cache, P.path = path, P.seq_lengths = seq_lengths, P.path_len = path_len;
    P.B = plan->B, P.H = plan->H, P.Lmax = plan->Lmax, P.t = t, P.row_bytes = plan->Dh * ffa_elem_size(plan->dtype);
    P.status = plan->status;
    P.page_table = page_table, P.max_pages = max_pages, P.page_rows = page_rows, P.pool_pages = pool_pages;
    r = ffa_k_tree_accept(P, static_cast<cudaStream_t>(stream));
    if (r != 0) return ffa_cuda_fail(r, "tree accept launch");
    ffa_count_launches(1);
    return FFA_OK;
}

}  // extern "C"
