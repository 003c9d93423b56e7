// C entries of eviction by accumulated attention weight and of beam search (include/ffa_c_api.h): argument checks and parameter
// fill.  (The accumulating decode step shares the decode steps' planner: ffa_attention_accumulate is in ffa_c_api.cu.)
#include <cuda_runtime.h>

#include <cstring>

#include "../../include/ffa_c_api.h"
#include "ffa_internal.h"
#include "ffa_plan.h"

namespace {

// rows a pair may have for ffa_evict: its bits and ranks (8 bytes per 32 rows) live in shared memory
constexpr int kMaxEvictRows = 1 << 19;

}  // namespace

extern "C" {

int ffa_evict(ffa_plan_t* plan, void* k_cache, void* v_cache, float* weights, int* positions, const int* rows, int max_rows, int keep,
              int recent, int first, int* kept, void* stream)
{
    if (plan == nullptr) return ffa_fail(FFA_ERR_ARG, "null plan");
    if (!k_cache || !v_cache || !weights || !positions || !rows || !kept) return ffa_fail(FFA_ERR_ARG, "null tensor pointer");
    if (!ffa_aligned16(k_cache) || !ffa_aligned16(v_cache)) return ffa_fail(FFA_ERR_ARG, "cache pointers must be 16-byte aligned");
    if (max_rows < 0 || max_rows > plan->Lmax) return ffa_fail(FFA_ERR_RANGE, "max_rows = %d outside [0, %d]", max_rows, plan->Lmax);
    if (max_rows > kMaxEvictRows) return ffa_fail(FFA_ERR_RANGE, "max_rows = %d exceeds the %d rows that one selection holds", max_rows, kMaxEvictRows);
    if (keep <= 0 || keep > plan->Lmax) return ffa_fail(FFA_ERR_RANGE, "keep = %d outside [1, %d]", keep, plan->Lmax);
    if (recent < 0 || first < 0 || (long long)recent + first > keep)
        return ffa_fail(FFA_ERR_RANGE, "need 0 <= recent (%d), 0 <= first (%d), recent + first <= keep (%d)", recent, first, keep);
    if (plan->offline) return ffa_fail(FFA_ERR_ARG, "this plan was created offline (planning only) and cannot launch");
    if (plan->ws == nullptr) return ffa_fail(FFA_ERR_WORKSPACE, "no workspace bound (ffa_workspace_bind)");
    if ((long long)plan->B * plan->H * ((keep + 31) / 32) >= (1LL << 31)) return ffa_fail(FFA_ERR_RANGE, "sizes exceed int range");
    FfaEvictParams P;
    std::memset(&P, 0, sizeof(P));
    P.k_cache = k_cache, P.v_cache = v_cache, P.weights = weights, P.positions = positions, P.rows = rows, P.kept = kept;
    P.B = plan->B, P.H = plan->H, P.Lmax = plan->Lmax, P.max_rows = max_rows, P.keep = keep, P.recent = recent, P.first = first;
    P.row_bytes = plan->Dh * ffa_elem_size(plan->dtype), P.status = plan->status;
    const int r = ffa_k_evict(P, static_cast<cudaStream_t>(stream));
    if (r != 0) return ffa_cuda_fail(r, "eviction launch");
    ffa_count_launches(max_rows > keep + 1 ? 2 : 1);
    return FFA_OK;
}

int ffa_beam_select(int dtype, int batch, int beams, int vocab, long long row_stride, const void* logits, const float* scores,
                    const unsigned char* finished, int pad_token, int num, float* out_scores, int* out_parents, int* out_tokens, void* stream)
{
    if (!ffa_dtype_ok(dtype)) return ffa_fail(FFA_ERR_DTYPE, "unsupported dtype code %d", dtype);
    if (batch <= 0 || vocab <= 0) return ffa_fail(FFA_ERR_RANGE, "batch and vocab must be positive");
    if (beams <= 0 || beams > kMaxBeams) return ffa_fail(FFA_ERR_RANGE, "beams = %d outside [1, %d]", beams, kMaxBeams);
    if (num <= 0 || num > kMaxBeamCandidates) return ffa_fail(FFA_ERR_RANGE, "num = %d outside [1, %d]", num, kMaxBeamCandidates);
    if ((long long)beams * vocab >= (1LL << 31) || batch > (1 << 27)) return ffa_fail(FFA_ERR_RANGE, "sizes exceed int range");
    if (row_stride < vocab) return ffa_fail(FFA_ERR_RANGE, "row stride %lld is smaller than the vocabulary (%d)", row_stride, vocab);
    if (pad_token < 0 || pad_token >= vocab) return ffa_fail(FFA_ERR_RANGE, "pad_token = %d outside [0, %d)", pad_token, vocab);
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return ffa_fail(FFA_ERR_ARG, "null tensor pointer");
    if (reinterpret_cast<uintptr_t>(logits) % ffa_elem_size(dtype) != 0) return ffa_fail(FFA_ERR_ARG, "logits must be aligned to its element type");
    FfaBeamParams P;
    std::memset(&P, 0, sizeof(P));
    P.logits = logits, P.scores = scores, P.finished = finished;
    P.out_scores = out_scores, P.out_parents = out_parents, P.out_tokens = out_tokens;
    P.row_stride = row_stride, P.batch = batch, P.beams = beams, P.vocab = vocab, P.num = num, P.pad_token = pad_token;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return ffa_cuda_fail(e, "device query");
    const int r = ffa_k_beam_select(dtype, P, sms, static_cast<cudaStream_t>(stream));
    if (r != 0) return ffa_cuda_fail(r, "beam selection launch");
    ffa_count_launches(1);
    return FFA_OK;
}

int ffa_cache_reorder(ffa_plan_t* plan, void* k_cache, void* v_cache, const int* parents, int beams, int first_row, int rows, void* stream)
{
    if (plan == nullptr) return ffa_fail(FFA_ERR_ARG, "null plan");
    if (!k_cache || !v_cache || !parents) return ffa_fail(FFA_ERR_ARG, "null tensor pointer");
    if (!ffa_aligned16(k_cache) || !ffa_aligned16(v_cache)) return ffa_fail(FFA_ERR_ARG, "cache pointers must be 16-byte aligned");
    if (beams <= 0 || beams > kMaxBeams) return ffa_fail(FFA_ERR_RANGE, "beams = %d outside [1, %d]", beams, kMaxBeams);
    if (plan->B % beams != 0) return ffa_fail(FFA_ERR_RANGE, "the batch (%d) is not a multiple of beams (%d)", plan->B, beams);
    if (first_row < 0 || rows < first_row || rows > plan->Lmax)
        return ffa_fail(FFA_ERR_RANGE, "need 0 <= first_row (%d) <= rows (%d) <= %d", first_row, rows, plan->Lmax);
    if (plan->offline) return ffa_fail(FFA_ERR_ARG, "this plan was created offline (planning only) and cannot launch");
    if (plan->ws == nullptr) return ffa_fail(FFA_ERR_WORKSPACE, "no workspace bound (ffa_workspace_bind)");
    if ((long long)plan->B * plan->H >= (1LL << 24)) return ffa_fail(FFA_ERR_RANGE, "sizes exceed int range");
    if (first_row == rows) return FFA_OK;
    FfaReorderParams P;
    std::memset(&P, 0, sizeof(P));
    P.k_cache = k_cache, P.v_cache = v_cache, P.parents = parents;
    P.groups = plan->B / beams, P.beams = beams, P.H = plan->H, P.Lmax = plan->Lmax, P.first = first_row, P.rows = rows;
    P.row_bytes = plan->Dh * ffa_elem_size(plan->dtype), P.status = plan->status;
    const int r = ffa_k_reorder(P, plan->sms, static_cast<cudaStream_t>(stream));
    if (r != 0) return ffa_cuda_fail(r, "cache reorder launch");
    ffa_count_launches(1);
    return FFA_OK;
}

}  // extern "C"
