// Launch glue of the tree attention: fp16 and bf16 on the tensor cores (ffa_tree_umma_kernel.cuh), fp32 on the CUDA cores
// (ffa_tree_kernel.cuh; the tensor cores round fp32 operands to tf32, and products of operands split into several such parts were not tried), and
// the acceptance of a path.
#include "ffa_tree_kernel.cuh"
#include "ffa_tree_umma_kernel.cuh"

#include "ffa_internal.h"
#include "ffa_launch.cuh"

using namespace ffa_dev;

namespace {

// fp32: the kernel whose warps own keys takes up to 16 query rows (its buffers and results would not fit at head_dim 256), the one
// whose threads own rows the others, with as few rows per thread (16 threads deep) as hold all, at most four
bool simt_few(int head_dim, int rows) { return head_dim <= 128 && rows <= 16; }
int simt_rt(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
template <int DH, typename F>
int with_rows(int rows, F&& f)
{
    if constexpr (DH <= 128) {
        if (simt_few(DH, rows)) return rows <= 8 ? f(ffa_tree_few_kernel<DH, 1>) : f(ffa_tree_few_kernel<DH, 2>);
    } else if (simt_rt(rows) == 1) {
        return f(ffa_tree_simt_kernel<DH, 1>);
    }
    return simt_rt(rows) <= 2 ? f(ffa_tree_simt_kernel<DH, 2>) : f(ffa_tree_simt_kernel<DH, 4>);
}
constexpr int kSmemPerSm = 228 * 1024;
int simt_smem(int head_dim, int rows)
{
    if (simt_few(head_dim, rows)) return few_smem(head_dim, rows <= 8 ? 1 : 2);
    const int bm = 16 * simt_rt(rows);
    return 4 * (bm * head_dim + kTreeKeys * (head_dim + 4) + kTreeKeys * head_dim + kTreeKeys * bm);
}

template <typename T, int DH, typename F>
int with_copies(int tile_rows, F&& f)
{
    switch (umma_rep(tile_rows)) {
        case 4: return f(ffa_tree_umma_kernel<T, DH, 4>);
        case 2: return f(ffa_tree_umma_kernel<T, DH, 2>);
        default: return f(ffa_tree_umma_kernel<T, DH, 1>);
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the driver's encoder, looked up once (nothing here links against the driver library)
EncodeTiled encoder()
{
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// rows of head_dim 16-bit elements, in boxes of 64 columns (128 swizzled bytes) and box_rows rows; columns behind head_dim and rows
// behind `rows` read as zeros
int encode(CUtensorMap* map, int dtype, const void* base, int head_dim, long long rows, int box_rows)
{
    const cuuint64_t dims[2] = {(cuuint64_t)head_dim, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)head_dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    const CUresult r = encoder()(map, dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base),
                                 dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <typename F>
int dispatch16(int dtype, int head_dim, F&& f)
{
    return dispatch(dtype, head_dim, [&](auto t, auto dh) -> int {
        if constexpr (sizeof(decltype(t)) == 2) return f(t, dh);
        else return (int)cudaErrorInvalidValue;
    });
}
template <typename F>
int dispatch32(int head_dim, F&& f)
{
    return dispatch(0, head_dim, [&](auto t, auto dh) -> int {
        if constexpr (sizeof(decltype(t)) == 4) return f(dh);
        else return (int)cudaErrorInvalidValue;
    });
}

template <typename T, int DH>
int merge(const FfaTreeParams& P, cudaStream_t stream)
{
    const long long rows = (long long)P.B * P.H * P.groups * P.tokens;
    return (int)launch_pdl(ffa_tree_merge_kernel<T, DH, sizeof(T) == 2>, (int)((rows + kMergeWarps - 1) / kMergeWarps), 32 * kMergeWarps, 0, 0, true, stream,
                           P);
}

}  // namespace

void ffa_k_tree_shape(int dtype, int head_dim, int rows, FfaTreeShape* s)
{
    if (dtype == 0) {
        const bool few = simt_few(head_dim, rows);
        s->tile_rows = few ? (rows <= 8 ? 8 : 16) : 16 * simt_rt(rows), s->tile_keys = kTreeKeys;
        const int fit = kSmemPerSm / (simt_smem(head_dim, rows) + 1024);
        // by registers: 168 and 255 a thread of 128; of 256 threads Dh 64 has 75 a thread with two rows to a thread and 134 with four (the
        // other head sizes: shared memory is the tighter limit, or the same)
        const int most = few ? (rows <= 8 ? 3 : 2) : head_dim == 64 ? (simt_rt(rows) == 4 ? 1 : 3) : 4;
        s->ctas_per_sm = fit > most ? most : fit;
        // S and O of a tile: 4 * rows * keys * Dh flops at about 55 % of an SM's 128 FMAs a cycle (30 % with a warp a scheduler), and two
        // memory latencies
        s->tile_us = 0.6 + 4.0 * s->tile_rows * kTreeKeys * head_dim / (2 * 128 * (few ? 0.3 : 0.55) * 1900);
    } else {
        const int tiles = (rows + kUmmaRows - 1) / kUmmaRows;   // of about equal height
        s->tile_rows = (rows + tiles - 1) / tiles, s->tile_keys = kUmmaKeys, s->ctas_per_sm = umma_ctas_per_sm(head_dim);
        // measured, one CTA to an SM: the chain S - softmax - O per tile, longer for Dh 256 by its products
        s->tile_us = head_dim > 128 ? 1.5 : umma_rep(s->tile_rows) == 1 ? 0.9 : 0.75;
    }
    s->row_tiles = (rows + s->tile_rows - 1) / s->tile_rows;
    s->part_rows = rows < s->tile_rows ? rows : s->tile_rows;
}

int ffa_k_tree_prepare(int dtype, int head_dim)
{
    if (dtype == 0)
        return dispatch32(head_dim, [&](auto dh) -> int {
            constexpr int DH = decltype(dh)::value;
            for (int rows : {8, 16, 32, 64}) {
                const int e = with_rows<DH>(rows, [&](auto kernel) {
                    return (int)cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, simt_smem(DH, rows));
                });
                if (e != 0) return e;
            }
            return 0;
        });
    if (encoder() == nullptr) return (int)cudaErrorNotSupported;
    return dispatch16(dtype, head_dim, [&](auto t, auto dh) -> int {
        using T = decltype(t);
        constexpr int DH = decltype(dh)::value;
        for (int rows : {32, 64, 128}) {
            const int e = with_copies<T, DH>(rows, [&](auto kernel) {
                return (int)cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, umma_smem(DH));
            });
            if (e != 0) return e;
        }
        return 0;
    });
}

int ffa_k_tree_attention(int dtype, int head_dim, const FfaTreeParams& P, cudaStream_t stream)
{
    const int rows = P.groups * P.tokens;
    const int grid = P.B * P.H * P.row_tiles * P.splits;
    if (dtype == 0)
        return dispatch32(head_dim, [&](auto dh) -> int {
            constexpr int DH = decltype(dh)::value;
            const int e = with_rows<DH>(rows, [&](auto kernel) { return (int)launch_pdl(kernel, grid, simt_few(DH, rows) ? 32 * kFewWarps : kTreeThreads, simt_smem(DH, rows), 0, true, stream, P); });
            return e != 0 || P.splits == 1 ? e : merge<float, DH>(P, stream);
        });
    FfaTreeUmmaParams U;
    U.p = P;
    const long long pairs = (long long)P.B * P.H;
    const long long cache_rows = P.page_table != nullptr ? (long long)P.pool_pages * P.H * P.page_rows : pairs * P.Lmax;
    int e = encode(&U.q, dtype, P.q, head_dim, pairs * rows, kQBoxRows);
    if (e == 0) e = encode(&U.k_new, dtype, P.k, head_dim, pairs * P.tokens, kUmmaKeys);
    if (e == 0) e = encode(&U.v_new, dtype, P.v, head_dim, pairs * P.tokens, kUmmaKeys);
    if (e == 0) e = encode(&U.k_cache, dtype, P.k_cache, head_dim, cache_rows, kUmmaKeys);
    if (e == 0) e = encode(&U.v_cache, dtype, P.v_cache, head_dim, cache_rows, kUmmaKeys);
    if (e != 0) return e;
    return dispatch16(dtype, head_dim, [&](auto t, auto dh) -> int {
        using T = decltype(t);
        constexpr int DH = decltype(dh)::value;
        const int r = with_copies<T, DH>(P.tile_rows, [&](auto kernel) {
            return (int)launch_pdl(kernel, grid, kUmmaThreads, umma_smem(DH), 0, true, stream, U);
        });
        return r != 0 || P.splits == 1 ? r : merge<T, DH>(P, stream);
    });
}

int ffa_k_tree_accept(const FfaAcceptParams& P, cudaStream_t stream)
{
    const int threads = (2 * P.row_bytes / 16 + 31) / 32 * 32;
    return (int)launch_pdl(ffa_tree_accept_kernel, P.B * P.H, threads, 0, 0, true, stream, P);
}
