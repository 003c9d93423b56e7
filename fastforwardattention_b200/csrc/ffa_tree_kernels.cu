// Launch glue of the tree attention kernels (ffa_tree_kernel.cuh).
#include "ffa_tree_kernel.cuh"

#include "ffa_internal.h"
#include "ffa_launch.cuh"

using namespace ffa_dev;

namespace {

// query rows per warp: a pair with at most 8 rows takes one per warp (eight times the CTA's warps share the tile's keys among
// fewer rows otherwise)
constexpr int kManyRows = 4;

template <typename T, int DH, typename F>
int with_rows(int rows, F&& f)
{
    return rows <= kTreeWarps ? f(ffa_tree_simt_kernel<T, DH, 1>) : f(ffa_tree_simt_kernel<T, DH, kManyRows>);
}

}  // namespace

int ffa_k_tree_rows(int dtype, int rows)
{
    (void)dtype;
    return rows <= kTreeWarps ? kTreeWarps : kTreeWarps * kManyRows;
}

int ffa_k_tree_smem(int dtype, int head_dim, int rows)
{
    const int rowb = head_dim * (dtype == 0 ? 4 : 2);
    return ffa_k_tree_rows(dtype, rows) * head_dim * 4 + 4 * kTreeKeys * (rowb + 16);
}

int ffa_k_tree_prepare(int dtype, int head_dim)
{
    return dispatch(dtype, head_dim, [&](auto t, auto dh) -> int {
        using T = decltype(t);
        constexpr int DH = decltype(dh)::value;
        for (int rows : {1, kTreeMaxRows}) {
            const int e = with_rows<T, DH>(rows, [&](auto kernel) {
                return (int)cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 ffa_k_tree_smem(dtype, DH, rows));
            });
            if (e != 0) return e;
        }
        return 0;
    });
}

int ffa_k_tree_attention(int dtype, int head_dim, const FfaTreeParams& P, cudaStream_t stream)
{
    return dispatch(dtype, head_dim, [&](auto t, auto dh) -> int {
        using T = decltype(t);
        constexpr int DH = decltype(dh)::value;
        const int rows = P.groups * P.tokens;
        const int grid = P.B * P.H * P.row_tiles * P.splits;
        return with_rows<T, DH>(rows, [&](auto kernel) {
            return (int)launch_pdl(kernel, grid, kTreeThreads, ffa_k_tree_smem(dtype, DH, rows), 0, true, stream, P);
        });
    });
}

int ffa_k_tree_accept(const FfaAcceptParams& P, cudaStream_t stream)
{
    const int threads = (2 * P.row_bytes / 16 + 31) / 32 * 32;
    ffa_tree_accept_kernel<<<(unsigned)(P.B * P.H), threads, 0, stream>>>(P);
    return (int)cudaGetLastError();
}
