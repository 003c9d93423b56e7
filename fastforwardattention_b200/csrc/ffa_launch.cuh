// Host-side helpers of the translation units that launch kernels: the switch over element type and head dimension, and the
// launch with programmatic overlap and thread-block clusters.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>
#include <type_traits>

namespace {

template <typename F>
int dispatch(int dtype, int head_dim, F&& f)
{
#define FFA_DH_SWITCH(T)                                        \
    switch (head_dim) {                                         \
        case 64: return f(T{}, std::integral_constant<int, 64>{});   \
        case 80: return f(T{}, std::integral_constant<int, 80>{});   \
        case 128: return f(T{}, std::integral_constant<int, 128>{}); \
        case 256: return f(T{}, std::integral_constant<int, 256>{}); \
        default: return (int)cudaErrorInvalidValue;             \
    }
    switch (dtype) {
        case 0: FFA_DH_SWITCH(float)
        case 1: FFA_DH_SWITCH(__half)
        case 2: FFA_DH_SWITCH(__nv_bfloat16)
        default: return (int)cudaErrorInvalidValue;
    }
#undef FFA_DH_SWITCH
}

// Launch -- when `overlap`, with the programmatic-serialisation attribute: the kernel may start while the previous
// kernel of the stream drains and waits at pdl_wait() before touching global memory -- and, when cluster > 1, as
// thread-block clusters of that many CTAs.
template <typename K, typename Params>
cudaError_t launch_pdl(K kernel, int grid, int threads, int smem, int cluster, bool overlap, cudaStream_t stream, const Params& P)
{
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (overlap) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)cluster, attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr, cfg.numAttrs = (unsigned)n;
    return cudaLaunchKernelEx(&cfg, kernel, P);
}

}  // namespace
