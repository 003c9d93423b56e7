// The plan behind the C ABI's opaque ffa_plan_t, and the helpers that the translation units with C entries share.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "../../include/ffa_c_api.h"
#include "ffa_internal.h"

struct ffa_plan {
    int dtype, B, H, Dh, Lmax, use_default, device, mode;
    int prune_path;  // 0 = choose, 1 = fused cluster kernel only, 2 = streaming kernel only
    bool accumulating;  // the call being planned is an accumulating step (ffa_attention_accumulate)
    int cluster_merge;  // 1 = merge split pairs inside a thread-block cluster when the cut allows it
    // answers of the occupancy query for cluster launches, keyed by (threads, shared memory, cluster size)
    struct { int threads, smem, cluster, clusters; } occ[8];
    int occ_n;
    bool offline;    // planning only: created from given device properties, never launches
    int sms, smem_per_cta, smem_per_sm;
    bool forced;
    ffa_launch_t force;
    // workspace carving
    void* ws;
    size_t ws_bytes;
    int* status;
    int* tickets;
    float* partials;
    float* scores;
    int max_grid;
    // output gather over peer memory
    int peer_world, peer_rank;
    void* peer_buf[FFA_MAX_PEERS];
    void* push_gathered;   // non-null: exact steps push their output rows to the peers (ffa_peer_push_target)
};

// Defined in ffa_c_api.cu: record the reason for a non-zero return (ffa_last_error) and return `code`; count a launch.
int ffa_fail(int code, const char* fmt, ...);
int ffa_cuda_fail(int cuda_error, const char* what);
void ffa_count_launches(int n);

inline int ffa_elem_size(int dtype) { return dtype == FFA_DTYPE_F32 ? 4 : 2; }
inline bool ffa_dtype_ok(int dtype) { return dtype == FFA_DTYPE_F32 || dtype == FFA_DTYPE_F16 || dtype == FFA_DTYPE_BF16; }
inline bool ffa_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t ffa_align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
