// What the host side of the attention (hnsw_attend.hip) and its kernels (hnsw_attend_kernels.h, built once for each row type) share.
#pragma once
#include "hnsw_cache.h"

namespace hnsw_amd {

struct AttendArgs {
    const uint8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    uint32_t n_blocks, n_heads, block_tokens, dim;
    const void* q;
    int64_t q_row_stride, q_head_stride;
    uint32_t n_rows, q_heads;
    const int32_t *table, *lens, *cu_q, *ids;
    uint32_t width, n_requests, n_ids, id_heads;
    int32_t causal, found;      // found: over the listed tokens `ids`
    float scale;
    void* out;
    float* lse;
    uint32_t group, lists;      // query heads that share a key head (a list), and lists that share a key head
    float group_inverse;
};

struct Partials {
    float* out;        // [n_rows][q_heads][n_splits][dim], divided by the split's sum
    float* lse;        // [n_rows][q_heads][n_splits], in base 2
    uint32_t n_splits, chunk;
};

constexpr uint32_t kTile = 32;            // tokens a wavefront takes at a time

// How a call's work is cut: units (rows) x heads x chunks of the items (tokens, or list entries).
struct Cut {
    bool tiles;                // through LDS tiles (attend_tile_kernel), or each wavefront by itself (attend_rows_kernel)
    uint32_t mt, waves;        // 16-row tiles of a wavefront, wavefronts of a workgroup
    uint32_t units, heads, chunk, n_splits;
};

// Launches the kernels of a call (arguments checked, device selected).
template <class T> void launch_attend(const AttendArgs& a, const Cut& cut, uint32_t codes, float* workspace, hipStream_t stream);

}  // namespace hnsw_amd
