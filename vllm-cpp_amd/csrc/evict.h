// evict.h -- internal launch interface of the eviction plan and of the row
// moves inside the pages (evict.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vcpp_attention.h"

namespace vcpp {

struct EvictPlanParams {
    const float* scores;       // [num_seqs][num_kv_heads][stride]
    const int32_t* positions;  // the same shape, or NULL
    const int32_t* context_lens;
    const int32_t* seen_lens;  // NULL: context_lens
    int64_t stride;
    int32_t num_seqs;
    int32_t num_kv_heads;
    int32_t max_len;
    int32_t budget;
    int32_t keep_first;
    int32_t keep_last;
    int32_t max_moves;
    int2* moves;               // [num_seqs][num_kv_heads][max_moves] (to, from)
    int32_t* move_counts;      // [num_seqs][num_kv_heads]
    int32_t* new_lens;         // [num_seqs]
    float* scores_out;
    int32_t* positions_out;    // NULL: none
};

// Rows moved inside the pages of one layer (evict) or of all layers (commit).
struct RowMoveParams {
    char* k;
    char* v;
    uint16_t* k_scale;
    uint16_t* v_scale;
    int64_t num_blocks;
    int64_t block_bytes;        // of a K (or V) page's stride
    int64_t layer_bytes;        // from one layer's pages to the next's
    int64_t scale_block_stride; // elements
    int64_t scale_layer_stride;
    int32_t block_size;
    int32_t num_kv_heads;
    int32_t row_bytes;          // of one head's row
    int32_t scaled;             // int8 pages
    int32_t num_layers;
    const int32_t* block_tables;
    int32_t max_blocks;
    int32_t num_seqs;
    // evict
    const int2* moves;          // [num_seqs][num_kv_heads][max_moves]
    const int32_t* move_counts;
    int32_t max_moves;
    // commit
    const int32_t* prefix_lens;
    const int32_t* accepted;    // [num_seqs][max_accepted]
    const int32_t* accept_lens;
    int32_t max_accepted;
    int32_t max_nodes;
};

hipError_t launch_evict_plan(const EvictPlanParams& p, hipStream_t stream);
hipError_t launch_evict_apply(const RowMoveParams& p, hipStream_t stream);
hipError_t launch_commit(const RowMoveParams& p, hipStream_t stream);

}  // namespace vcpp
