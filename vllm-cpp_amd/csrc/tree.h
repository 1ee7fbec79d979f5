// tree.h -- internal launch interface of the draft-tree attention and of the
// accumulated attention weights (tree.hip, mass.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vcpp_attention.h"

namespace vcpp {

// Most nodes of one tree (four 64-bit mask words).
constexpr int kMaxTreeNodes = 256;

struct TreeParams {
    // KV pages (see vcpp_kv_pages)
    const void* k;
    const void* v;
    const uint16_t* k_scale;
    const uint16_t* v_scale;
    int64_t num_blocks;
    int64_t block_stride;
    int64_t scale_block_stride;
    int32_t block_size;
    int32_t num_kv_heads;
    int32_t head_dim;
    int32_t kv_dtype;
    // queries (fp16 [rows][num_heads][head_dim])
    const uint16_t* q;
    int32_t num_heads;
    int32_t group;  // num_heads / num_kv_heads
    // sequences
    const int32_t* block_tables;  // [num_seqs][max_blocks]
    const int32_t* q_start;       // [num_seqs + 1]
    const int32_t* prefix_lens;   // [num_seqs]
    const uint64_t* mask;         // [rows][mask_words], NULL: a chain
    int32_t mask_words;
    int32_t max_blocks;
    int32_t num_seqs;
    int32_t max_nodes;
    int32_t max_len;   // max_prefix_len + max_nodes: positions at or past it are not attended
    float scale_log2;  // log2(e) / sqrt(head_dim)
    uint64_t bs_magic; // ceil(2^40 / block_size): pos / block_size = (pos * bs_magic) >> 40
    // attention: fp32 outputs, and each row's log-sum-exp (NULL: none)
    float* out;
    float* lse;
    // Key split (attention): the units (sequence, row tile), each as long as its
    // key blocks, are cut into `ranges` equal ranges (TreeRanges).
    int32_t ranges;
    int32_t table_cap; // 16-position tiles of a range's longest piece
    int64_t rows_cap;  // num_seqs * max_nodes
    float* ws_o;       // [ranges][2][num_kv_heads][tile rows][head_dim]
    float2* ws_ml;     // [ranges][2][num_kv_heads][tile rows] (exponent in log2 units, sum)
    // Position split (weights): parts of part_len positions.
    int32_t part_len;
    int32_t parts;
    int32_t head_waves;  // kv heads of a workgroup where a head has at most kMassOneRows rows (divides num_kv_heads)
    // weights: each row's log-sum-exp and the sums [num_seqs][num_kv_heads][score_stride]
    const float* lse_in;
    float* scores;
    int64_t score_stride;
};

// Key blocks (32 positions) of a range, at least: a call that has fewer is cut
// into fewer ranges.
constexpr int kTreeMinBlocks = 4;
// Rows of a kv head up to which a wave of the weights' kernel keeps them in registers.
constexpr int kMassOneRows = 16;
// Rows (node, head of the group) of one workgroup for trees of `rows` rows.
int tree_tile_rows(int kv_dtype, int head_dim, int rows);
// Workgroups of that tile a CU holds at once.
int tree_wgs_per_cu(int kv_dtype, int head_dim, int rows);
hipError_t launch_tree(const TreeParams& p, hipStream_t stream);
hipError_t launch_mass(const TreeParams& p, hipStream_t stream);

}  // namespace vcpp
