// api_tree.cpp -- extern "C" entry points of drafted decoding and of the
// bounded cache (include/vcpp_attention.h): argument checks, the key split's
// size and launch parameters.  Kernels: tree.hip, mass.hip, evict.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "evict.h"
#include "tree.h"
#include "vcpp_attention.h"

namespace vcpp {
// api.cpp
int record_error(int code, const char* msg);
int check_kv_pages(const vcpp_kv_pages* kv);
void clear_error();
int compute_units();
}  // namespace vcpp

namespace {

static_assert(vcpp::kMaxTreeNodes == VCPP_MAX_TREE_NODES, "tree size");

// Longest context of these calls: pos / block_size as a product (tree.h) stays
// below 2^63.
constexpr int64_t kMaxLen = 1 << 24;

int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return vcpp::record_error(code, buf);
}

int hip_fail(hipError_t e, const char* what) { return fail(VCPP_E_HIP, "%s: %s", what, hipGetErrorString(e)); }

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Cut of a tree call (TreeRanges) and the partials' place in the workspace.
struct TreeSplit {
    int64_t blocks;  // of one sequence's row tiles
    int32_t ranges, table_cap;
    size_t off_ml, bytes;
};

// Ranges: one per workgroup (and kv head) that the GPU holds at once, fewer
// where the bounds allow fewer than kTreeMinBlocks blocks each, more where a
// range's tile table in LDS would pass kMaxRange blocks (8 or 16 KB).
constexpr int64_t kMaxRange = 512;

TreeSplit tree_split(const vcpp_kv_pages* kv, int32_t num_seqs, int32_t max_nodes, int32_t max_prefix_len,
                     int32_t num_heads) {
    TreeSplit t{};
    const int rows = max_nodes * (num_heads / kv->num_kv_heads);
    const int tile = vcpp::tree_tile_rows(kv->dtype, kv->head_dim, rows);
    const int64_t blocks = ((int64_t)max_prefix_len + max_nodes + 31) / 32;
    t.blocks = (rows + tile - 1) / tile * blocks;
    const int64_t most = num_seqs * t.blocks;  // upper bound of the axis
    const int64_t slots = (int64_t)vcpp::compute_units() * vcpp::tree_wgs_per_cu(kv->dtype, kv->head_dim, rows);
    int64_t R = std::min(std::max<int64_t>(1, slots / kv->num_kv_heads), std::max<int64_t>(1, most / vcpp::kTreeMinBlocks));
    // (a piece is no longer than its sequence, nor than its range)
    if (blocks > kMaxRange - 4) R = std::max(R, (most + kMaxRange - 5) / (kMaxRange - 4));
    t.ranges = (int32_t)std::min<int64_t>(R, INT32_MAX);
    const int64_t longest = std::min(blocks, std::max<int64_t>((most + R - 1) / R, 2 * vcpp::kTreeMinBlocks) + 1);
    t.table_cap = (int32_t)(2 * longest);
    if (t.ranges > 1) {
        const size_t n = (size_t)t.ranges * 2 * kv->num_kv_heads * tile;
        t.off_ml = align256(n * kv->head_dim * sizeof(float));
        t.bytes = t.off_ml + align256(n * sizeof(float2));
    }
    return t;
}

int check_tree(const vcpp_kv_pages* kv, const uint16_t* q, const int32_t* block_tables, int32_t max_blocks_per_seq,
               const int32_t* q_start, const int32_t* prefix_lens, const uint64_t* tree_mask, int32_t mask_words,
               int32_t num_seqs, int32_t max_nodes, int32_t max_prefix_len, int32_t num_heads) {
    const int rc = vcpp::check_kv_pages(kv);
    if (rc != VCPP_OK) return rc;
    if (kv->dtype == VCPP_KV_F32)
        return fail(VCPP_E_UNSUPPORTED, "tree attention supports fp16, int8 and fp8 pages (got fp32)");
    if (kv->head_dim != 64 && kv->head_dim != 80 && kv->head_dim != 128)
        return fail(VCPP_E_UNSUPPORTED, "tree attention head_dim %d (64, 80 or 128)", kv->head_dim);
    if (num_heads <= 0 || num_heads % kv->num_kv_heads != 0)
        return fail(VCPP_E_INVALID, "num_heads %d is not a positive multiple of num_kv_heads %d", num_heads,
                    kv->num_kv_heads);
    if (num_seqs < 0 || max_nodes < 0 || max_prefix_len < 0)
        return fail(VCPP_E_INVALID, "num_seqs, max_nodes and max_prefix_len must be >= 0");
    if (max_nodes > VCPP_MAX_TREE_NODES)
        return fail(VCPP_E_UNSUPPORTED, "max_nodes %d exceeds %d", max_nodes, VCPP_MAX_TREE_NODES);
    if ((int64_t)max_prefix_len + max_nodes > kMaxLen)
        return fail(VCPP_E_UNSUPPORTED, "max_prefix_len %d too long", max_prefix_len);
    if (num_seqs == 0 || max_nodes == 0) return VCPP_OK;
    if (tree_mask && (mask_words <= 0 || mask_words * (int64_t)64 < max_nodes))
        return fail(VCPP_E_INVALID, "mask_words %d holds fewer than max_nodes %d bits", mask_words, max_nodes);
    if (!q || !q_start || !prefix_lens) return fail(VCPP_E_INVALID, "q/q_start/prefix_lens is NULL");
    if (reinterpret_cast<uintptr_t>(q) % 16 != 0) return fail(VCPP_E_INVALID, "q must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(tree_mask) % 8 != 0) return fail(VCPP_E_INVALID, "tree_mask must be 8-byte aligned");
    if (max_blocks_per_seq <= 0 || !block_tables) return fail(VCPP_E_INVALID, "block_tables missing");
    if ((int64_t)num_seqs * max_nodes > INT32_MAX || num_heads > 65535)
        return fail(VCPP_E_UNSUPPORTED, "too many rows or heads");
    return VCPP_OK;
}

vcpp::TreeParams tree_params(const vcpp_kv_pages* kv, const uint16_t* q, const int32_t* block_tables,
                             int32_t max_blocks_per_seq, const int32_t* q_start, const int32_t* prefix_lens,
                             const uint64_t* tree_mask, int32_t mask_words, int32_t num_seqs, int32_t max_nodes,
                             int32_t max_prefix_len, int32_t num_heads) {
    vcpp::TreeParams p{};
    p.k = kv->k;
    p.v = kv->v;
    p.k_scale = kv->k_scale;
    p.v_scale = kv->v_scale;
    p.num_blocks = kv->num_blocks;
    p.block_stride = kv->block_stride;
    p.scale_block_stride = kv->scale_block_stride;
    p.block_size = kv->block_size;
    p.num_kv_heads = kv->num_kv_heads;
    p.head_dim = kv->head_dim;
    p.kv_dtype = kv->dtype;
    p.q = q;
    p.num_heads = num_heads;
    p.group = num_heads / kv->num_kv_heads;
    p.block_tables = block_tables;
    p.q_start = q_start;
    p.prefix_lens = prefix_lens;
    p.mask = tree_mask;
    p.mask_words = mask_words;
    p.max_blocks = max_blocks_per_seq;
    p.num_seqs = num_seqs;
    p.max_nodes = max_nodes;
    p.max_len = max_prefix_len + max_nodes;
    p.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)kv->head_dim));
    p.bs_magic = ((1ull << 40) + kv->block_size - 1) / kv->block_size;
    p.rows_cap = (int64_t)num_seqs * max_nodes;
    return p;
}

// Workgroups of a grid whose cells (sequence, part) are dealt to the 8 XCDs.
bool grid_fits(int64_t cells, int64_t per_cell, int64_t threads) {
    return (cells + 7) / 8 * 8 * per_cell * threads < ((int64_t)1 << 31);
}

int move_params(const vcpp_kv_pages* kv, const int32_t* block_tables, int32_t max_blocks_per_seq, int32_t num_seqs,
                vcpp::RowMoveParams& p) {
    const int rc = vcpp::check_kv_pages(kv);
    if (rc != VCPP_OK) return rc;
    if (num_seqs < 0) return fail(VCPP_E_INVALID, "num_seqs must be >= 0");
    if (num_seqs > 0 && (max_blocks_per_seq <= 0 || !block_tables)) return fail(VCPP_E_INVALID, "block_tables missing");
    const int esize = kv->dtype == VCPP_KV_F32 ? 4 : kv->dtype == VCPP_KV_F16 ? 2 : 1;
    p.k = static_cast<char*>(const_cast<void*>(kv->k));
    p.v = static_cast<char*>(const_cast<void*>(kv->v));
    p.k_scale = const_cast<uint16_t*>(kv->k_scale);
    p.v_scale = const_cast<uint16_t*>(kv->v_scale);
    p.num_blocks = kv->num_blocks;
    p.block_bytes = kv->block_stride * esize;
    p.scale_block_stride = kv->scale_block_stride;
    p.block_size = kv->block_size;
    p.num_kv_heads = kv->num_kv_heads;
    p.row_bytes = kv->head_dim * esize;
    p.scaled = kv->dtype == VCPP_KV_I8;
    p.num_layers = 1;
    p.block_tables = block_tables;
    p.max_blocks = max_blocks_per_seq;
    p.num_seqs = num_seqs;
    return VCPP_OK;
}

}  // namespace

extern "C" {

size_t vcpp_tree_workspace_size(const vcpp_kv_pages* kv, int32_t num_seqs, int32_t max_nodes, int32_t max_prefix_len,
                                int32_t num_heads) {
    if (!kv || kv->num_kv_heads <= 0 || num_heads <= 0 || num_heads % kv->num_kv_heads != 0 || num_seqs <= 0 ||
        max_nodes <= 0 || max_nodes > VCPP_MAX_TREE_NODES || max_prefix_len < 0)
        return 0;
    return tree_split(kv, num_seqs, max_nodes, max_prefix_len, num_heads).bytes;
}

int vcpp_paged_tree_attention(const vcpp_kv_pages* kv, const uint16_t* q, float* out, float* lse,
                              const int32_t* block_tables, int32_t max_blocks_per_seq, const int32_t* q_start,
                              const int32_t* prefix_lens, const uint64_t* tree_mask, int32_t mask_words,
                              int32_t num_seqs, int32_t max_nodes, int32_t max_prefix_len, int32_t num_heads,
                              void* workspace, size_t workspace_bytes, void* stream) {
    vcpp::clear_error();
    const int rc = check_tree(kv, q, block_tables, max_blocks_per_seq, q_start, prefix_lens, tree_mask, mask_words,
                              num_seqs, max_nodes, max_prefix_len, num_heads);
    if (rc != VCPP_OK || num_seqs == 0 || max_nodes == 0) return rc;
    if (!out) return fail(VCPP_E_INVALID, "out is NULL");
    if (reinterpret_cast<uintptr_t>(out) % 16 != 0) return fail(VCPP_E_INVALID, "out must be 16-byte aligned");
    // (32-bit places: a row's byte offset in its 16-position tile, 27 bits, and
    // the key blocks of 64 sequences' row tiles)
    if ((int64_t)kv->num_kv_heads * kv->head_dim * (kv->dtype == VCPP_KV_F16 ? 2 : 1) > 1 << 23)
        return fail(VCPP_E_UNSUPPORTED, "too many kv heads (%d of %d dims)", kv->num_kv_heads, kv->head_dim);
    const TreeSplit t = tree_split(kv, num_seqs, max_nodes, max_prefix_len, num_heads);
    if (t.blocks * std::min(num_seqs, 64) > INT32_MAX)
        return fail(VCPP_E_UNSUPPORTED, "too many heads or positions for one launch");
    if (!grid_fits(t.ranges, kv->num_kv_heads, 256) || !grid_fits((int64_t)num_seqs * max_nodes, 1, 256))
        return fail(VCPP_E_UNSUPPORTED, "too many sequences, heads or positions for one launch");
    if (t.bytes > 0 && (!workspace || workspace_bytes < t.bytes))
        return fail(VCPP_E_WORKSPACE, "tree attention needs %zu workspace bytes, got %zu", t.bytes,
                    workspace ? workspace_bytes : (size_t)0);
    if (t.bytes > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(VCPP_E_INVALID, "workspace must be 16-byte aligned");
    vcpp::TreeParams p = tree_params(kv, q, block_tables, max_blocks_per_seq, q_start, prefix_lens, tree_mask,
                                     mask_words, num_seqs, max_nodes, max_prefix_len, num_heads);
    p.out = out;
    p.lse = lse;
    p.ranges = t.ranges;
    p.table_cap = t.table_cap;
    if (t.bytes > 0) {
        p.ws_o = static_cast<float*>(workspace);
        p.ws_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + t.off_ml);
    }
    const hipError_t e = vcpp::launch_tree(p, static_cast<hipStream_t>(stream));
    return e != hipSuccess ? hip_fail(e, "tree attention launch") : VCPP_OK;
}

int vcpp_attention_mass(const vcpp_kv_pages* kv, const uint16_t* q, const float* lse, float* scores,
                        int64_t score_stride, const int32_t* block_tables, int32_t max_blocks_per_seq,
                        const int32_t* q_start, const int32_t* prefix_lens, const uint64_t* tree_mask,
                        int32_t mask_words, int32_t num_seqs, int32_t max_nodes, int32_t max_prefix_len,
                        int32_t num_heads, void* stream) {
    vcpp::clear_error();
    const int rc = check_tree(kv, q, block_tables, max_blocks_per_seq, q_start, prefix_lens, tree_mask, mask_words,
                              num_seqs, max_nodes, max_prefix_len, num_heads);
    if (rc != VCPP_OK || num_seqs == 0 || max_nodes == 0) return rc;
    if (!lse || !scores) return fail(VCPP_E_INVALID, "lse/scores is NULL");
    if (score_stride < (int64_t)max_prefix_len + max_nodes)
        return fail(VCPP_E_INVALID, "score_stride %lld is below max_prefix_len + max_nodes", (long long)score_stride);
    vcpp::TreeParams p = tree_params(kv, q, block_tables, max_blocks_per_seq, q_start, prefix_lens, tree_mask,
                                     mask_words, num_seqs, max_nodes, max_prefix_len, num_heads);
    p.lse_in = lse;
    p.scores = scores;
    p.score_stride = score_stride;
    // Heads of few rows: a workgroup reads head_waves heads next to each other, so
    // that the 128-byte lines two heads share are used while they are near; up to
    // 16 workgroups a CU.  More rows: 6 a CU (each stages its rows again; 32 nodes
    // on 4 int8 sequences of 4000..16000 23.2 us against 25.5 at 16).  An odd number of
    // parts spreads every sequence's parts over the 8 XCDs (a cell's XCD is its index
    // mod 8): 64 decoding sequences 55.6 -> 50.2 us, the windows 33.4 -> 26.3.
    const bool one = (int64_t)max_nodes * p.group <= vcpp::kMassOneRows;
    p.head_waves = !one ? 1 : kv->num_kv_heads % 4 == 0 ? 4 : kv->num_kv_heads % 2 == 0 ? 2 : 1;
    const int32_t step = 256 / p.head_waves;  // positions of a workgroup's step
    const int64_t items = (int64_t)num_seqs * (kv->num_kv_heads / p.head_waves);
    const int64_t want = std::max<int64_t>(1, (one ? 16 : 6) * (int64_t)vcpp::compute_units() / items);
    p.part_len = (int32_t)((p.max_len + want - 1) / want + step - 1) / step * step;
    p.parts = (p.max_len + p.part_len - 1) / p.part_len | 1;
    if (!grid_fits((int64_t)num_seqs * p.parts, kv->num_kv_heads, 256))
        return fail(VCPP_E_UNSUPPORTED, "too many sequences, heads or positions for one launch");
    const hipError_t e = vcpp::launch_mass(p, static_cast<hipStream_t>(stream));
    return e != hipSuccess ? hip_fail(e, "attention mass launch") : VCPP_OK;
}

int vcpp_kv_commit(const vcpp_kv_pages* kv, const int32_t* block_tables, int32_t max_blocks_per_seq,
                   const int32_t* prefix_lens, const int32_t* accepted, const int32_t* accept_lens, int32_t num_seqs,
                   int32_t max_accepted, int32_t max_nodes, int32_t num_layers, int64_t layer_stride,
                   int64_t scale_layer_stride, void* stream) {
    vcpp::clear_error();
    vcpp::RowMoveParams p{};
    const int rc = move_params(kv, block_tables, max_blocks_per_seq, num_seqs, p);
    if (rc != VCPP_OK) return rc;
    if (max_accepted < 0 || max_nodes < 0 || num_layers < 0)
        return fail(VCPP_E_INVALID, "max_accepted, max_nodes and num_layers must be >= 0");
    if (max_accepted > VCPP_MAX_TREE_NODES || max_nodes > VCPP_MAX_TREE_NODES)
        return fail(VCPP_E_UNSUPPORTED, "max_accepted %d or max_nodes %d exceeds %d", max_accepted, max_nodes,
                    VCPP_MAX_TREE_NODES);
    if (num_seqs > 65535 || num_layers > 65535) return fail(VCPP_E_UNSUPPORTED, "too many sequences or layers");
    if (num_seqs == 0 || max_accepted == 0 || max_nodes == 0 || num_layers == 0) return VCPP_OK;
    if (!prefix_lens || !accepted || !accept_lens) return fail(VCPP_E_INVALID, "prefix_lens/accepted/accept_lens is NULL");
    const int64_t page = (int64_t)kv->block_size * kv->num_kv_heads * kv->head_dim;
    const int64_t esize = p.row_bytes / kv->head_dim;
    if (num_layers > 1) {
        if (layer_stride < 0 ? -layer_stride < page : layer_stride < page)
            return fail(VCPP_E_INVALID, "layer_stride %lld smaller than one page", (long long)layer_stride);
        if (layer_stride * esize % (esize == 1 ? 8 : 16) != 0)
            return fail(VCPP_E_INVALID, "layer_stride must keep pages %d-byte aligned", esize == 1 ? 8 : 16);
        if (p.scaled && (scale_layer_stride < 0 ? -scale_layer_stride : scale_layer_stride) <
                            (int64_t)kv->num_kv_heads * kv->block_size)
            return fail(VCPP_E_INVALID, "scale_layer_stride %lld smaller than one page", (long long)scale_layer_stride);
        p.layer_bytes = layer_stride * esize;
        p.scale_layer_stride = scale_layer_stride;
    }
    p.num_layers = num_layers;
    p.prefix_lens = prefix_lens;
    p.accepted = accepted;
    p.accept_lens = accept_lens;
    p.max_accepted = max_accepted;
    p.max_nodes = max_nodes;
    const hipError_t e = vcpp::launch_commit(p, static_cast<hipStream_t>(stream));
    return e != hipSuccess ? hip_fail(e, "commit launch") : VCPP_OK;
}

int vcpp_kv_evict_plan(const float* scores, const int32_t* positions, int64_t stride, const int32_t* context_lens,
                       const int32_t* seen_lens, int32_t num_seqs, int32_t num_kv_heads, int32_t max_context_len,
                       int32_t budget, int32_t keep_first, int32_t keep_last, int32_t* moves, int32_t max_moves,
                       int32_t* move_counts, int32_t* new_lens, float* scores_out, int32_t* positions_out,
                       void* stream) {
    vcpp::clear_error();
    if (num_seqs < 0 || max_context_len < 0) return fail(VCPP_E_INVALID, "num_seqs and max_context_len must be >= 0");
    if (num_kv_heads <= 0) return fail(VCPP_E_INVALID, "num_kv_heads must be positive");
    if (budget <= 0) return fail(VCPP_E_INVALID, "budget must be positive");
    if (keep_first < 0 || keep_last < 0 || (int64_t)keep_first + keep_last > budget)
        return fail(VCPP_E_INVALID, "keep_first %d + keep_last %d must be within the budget %d", keep_first, keep_last,
                    budget);
    if (stride < max_context_len) return fail(VCPP_E_INVALID, "stride %lld is below max_context_len", (long long)stride);
    const int64_t most = std::max<int64_t>(0, std::min<int64_t>(budget, (int64_t)max_context_len - budget));
    if (max_moves < most)
        return fail(VCPP_E_INVALID, "max_moves %d is below min(budget, max_context_len - budget) = %lld", max_moves,
                    (long long)most);
    if (max_context_len > kMaxLen) return fail(VCPP_E_UNSUPPORTED, "max_context_len %d too long", max_context_len);
    if ((int64_t)num_seqs * num_kv_heads > (1 << 20)) return fail(VCPP_E_UNSUPPORTED, "too many sequences x kv heads");
    if (num_seqs == 0) return VCPP_OK;
    if (!scores || !context_lens || !move_counts || !new_lens || !scores_out || (most > 0 && !moves))
        return fail(VCPP_E_INVALID, "scores/context_lens/moves/move_counts/new_lens/scores_out is NULL");
    if (new_lens == context_lens || new_lens == seen_lens)
        return fail(VCPP_E_INVALID, "new_lens must not be context_lens or seen_lens");
    vcpp::EvictPlanParams p{};
    p.scores = scores;
    p.positions = positions;
    p.context_lens = context_lens;
    p.seen_lens = seen_lens;
    p.stride = stride;
    p.num_seqs = num_seqs;
    p.num_kv_heads = num_kv_heads;
    p.max_len = max_context_len;
    p.budget = budget;
    p.keep_first = keep_first;
    p.keep_last = keep_last;
    p.max_moves = max_moves;
    p.moves = reinterpret_cast<int2*>(moves);
    p.move_counts = move_counts;
    p.new_lens = new_lens;
    p.scores_out = scores_out;
    p.positions_out = positions_out;
    const hipError_t e = vcpp::launch_evict_plan(p, static_cast<hipStream_t>(stream));
    return e != hipSuccess ? hip_fail(e, "evict plan launch") : VCPP_OK;
}

int vcpp_kv_evict_apply(const vcpp_kv_pages* kv, const int32_t* block_tables, int32_t max_blocks_per_seq,
                        const int32_t* moves, int32_t max_moves, const int32_t* move_counts, int32_t num_seqs,
                        void* stream) {
    vcpp::clear_error();
    vcpp::RowMoveParams p{};
    const int rc = move_params(kv, block_tables, max_blocks_per_seq, num_seqs, p);
    if (rc != VCPP_OK) return rc;
    if (max_moves < 0) return fail(VCPP_E_INVALID, "max_moves must be >= 0");
    if (max_moves > kMaxLen) return fail(VCPP_E_UNSUPPORTED, "max_moves %d too many", max_moves);
    if ((int64_t)num_seqs * kv->num_kv_heads > 65535) return fail(VCPP_E_UNSUPPORTED, "too many sequences x kv heads");
    if (num_seqs == 0 || max_moves == 0) return VCPP_OK;
    if (!moves || !move_counts) return fail(VCPP_E_INVALID, "moves/move_counts is NULL");
    if (reinterpret_cast<uintptr_t>(moves) % 8 != 0) return fail(VCPP_E_INVALID, "moves must be 8-byte aligned");
    p.moves = reinterpret_cast<const int2*>(moves);
    p.move_counts = move_counts;
    p.max_moves = max_moves;
    const hipError_t e = vcpp::launch_evict_apply(p, static_cast<hipStream_t>(stream));
    return e != hipSuccess ? hip_fail(e, "evict apply launch") : VCPP_OK;
}

}  // extern "C"
