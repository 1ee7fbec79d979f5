// tree_mask.h -- which of 32 consecutive positions a row of a draft tree sees.
#pragma once

#include "device_common.h"
#include "tree.h"

namespace vcpp {

namespace {

// One sequence of a call, its values clamped to what the call announced.
struct TreeSeq {
    int q0, n;       // first row, nodes
    int64_t prefix;  // positions in front of the tree
    int end;         // positions attended: min(prefix + n, max_len)
    __device__ __forceinline__ TreeSeq(const TreeParams& p, int s) {
        q0 = p.q_start[s];
        n = min(max(p.q_start[s + 1] - q0, 0), p.max_nodes);
        prefix = max(p.prefix_lens[s], 0);
        end = (int)min(prefix + n, (int64_t)p.max_len);
        if (q0 < 0 || (int64_t)q0 + n > p.rows_cap) n = 0, end = 0;
    }
};

// Positions pos .. pos + 31 that node t of the sequence sees, bit b for
// position pos + b: all of the prefix, the nodes of t's mask row (words at
// `row`; NULL: nodes 0 .. t), nothing at or past `end`.
__device__ __forceinline__ uint32_t tree_window(const TreeParams& p, const TreeSeq& q, const uint64_t* row, int t,
                                                int pos) {
    const int64_t base = pos - q.prefix;  // node of bit 0 (negative: in the prefix)
    uint32_t w;
    if (base <= -32) {
        w = ~0u;
    } else if (row) {
        if (base < 0) {
            w = (uint32_t)(row[0] << (int)-base) | ((1u << (int)-base) - 1);
        } else {
            const int at = (int)(base >> 6), sh = (int)(base & 63);
            w = at < p.mask_words ? (uint32_t)(row[at] >> sh) : 0u;
            if (sh > 32 && at + 1 < p.mask_words) w |= (uint32_t)(row[at + 1] << (64 - sh));
        }
    } else {
        const int64_t k = t - base + 1;  // bits 0 .. k - 1
        w = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << (int)k) - 1;
    }
    const int left = q.end - pos;
    return left >= 32 ? w : left <= 0 ? 0u : w & ((1u << left) - 1);
}

}  // namespace

}  // namespace vcpp
