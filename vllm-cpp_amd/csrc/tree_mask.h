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
    int plain;       // positions that every row sees: min(prefix, end)
    __device__ __forceinline__ TreeSeq(const TreeParams& p, int s) {
        q0 = p.q_start[s];
        n = min(max(p.q_start[s + 1] - q0, 0), p.max_nodes);
        prefix = max(p.prefix_lens[s], 0);
        end = (int)min(prefix + n, (int64_t)p.max_len);
        plain = (int)min(prefix, (int64_t)end);
        if (q0 < 0 || (int64_t)q0 + n > p.rows_cap) n = 0, end = 0;
    }
};

// The cut of a call's work.  Unit (s, u) is row tile u of sequence s, as long as
// the sequence's key blocks; units follow each other on one axis of `total`
// blocks, and range r of R covers blocks total r / R .. total (r + 1) / R - 1.
// Every wave forms this by itself, 64 sequences at a time.
struct TreeRanges {
    int64_t total;
    int R;
    // Row tiles and key blocks of sequence s (0 past the last).
    __device__ static __forceinline__ void unit(const TreeParams& p, int rows, int s, int& tiles, int& blocks) {
        tiles = blocks = 0;
        if (s < p.num_seqs) {
            const TreeSeq q(p, s);
            tiles = (q.n * p.group + rows - 1) / rows;
            blocks = (q.end + 31) / 32;
        }
    }
    __device__ __forceinline__ TreeRanges(const TreeParams& p, int rows, int lane) : total(0) {
        for (int s0 = 0; s0 < p.num_seqs; s0 += kWave) {
            int tiles, blocks;
            unit(p, rows, s0 + lane, tiles, blocks);
            total += wave_sum(tiles * blocks);
        }
        R = (int)max((int64_t)1, min((int64_t)p.ranges, total / kTreeMinBlocks));
    }
    __device__ __forceinline__ int64_t start(int r) const { return total * r / R; }
    __device__ __forceinline__ int range_of(int64_t x) const { return (int)(((x + 1) * R - 1) / total); }
    // The sequence whose units hold block x, and its first block.
    __device__ __forceinline__ int seq_of(const TreeParams& p, int rows, int lane, int64_t x, int64_t& first) const {
        int64_t base = 0;
        for (int s0 = 0; s0 < p.num_seqs; s0 += kWave) {
            int tiles, blocks;
            unit(p, rows, s0 + lane, tiles, blocks);
            const int incl = wave_incl_scan(tiles * blocks);
            const int all = __builtin_amdgcn_readlane(incl, 63);
            if (x < base + all) {
                const int at = __builtin_ctzll(__ballot(base + incl > x));
                first = base + (at > 0 ? __builtin_amdgcn_readlane(incl, at - 1) : 0);
                return s0 + at;
            }
            base += all;
        }
        first = 0;
        return 0;  // (x < total: not reached)
    }
    // The first block of sequence s.
    __device__ __forceinline__ int64_t first_of(const TreeParams& p, int rows, int lane, int s) const {
        int64_t base = 0;
        for (int s0 = 0; s0 < s; s0 += kWave) {
            int tiles, blocks;
            unit(p, rows, s0 + lane, tiles, blocks);
            base += wave_sum(s0 + lane < s ? tiles * blocks : 0);
        }
        return base;
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
