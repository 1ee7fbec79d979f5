// tree_mask.h -- which of 32 consecutive positions a row of a draft tree sees.
#pragma once

#include "device_common.h"
#include "tree.h"

namespace vcpp {

namespace {

// One sequence of a call, its values clamped to what the call announced.
struct TreeSeq {
    int q0, n;   // first row, nodes
    int prefix;  // positions in front of the tree
    int end;     // positions attended: min(prefix + n, max_len)
    int plain;   // positions that every row sees: min(prefix, end)
    __device__ __forceinline__ TreeSeq() : q0(0), n(0), prefix(0), end(0), plain(0) {}
    __device__ __forceinline__ TreeSeq(const TreeParams& p, int s) {
        const int a = p.q_start[s], b = p.q_start[s + 1], c = p.prefix_lens[s];
        q0 = a;
        n = min(max(b - a, 0), p.max_nodes);
        prefix = min(max(c, 0), INT32_MAX - kMaxTreeNodes);
        if (q0 < 0 || (int64_t)q0 + n > p.rows_cap) n = 0;
        end = n > 0 ? min(prefix + n, p.max_len) : 0;
        plain = min(prefix, end);
    }
};

// a / b for 0 <= a, 0 < b: 32 bits where they hold both (the usual call; a
// 64-bit division is 140 scalar instructions).
__device__ __forceinline__ int64_t div_any(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
    return a / b;
}

// The cut of a call's work.  Unit (s, u) is row tile u of sequence s, as long as
// the sequence's key blocks; units follow each other on one axis of `total`
// blocks, and range r of R covers blocks total r / R .. total (r + 1) / R - 1.
// Every wave forms this by itself, 64 sequences at a time.
struct TreeRanges {
    const TreeParams& p;
    int rows, lane;
    int64_t total;
    int R;
    int at;          // sequences at .. at + 63 are in the lanes
    TreeSeq mine;    // this lane's sequence,
    int work, incl;  // its blocks over all row tiles, and their sum up to it
    __device__ __forceinline__ void load(int s0) {
        at = s0;
        mine = s0 + lane < p.num_seqs ? TreeSeq(p, s0 + lane) : TreeSeq();
        work = (mine.n * p.group + rows - 1) / rows * ((mine.end + 31) / 32);
        incl = wave_incl_scan(work);
    }
    __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(incl, 63); }
    __device__ __forceinline__ TreeRanges(const TreeParams& p_, int rows_, int lane_)
        : p(p_), rows(rows_), lane(lane_), total(0) {
        for (int s0 = 0; s0 < p.num_seqs; s0 += kWave) {
            load(s0);
            total += all();
        }
        R = (int)max((int64_t)1, min((int64_t)p.ranges, total / kTreeMinBlocks));
    }
    __device__ __forceinline__ int64_t start(int r) const { return div_any(total * r, R); }
    __device__ __forceinline__ int range_of(int64_t x) const { return (int)div_any((x + 1) * R - 1, total); }
    // The sequence whose units hold block x < total, and its first block.
    __device__ __forceinline__ int seq_of(int64_t x, int64_t& first) {
        int64_t base = 0;
        for (int s0 = 0; s0 < p.num_seqs; s0 += kWave) {
            if (p.num_seqs > kWave) load(s0);
            if (x < base + all()) {
                const int i = __builtin_ctzll(__ballot(base + incl > x));
                first = base + __builtin_amdgcn_readlane(incl, i) - __builtin_amdgcn_readlane(work, i);
                return s0 + i;
            }
            base += all();
        }
        first = 0;
        return 0;  // (not reached)
    }
    // The first block of sequence s.
    __device__ __forceinline__ int64_t first_of(int s) {
        int64_t base = 0;
        for (int s0 = 0; s0 + kWave <= s; s0 += kWave) {
            load(s0);
            base += all();
        }
        if (s < at || s >= at + kWave) load(s / kWave * kWave);
        return base + __builtin_amdgcn_readlane(incl, s - at) - __builtin_amdgcn_readlane(work, s - at);
    }
};

// Positions pos .. pos + 31 that node t of the sequence sees, bit b for
// position pos + b: all of the prefix, the nodes of t's mask row (words at
// `row`; NULL: nodes 0 .. t), nothing at or past `end`.
__device__ __forceinline__ uint32_t tree_window(const TreeParams& p, const TreeSeq& q, const uint64_t* row, int t,
                                                int pos) {
    const int base = pos - q.prefix;  // node of bit 0 (negative: in the prefix)
    uint32_t w;
    if (base <= -32) {
        w = ~0u;
    } else if (row) {
        if (base < 0) {
            w = (uint32_t)(row[0] << -base) | ((1u << -base) - 1);
        } else {
            const int at = base >> 6, sh = base & 63;
            w = at < p.mask_words ? (uint32_t)(row[at] >> sh) : 0u;
            if (sh > 32 && at + 1 < p.mask_words) w |= (uint32_t)(row[at + 1] << (64 - sh));
        }
    } else {
        const int k = t - base + 1;  // bits 0 .. k - 1
        w = k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1;
    }
    const int left = q.end - pos;
    return left >= 32 ? w : left <= 0 ? 0u : w & ((1u << left) - 1);
}

}  // namespace

}  // namespace vcpp
