// evict.hip -- a bounded KV cache: which positions of each kv head stay
// (evict_plan_kernel), and the rows that move for it (evict_apply_kernel); the
// rows of an accepted draft path moved into place (commit_kernel).
#include "evict.h"

#include <algorithm>

#include "device_common.h"

namespace vcpp {

namespace {

// ---- plan -------------------------------------------------------------------
//
// A workgroup owns one (sequence, kv head).  Scores become 32-bit keys whose
// unsigned order is the keeping order (a protected position above every score,
// NaN below every one); the budget-th largest key is found digit by digit from
// the top (radix select: a histogram of the next 8 bits over the keys that
// share the digits found so far), equal keys are kept in slot order, and the
// j-th hole among the first `budget` slots takes the j-th kept slot behind
// them.  Ranks come from ballots: each wave walks a contiguous run of slots, 64
// at a time, and only the waves' totals meet in LDS.
//
// Rows of up to 32768 slots (evict_plan_kernel) keep their keys in LDS; longer
// ones (evict_plan_long_kernel) read them again for every pass.  What bounds it
// is the chain of passes with a barrier each: 512 rows of 2064 slots 9.7 us, 32
// rows of 16384 18.8.

constexpr int kPlanLdsKeys = 32768;

struct PlanRow {
    const float* scores;
    const int32_t* positions;
    int64_t shift;  // seen - len: a slot that was only appended holds position slot + shift
    int64_t first, last;  // protected: position < first or >= last

    __device__ __forceinline__ int64_t position(int slot) const {
        const int32_t x = positions ? positions[slot] : -1;
        return x >= 0 ? (int64_t)x : slot + shift;
    }
    __device__ __forceinline__ uint32_t key_of(float score, int64_t at) const {
        const float x = score + 0.f;  // (-0 ranks with +0)
        const uint32_t b = __float_as_uint(x);
        if (at < first || at >= last) return 0xFFFFFFFFu;
        return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
    }
    __device__ __forceinline__ uint32_t key(int slot) const { return key_of(scores[slot], position(slot)); }
};

// The budget-th largest key's digit at bit d, from the histogram of the keys
// that share the digits above it: one wave, four bins a lane from the top.
// got: {the digit, keys still to take from its bin, keys in its bin}.
__device__ __forceinline__ void find_digit(const uint32_t* hist, int left, int lane, uint32_t* got) {
    int n[4], all = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) all += n[j] = (int)hist[255 - 4 * lane - j];
    int before = wave_excl_scan(all, lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (before < left && before + n[j] >= left) got[0] = 255 - 4 * lane - j, got[1] = left - before, got[2] = n[j];
        before += n[j];
    }
}

__device__ __forceinline__ int mbcnt64(uint64_t m) {  // set bits below this lane
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}

// At most kPlanLdsKeys slots.  Slots in groups of 64: a group's kept slots are
// one ballot in LDS, ranks are scans of the groups' counts.  The select ends at
// the first digit whose whole bin stays (distinct scores: after two of four).
//
// The first digit is a score's sign and seven bits of its exponent: most scores
// share a few bins, and LDS atomics on one word queue up.  Its histogram is
// counted while the keys are made, in kPlanCopies copies on different banks.
constexpr int kPlanCopies = 8;
constexpr int kPlanCopy = 257;                        // words of a copy
constexpr int kPlanHoles = kPlanCopies * kPlanCopy;   // holes whose slots are in LDS too (behind the select)

template <int T>
__global__ __launch_bounds__(T) void evict_plan_kernel(EvictPlanParams p) {
    constexpr int W = T / 64, GROUPS = kPlanLdsKeys / 64;
    extern __shared__ uint32_t plan_keys[];
    __shared__ uint64_t kept_s[GROUPS];
    __shared__ int hole0[GROUPS], filler0[GROUPS];  // holes and fillers before each group
    __shared__ int holes_s[kPlanHoles];  // (first the first digit's histograms)
    __shared__ uint32_t hist[4][256];
    uint32_t* const copies = reinterpret_cast<uint32_t*>(holes_s);
    __shared__ uint32_t found[3];
    __shared__ int total_s;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int s = blockIdx.x / p.num_kv_heads, h = blockIdx.x - s * p.num_kv_heads;
    const int len = min(max(p.context_lens[s], 0), p.max_len);
    const int64_t base = (int64_t)blockIdx.x * p.stride;
    const int64_t seen = p.seen_lens ? (int64_t)p.seen_lens[s] : (int64_t)len;
    const PlanRow row{p.scores + base, p.positions ? p.positions + base : nullptr, seen - len, p.keep_first,
                      seen - p.keep_last};
    float* so = p.scores_out + base;
    int32_t* po = p.positions_out ? p.positions_out + base : nullptr;
    const int budget = p.budget, keep = min(len, budget);
    if (h == 0 && tid == 0) p.new_lens[s] = keep;
    const bool cut = len > budget;
    if (cut) {
        for (int i = tid; i < 4 * 256; i += T) (&hist[0][0])[i] = 0;
        for (int i = tid; i < kPlanHoles; i += T) copies[i] = 0;
        __syncthreads();
    }
    // The state in front of the budget as it is (holes are overwritten by the
    // moves), and the keys.  (Eight slots are loaded before any is stored: the
    // stores may alias the loads, so that the compiler keeps their order.)
    constexpr int AT = 8;
    for (int i0 = tid; i0 < len; i0 += AT * T) {
        float x[AT];
        int32_t at[AT];
#pragma unroll
        for (int j = 0; j < AT; ++j) {
            const int i = min(i0 + j * T, len - 1);
            x[j] = row.scores[i];
            at[j] = row.positions ? row.positions[i] : -1;
        }
#pragma unroll
        for (int j = 0; j < AT; ++j) {
            const int i = i0 + j * T;
            if (i >= len) break;
            const int pos = at[j] >= 0 ? at[j] : (int)(i + row.shift);
            if (cut) {
                const uint32_t k = row.key_of(x[j], pos);
                plan_keys[i] = k;
                atomicAdd(&copies[tid % kPlanCopies * kPlanCopy + (k >> 24)], 1u);
            }
            if (i < keep) {
                so[i] = x[j];
                if (po) po[i] = pos;
            }
        }
    }
    int count = 0;
    if (cut) {
        uint32_t limit = 0, ties = 0;  // keys above `limit` stay, and `ties` of the equal ones, in slot order
        int left = budget;
        bool all_equal = false;        // every equal one stays
        __syncthreads();
        for (int d = 24, n = 0; d >= 0; d -= 8, ++n) {
            if (d == 24) {
                if (tid < 256) {
                    uint32_t sum = 0;
#pragma unroll
                    for (int c = 0; c < kPlanCopies; ++c) sum += copies[c * kPlanCopy + tid];
                    hist[0][tid] = sum;
                }
            } else {
                for (int i = tid; i < len; i += T) {
                    const uint32_t k = plan_keys[i];
                    if ((k ^ limit) >> (d + 8) == 0) atomicAdd(&hist[n][k >> d & 255], 1u);
                }
            }
            __syncthreads();
            if (wave == 0) find_digit(hist[n], left, lane, found);
            __syncthreads();
            limit |= found[0] << d;
            left = (int)found[1];
            if (found[1] == found[2]) {  // (the last digit: `left` equal keys, all of them kept)
                all_equal = true;
                break;
            }
        }
        ties = (uint32_t)left;
        const int groups = (len + 63) / 64;
        const auto valid = [&](int g) { return len - 64 * g >= 64 ? ~0ull : (1ull << (len - 64 * g)) - 1; };
        if (all_equal) {  // key >= limit (digits below the found one are 0)
            for (int g = wave; g < groups; g += W) {
                const int i = 64 * g + lane;
                const uint64_t k = __ballot(i < len && plan_keys[min(i, len - 1)] >= limit);
                if (lane == 0) kept_s[g] = k;
            }
        } else {  // equal keys by their rank: counts of the groups first
            for (int g = wave; g < groups; g += W) {
                const int i = 64 * g + lane;
                const int n = __popcll(__ballot(i < len && plan_keys[min(i, len - 1)] == limit));
                if (lane == 0) hole0[g] = n;
            }
            __syncthreads();
            if (wave == 0) {
                int before = 0;
                for (int g = 0; g < groups; g += 64) {
                    const int n = g + lane < groups ? hole0[g + lane] : 0, incl = wave_incl_scan(n);
                    if (g + lane < groups) filler0[g + lane] = before + incl - n;
                    before += __builtin_amdgcn_readlane(incl, 63);
                }
            }
            __syncthreads();
            for (int g = wave; g < groups; g += W) {
                const int i = 64 * g + lane;
                const uint32_t k = i < len ? plan_keys[i] : 0u;
                const uint64_t e = __ballot(i < len && k == limit);
                const bool stays = i < len && (k > limit || (k == limit && filler0[g] + mbcnt64(e) < (int)ties));
                const uint64_t b = __ballot(stays);
                if (lane == 0) kept_s[g] = b;
            }
        }
        __syncthreads();
        const auto in_front = [&](int g) {  // slots of group g below the budget
            const int n = budget - 64 * g;
            return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
        };
        if (wave == 0) {
            int hb = 0, fb = 0;
            for (int g = 0; g < groups; g += 64) {
                const int gl = g + lane;
                int nh = 0, nf = 0;
                if (gl < groups) {
                    const uint64_t k = kept_s[gl], f = in_front(gl);
                    nh = __popcll(~k & f & valid(gl));
                    nf = __popcll(k & ~f);
                }
                const int ih = wave_incl_scan(nh), jf = wave_incl_scan(nf);
                if (gl < groups) hole0[gl] = hb + ih - nh, filler0[gl] = fb + jf - nf;
                hb += __builtin_amdgcn_readlane(ih, 63);
                fb += __builtin_amdgcn_readlane(jf, 63);
            }
            if (lane == 0) total_s = hb;
        }
        __syncthreads();
        count = min(total_s, p.max_moves);
        int2* moves = p.moves + (int64_t)blockIdx.x * p.max_moves;
        const bool in_lds = count <= kPlanHoles;
        for (int g = wave; 64 * g < budget; g += W) {
            const uint64_t a = ~kept_s[g] & in_front(g) & valid(g);
            const int r = hole0[g] + mbcnt64(a);
            if (a >> lane & 1 && r < count) {
                if (in_lds) holes_s[r] = 64 * g + lane;
                else moves[r].x = 64 * g + lane;
            }
        }
        __threadfence_block();
        __syncthreads();
        constexpr int FG = 4;  // groups at once
        for (int g0 = budget / 64 + wave; g0 < groups; g0 += FG * W) {
            float x[FG];
            int32_t pos[FG];
            int rank[FG];
#pragma unroll
            for (int j = 0; j < FG; ++j) {
                const int g = g0 + j * W, from = 64 * g + lane;
                rank[j] = -1;
                if (g >= groups) continue;
                const uint64_t b = kept_s[g] & ~in_front(g);
                const int r = filler0[g] + mbcnt64(b);
                if (!(b >> lane & 1) || r >= count) continue;
                rank[j] = r;
                x[j] = row.scores[from];
                pos[j] = row.positions ? row.positions[from] : -1;
            }
#pragma unroll
            for (int j = 0; j < FG; ++j) {
                const int r = rank[j], from = 64 * (g0 + j * W) + lane;
                if (r < 0) continue;
                const int to = in_lds ? holes_s[r] : moves[r].x;
                if (in_lds) moves[r] = make_int2(to, from);
                else moves[r].y = from;
                so[to] = x[j];
                if (po) po[to] = pos[j] >= 0 ? pos[j] : (int)(from + row.shift);
            }
        }
        __syncthreads();  // (scores_out may be scores: sources are read before they are cleared)
    }
    if (tid == 0) p.move_counts[blockIdx.x] = count;
    for (int i = keep + tid; i < p.max_len; i += T) {
        so[i] = 0.f;
        if (po) po[i] = -1;
    }
}

template <int T>
__global__ __launch_bounds__(T) void evict_plan_long_kernel(EvictPlanParams p) {
    constexpr int W = T / 64;
    __shared__ uint32_t hist[256];
    __shared__ uint32_t found[3];
    __shared__ int tot[3][W];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int s = blockIdx.x / p.num_kv_heads, h = blockIdx.x - s * p.num_kv_heads;
    const int len = min(max(p.context_lens[s], 0), p.max_len);
    const int64_t base = (int64_t)blockIdx.x * p.stride;
    const int64_t seen = p.seen_lens ? (int64_t)p.seen_lens[s] : (int64_t)len;
    const PlanRow row{p.scores + base, p.positions ? p.positions + base : nullptr, seen - len, p.keep_first,
                      seen - p.keep_last};
    float* so = p.scores_out + base;
    int32_t* po = p.positions_out ? p.positions_out + base : nullptr;
    const int budget = p.budget, keep = min(len, budget);
    if (h == 0 && tid == 0) p.new_lens[s] = keep;
    // This wave's slots: whole groups of 64.
    const int run = ((len + 63) / 64 + W - 1) / W * 64;
    const int lo = min(wave * run, len), hi = min(lo + run, len);

    uint32_t limit = 0;  // keys above it stay
    int ties = 0;        // slots of equal keys that stay, in slot order
    int count = 0;       // moves
    if (len > budget) {
        const auto key = [&](int i) { return row.key(i); };
        int left = budget;
        for (int d = 24; d >= 0; d -= 8) {
            __syncthreads();
            for (int i = tid; i < 256; i += T) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < len; i += T) {
                const uint32_t k = key(i);
                if (d == 24 || (k ^ limit) >> (d + 8) == 0) atomicAdd(&hist[k >> d & 255], 1u);
            }
            __syncthreads();
            if (wave == 0) find_digit(hist, left, lane, found);
            __syncthreads();
            limit |= found[0] << d;
            left = (int)found[1];
        }
        // `left` of the slots whose key is the limit stay.
        ties = left;
        int eq = 0;
        for (int i = lo; i < hi; i += 64) eq += __popcll(__ballot(i + lane < hi && key(i + lane) == limit));
        if (lane == 0) tot[0][wave] = eq;
        __syncthreads();
        int eq0 = 0;
        for (int w = 0; w < wave; ++w) eq0 += tot[0][w];
        // Kept slots of the 64 at i, from the number of equal keys before them.
        const auto kept = [&](int i, int& equal) {
            const bool in = i + lane < hi;
            const uint32_t k = in ? key(i + lane) : 0u;
            const uint64_t e = __ballot(in && k == limit);
            const int at = equal + mbcnt64(e);
            equal += __popcll(e);
            return __ballot(in && (k > limit || (k == limit && at < ties)));
        };
        const auto in_front = [&](int i) {  // slots of the 64 at i that are below the budget
            return budget - i >= 64 ? ~0ull : budget <= i ? 0ull : (1ull << (budget - i)) - 1;
        };
        const auto valid = [&](int i) { return hi - i >= 64 ? ~0ull : (1ull << (hi - i)) - 1; };
        int equal = eq0, holes = 0, fillers = 0;
        for (int i = lo; i < hi; i += 64) {
            const uint64_t k = kept(i, equal), f = in_front(i);
            holes += __popcll(~k & f & valid(i));
            fillers += __popcll(k & ~f);
        }
        if (lane == 0) tot[1][wave] = holes, tot[2][wave] = fillers;
        __syncthreads();
        int hole = 0, filler = 0;
        for (int w = 0; w < W; ++w) {
            if (w < wave) hole += tot[1][w], filler += tot[2][w];
            count += tot[1][w];
        }
        int2* moves = p.moves + (int64_t)blockIdx.x * p.max_moves;
        equal = eq0;
        for (int i = lo; i < hi; i += 64) {
            const uint64_t k = kept(i, equal), f = in_front(i), v = valid(i);
            const uint64_t a = ~k & f & v, b = k & ~f;
            const int ra = hole + mbcnt64(a);
            const int rb = filler + mbcnt64(b);
            if (a >> lane & 1 && ra < p.max_moves) moves[ra].x = i + lane;
            if (b >> lane & 1 && rb < p.max_moves) moves[rb].y = i + lane;
            if (k & f & 1ull << lane) {
                const int slot = i + lane;
                const float x = row.scores[slot];
                const int at = (int)row.position(slot);
                so[slot] = x;
                if (po) po[slot] = at;
            }
            hole += __popcll(a);
            filler += __popcll(b);
        }
        count = min(count, p.max_moves);
        __threadfence_block();
        __syncthreads();
        // (scores_out may be scores: sources lie behind the budget, targets in front of it)
        for (int j = tid; j < count; j += T) {
            const int2 m = moves[j];
            const float x = row.scores[m.y];
            const int at = (int)row.position(m.y);
            so[m.x] = x;
            if (po) po[m.x] = at;
        }
        __syncthreads();
    } else {
        for (int i = tid; i < len; i += T) {
            const float x = row.scores[i];
            const int at = (int)row.position(i);
            so[i] = x;
            if (po) po[i] = at;
        }
    }
    if (tid == 0) p.move_counts[blockIdx.x] = count;
    for (int i = keep + tid; i < p.max_len; i += T) {
        so[i] = 0.f;
        if (po) po[i] = -1;
    }
}

// ---- moves ------------------------------------------------------------------

// Physical slot of a position: its block's byte offset and its place in it;
// false where the table or the pool has none.
__device__ __forceinline__ bool place(const RowMoveParams& p, const int32_t* table, int64_t pos, int& bid, int& at) {
    if (pos < 0 || pos >= (int64_t)p.max_blocks * p.block_size) return false;
    const uint32_t x = (uint32_t)pos, lb = x / (uint32_t)p.block_size;  // (positions are below 2^31 + 256)
    bid = table[lb];
    at = (int)(x - lb * (uint32_t)p.block_size);
    return bid >= 0 && (int64_t)bid < p.num_blocks;
}

// A thread moves one 16-byte piece of one row: sources and targets of a plan
// are disjoint, so the moves need no order.  Bound by the lines it touches: a
// head's fp16 row of 80 is 160 bytes at any place, 2 or 3 lines of 128 each way
// (4 prompts cut to 4096 rows, 53 MB: 18 us where whole lines would take 10).
__global__ __launch_bounds__(256) void evict_apply_kernel(RowMoveParams p) {
    const int s = blockIdx.y / p.num_kv_heads, h = blockIdx.y - s * p.num_kv_heads;
    const int pieces = p.row_bytes / 16, per = 2 * pieces;  // K's, then V's
    const int count = min(max(p.move_counts[blockIdx.y], 0), p.max_moves);
    const int32_t* table = p.block_tables + (int64_t)s * p.max_blocks;
    const int2* moves = p.moves + (int64_t)blockIdx.y * p.max_moves;
    // (32-bit indexes and divisions: 0 .. 2^24 moves of at most 64 pieces.)
    const uint32_t items = (uint32_t)count * (uint32_t)per;
    for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < items; i += gridDim.x * 256u) {
        const int j = (int)(i / (uint32_t)per), piece = (int)(i - (uint32_t)(j * per));
        const int2 m = moves[j];
        int tb, ta, fb, fa;
        if (!place(p, table, m.x, tb, ta) || !place(p, table, m.y, fb, fa)) continue;
        const bool isv = piece >= pieces;
        char* base = isv ? p.v : p.k;
        const int64_t in = (int64_t)(isv ? piece - pieces : piece) * 16 + (int64_t)h * p.row_bytes;
        const int64_t row = (int64_t)p.num_kv_heads * p.row_bytes;
        *reinterpret_cast<i4*>(base + tb * p.block_bytes + ta * row + in) =
            *reinterpret_cast<const i4*>(base + fb * p.block_bytes + fa * row + in);
        if (p.scaled && (piece == 0 || piece == pieces)) {
            uint16_t* sc = isv ? p.v_scale : p.k_scale;
            sc[tb * p.scale_block_stride + (int64_t)h * p.block_size + ta] =
                sc[fb * p.scale_block_stride + (int64_t)h * p.block_size + fa];
        }
    }
}

// A workgroup owns a column slice of one layer's K or V rows of one sequence,
// and holds every accepted row's slice in registers before it writes any:
// sources may be other rows' targets.  One round trip: 64 layers of one
// sequence 4.0 us, 16 layers of 32 (8 rows each) 8.6 us.
constexpr int kCommitRegs = 8;
constexpr int kCommitItems = 256 * kCommitRegs;

__global__ __launch_bounds__(256) void commit_kernel(RowMoveParams p, int width, int slices, int scale_width) {
    const int slice = blockIdx.x >> 1, isv = blockIdx.x & 1, s = blockIdx.y, layer = blockIdx.z;
    const int n = min(max(p.accept_lens[s], 0), p.max_accepted);
    const int64_t prefix = max(p.prefix_lens[s], 0);
    const int32_t* table = p.block_tables + (int64_t)s * p.max_blocks;
    const int32_t* accepted = p.accepted + (int64_t)s * p.max_accepted;
    const int64_t row = (int64_t)p.num_kv_heads * p.row_bytes;
    const bool scales = slice >= slices;
    const int w = scales ? scale_width : width;
    const int col0 = (scales ? slice - slices : slice) * w;
    const int cols = scales ? p.num_kv_heads : (int)(row / 16);
    char* base = (isv ? p.v : p.k) + layer * p.layer_bytes;
    uint16_t* sbase = (isv ? p.v_scale : p.k_scale) + layer * p.scale_layer_stride;
    i4 data[kCommitRegs];
    int64_t to[kCommitRegs];
#pragma unroll
    for (int r = 0; r < kCommitRegs; ++r) {
        to[r] = -1;
        const int i = threadIdx.x + 256 * r;
        const int j = i / w, col = col0 + i - j * w;
        if (j >= n || col >= cols) continue;
        const int a = accepted[j];
        int tb, ta, fb, fa;
        if (a < 0 || a >= p.max_nodes || a == j) continue;
        if (!place(p, table, prefix + j, tb, ta) || !place(p, table, prefix + a, fb, fa)) continue;
        if (scales) {
            to[r] = tb * p.scale_block_stride + (int64_t)col * p.block_size + ta;
            data[r].x = sbase[fb * p.scale_block_stride + (int64_t)col * p.block_size + fa];
        } else {
            to[r] = tb * p.block_bytes + ta * row + (int64_t)col * 16;
            data[r] = *reinterpret_cast<const i4*>(base + fb * p.block_bytes + fa * row + (int64_t)col * 16);
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): every load is back before any wave stores
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kCommitRegs; ++r) {
        if (to[r] < 0) continue;
        if (scales) sbase[to[r]] = (uint16_t)data[r].x;
        else *reinterpret_cast<i4*>(base + to[r]) = data[r];
    }
}

}  // namespace

// Threads by the row's length (us with 256 / 512 / 1024 threads): 512 rows of
// 2064 slots 12.5 / 11.0 / 11.2, 4096 rows of them 48 / 44 / 58, 128 rows of 4090
// 15.4 / 11.5 / 10.5, 4096 rows of 900 slots 24 / 28 / 45.
hipError_t launch_evict_plan(const EvictPlanParams& p, hipStream_t stream) {
    const dim3 grid((uint32_t)(p.num_seqs * p.num_kv_heads));
    if (p.max_len > kPlanLdsKeys) {
        evict_plan_long_kernel<1024><<<grid, dim3(1024), 0, stream>>>(p);
    } else if (p.max_len > 4096) {
        const hipError_t e = hipFuncSetAttribute((const void*)evict_plan_kernel<1024>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, kPlanLdsKeys * 4);
        if (e != hipSuccess) return e;
        evict_plan_kernel<1024><<<grid, dim3(1024), p.max_len * 4, stream>>>(p);
    } else if (p.max_len > 1024) {
        evict_plan_kernel<512><<<grid, dim3(512), p.max_len * 4, stream>>>(p);
    } else {
        evict_plan_kernel<256><<<grid, dim3(256), p.max_len * 4, stream>>>(p);
    }
    return hipGetLastError();
}

hipError_t launch_evict_apply(const RowMoveParams& p, hipStream_t stream) {
    const int64_t items = (int64_t)p.max_moves * 2 * (p.row_bytes / 16);
    const int64_t rows = (int64_t)p.num_seqs * p.num_kv_heads;
    const int64_t need = (items + 255) / 256;
    const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>(need, 8192 / std::max<int64_t>(1, rows)));
    evict_apply_kernel<<<dim3((uint32_t)wgs, (uint32_t)rows), dim3(256), 0, stream>>>(p);
    return hipGetLastError();
}

hipError_t launch_commit(const RowMoveParams& p, hipStream_t stream) {
    const int cols = (int)((int64_t)p.num_kv_heads * p.row_bytes / 16);
    const int width = std::min(cols, kCommitItems / p.max_accepted);
    const int slices = (cols + width - 1) / width;
    const int scale_width = std::min(p.num_kv_heads, kCommitItems / p.max_accepted);
    const int scale_slices = p.scaled ? (p.num_kv_heads + scale_width - 1) / scale_width : 0;
    const dim3 grid((uint32_t)(2 * (slices + scale_slices)), (uint32_t)p.num_seqs, (uint32_t)p.num_layers);
    commit_kernel<<<grid, dim3(256), 0, stream>>>(p, width, slices, scale_width);
    return hipGetLastError();
}

}  // namespace vcpp
