// mass.hip -- the softmax weights of a step's queries, added up per kv head
// and cache position: scores[s][g][j] += sum over the rows (node i, head h of
// group g) that see position j of exp(q_i . k_j / sqrt(D) - lse_i).
//
// With the rows' log-sum-exp given, every position is independent: no running
// maximum, no merge, and each sum is formed by one wave in a fixed order (no
// atomics, the same bits every time).  A wave owns 64 positions at a time;
// S[16 rows][16 positions] = Q x K^T comes from 16x16x32 f16 products with the
// rows along a lane's accumulators, so that a lane sums its position's weights
// in registers and only the four lane groups meet at the end.  K goes straight
// from its pages to the product's operands (a lane's 16 bytes are 16 bytes of
// its position's row): each row of K is read once per kv head.
//
// A decode step (few rows) is bound by the K bytes: their operand stays in
// registers and the waves of a workgroup take neighbouring heads (64 sequences
// of 128..4096 fp16 tokens, 64 heads over 8 kv heads of 80: 173 MB cold in 44.5
// us, 3.9 TB/s with the launch; a head per workgroup 50.2).  Many rows are bound by
// the products and exponentials: the rows' operands and log-sum-exps are staged
// in LDS, 128 rows at a time.  K loads a step ahead of the products measured
// slower in both (59 us and 42 against 50 and 26: the registers cost waves).
#include "device_common.h"
#include "tree.h"
#include "tree_mask.h"

namespace vcpp {

namespace {

constexpr int kMassTiles = 4;                   // 16-position tiles of a wave
constexpr int kMassKeys = 16 * kMassTiles;      // positions of a wave
constexpr int kMassWaves = 4;

// Operand k slices of a row: 8 dims of lane group g in slice i.  fp16 pages:
// dims 32 i + 8 g.  Byte pages: 16 consecutive bytes of a lane serve two
// slices.  A 16-dim rest (D = 80) fills lane groups 0 and 1 of a last slice.
template <int KV, int D>
struct MassDims {
    static constexpr int NC = D / 32, REM = (D % 32) / 16, NS = NC + REM;
    __device__ static __forceinline__ int dim(int i, int g) {
        if (i == NC) return 32 * NC + 8 * g;  // (g < 2)
        return KV == VCPP_KV_F16 ? 32 * i + 8 * g : 64 * (i >> 1) + 16 * g + 8 * (i & 1);
    }
};

template <int KV, int D>
__device__ __forceinline__ void load_k(const TreeParams& p, int64_t row, int g, h8 (&k)[MassDims<KV, D>::NS]) {
    using M = MassDims<KV, D>;
    if constexpr (KV == VCPP_KV_F16) {
        const _Float16* b = static_cast<const _Float16*>(p.k) + row;
#pragma unroll
        for (int i = 0; i < M::NS; ++i)
            k[i] = i < M::NC || g < 2 ? *reinterpret_cast<const h8*>(b + M::dim(i, g)) : h8{};
    } else {
        const uint8_t* b = static_cast<const uint8_t*>(p.k) + row;
#pragma unroll
        for (int i = 0; i < M::NC; i += 2) {
            const i4 x = *reinterpret_cast<const i4*>(b + M::dim(i, g));
            k[i] = bytes8_to_h8<KV>((uint32_t)x.x, (uint32_t)x.y);
            k[i + 1] = bytes8_to_h8<KV>((uint32_t)x.z, (uint32_t)x.w);
        }
        if constexpr (M::REM) {
            i2 x = {0, 0};
            if (g < 2) x = *reinterpret_cast<const i2*>(b + M::dim(M::NC, g));
            k[M::NC] = g < 2 ? bytes8_to_h8<KV>((uint32_t)x.x, (uint32_t)x.y) : h8{};
        }
    }
}

// Rows (node, head of the group) held in LDS at a time.
constexpr int kMassRows = 128;

// ONE: at most kMassOneRows rows.  The next positions' block ids are loaded
// beside this step's K.  Four waves a SIMD where the registers allow it without
// scratch (decode 46.8 -> 44.5 us).
template <int KV, int D, bool ONE>
__global__ __launch_bounds__(64 * kMassWaves, D == 64 || (ONE && D == 80 && KV == VCPP_KV_F16) ? 4 : 3) void mass_kernel(TreeParams p) {
    using MD = MassDims<KV, D>;
    constexpr bool SCALED = KV == VCPP_KV_I8;
    constexpr int RBS = ONE ? 1 : kMassRows / 16;
    __shared__ __attribute__((aligned(16))) h8 q_s[ONE ? 1 : RBS][MD::NS][kWave];     // operands as the lanes hold them
    __shared__ __attribute__((aligned(16))) float shift_s[RBS * 16];        // log-sum-exps in log2 units
    __shared__ uint64_t win_s[kMassWaves][RBS * 16];                        // windows of each wave's 64 positions
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, c = lane & 15;
    // The kv heads of one (sequence, part) share an XCD (and its L2's lines).
    const int jj = blockIdx.x >> 3;
    // ONE: head_waves waves take that many heads next to each other, and the same
    // positions; else the waves take 64 positions each of one head.
    const int hw = ONE ? p.head_waves : 1, lanes_of = ONE ? p.num_kv_heads / hw : p.num_kv_heads;
    const int cell = (jj / lanes_of) * 8 + (blockIdx.x & 7);
    const int kvh = ONE ? jj % lanes_of * hw + wave % hw : jj % lanes_of;
    const int at = ONE ? wave / hw : wave;
    const int s = cell / p.parts, part = cell - s * p.parts;
    if (s >= p.num_seqs) return;
    const TreeSeq sq(p, s);
    const int G = p.group, M = sq.n * G;
    const int k_lo = part * p.part_len, k_hi = min(k_lo + p.part_len, sq.end);
    if (M == 0 || k_lo >= k_hi) return;  // whole workgroup
    const int32_t* table = p.block_tables + (int64_t)s * p.max_blocks;
    float* out = p.scores + ((int64_t)s * p.num_kv_heads + kvh) * p.score_stride;

    // Slice i of lane group gg of a row's operand, and the row's log-sum-exp in
    // log2 units (rows past the last, and rows that saw nothing, add exp2(-inf)).
    auto q_of = [&](int row, int i, int gg) {
        const int t = row / G;
        return row < M && (i < MD::NC || gg < 2)
                   ? *reinterpret_cast<const h8*>(
                         reinterpret_cast<const _Float16*>(p.q) +
                         ((int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G)) * D + MD::dim(i, gg))
                   : h8{};
    };
    auto shift_of = [&](int row) {
        const int t = row / G;
        const float x = row < M ? p.lse_in[(int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G)]
                                : -__builtin_inff();
        return x != -__builtin_inff() ? x * kLog2e : __builtin_inff();
    };
    // Rows r0 .. r0 + 16 RBS - 1 into LDS.
    auto stage = [&](int r0) {
        const int units = (min(M - r0, 16 * RBS) + 15) / 16 * MD::NS * kWave;
        constexpr int EACH = (RBS * MD::NS + kMassWaves - 1) / kMassWaves;  // a thread's units, loaded at once
        h8 v[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int u = threadIdx.x + 64 * kMassWaves * j;
            const int l = u & 63, i = u / kWave % MD::NS, rb = u / (kWave * MD::NS);
            v[j] = u < units ? q_of(r0 + 16 * rb + (l & 15), i, l >> 4) : h8{};
        }
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int u = threadIdx.x + 64 * kMassWaves * j;
            if (u < units) (&q_s[0][0][0])[u] = v[j];
        }
        for (int i = threadIdx.x; i < RBS * 16; i += 64 * kMassWaves) shift_s[i] = shift_of(r0 + i);
        __syncthreads();
    };
    // This lane's position of the wave's 64 at k0: its block id (-1: none).
    auto block_of = [&](int k0, int& slot) {
        const int pos = k0 + lane;
        const int lb = (int)(((uint64_t)(uint32_t)pos * p.bs_magic) >> 40);
        slot = pos - lb * p.block_size;
        const int bid = pos < k_hi && lb < p.max_blocks ? table[lb] : -1;
        return bid >= 0 && (int64_t)bid < p.num_blocks ? bid : -1;
    };
    const bool several = !ONE && M > 16 * RBS;
    const int step = kMassKeys * kMassWaves / hw;
    int slot = 0, bid = block_of(k_lo + kMassKeys * at, slot);
    h8 q1[MD::NS];
    f4 shift1 = {0.f, 0.f, 0.f, 0.f};
    for (int base = k_lo; base < k_hi; base += step) {  // (whole workgroup)
        const int k0 = base + kMassKeys * at;
        const bool have = bid >= 0;
        h8 k[kMassTiles][MD::NS];
        float ksc[kMassTiles];
        const int64_t my_row = (int64_t)bid * p.block_stride + ((int64_t)slot * p.num_kv_heads + kvh) * D;
        float my_scale = 0.f;
        if constexpr (SCALED)
            if (have)
                my_scale = (float)__builtin_bit_cast(
                    _Float16, p.k_scale[(int64_t)bid * p.scale_block_stride + (int64_t)kvh * p.block_size + slot]);
        const float before = have ? out[k0 + lane] : 0.f;
#pragma unroll
        for (int kt = 0; kt < kMassTiles; ++kt) {
            const int from = 16 * kt + c;
            const int64_t row = (int64_t)(uint32_t)__shfl((int)my_row, from) | (int64_t)__shfl((int)(my_row >> 32), from) << 32;
            if (__shfl((int)have, from)) load_k<KV, D>(p, row, g, k[kt]);
            else
#pragma unroll
                for (int i = 0; i < MD::NS; ++i) k[kt][i] = h8{};
        }
        if (base + step < k_hi) bid = block_of(k0 + step, slot);
#pragma unroll
        for (int kt = 0; kt < kMassTiles; ++kt) {
            ksc[kt] = p.scale_log2;
            if constexpr (SCALED) ksc[kt] *= shfl(my_scale, 16 * kt + c);
        }
        const bool masked = k0 + kMassKeys > sq.plain;
        float sum[kMassTiles] = {0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < M; r0 += 16 * RBS) {
            if constexpr (ONE) {
                if (base == k_lo) {  // (behind the first K loads)
#pragma unroll
                    for (int i = 0; i < MD::NS; ++i) q1[i] = q_of(c, i, g);
#pragma unroll
                    for (int r = 0; r < 4; ++r) shift1[r] = shift_of(4 * g + r);
                }
            } else if (several || base == k_lo) {
                if (r0 > 0 || base > k_lo) __syncthreads();
                stage(r0);
            }
            const int rows = min(M - r0, 16 * RBS);
            if (masked) {
                for (int i = lane; i < (rows + 15) / 16 * 16; i += kWave) {
                    const int row = r0 + i, t = row / G;
                    const uint64_t* mrow = p.mask ? p.mask + (int64_t)(sq.q0 + t) * p.mask_words : nullptr;
                    win_s[wave][i] = row >= M ? 0
                                              : (uint64_t)tree_window(p, sq, mrow, t, k0 + 32) << 32 |
                                                    tree_window(p, sq, mrow, t, k0);
                }
                asm volatile("" ::: "memory");  // (one wave's LDS accesses are in order)
            }
            for (int rb = 0; rb < (ONE ? 1 : (rows + 15) / 16); ++rb) {
                h8 q[MD::NS];
                f4 shift;
                if constexpr (ONE) {
#pragma unroll
                    for (int i = 0; i < MD::NS; ++i) q[i] = q1[i];
                    shift = shift1;
                } else {
#pragma unroll
                    for (int i = 0; i < MD::NS; ++i) q[i] = q_s[rb][i][lane];
                    shift = *reinterpret_cast<const f4*>(&shift_s[16 * rb + 4 * g]);
                }
                f4 x[kMassTiles];
#pragma unroll
                for (int kt = 0; kt < kMassTiles; ++kt) {
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < MD::NS; ++i) acc = mfma32(q[i], k[kt][i], acc);
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[kt][r] = fmaf(acc[r], ksc[kt], -shift[r]);
                }
                if (masked) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint64_t w = win_s[wave][16 * rb + 4 * g + r] >> c;
#pragma unroll
                        for (int kt = 0; kt < kMassTiles; ++kt)
                            x[kt][r] = (w >> (16 * kt)) & 1 ? x[kt][r] : -__builtin_inff();
                    }
                }
#pragma unroll
                for (int kt = 0; kt < kMassTiles; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sum[kt] += fast_exp2(x[kt][r]);
            }
        }
        // The four lane groups' sums; group g writes tile g.
        float mine = 0.f;
#pragma unroll
        for (int kt = 0; kt < kMassTiles; ++kt) {
            float y = sum[kt];
            y += shfl_xor(y, 32);
            y += shfl_xor(y, 16);
            if (g == kt) mine = y;
        }
        if (have) out[k0 + lane] = before + mine;
    }
}

template <int KV, int D>
hipError_t launch_mass_dim(const TreeParams& p, hipStream_t stream) {
    const int64_t cells = (int64_t)p.num_seqs * p.parts;
    const bool one = p.max_nodes * p.group <= kMassOneRows;
    const int64_t grid = (cells + 7) / 8 * 8 * (one ? p.num_kv_heads / p.head_waves : p.num_kv_heads);
    if (one)
        mass_kernel<KV, D, true><<<dim3((uint32_t)grid), dim3(64 * kMassWaves), 0, stream>>>(p);
    else
        mass_kernel<KV, D, false><<<dim3((uint32_t)grid), dim3(64 * kMassWaves), 0, stream>>>(p);
    return hipGetLastError();
}

template <int KV>
hipError_t launch_mass_kv(const TreeParams& p, hipStream_t stream) {
    switch (p.head_dim) {
        case 64: return launch_mass_dim<KV, 64>(p, stream);
        case 80: return launch_mass_dim<KV, 80>(p, stream);
        case 128: return launch_mass_dim<KV, 128>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_mass(const TreeParams& p, hipStream_t stream) {
    switch (p.kv_dtype) {
        case VCPP_KV_F16: return launch_mass_kv<VCPP_KV_F16>(p, stream);
        case VCPP_KV_I8: return launch_mass_kv<VCPP_KV_I8>(p, stream);
        case VCPP_KV_FP8: return launch_mass_kv<VCPP_KV_FP8>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace vcpp
