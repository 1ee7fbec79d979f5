// tree.hip -- attention of trees of drafted tokens over paged prefixes.
//
// Row (node i, query head h) of a sequence with prefix p sees positions
// 0 .. p - 1 and the positions p + a of the nodes a in node i's mask row:
//   x_j = q . k_j / sqrt(D),  out = sum_j e^(x_j - m) v_j / sum_j e^(x_j - m),
//   lse = m + ln sum_j e^(x_j - m)
// with the skip rules of src/paged_attention.cpp:11-90 (missing and invalid
// blocks) and zeros (lse -inf) for a row that sees nothing.
//
// Work decomposition: the rows of one kv head (node-major, its group's heads
// next to each other) are cut into tiles of WR waves x RB blocks of 16 rows,
// the positions into parts of part_len; a workgroup owns (sequence, part, kv
// head, row tile).  Keys stream in blocks of 32 through a ring of LDS stages
// filled by direct-to-LDS DMA.  Per key block and 16 rows:
//   S^T[32 keys][16 rows] = K x Q^T   (16x16x32 f16)
//   P = exp2(S scale - m)             (fp32)
//   O[16 rows][D] += P x V            (16x16x32 f16, twice)
// Verification has to reproduce what a decode of the accepted tokens computes,
// so P is not rounded to fp16: it enters the matrix product as the sum of two
// fp16 numbers (22 bits of it), and the row sums are fp32 sums of P itself.
// The running exponent leaves 11 bits of headroom below fp16's largest power
// (P <= 2^15), so that the low part of a P of 2^-16 of the row's largest still
// has 19 bits; it moves when a row's largest score grows by more than 2^4.
// int8 pages: K and V are exact fp16 integers; the key's K scale multiplies
// the score, its V scale P (over a running power of two, so that any scale
// keeps P in fp16's range).
#include "prefill_body.h"
#include "profile.h"
#include "tree.h"
#include "tree_mask.h"

namespace vcpp {

namespace {

constexpr float kHead = 11.f;         // log2 of the P that a row's running maximum maps to
constexpr float kTopP = 32768.f;      // 2^15: largest P
constexpr float kTopLog = 15.f;


// Natural log-sum-exp of a row of exponent m (log2 units) and sum l.
__device__ __forceinline__ float row_lse(float m, float l) {
    return l == 0.f ? -__builtin_inff() : (m + __log2f(l)) * 0.6931471805599453f;
}

// x where bit b of w is set, else -inf: a select on integers (compares would
// hold a pair of scalar registers for every element of a block).
__device__ __forceinline__ float seen_or_inf(float x, uint32_t w, int b) {
    const int m = __builtin_amdgcn_sbfe((int)w, b, 1);
    return __int_as_float((__float_as_int(x) & m) | ((int)0xFF800000u & ~m));
}

template <int KV, int D, int RB_, int WR_, int ST>
struct TreeDims {
    static constexpr bool BYTES = KV != VCPP_KV_F16;
    static constexpr bool SCALED = KV == VCPP_KV_I8;
    using DD = DmaDims<D>;
    using ID = ByteDims<D, SCALED>;
    static constexpr int RB = RB_, WR = WR_;
    static constexpr int ROWS = 16 * RB * WR;
    static constexpr int STAGES = ST;
    static constexpr int RSTAGE = BYTES ? ID::STAGE : DD::STAGE;  // bytes of a ring stage
    static constexpr int NINST = BYTES ? ID::NINST : DD::NINST;   // DMA instructions per stage
    static constexpr int PERW = (NINST + WR - 1) / WR;
    static constexpr int AREA = STAGES * RSTAGE;
    static constexpr int NF16 = !BYTES ? STAGES : WR > 1 ? 2 : 1;  // fp16 blocks
    static constexpr int F16BASE = BYTES ? AREA : 0;
    // Marks of drafted V values that are not finite (not int8): [0] any in this
    // piece, [1] any in this block, then a 32-key word per dim, then a bit per
    // (row, dim) of the tile.
    static constexpr int DW = (D + 31) / 32;
    static constexpr int MARKS = AREA + (BYTES ? NF16 * DD::STAGE : 0);
    static constexpr int TABLE = MARKS + (SCALED ? 0 : (2 + D + ROWS * DW) * 4);
    static_assert(STAGES >= 3 && (STAGES - 1) * PERW < 64, "ring depth");
};

template <int N>
__device__ __forceinline__ void wait_dma(bool full) {  // N instructions of this wave may stay in flight
    if (full) wait_vmcnt<N>();
    else wait_vmcnt<0>();
}

template <int WR>
__device__ __forceinline__ void tree_barrier() {
    if constexpr (WR > 1) __syncthreads();
    else asm volatile("" ::: "memory");  // one wave: its LDS accesses are in order
}

#ifndef T_OCC
#define T_OCC 2
#endif
#ifndef T_RB
#define T_RB 2
#endif
#ifndef T_ST
#define T_ST 4
#endif
template <int KV, int D, int RB, int WR, int ST>
__global__ __launch_bounds__(64 * WR, T_OCC) void tree_kernel(TreeParams p) {
    using T = TreeDims<KV, D, RB, WR, ST>;
    using DD = typename T::DD;
    using ID = typename T::ID;
    constexpr bool BYTES = T::BYTES, SCALED = T::SCALED;
    constexpr int NC32 = PDims<D>::NC32, NT = PDims<D>::NT, REM = PDims<D>::REM;
    extern __shared__ __attribute__((aligned(16))) char tree_lds[];
    lds_char* lds = (lds_char*)tree_lds;
    const uint32_t lds_addr = (uint32_t)(uintptr_t)lds;
    __attribute__((address_space(3))) int32_t* table_s =
        reinterpret_cast<__attribute__((address_space(3))) int32_t*>(lds + T::TABLE);
    __attribute__((address_space(3))) uint32_t* marks =
        reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(lds + T::MARKS);
    __attribute__((address_space(3))) uint32_t* bad_dims = marks + 2;
    __attribute__((address_space(3))) uint32_t* bad_outs = bad_dims + D;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    // Consecutive workgroups go to the 8 XCDs in turn: the kv heads of one
    // range share an XCD, whose L2 then holds the lines that neighbouring
    // heads' rows share.
    const int jj = blockIdx.x >> 3;
    const int kvh = jj % p.num_kv_heads;
    const int range = (jj / p.num_kv_heads) * 8 + (blockIdx.x & 7);
    const TreeRanges cut(p, T::ROWS, lane);
    if (range >= cut.R || cut.total == 0) return;  // whole workgroup
    const int64_t lo = cut.start(range), hi = cut.start(range + 1);
    int64_t first;  // first block of sequence s
    int s = cut.seq_of(p, T::ROWS, lane, lo, first);
    const int G = p.group;
    int64_t at_block = lo;
    while (at_block < hi) {  // the range's pieces, one per unit
    const TreeSeq sq(p, s);
    const int M = sq.n * G;
    const int tiles = (M + T::ROWS - 1) / T::ROWS, blocks = (sq.end + 31) / 32;
    if (at_block >= first + (int64_t)tiles * blocks) {  // next sequence
        first += (int64_t)tiles * blocks;
        ++s;
        continue;
    }
    const int rt = (int)((at_block - first) / blocks);
    const int64_t unit0 = first + (int64_t)rt * blocks;  // the unit's first block
    const int kb_lo = (int)(at_block - unit0);
    const int kb_hi = (int)min((int64_t)blocks, hi - unit0);
    const bool whole = kb_lo == 0 && kb_hi == blocks;
    const int64_t piece = (int64_t)range * 2 + (at_block > lo ? 1 : 0);  // partials' place (not whole)
    at_block = unit0 + kb_hi;
    const int row0 = rt * T::ROWS;
    const int k_lo = kb_lo * kKBlk, k_hi = min(kb_hi * kKBlk, sq.end);

    // Q fragments (B operand): row row0 + 16 (RB wave + rb) + c
    h8 qa[RB][NC32 > 0 ? NC32 : 1];
    h8 qr[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * (RB * wave + rb) + c;
        const bool ok = row < M;
        const int t = ok ? row / G : 0;
        const _Float16* qrow = reinterpret_cast<const _Float16*>(p.q) +
                               ((int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (ok ? row - t * G : 0)) * D;
#pragma unroll
        for (int cc = 0; cc < NC32; ++cc)
            qa[rb][cc] = ok ? *reinterpret_cast<const h8*>(qrow + 32 * cc + 8 * g) : h8{};
        if constexpr (REM) qr[rb] = ok && g < 2 ? *reinterpret_cast<const h8*>(qrow + 32 * NC32 + 8 * g) : h8{};
    }
    if (tid < T::NF16)
        *reinterpret_cast<__attribute__((address_space(3))) h8*>(lds + T::F16BASE + tid * DD::STAGE + DD::ZERO) = h8{};
    if constexpr (!SCALED)
        for (int i = tid; i < 2 + D + T::ROWS * T::DW; i += 64 * WR) marks[i] = 0;
    // The piece's block ids (-1: missing or outside the pool).
    const int32_t* table = p.block_tables + (int64_t)s * p.max_blocks;
    const int lb0 = k_lo / p.block_size;
    const int npages = min((k_hi - 1) / p.block_size + 1 - lb0, p.table_cap);
    int bad = 0;
    for (int i = tid; i < npages; i += 64 * WR) {
        const int bid = lb0 + i < p.max_blocks ? table[lb0 + i] : -1;
        const bool ok = bid >= 0 && (int64_t)bid < p.num_blocks;
        table_s[i] = ok ? bid : -1;
        bad |= !ok;
    }
    const bool any_bad = __syncthreads_or(bad) != 0;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the ring's DMA is not in the compiler's count

    // DMA: instruction j = wave + WR i fills slots 64 j + lane of a stage (see
    // prefill_tile for the layouts).
    const int my_inst = T::NINST % WR == 0 || wave < T::NINST % WR ? T::PERW : T::PERW - 1;
    const int dkey = BYTES ? lane & 31 : (lane & 31) ^ ((lane >> 5) * kSwz);
    auto issue = [&](int kb) {
        const uint32_t sbase = lds_addr + (kb % T::STAGES) * T::RSTAGE;
        const int pos = kb * kKBlk + dkey;
        int64_t off = -1, soff = 0;
        if (pos < k_hi) {
            const int lb = (int)(((uint64_t)(uint32_t)pos * p.bs_magic) >> 40);
            const int bid = table_s[lb - lb0];
            if (bid >= 0) {
                const int slot = pos - lb * p.block_size;
                off = (int64_t)bid * p.block_stride + ((int64_t)slot * p.num_kv_heads + kvh) * D;
                if constexpr (!BYTES) off = off * 2 + (lane >> 5) * 16;
                if constexpr (SCALED)
                    soff = ((int64_t)bid * p.scale_block_stride + (int64_t)kvh * p.block_size + slot) * 2;
            }
        }
#pragma unroll
        for (int i = 0; i < T::PERW; ++i) {
            if (i < my_inst) {
                const int j = wave + WR * i;
                const uint32_t dst = __builtin_amdgcn_readfirstlane(sbase + j * 1024);
                if constexpr (!BYTES) {
                    const int which = j >= DD::REGION / 64;
                    const int cp = j - which * (DD::REGION / 64);
                    const char* base = static_cast<const char*>(which ? p.v : p.k) + cp * 32;
                    dma16(off >= 0 ? (const void*)(base + off) : (const void*)kZeroChunk, dst);
                } else if (j < ID::NDATA) {
                    const int sl = 64 * j + lane;
                    const int which = sl >= ID::REGION;
                    const int ch = (sl - which * ID::REGION) >> 5;
                    const char* base = static_cast<const char*>(which ? p.v : p.k) + ch * 16;
                    dma16(off >= 0 ? (const void*)(base + off) : (const void*)kZeroChunk, dst);
                } else {
                    const char* base = reinterpret_cast<const char*>(lane >> 5 ? p.v_scale : p.k_scale);
                    dma2(off >= 0 ? (const void*)(base + soff) : (const void*)kZeroChunk,
                         __builtin_amdgcn_readfirstlane(sbase + ID::SCALES));
                }
            }
        }
    };
    // Byte block kb -> fp16 values (int8: exact integers); its scales -> fp32
    // (K's times log2(e) / sqrt(D)).
    auto widen = [&](int kb) {
        lds_char* st = lds + (kb % T::STAGES) * T::RSTAGE;
        if constexpr (SCALED) {
            if (tid < 64) {
                lds_char* sw = st + ID::SCALES + tid * 4;
                const float x = (float)__builtin_bit_cast(
                    _Float16, *reinterpret_cast<__attribute__((address_space(3))) const uint16_t*>(sw));
                *reinterpret_cast<__attribute__((address_space(3))) float*>(sw) = tid < 32 ? x * p.scale_log2 : x;
            }
        }
        lds_char* dst0 = lds + T::AREA + (kb % T::NF16) * DD::STAGE;
#pragma unroll 2
        for (int u0 = 0; u0 < ID::UNITS; u0 += 64 * WR) {
            const int u = u0 + tid;
            if (ID::UNITS % (64 * WR) == 0 || u < ID::UNITS) {
                const int which = u >= ID::REGION;
                const int q = u - which * ID::REGION;
                const int ch = q >> 5, key = q & 31;
                const i4 raw = *reinterpret_cast<__attribute__((address_space(3))) i4*>(st + u * 16);
                lds_char* dst = dst0 + which * DD::REGION * 16;
                *reinterpret_cast<__attribute__((address_space(3))) h8*>(dst + slot_of(2 * ch, key) * 16) =
                    bytes8_to_h8<KV>((uint32_t)raw.x, (uint32_t)raw.y);
                *reinterpret_cast<__attribute__((address_space(3))) h8*>(dst + slot_of(2 * ch + 1, key) * 16) =
                    bytes8_to_h8<KV>((uint32_t)raw.z, (uint32_t)raw.w);
            }
        }
    };

    // A drafted V row that is not finite must not reach the rows that do not see
    // it (0 x inf in the matrix product): such values of block kb are replaced
    // by 0 in LDS, and the outputs that attend them are marked, to become NaN
    // at the end.  (Only blocks that reach into a tree; in registers and
    // unrolled this cost the main loop 60 of them.)
    auto scrub = [&](int kb) {
        lds_char* vs = (BYTES ? lds + T::AREA + (kb % T::NF16) * DD::STAGE : lds + (kb % T::STAGES) * DD::STAGE) +
                       DD::REGION * 16;
#pragma unroll 1
        for (int u = tid; u < DD::REGION; u += 64 * WR) {
            const int ch = u >> 5, key = (u & 31) ^ ((ch & 1) * kSwz);
            __attribute__((address_space(3))) uint16_t* e =
                reinterpret_cast<__attribute__((address_space(3))) uint16_t*>(vs + u * 16);
#pragma unroll 1
            for (int i = 0; i < 8; ++i)
                if ((e[i] & 0x7C00u) == 0x7C00u) {
                    e[i] = 0;
                    marks[0] = marks[1] = 1;
                    __hip_atomic_fetch_or(&bad_dims[8 * ch + i], 1u << key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                }
        }
        __syncthreads();
        if (marks[1]) {
#pragma unroll 1
            for (int i = tid; i < T::ROWS; i += 64 * WR) {
                const int row = row0 + i, t = row / G;
                if (row >= M) continue;
                const uint32_t w = tree_window(
                    p, sq, p.mask ? p.mask + (int64_t)(sq.q0 + t) * p.mask_words : nullptr, t, kb * kKBlk);
                for (int d = 0; d < D; ++d)
                    if (w & bad_dims[d]) bad_outs[i * T::DW + d / 32] |= 1u << (d & 31);
            }
            __syncthreads();
            for (int i = 1 + tid; i < 2 + D; i += 64 * WR) marks[i] = 0;
            __syncthreads();
        }
    };

    f4 o[RB][NT];
    float lsum[RB], m_run[RB];  // (m_run: the exponent that maps to P = 1)
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int t = 0; t < NT; ++t) o[rb][t] = f4{0.f, 0.f, 0.f, 0.f};
        lsum[rb] = 0.f;
        m_run[rb] = kMaxSeed;
    }
    float vcap = 0.f, vinv = 0.f;  // int8: power of two at or above every finite V scale so far, and its inverse

    const int kbase = (32 * g + (c ^ ((g & 1) * kSwz))) * 16;
    const int rpar = (4 * NC32 + g) & 1;
    const int krb0 = g < 2 ? ((4 * NC32 + g) * 32 + (c ^ (rpar * kSwz))) * 16 : DD::ZERO;
    const int krb1 = g < 2 ? krb0 + 16 * 16 : krb0;
    const int vpar = (c >> 1) & 1;
    const int vbase = DD::REGION * 16 + (((c & 3) >> 1) * 32 + ((4 * g + (c >> 2)) ^ (vpar * kSwz))) * 16 + 8 * (c & 1);

    // One body for masked and free blocks (the mask's parts behind uniform
    // branches): two inlined forms held 50 registers more and spilled.
    auto compute = [&](int kb, const bool masked) {
        lds_char* sb = BYTES ? lds + T::AREA + (kb % T::NF16) * DD::STAGE : lds + (kb % T::STAGES) * DD::STAGE;
        const int key0 = kb * kKBlk;
        h8 ka[2][NC32 > 0 ? NC32 : 1];
        h8 kr[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int cc = 0; cc < NC32; ++cc)
                ka[kt][cc] = *reinterpret_cast<__attribute__((address_space(3))) h8*>(sb + kbase + (128 * cc + 16 * kt) * 16);
            if constexpr (REM)
                kr[kt] = *reinterpret_cast<__attribute__((address_space(3))) h8*>(sb + (kt ? krb1 : krb0));
        }
        // Scales of this lane's keys 16 kt + 4 g + r.
        float ksc[2][4], vsc[2][4];
        if constexpr (SCALED) {
            const lds_char* sp = lds + (kb % T::STAGES) * T::RSTAGE + ID::SCALES;
            float top = 0.f;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const f4 a = *reinterpret_cast<__attribute__((address_space(3))) const f4*>(sp + (16 * kt + 4 * g) * 4);
                const f4 b = *reinterpret_cast<__attribute__((address_space(3))) const f4*>(sp + (32 + 16 * kt + 4 * g) * 4);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    ksc[kt][r] = a[r];
                    vsc[kt][r] = b[r];
                    const float x = fabsf(b[r]);
                    if (x < 65536.f) top = fmaxf(top, x);  // (finite)
                }
            }
            if (__any(top > vcap)) {
                top = fmaxf(top, shfl_xor(top, 16));
                top = fmaxf(top, shfl_xor(top, 32));
                const uint32_t up = (__float_as_uint(top) + 0x7FFFFFu) & 0x7F800000u;  // (fp16 scales are normal in fp32)
                const float cap = fmaxf(__uint_as_float(up), vcap);
                const float down = vcap / cap;
                vcap = cap;
                vinv = 1.f / cap;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[rb][t] *= down;
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) vsc[kt][r] *= vinv;
        }
        uint32_t win[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) win[rb] = ~0u;
        if (masked) {
            uint32_t pages = ~0u;  // positions on missing pages leave
            if (any_bad) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const int k16 = key0 + 16 * kt;
                    if (k16 < k_hi && table_s[k16 / p.block_size - lb0] < 0) pages &= kt ? 0xFFFFu : 0xFFFF0000u;
                }
            }
            const bool tree = key0 + kKBlk > sq.plain;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                if (tree) {
                    const int row = row0 + 16 * (RB * wave + rb) + c, node = row / G;
                    win[rb] = row < M ? tree_window(p, sq, p.mask ? p.mask + (int64_t)(sq.q0 + node) * p.mask_words : nullptr,
                                                    node, key0)
                                      : 0u;
                }
                win[rb] &= pages;
            }
        }
        f4 sc[RB][2];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int cc = 0; cc < NC32; ++cc) acc = mfma32(ka[kt][cc], qa[rb][cc], acc);
                if constexpr (REM) acc = mfma32(kr[kt], qr[rb], acc);
                sc[rb][kt] = acc;
            }
        // (V's registers after K's: both at once pass 256 at head_dim 128)
        __builtin_amdgcn_sched_barrier(0);
        h8 vb[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const h4 lo = read_tr(sb + vbase + 64 * t * 16);
            const h4 hi = read_tr(sb + vbase + (64 * t + 16) * 16);
            vb[t] = h8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float pf[2][4];
            const uint32_t w4 = win[rb] >> (4 * g);
            auto exps = [&]() {
                float b = 0.f;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        pf[kt][r] = fmaf(sc[rb][kt][r], SCALED ? ksc[kt][r] : p.scale_log2, -m_run[rb]);
                if (masked)
#pragma unroll
                    for (int e = 0; e < 8; ++e) pf[e >> 2][e & 3] = seen_or_inf(pf[e >> 2][e & 3], w4, 16 * (e >> 2) + (e & 3));
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        pf[kt][r] = fast_exp2(pf[kt][r]);
                        b += pf[kt][r];
                    }
                return b;
            };
            float bs = exps();
            if (__builtin_expect(__any(!(bs <= kTopP)), 0)) {  // a score past the headroom (inf and NaN too)
                float ml = -__builtin_inff();
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float x = sc[rb][kt][r] * (SCALED ? ksc[kt][r] : p.scale_log2);
                        ml = vmax(ml, seen_or_inf(x, w4, 16 * kt + r));
                    }
                ml = max_over_groups(ml);
                const bool grow = ml > m_run[rb] + kTopLog;  // uniform per row
                const float m_new = grow ? ml - kHead : m_run[rb];
                const float alpha = fast_exp2(m_run[rb] - m_new);
                m_run[rb] = m_new;
                lsum[rb] *= alpha;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float a = shfl(alpha, 4 * g + r);
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[rb][t][r] *= a;
                }
                bs = exps();
            }
            lsum[rb] += bs;
            h8 ph, pl;
            if constexpr (SCALED) {
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e >> 2][e & 3] *= vsc[e >> 2][e & 3];
                if (masked)  // (the scale of a row that is not seen may be anything)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        pf[e >> 2][e & 3] = __int_as_float(__float_as_int(pf[e >> 2][e & 3]) &
                                                           __builtin_amdgcn_sbfe((int)w4, 16 * (e >> 2) + (e & 3), 1));
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = pf[kt][r];
                    if constexpr (SCALED) {
                        // Both parts come from the rounded product: fused with
                        // it, the high part may round another way than the one
                        // that the low part is the rest of.
                        asm("" : "+v"(x));
                    }
                    const _Float16 h = (_Float16)x;
                    ph[4 * kt + r] = h;
                    pl[4 * kt + r] = (_Float16)(x - (float)h);
                }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                o[rb][t] = mfma32(ph, vb[t], o[rb][t]);
                o[rb][t] = mfma32(pl, vb[t], o[rb][t]);
            }
        }
    };

    // Blocks in front of the tree (and on valid pages) need no mask.
    const int free_hi = any_bad ? kb_lo : max(kb_lo, min(kb_hi, sq.plain / kKBlk));
    const bool busy = row0 + 16 * RB * wave < M;  // (a wave past the last row only moves data)
    constexpr int S = T::STAGES;
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
        if (kb_lo + i < kb_hi) issue(kb_lo + i);
    // Before block kb is used: the blocks after it that may stay in flight.
    auto land = [&](int kb) {
        if (my_inst == T::PERW) wait_dma<(S - 2) * T::PERW>(kb + S - 2 < kb_hi);
        else wait_dma<(S - 2) * (T::PERW - 1)>(kb + S - 2 < kb_hi);
    };
    if constexpr (BYTES && WR > 1) {
        land(kb_lo);
        __syncthreads();
        if (kb_lo < kb_hi) widen(kb_lo);
    }
    auto step = [&](int kb) {
        if constexpr (BYTES && WR > 1) {
            // block kb + 1 landed for every wave, kb widened, kb - 1 used up
            if (my_inst == T::PERW) wait_dma<(S - 3) * T::PERW>(kb + S - 2 < kb_hi);
            else wait_dma<(S - 3) * (T::PERW - 1)>(kb + S - 2 < kb_hi);
            __syncthreads();
            if (kb + S - 1 < kb_hi) issue(kb + S - 1);
            if (kb + 1 < kb_hi) widen(kb + 1);
        } else {
            land(kb);
            tree_barrier<WR>();  // block kb landed for every wave, kb - 1 used up
            if (kb + S - 1 < kb_hi) issue(kb + S - 1);
            if constexpr (BYTES) {
                widen(kb);
                tree_barrier<WR>();
            }
        }
    };
    for (int kb = kb_lo; kb < kb_hi; ++kb) {
        step(kb);
        if constexpr (!SCALED)
            if (kb * kKBlk + kKBlk > sq.plain) scrub(kb);
        if (busy) compute(kb, kb >= free_hi);
    }

    const float vmul = SCALED ? vcap : 1.f;
    const int64_t pbase = (piece * p.num_kv_heads + kvh) * T::ROWS;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float l = sum_over_groups(lsum[rb]);  // row c
        const int w16 = 16 * (RB * wave + rb);
        if (g == 0 && row0 + w16 + c < M) {
            const int row = row0 + w16 + c, t = row / G;
            if (!whole) p.ws_ml[pbase + w16 + c] = make_float2(m_run[rb], l);
            else if (p.lse)
                p.lse[(int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G)] = row_lse(m_run[rb], l);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + w16 + 4 * g + r;
            const float lr = shfl(l, 4 * g + r);
            const float mul = !whole ? vmul : lr == 0.f ? 0.f : vmul / lr;
            if (row < M) {
                const int t = row / G;
                float* orow = !whole ? p.ws_o + (pbase + w16 + 4 * g + r) * D
                                     : p.out + ((int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G)) * D;
#pragma unroll
                for (int tt = 0; tt < NT; ++tt) orow[16 * tt + c] = o[rb][tt][r] * mul;
            }
        }
    }
    if constexpr (!SCALED)
        if (marks[0]) {
#pragma unroll 1
            for (int i = lane; i < 16 * RB * D; i += 64) {
                const int w = 16 * RB * wave + i / D, d = i % D, row = row0 + w, t = row / G;
                if (row >= M || !(bad_outs[w * T::DW + d / 32] >> (d & 31) & 1)) continue;
                (!whole ? p.ws_o + (pbase + w) * D
                        : p.out + ((int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G)) * D)[d] = __builtin_nanf("");
            }
        }
    if constexpr (WR > 1) __syncthreads();  // the ring and the block ids are free for the next piece
    }  // pieces
}

// Joins the pieces of each row that a range's end cut: thread (row, head, 4 dims).
template <int ROWS>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
    const int s = blockIdx.x / p.max_nodes, t = blockIdx.x - s * p.max_nodes;
    const TreeSeq sq(p, s);
    if (t >= sq.n) return;
    const TreeRanges cut(p, ROWS, threadIdx.x & 63);
    const int64_t first = cut.first_of(p, ROWS, threadIdx.x & 63, s);
    const int D4 = p.head_dim / 4;
    const int e = blockIdx.y * 256 + threadIdx.x;
    const int h = e / D4, d = e - h * D4;
    if (h >= p.num_heads) return;
    const int kvh = h / p.group, row = t * p.group + (h - kvh * p.group);
    const int blocks = (sq.end + 31) / 32;
    const int64_t unit0 = first + (int64_t)(row / ROWS) * blocks;
    const int r0 = cut.range_of(unit0), r1 = cut.range_of(unit0 + blocks - 1);
    if (r0 == r1) return;  // whole in one range
    const int64_t head0 = (int64_t)kvh * ROWS + row % ROWS, step = (int64_t)p.num_kv_heads * ROWS;
    const int64_t at0 = (r0 * 2 + (cut.start(r0) < unit0 ? 1 : 0)) * step + head0;
    const auto at = [&](int r) { return r == r0 ? at0 : r * 2 * step + head0; };
    float m = kMaxSeed;
    for (int r = r0; r <= r1; ++r) m = fmaxf(m, p.ws_ml[at(r)].x);
    float l = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    for (int r = r0; r <= r1; ++r) {
        const float2 ml = p.ws_ml[at(r)];
        const float w = fast_exp2(ml.x - m);
        l += ml.y * w;
        o += *reinterpret_cast<const f4*>(p.ws_o + (at(r) * D4 + d) * 4) * w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t to = (int64_t)(sq.q0 + t) * p.num_heads + h;
    *reinterpret_cast<f4*>(p.out + (to * D4 + d) * 4) = o * inv;
    if (d == 0 && p.lse) p.lse[to] = row_lse(m, l);
}

template <int KV, int D, int RB, int WR, int ST>
hipError_t launch_tile(const TreeParams& p, hipStream_t stream) {
    using T = TreeDims<KV, D, RB, WR, ST>;
    const size_t lds = T::TABLE + (size_t)p.table_cap * 4;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)tree_kernel<KV, D, RB, WR, ST>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int64_t grid = (int64_t)(p.ranges + 7) / 8 * 8 * p.num_kv_heads;
    tree_kernel<KV, D, RB, WR, ST><<<dim3((uint32_t)grid), dim3(64 * WR), lds, stream>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.ranges == 1) return e;
    const uint32_t chunks = (uint32_t)((p.num_heads * (p.head_dim / 4) + 255) / 256);
    tree_merge_kernel<T::ROWS><<<dim3((uint32_t)(p.num_seqs * p.max_nodes), chunks), dim3(256), 0, stream>>>(p);
    return hipGetLastError();
}

// Tiles of a shape: RB row blocks per wave and WR waves by the rows of a tree.
template <int KV, int D>
hipError_t launch_shape(const TreeParams& p, hipStream_t stream) {
    constexpr int RB = D <= 80 ? T_RB : 2;
    switch (tree_tile_rows(KV, D, p.max_nodes * p.group)) {
        case 16: return launch_tile<KV, D, 1, 1, 3>(p, stream);
        case 32: return launch_tile<KV, D, 2, 1, 3>(p, stream);
        case 64: return launch_tile<KV, D, RB, 4 / RB, 3>(p, stream);
        case 128: return launch_tile<KV, D, RB, 8 / RB, T_ST>(p, stream);
        default: return launch_tile<KV, D, RB, 4, T_ST>(p, stream);
    }
}

template <int KV>
hipError_t launch_dim(const TreeParams& p, hipStream_t stream) {
    switch (p.head_dim) {
        case 64: return launch_shape<KV, 64>(p, stream);
        case 80: return launch_shape<KV, 80>(p, stream);
        case 128: return launch_shape<KV, 128>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

int tree_tile_rows(int kv_dtype, int head_dim, int rows) {
    const int most = 64 * (head_dim <= 80 ? T_RB : 2);
    for (int t = 16; t < most; t *= 2)
        if (rows <= t) return t;
    return most;
}

int tree_wgs_per_cu(int kv_dtype, int head_dim, int rows) {
    const int t = tree_tile_rows(kv_dtype, head_dim, rows);
    return t <= (head_dim <= 80 ? 64 : 32) ? 4 : 2;
}

hipError_t launch_tree(const TreeParams& p, hipStream_t stream) {
    switch (p.kv_dtype) {
        case VCPP_KV_F16: return launch_dim<VCPP_KV_F16>(p, stream);
        case VCPP_KV_I8: return launch_dim<VCPP_KV_I8>(p, stream);
        case VCPP_KV_FP8: return launch_dim<VCPP_KV_FP8>(p, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace vcpp
