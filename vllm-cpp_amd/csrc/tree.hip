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

typedef uint16_t us8 __attribute__((ext_vector_type(8)));

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
    static constexpr int TABLE = AREA + (BYTES ? NF16 * DD::STAGE : 0);
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

template <int KV, int D, int RB, int WR, int ST>
__global__ __launch_bounds__(64 * WR) void tree_kernel(TreeParams p) {
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

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    // Consecutive workgroups go to the 8 XCDs in turn: the kv heads and row
    // tiles of one (sequence, part) share an XCD, whose L2 then holds the
    // lines that neighbouring heads' rows share.
    const int per = p.num_kv_heads * p.row_tiles;
    const int jj = blockIdx.x >> 3;
    const int cell = (jj / per) * 8 + (blockIdx.x & 7);
    const int within = jj % per;
    const int part = cell / p.num_seqs, s = cell - part * p.num_seqs;
    if (part >= p.parts) return;  // whole workgroup
    const int kvh = within / p.row_tiles, rt = within - kvh * p.row_tiles;
    const TreeSeq sq(p, s);
    const int G = p.group, M = sq.n * G;
    const int row0 = rt * T::ROWS;
    const int k_lo = part * p.part_len;
    if (row0 >= M || (part > 0 && k_lo >= sq.end)) return;  // whole workgroup
    const int k_hi = min(k_lo + p.part_len, sq.end);
    const int kb_lo = k_lo / kKBlk, kb_hi = (k_hi + kKBlk - 1) / kKBlk;

    // Q fragments (B operand): row row0 + 16 (RB wave + rb) + c
    h8 qa[RB][NC32 > 0 ? NC32 : 1];
    h8 qr[RB];
    int node[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * (RB * wave + rb) + c;
        const bool ok = row < M;
        const int t = ok ? row / G : 0;
        node[rb] = ok ? t : -1;
        const _Float16* qrow = reinterpret_cast<const _Float16*>(p.q) +
                               ((int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (ok ? row - t * G : 0)) * D;
#pragma unroll
        for (int cc = 0; cc < NC32; ++cc)
            qa[rb][cc] = ok ? *reinterpret_cast<const h8*>(qrow + 32 * cc + 8 * g) : h8{};
        if constexpr (REM) qr[rb] = ok && g < 2 ? *reinterpret_cast<const h8*>(qrow + 32 * NC32 + 8 * g) : h8{};
    }
    if (tid < T::NF16)
        *reinterpret_cast<__attribute__((address_space(3))) h8*>(lds + T::F16BASE + tid * DD::STAGE + DD::ZERO) = h8{};
    // The part's block ids (-1: missing or outside the pool).
    const int32_t* table = p.block_tables + (int64_t)s * p.max_blocks;
    const int lb0 = k_lo / p.block_size;
    const int npages = k_hi > k_lo ? (k_hi - 1) / p.block_size + 1 - lb0 : 0;
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
#pragma unroll
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

    auto compute = [&](int kb, auto masked_tag) {
        constexpr bool MASKED = decltype(masked_tag)::value;
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
        h8 vb[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const h4 lo = read_tr(sb + vbase + 64 * t * 16);
            const h4 hi = read_tr(sb + vbase + (64 * t + 16) * 16);
            vb[t] = h8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
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
        bool tile_ok[2] = {true, true};
        if constexpr (MASKED) {
            if (any_bad) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const int k16 = key0 + 16 * kt;
                    tile_ok[kt] = k16 < k_hi && table_s[k16 / p.block_size - lb0] >= 0;
                }
            }
        }
        uint32_t win[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            win[rb] = 0;
            if constexpr (MASKED) {
                if (node[rb] >= 0) {
                    const uint64_t* mrow = p.mask ? p.mask + (int64_t)(sq.q0 + node[rb]) * p.mask_words : nullptr;
                    win[rb] = tree_window(p, sq, mrow, node[rb], key0);
                }
                if (!tile_ok[0]) win[rb] &= 0xFFFF0000u;
                if (!tile_ok[1]) win[rb] &= 0x0000FFFFu;
            }
        }
        // A drafted V row that is not finite must not reach the rows that do not
        // see it (0 x inf in the matrix product): such values leave the product,
        // and the rows that do see them get NaN where a product of the rows'
        // visible bits and the values' flags is not zero.
        if constexpr (MASKED && !SCALED) {
            uint32_t any = 0;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const us8 e = __builtin_bit_cast(us8, vb[t]) & (uint16_t)0x7C00;
                const i4 w = __builtin_bit_cast(i4, (us8)(e == (uint16_t)0x7C00));
                any |= (uint32_t)(w.x | w.y | w.z | w.w);
            }
            if (__any(any != 0)) {
                h8 seen[RB];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        seen[rb][e] = (_Float16)(int)(win[rb] >> (16 * (e >> 2) + 4 * g + (e & 3)) & 1);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const us8 x = __builtin_bit_cast(us8, vb[t]);
                    const us8 not_fin = (us8)((x & (uint16_t)0x7C00) == (uint16_t)0x7C00);
                    const h8 flag = __builtin_bit_cast(h8, (us8)(not_fin & (uint16_t)0x3C00));
                    vb[t] = __builtin_bit_cast(h8, (us8)(x & ~not_fin));
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        const f4 hit = mfma32(seen[rb], flag, f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[rb][t][r] = hit[r] > 0.f ? __builtin_nanf("") : o[rb][t][r];
                    }
                }
            }
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float sc[2][4], pf[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int cc = 0; cc < NC32; ++cc) acc = mfma32(ka[kt][cc], qa[rb][cc], acc);
                if constexpr (REM) acc = mfma32(kr[kt], qr[rb], acc);
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[kt][r] = acc[r];
            }
            const uint32_t w4 = win[rb] >> (4 * g);
            auto exps = [&]() {
                float b = 0.f;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float x = fmaf(sc[kt][r], SCALED ? ksc[kt][r] : p.scale_log2, -m_run[rb]);
                        if constexpr (MASKED) x = (w4 >> (16 * kt + r)) & 1 ? x : -__builtin_inff();
                        pf[kt][r] = fast_exp2(x);
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
                        float x = sc[kt][r] * (SCALED ? ksc[kt][r] : p.scale_log2);
                        if constexpr (MASKED) x = (w4 >> (16 * kt + r)) & 1 ? x : -__builtin_inff();
                        ml = vmax(ml, x);
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
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = pf[kt][r];
                    if constexpr (SCALED) {
                        x *= vsc[kt][r];
                        if constexpr (MASKED) x = (w4 >> (16 * kt + r)) & 1 ? x : 0.f;
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
    const int free_hi = any_bad ? kb_lo : (int)max((int64_t)kb_lo, min((int64_t)kb_hi, sq.prefix / kKBlk));
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
    for (int kb = kb_lo; kb < free_hi; ++kb) {
        step(kb);
        compute(kb, std::false_type{});
    }
    for (int kb = free_hi; kb < kb_hi; ++kb) {
        step(kb);
        compute(kb, std::true_type{});
    }

    const float vmul = SCALED ? vcap : 1.f;
    const bool split = p.parts > 1;
    const int64_t pbase = (int64_t)part * p.rows_cap;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float l = sum_over_groups(lsum[rb]);  // row c
        const int r16 = row0 + 16 * (RB * wave + rb);
        if (g == 0 && r16 + c < M) {
            const int t = (r16 + c) / G;
            const int64_t at = (int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (r16 + c - t * G);
            if (split) p.ws_ml[pbase * p.num_heads + at] = make_float2(m_run[rb], l);
            else if (p.lse) p.lse[at] = l == 0.f ? -__builtin_inff() : (m_run[rb] + __log2f(l)) * 0.6931471805599453f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = r16 + 4 * g + r;
            const float lr = shfl(l, 4 * g + r);
            const float mul = split ? vmul : lr == 0.f ? 0.f : vmul / lr;
            if (row < M) {
                const int t = row / G;
                const int64_t at = (int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G);
                float* orow = split ? p.ws_o + (pbase * p.num_heads + at) * D : p.out + at * D;
#pragma unroll
                for (int tt = 0; tt < NT; ++tt) orow[16 * tt + c] = o[rb][tt][r] * mul;
            }
        }
    }
}

// Joins the parts of each row: thread (row, head, 4 dims).
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
    const int s = blockIdx.x / p.max_nodes, t = blockIdx.x - s * p.max_nodes;
    const TreeSeq sq(p, s);
    if (t >= sq.n) return;
    const int D4 = p.head_dim / 4;
    const int e = blockIdx.y * 256 + threadIdx.x;
    const int h = e / D4, d = e - h * D4;
    if (h >= p.num_heads) return;
    const int64_t at = (int64_t)(sq.q0 + t) * p.num_heads + h, step = p.rows_cap * p.num_heads;
    const int live = max(1, (sq.end + p.part_len - 1) / p.part_len);
    float m = kMaxSeed;
    for (int k = 0; k < live; ++k) m = fmaxf(m, p.ws_ml[k * step + at].x);
    float l = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < live; ++k) {
        const float2 ml = p.ws_ml[k * step + at];
        const float w = fast_exp2(ml.x - m);
        l += ml.y * w;
        o += *reinterpret_cast<const f4*>(p.ws_o + ((k * step + at) * D4 + d) * 4) * w;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<f4*>(p.out + (at * D4 + d) * 4) = o * inv;
    if (d == 0 && p.lse) p.lse[at] = l == 0.f ? -__builtin_inff() : (m + __log2f(l)) * 0.6931471805599453f;
}

template <int KV, int D, int RB, int WR, int ST>
hipError_t launch_tile(const TreeParams& p, hipStream_t stream) {
    using T = TreeDims<KV, D, RB, WR, ST>;
    const int entries = p.part_len / p.block_size + 2;
    const size_t lds = T::TABLE + (size_t)entries * 4;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)tree_kernel<KV, D, RB, WR, ST>,
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int64_t cells = (int64_t)p.num_seqs * p.parts;
    const int64_t grid = (cells + 7) / 8 * 8 * p.num_kv_heads * p.row_tiles;
    tree_kernel<KV, D, RB, WR, ST><<<dim3((uint32_t)grid), dim3(64 * WR), lds, stream>>>(p);
    return hipGetLastError();
}

// Tiles of a shape: RB row blocks per wave and WR waves by the rows of a tree.
template <int KV, int D>
hipError_t launch_shape(const TreeParams& p, hipStream_t stream) {
    switch (tree_tile_rows(KV, D, p.max_nodes * p.group)) {
        case 16: return launch_tile<KV, D, 1, 1, 3>(p, stream);
        case 32: return launch_tile<KV, D, 2, 1, 3>(p, stream);
        case 64: return D <= 80 ? launch_tile<KV, D, D <= 80 ? 4 : 2, D <= 80 ? 1 : 2, 3>(p, stream)
                                : launch_tile<KV, D, 2, 2, 3>(p, stream);
        case 128: return D <= 80 ? launch_tile<KV, D, D <= 80 ? 4 : 2, D <= 80 ? 2 : 4, 4>(p, stream)
                                 : launch_tile<KV, D, 2, 4, 4>(p, stream);
        default: return launch_tile<KV, D, D <= 80 ? 4 : 2, 4, 4>(p, stream);
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
    const int most = head_dim <= 80 ? 256 : 128;
    for (int t = 16; t < most; t *= 2)
        if (rows <= t) return t;
    return most;
}

int tree_wgs_per_cu(int kv_dtype, int head_dim, int rows) {
    const int t = tree_tile_rows(kv_dtype, head_dim, rows);
    return t <= (head_dim <= 80 ? 64 : 32) ? 4 : 2;
}

hipError_t launch_tree(const TreeParams& p, hipStream_t stream) {
    hipError_t e;
    switch (p.kv_dtype) {
        case VCPP_KV_F16: e = launch_dim<VCPP_KV_F16>(p, stream); break;
        case VCPP_KV_I8: e = launch_dim<VCPP_KV_I8>(p, stream); break;
        case VCPP_KV_FP8: e = launch_dim<VCPP_KV_FP8>(p, stream); break;
        default: return hipErrorInvalidValue;
    }
    if (e != hipSuccess || p.parts <= 1) return e;
    const uint32_t chunks = (uint32_t)((p.num_heads * (p.head_dim / 4) + 255) / 256);
    tree_merge_kernel<<<dim3((uint32_t)(p.num_seqs * p.max_nodes), chunks), dim3(256), 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace vcpp
