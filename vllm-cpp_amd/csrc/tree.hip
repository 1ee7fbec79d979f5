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
// next to each other) are cut into tiles of WR waves x RB blocks of 16 rows.
// All units (sequence, row tile), each as long as its 32-key blocks, lie on one
// axis that is cut into equal ranges, one per workgroup the GPU holds and kv
// head (tree_mask.h): uneven sequences cost no one a tail.  A unit that range
// ends cut leaves partial results (exponent, sum, outputs) in the workspace,
// which a second kernel merges.  Keys stream through a ring of LDS stages filled
// by direct-to-LDS DMA.  Per key block and 16 rows:
//   S^T[32 keys][16 rows] = K x Q^T   (16x16x32 f16)
//   P = exp2(S scale - m)             (fp32)
//   O[16 rows][D] += P x V            (16x16x32 f16, twice)
// Verification has to reproduce what a decode of the accepted tokens computes,
// so P is not rounded to fp16: it enters the matrix product as the sum of two
// fp16 numbers (22 bits of it), and the row sums are fp32 sums of P itself.
// The running exponent leaves 11 bits of headroom below fp16's largest power
// (P <= 2^15), so that the low part of a P of 2^-16 of the row's largest still
// has 19 bits; it moves when a row's largest score grows by more than 2^4.
// What bounds it, 64 heads over 8 kv heads of 80: 16 nodes on 32 fp16 sequences
// of 128..4096 take 76 us, of which the ring without products takes 49 (210 MB)
// and the merge 12; 64 nodes on 8 FP8 sequences of 8000..16384 take 233 us, of
// which the products (three per key and row: S, P's high and low part) are 108
// at a large matrix product's rate, and the rest the softmax and the widening on
// the vector units beside them.
// int8 pages: K and V are exact fp16 integers; the key's K scale multiplies
// the score, its V scale P (whose exponent is lowered by a running power of two
// at or above the scales, so that any scale keeps the product in range).
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

// dma16 without the normal allocation policy, for lines that are read once: 16
// nodes on 32 fp16 sequences of 128..4096 tokens, 32 heads over 8 of 128, 92 ->
// 82 us.  (Lines that neighbouring heads or row tiles read again: 64 nodes on FP8
// pages of 80 dims 250 -> 263.)
__device__ __forceinline__ void dma16_once(const void* src, uint32_t lds_base) {
    uint32_t saved;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %2, off nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved) : "s"(lds_base), "v"(src) : "memory");
}

// Eight numbers as sums of two fp16 numbers each: the nearest ones (hi), and
// the rests rounded (lo; v_fma_mix: one instruction forms x - hi and rounds
// it).  One asm block: a half-register write needs one instruction between it
// and whatever reads the register, which the compiler does not see here.
__device__ __forceinline__ void split8(const float (&x)[8], h8& hi, h8& lo) {
    h2 h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = h2{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
    asm("v_fma_mixlo_f16 %0, %4, -1.0, %8 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixlo_f16 %1, %5, -1.0, %10 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixlo_f16 %2, %6, -1.0, %12 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixlo_f16 %3, %7, -1.0, %14 op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %0, %4, -1.0, %9 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %1, %5, -1.0, %11 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %2, %6, -1.0, %13 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "v_fma_mixhi_f16 %3, %7, -1.0, %15 op_sel:[1,0,0] op_sel_hi:[1,0,0]\n\t"
        "s_nop 1"
        : "=&v"(l[0]), "=&v"(l[1]), "=&v"(l[2]), "=&v"(l[3]), "+v"(h[0]), "+v"(h[1]), "+v"(h[2]), "+v"(h[3])
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi[2 * i] = h[i][0], hi[2 * i + 1] = h[i][1];
        lo[2 * i] = l[i][0], lo[2 * i + 1] = l[i][1];
    }
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
    // Every 128-byte line is read by one workgroup only: rows are whole lines, and
    // a tree is one row tile.
    static constexpr bool ONCE = D * (BYTES ? 1 : 2) % 128 == 0 && ROWS < 256;
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
    // Windows (tree_window) of the tile's rows on the key blocks that reach into
    // a tree: at most 9.
    static constexpr int WINDOWS = MARKS + (SCALED ? 0 : (2 + D + ROWS * DW) * 4);
    static constexpr int SEQS = WINDOWS + (kMaxTreeNodes / kKBlk + 1) * ROWS * 4;  // the (at most 64) sequences
    static constexpr int TABLE = (SEQS + kWave * (int)sizeof(TreeSeq) + 7) & ~7;
    static_assert(STAGES >= 3 && (STAGES - 1) * PERW < 64, "ring depth");
};

// LDS layout of a K (or V) block: rows of NCH 16-byte chunks.  Rows of 8 or 16
// chunks start on the same banks; there a row's chunks are permuted by its
// number (chunk ^ (row & 7)), which spreads both the K fragments' 16 rows and
// the transposing V reads' rows over the banks.
constexpr bool is_pow2(int n) { return (n & (n - 1)) == 0; }
template <int NCH>
__device__ __forceinline__ int chunk_at(int row, int pos) {
    return is_pow2(NCH) ? pos ^ (row & 7) : pos;
}
template <int NCH>
__device__ __forceinline__ int slot_at(int row, int chunk) {
    return row * NCH + chunk_at<NCH>(row, chunk);
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
    return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
           (int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32;
}

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

// Row blocks per wave (RB), waves (WR) and ring stages (ST) of a tile of `ROWS`
// rows.  One row block a wave while the tile is small: 8 nodes of 8-head groups
// (64 rows) on 32 sequences of 128..4096 tokens 55 us against 73 with two.
// Four (two for int8 and head_dim 128, whose registers hold no more) once the
// matrix products are the time: fewer fragment reads and barriers a product.
template <int KV, int D, int ROWS>
struct TreeTile {
    static constexpr int RB = ROWS <= 64 ? 1 : ROWS == 128 ? 2 : D == 64 || (D == 80 && KV != VCPP_KV_I8) ? 4 : 2;
    static constexpr int WR = ROWS / 16 / RB;
    static constexpr int ST = ROWS <= 64 ? 3 : 4;
};

template <int KV, int D, int RB, int WR, int ST>
__global__ __launch_bounds__(64 * WR, RB == 1 && D <= 80 ? 3 : 2) void tree_kernel(TreeParams p) {
    using T = TreeDims<KV, D, RB, WR, ST>;
    using DD = typename T::DD;
    using ID = typename T::ID;
    constexpr bool BYTES = T::BYTES, SCALED = T::SCALED;
    constexpr int NC32 = PDims<D>::NC32, NT = PDims<D>::NT, REM = PDims<D>::REM;
    extern __shared__ __attribute__((aligned(16))) char tree_lds[];
    lds_char* lds = (lds_char*)tree_lds;
    const uint32_t lds_addr = (uint32_t)(uintptr_t)lds;
    __attribute__((address_space(3))) int64_t* table_s =
        reinterpret_cast<__attribute__((address_space(3))) int64_t*>(lds + T::TABLE);
    __attribute__((address_space(3))) uint32_t* marks =
        reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(lds + T::MARKS);
    __attribute__((address_space(3))) uint32_t* windows =
        reinterpret_cast<__attribute__((address_space(3))) uint32_t*>(lds + T::WINDOWS);
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
    TreeRanges cut(p, T::ROWS, lane);
    if (range >= cut.R || cut.total == 0) return;  // whole workgroup
    const int64_t lo = cut.start(range), hi = cut.start(range + 1);
    int64_t first;  // first block of sequence s
    int s = cut.seq_of(lo, first);
    // (in LDS: in the lanes they would hold registers through the loop)
    __attribute__((address_space(3))) int32_t* seqs =
        reinterpret_cast<__attribute__((address_space(3))) int32_t*>(lds + T::SEQS);
    if (p.num_seqs <= kWave && wave == 0) {
        const int v[5] = {cut.mine.q0, cut.mine.n, cut.mine.prefix, cut.mine.end, cut.mine.plain};
#pragma unroll
        for (int i = 0; i < 5; ++i) seqs[5 * lane + i] = v[i];
    }
    __syncthreads();
    const int G = p.group;
    int64_t at_block = lo;
    while (at_block < hi) {  // the range's pieces, one per unit
    TreeSeq sq;
    if (p.num_seqs <= kWave) {
        sq.q0 = __builtin_amdgcn_readfirstlane(seqs[5 * s]);
        sq.n = __builtin_amdgcn_readfirstlane(seqs[5 * s + 1]);
        sq.prefix = __builtin_amdgcn_readfirstlane(seqs[5 * s + 2]);
        sq.end = __builtin_amdgcn_readfirstlane(seqs[5 * s + 3]);
        sq.plain = __builtin_amdgcn_readfirstlane(seqs[5 * s + 4]);
    } else {
        sq = TreeSeq(p, s);
    }
    const int M = sq.n * G;
    const int tiles = (M + T::ROWS - 1) / T::ROWS, blocks = (sq.end + 31) / 32;
    if (at_block >= first + (int64_t)tiles * blocks) {  // next sequence
        first += (int64_t)tiles * blocks;
        ++s;
        continue;
    }
    const int rt = (int)((uint32_t)(at_block - first) / (uint32_t)blocks);  // (a sequence's blocks: below 2^31)
    const int64_t unit0 = first + (int64_t)rt * blocks;  // the unit's first block
    const int kb_lo = (int)(at_block - unit0);
    const int kb_hi = (int)min((int64_t)blocks, hi - unit0);
    const bool whole = kb_lo == 0 && kb_hi == blocks;
    const int64_t piece = (int64_t)range * 2 + (at_block > lo ? 1 : 0);  // partials' place (not whole)
    at_block = unit0 + kb_hi;
    const int row0 = rt * T::ROWS;
    const int k_lo = kb_lo * kKBlk, k_hi = min(kb_hi * kKBlk, sq.end);

    // Q fragments (B operand): row row0 + 16 (WR rb + wave) + c (a tile that is
    // not full keeps every wave busy)
    h8 qa[RB][NC32 > 0 ? NC32 : 1];
    h8 qr[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = row0 + 16 * (WR * rb + wave) + c;
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
    const int tree_kb = sq.plain / kKBlk;  // first block that reaches into the tree
    for (int i = tid + max(0, kb_lo - tree_kb) * T::ROWS; i < (kb_hi - tree_kb) * T::ROWS; i += 64 * WR) {
        const int row = row0 + i % T::ROWS, t = row / G;
        windows[i] = row < M ? tree_window(p, sq, p.mask ? p.mask + (int64_t)(sq.q0 + t) * p.mask_words : nullptr, t,
                                           (tree_kb + i / T::ROWS) * kKBlk)
                             : 0u;
    }
    // Byte offsets in the pool of the piece's 16-position tiles (a tile lies in
    // one page), this kv head's rows; -1: missing or outside the pool.  int8:
    // those of their scales behind them.
    const int32_t* table = p.block_tables + (int64_t)s * p.max_blocks;
    const int ntiles = min(2 * (kb_hi - kb_lo), p.table_cap);
    int bad = 0;
    for (int i = tid; i < ntiles; i += 64 * WR) {
        const int pos = k_lo + 16 * i;
        const int lb = (int)(((uint64_t)(uint32_t)pos * p.bs_magic) >> 40), slot = pos - lb * p.block_size;
        const int bid = pos < k_hi && lb < p.max_blocks ? table[lb] : -1;
        const bool ok = bid >= 0 && (int64_t)bid < p.num_blocks;
        constexpr int ES = BYTES ? 1 : 2;
        table_s[i] = ok ? ((int64_t)bid * p.block_stride + ((int64_t)slot * p.num_kv_heads + kvh) * D) * ES : -1;
        if constexpr (SCALED)
            table_s[p.table_cap + i] = ((int64_t)bid * p.scale_block_stride + (int64_t)kvh * p.block_size + slot) * 2;
        bad |= pos < k_hi && !ok;
    }
    const bool any_bad = __syncthreads_or(bad) != 0;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the ring's DMA is not in the compiler's count

    // DMA: instruction j = wave + WR i fills slots 64 j + lane of a stage, K's
    // rows and then V's, NCHB 16-byte chunks each: neighbouring lanes read
    // neighbouring bytes.  (Chunks key by key, as prefill_tile lays them out,
    // make every lane of an instruction a request of its own: one node on
    // 64 fp16 sequences of 128..4096 tokens 101 -> 87 us.)  lo: the lane's byte
    // offset in its tile, its row in the top 5 bits.  Positions past the piece
    // and missing tiles read zeros.
    const int my_inst = T::NINST % WR == 0 || wave < T::NINST % WR ? T::PERW : T::PERW - 1;
    const uint32_t row_bytes = (uint32_t)p.num_kv_heads * D * (BYTES ? 1 : 2);
    constexpr int NCHB = BYTES ? ID::NCH : DD::NCH, REGB = kKBlk * NCHB;
    uint32_t lo_at[T::PERW];
#pragma unroll
    for (int i = 0; i < T::PERW; ++i) {
        const int n = 64 * (wave + WR * i) + lane, q = n >= REGB ? n - REGB : n;
        const int row = (q / NCHB) & 31, pos = q % NCHB;
        lo_at[i] = (uint32_t)row << 27 | ((row & 15) * row_bytes + (BYTES ? pos : chunk_at<NCHB>(row, pos)) * 16);
    }
    int wr_at = 0, rd_at = 0;  // byte offsets of the ring stages to fill and to use next
    const auto next = [](int at) { return at + T::RSTAGE == T::AREA ? 0 : at + T::RSTAGE; };
    auto issue = [&](int kb) {
        const uint32_t sbase = lds_addr + wr_at;
        wr_at = next(wr_at);
        const int ti = 2 * (kb - kb_lo);
        const int64_t t0 = uniform64(table_s[ti]), t1 = uniform64(table_s[ti + 1]);
        const bool full = t0 >= 0 && t1 >= 0 && (kb + 1) * kKBlk <= k_hi;
#pragma unroll
        for (int i = 0; i < T::PERW; ++i) {
            if (i < my_inst) {
                const int j = wave + WR * i;
                const uint32_t dst = __builtin_amdgcn_readfirstlane(sbase + j * 1024);
                if (2 * REGB / 64 > j) {
                    const bool isv = REGB % 64 == 0 ? j >= REGB / 64 : 64 * j + lane >= REGB;
                    const int64_t at = (int32_t)lo_at[i] < 0 ? t1 : t0;
                    const char* src = static_cast<const char*>(isv ? p.v : p.k) + at + (lo_at[i] & 0x7FFFFFFu);
                    if (!full && (at < 0 || kb * kKBlk + (int)(lo_at[i] >> 27) >= k_hi))
                        src = reinterpret_cast<const char*>(kZeroChunk);
                    if constexpr (T::ONCE) dma16_once(src, dst);
                    else dma16(src, dst);
                } else if constexpr (SCALED) {
                    const int key = lane & 31;
                    const bool ok = (key < 16 ? t0 : t1) >= 0 && kb * kKBlk + key < k_hi;
                    const char* sb = reinterpret_cast<const char*>(lane >> 5 ? p.v_scale : p.k_scale);
                    dma2(ok ? (const void*)(sb + table_s[p.table_cap + ti + (key >> 4)] + 2 * (key & 15)) : (const void*)kZeroChunk,
                         __builtin_amdgcn_readfirstlane(sbase + ID::SCALES));
                }
            }
        }
    };
    // Byte block kb -> fp16 values (int8: exact integers); its scales -> fp32
    // (K's times log2(e) / sqrt(D)).
    auto widen = [&](int kb, int at) {
        lds_char* st = lds + at;
        if constexpr (SCALED) {
            if (tid < 64) {
                lds_char* sw = st + ID::SCALES + tid * 4;
                const float x = (float)__builtin_bit_cast(
                    _Float16, *reinterpret_cast<__attribute__((address_space(3))) const uint16_t*>(sw));
                *reinterpret_cast<__attribute__((address_space(3))) float*>(sw) = tid < 32 ? x * p.scale_log2 : x;
            }
        }
        lds_char* dst0 = lds + T::AREA + (kb % T::NF16) * DD::STAGE;
        const auto unit = [&](int u, lds_char* dst, int slot) {  // raw unit u to slots `slot` and the row's next chunk
            const i4 raw = *reinterpret_cast<__attribute__((address_space(3))) i4*>(st + u * 16);
            *reinterpret_cast<__attribute__((address_space(3))) h8*>(dst + slot * 16) =
                bytes8_to_h8<KV>((uint32_t)raw.x, (uint32_t)raw.y);
            *reinterpret_cast<__attribute__((address_space(3))) h8*>(dst + (is_pow2(DD::NCH) ? slot ^ 1 : slot + 1) * 16) =
                bytes8_to_h8<KV>((uint32_t)raw.z, (uint32_t)raw.w);
        };
        if constexpr (ID::REGION % (64 * WR) == 0) {  // a thread's units are 64 WR / NCH keys apart, K's then V's
            constexpr int EACH = ID::REGION / (64 * WR), STEP = 64 * WR / ID::NCH;
            const int slot = slot_at<DD::NCH>(tid / ID::NCH, 2 * (tid % ID::NCH));
#pragma unroll
            for (int i = 0; i < 2 * EACH; ++i)
                unit(tid + 64 * WR * i, dst0 + (i / EACH * DD::REGION + i % EACH * STEP * DD::NCH) * 16, slot);
        } else {
#pragma unroll 1
            for (int u = tid; u < ID::UNITS; u += 64 * WR) {
                const int which = u >= ID::REGION, q = u - which * ID::REGION;
                unit(u, dst0 + which * DD::REGION * 16, slot_at<DD::NCH>(q / ID::NCH, 2 * (q % ID::NCH)));
            }
        }
    };

    // A drafted V row that is not finite must not reach the rows that do not see
    // it (0 x inf in the matrix product): such values of block kb are replaced
    // by 0 in LDS, and the outputs that attend them are marked, to become NaN
    // at the end.  (Only blocks that reach into a tree; in registers and
    // unrolled this cost the main loop 60 of them.)
    auto scrub = [&](int kb) {
        lds_char* vs = (BYTES ? lds + T::AREA + (kb % T::NF16) * DD::STAGE : lds + rd_at) + DD::REGION * 16;
#pragma unroll 1
        for (int u = tid; u < DD::REGION; u += 64 * WR) {
            const int key = u / DD::NCH, ch = chunk_at<DD::NCH>(key, u % DD::NCH);
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
                const uint32_t w = windows[(kb - tree_kb) * T::ROWS + i];
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
    // int8: a power of two 2^vexp at or above every finite V scale so far
    // divides P (it is part of m_run), so that P times a scale stays in range.
    float vcap = 0x1p-24f, vexp = -24.f, p_top = SCALED ? kTopP * 0x1p24f : kTopP;

    // LDS byte offsets of this lane's fragment reads.  K: row 16 kt + c, chunks
    // 4 cc + g; V: rows 16 hh + 4 g + c / 4, half c & 1 of chunk 2 t + (c & 3) / 2.
    constexpr int ROWB = DD::NCH * 16;
    constexpr int NK = is_pow2(DD::NCH) ? 2 : 1, NV = is_pow2(DD::NCH) ? 4 : 1;  // (constant steps without a permutation)
    int kat[NK], vat[NV];
#pragma unroll
    for (int i = 0; i < NK; ++i) kat[i] = slot_at<DD::NCH>(c, 4 * i + g) * 16;
    // The 16-dim rest (D = 80) of lane groups 2 and 3 is the stage's zero slot.
    const int krest0 = g < 2 ? c * ROWB + (4 * NC32 + g) * 16 : DD::ZERO, krest1 = g < 2 ? krest0 + 16 * ROWB : krest0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        vat[i] = DD::REGION * 16 + slot_at<DD::NCH>(4 * g + (c >> 2), 2 * i + ((c & 3) >> 1)) * 16 + 8 * (c & 1);

    const int live = (M - row0 - 16 * wave + 16 * WR - 1) / (16 * WR);  // this wave's row blocks that hold rows (<= 0: none)
    // One key block (K and V at `at`) for this wave's rows, SG row blocks at a
    // time.  One body for masked and free blocks (the mask's parts behind
    // uniform branches): two inlined forms held 50 registers more and spilled.
    auto compute = [&](int kb, const bool masked, lds_char* at) {
        h8 ka[2][NC32 > 0 ? NC32 : 1];
        h8 kr[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int cc = 0; cc < NC32; ++cc)
                ka[kt][cc] = *reinterpret_cast<__attribute__((address_space(3))) h8*>(at + kat[cc % NK] + (cc / NK) * NK * 64 +
                                                                                      kt * 16 * ROWB);
            if constexpr (REM)
                kr[kt] = *reinterpret_cast<__attribute__((address_space(3))) h8*>(at + (kt ? krest1 : krest0));
        }
        // Scales of this lane's keys 16 kt + 4 g + r (V's: behind them), read
        // where they are used.
        const auto scale4 = [&](int kt, bool v) {
            return *reinterpret_cast<__attribute__((address_space(3))) const f4*>(lds + rd_at + ID::SCALES +
                                                                                  ((v ? 32 : 0) + 16 * kt + 4 * g) * 4);
        };
        f4 ks[2];
        float top = 0.f;
        if constexpr (SCALED) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                ks[kt] = scale4(kt, false);
                const f4 b = scale4(kt, true);
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(b[r]) < 65536.f ? fabsf(b[r]) : 0.f);  // (finite ones)
            }
        }
        // Bits 16 kt + r: key 16 kt + 4 g + r is seen by row c of row block rb.
        const auto seen = [&](int rb) {
            uint32_t w = ~0u;
            if (any_bad) {  // positions on missing pages leave
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    if (table_s[2 * (kb - kb_lo) + kt] < 0) w &= kt ? 0xFFFFu : 0xFFFF0000u;
            }
            if (kb >= tree_kb) w &= windows[(kb - tree_kb) * T::ROWS + 16 * (WR * rb + wave) + c];
            return w >> (4 * g);
        };
        constexpr int SG = 1;
        h8 vb[NT];
#pragma unroll
        for (int r0 = 0; r0 < RB; r0 += SG) {
            if (r0 >= live) break;
            f4 sc[SG][2];
#pragma unroll
            for (int i = 0; i < SG; ++i)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int cc = 0; cc < NC32; ++cc) acc = mfma32(ka[kt][cc], qa[r0 + i][cc], acc);
                    if constexpr (REM) acc = mfma32(kr[kt], qr[r0 + i], acc);
                    sc[i][kt] = acc;
                }
            if (r0 == 0) {
                // (V's registers after K's: both at once pass 256 at head_dim 128)
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const h4 lo = read_tr(at + vat[t % NV] + (t / NV) * NV * 32);
                    const h4 hi = read_tr(at + vat[t % NV] + (t / NV) * NV * 32 + 16 * ROWB);
                    vb[t] = h8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                }
            }
            // (behind the first products: the scales' way out of LDS is covered)
            if (SCALED && r0 == 0 && __builtin_expect(__any(top > vcap), 0)) {
                asm volatile("" : "+v"(top));  // (a branch: as selects its products run for every block)
                top = fmaxf(top, shfl_xor(top, 16));
                top = fmaxf(top, shfl_xor(top, 32));
                const uint32_t up = (__float_as_uint(top) + 0x7FFFFFu) & 0x7F800000u;  // (fp16 scales are normal in fp32)
                const float cap = fmaxf(__uint_as_float(up), vcap);
                const float down = vcap / cap, by = (float)((int)(__float_as_uint(cap) >> 23) - 127) - vexp;
                vcap = cap;
                vexp += by;
                p_top = kTopP / cap;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    m_run[rb] += by;
                    lsum[rb] *= down;
#pragma unroll
                    for (int t = 0; t < NT; ++t) o[rb][t] *= down;
                }
            }
            float pf[SG][8], bs[SG];
            auto exps = [&](int i) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        pf[i][4 * kt + r] = fmaf(sc[i][kt][r], SCALED ? ks[kt][r] : p.scale_log2, -m_run[r0 + i]);
                }
                if (masked) {
                    uint32_t w = seen(r0 + i);
                    asm volatile("" : "+v"(w));  // (nothing below is hoisted out of the branch)
#pragma unroll
                    for (int e = 0; e < 8; ++e) pf[i][e] = seen_or_inf(pf[i][e], w, 16 * (e >> 2) + (e & 3));
                }
                bs[i] = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    pf[i][e] = fast_exp2(pf[i][e]);
                    bs[i] += pf[i][e];
                }
            };
            bool cross = false;  // a score past the headroom (inf and NaN too)
#pragma unroll
            for (int i = 0; i < SG; ++i) {
                exps(i);
                cross |= !(bs[i] <= p_top);
            }
            if (__builtin_expect(__any(cross), 0)) {
#pragma unroll
                for (int i = 0; i < SG; ++i) {
                    const int rb = r0 + i;
                    float ml = -__builtin_inff();
                    const uint32_t w = masked ? seen(rb) : ~0u;
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            ml = vmax(ml, seen_or_inf(sc[i][kt][r] * (SCALED ? ks[kt][r] : p.scale_log2), w, 16 * kt + r));
                    }
                    ml = max_over_groups(ml);
                    if constexpr (SCALED) ml += vexp;
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
                    exps(i);
                }
            }
#pragma unroll
            for (int i = 0; i < SG; ++i) {
                const int rb = r0 + i;
                lsum[rb] += bs[i];
                h8 ph, pl;
                if constexpr (SCALED) {
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) {
                        const f4 vs = scale4(kt, true);
#pragma unroll
                        for (int r = 0; r < 4; ++r) pf[i][4 * kt + r] *= vs[r];
                    }
                    if (masked) {  // (the scale of a row that is not seen may be anything)
                        uint32_t w = seen(rb);
                        asm volatile("" : "+v"(w));
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            pf[i][e] = __int_as_float(__float_as_int(pf[i][e]) &
                                                      __builtin_amdgcn_sbfe((int)w, 16 * (e >> 2) + (e & 3), 1));
                    }
                }
                split8(pf[i], ph, pl);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    o[rb][t] = mfma32(ph, vb[t], o[rb][t]);
                    o[rb][t] = mfma32(pl, vb[t], o[rb][t]);
                }
            }
        }
    };

    // Blocks in front of the tree (and on valid pages) need no mask.
    const int free_hi = any_bad ? kb_lo : max(kb_lo, min(kb_hi, tree_kb));
    constexpr int S = T::STAGES;
#pragma unroll
    for (int i = 0; i < S - 1; ++i)
        if (kb_lo + i < kb_hi) issue(kb_lo + i);
    // Waits for block kb; of the blocks issued, up to `last`, those after it may
    // stay in flight (the count is exact only while whole rounds follow).
    auto land = [&](int kb, int last, auto in_flight) {
        constexpr int N = decltype(in_flight)::value;
        if (my_inst == T::PERW) wait_dma<N * T::PERW>(kb + N <= last);
        else wait_dma<N * (T::PERW - 1)>(kb + N <= last);
    };
    const int top = kb_hi - 1;
    if constexpr (BYTES && WR > 1) {
        land(kb_lo, min(kb_lo + S - 2, top), std::integral_constant<int, S - 2>{});
        __syncthreads();
        widen(kb_lo, 0);
    }
    for (int kb = kb_lo; kb < kb_hi; ++kb) {
        if constexpr (BYTES && WR > 1) {
            // block kb + 1 landed for every wave, kb widened, kb - 1 used up
            land(kb + 1, min(kb + S - 2, top), std::integral_constant<int, S - 3>{});
            __syncthreads();
            if (kb + S - 1 < kb_hi) issue(kb + S - 1);
            if (kb + 1 < kb_hi) widen(kb + 1, next(rd_at));
        } else {
            land(kb, min(kb + S - 2, top), std::integral_constant<int, S - 2>{});
            tree_barrier<WR>();  // block kb landed for every wave, kb - 1 used up
            if (kb + S - 1 < kb_hi) issue(kb + S - 1);
            if constexpr (BYTES) {
                widen(kb, rd_at);
                tree_barrier<WR>();
            }
        }
        if constexpr (!SCALED)
            if (kb >= tree_kb) scrub(kb);
        if (live > 0)
            compute(kb, kb >= free_hi, BYTES ? lds + T::AREA + (kb % T::NF16) * DD::STAGE : lds + rd_at);
        rd_at = next(rd_at);
    }

    const int64_t pbase = (piece * p.num_kv_heads + kvh) * T::ROWS;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float l = sum_over_groups(lsum[rb]);  // row c
        const int w16 = 16 * (WR * rb + wave);
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
            const float mul = !whole ? 1.f : lr == 0.f ? 0.f : 1.f / lr;
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
                const int w = 16 * (WR * (i / (16 * D)) + wave) + i / D % 16, d = i % D, row = row0 + w, t = row / G;
                if (row >= M || !(bad_outs[w * T::DW + d / 32] >> (d & 31) & 1)) continue;
                (!whole ? p.ws_o + (pbase + w) * D
                        : p.out + ((int64_t)(sq.q0 + t) * p.num_heads + kvh * G + (row - t * G)) * D)[d] = __builtin_nanf("");
            }
        }
    if constexpr (WR > 1) __syncthreads();  // the ring and the block ids are free for the next piece
    }  // pieces
}

// The pieces of a row that ranges' ends cut: their places in the workspace.
template <int ROWS>
struct TreePieces {
    int r0, r1;       // ranges (equal: the row is whole, written in place)
    int64_t at0, step, head0;
    __device__ __forceinline__ TreePieces(const TreeParams& p, const TreeRanges& cut, int64_t first, int blocks, int kvh,
                                          int row) {
        const int64_t unit0 = first + (int64_t)(row / ROWS) * blocks;
        r0 = cut.range_of(unit0);
        r1 = cut.range_of(unit0 + blocks - 1);
        head0 = (int64_t)kvh * ROWS + row % ROWS;
        step = (int64_t)p.num_kv_heads * ROWS;
        at0 = (r0 * 2 + (cut.start(r0) < unit0 ? 1 : 0)) * step + head0;
    }
    __device__ __forceinline__ int64_t at(int r) const { return r == r0 ? at0 : r * 2 * step + head0; }
};

// Joins rows of few pieces: thread (row, head, 4 dims), four pieces' sums and
// outputs loaded at once.
template <int ROWS, int D>
__global__ __launch_bounds__(256) void tree_merge_few_kernel(TreeParams p) {
    constexpr int D4 = D / 4, AT = 4;
    const int s = blockIdx.x / p.max_nodes, t = blockIdx.x - s * p.max_nodes;
    const TreeSeq sq(p, s);
    if (t >= sq.n) return;
    TreeRanges cut(p, ROWS, threadIdx.x & 63);
    const int64_t first = cut.first_of(s);
    const int e = blockIdx.y * 256 + threadIdx.x;
    const int h = e / D4, d = e - h * D4;
    if (h >= p.num_heads) return;
    const int kvh = h / p.group;
    const TreePieces<ROWS> pc(p, cut, first, (sq.end + 31) / 32, kvh, t * p.group + (h - kvh * p.group));
    if (pc.r0 == pc.r1) return;
    float m = kMaxSeed, l = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
    for (int r = pc.r0; r <= pc.r1; r += AT) {
        float2 ml[AT];
        f4 x[AT];
#pragma unroll
        for (int i = 0; i < AT; ++i) {
            const int64_t at = pc.at(min(r + i, pc.r1));
            ml[i] = p.ws_ml[at];
            x[i] = *reinterpret_cast<const f4*>(p.ws_o + (at * D4 + d) * 4);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < AT; ++i) top = fmaxf(top, ml[i].x);
        const float down = fast_exp2(m - top);
        m = top;
        l *= down;
        o *= down;
#pragma unroll
        for (int i = 0; i < AT; ++i) {
            if (r + i > pc.r1) continue;
            const float w = fast_exp2(ml[i].x - m);
            l += ml[i].y * w;
            o += x[i] * w;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t to = (int64_t)(sq.q0 + t) * p.num_heads + h;
    *reinterpret_cast<f4*>(p.out + (to * D4 + d) * 4) = o * inv;
    if (d == 0 && p.lse) p.lse[to] = row_lse(m, l);
}

// Joins rows of many pieces.  A wave takes `heads` heads of one row after
// another; its lanes hold the pieces' (exponent, sum) 64 at a time, and then
// slices of the pieces' outputs, 4 dims a lane, whose loads do not wait for
// each other: 65 pieces (32768 tokens, 16 nodes, 64/8 heads of 80) 13 us
// against 48 with a thread per 4 dims walking them one by one.
template <int ROWS, int D>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p, int heads) {
    constexpr int D4 = D / 4, SL = kWave / D4;  // lanes of a row, pieces at once
    const int s = blockIdx.x / p.max_nodes, t = blockIdx.x - s * p.max_nodes;
    const int lane = threadIdx.x & 63;
    const TreeSeq sq(p, s);
    if (t >= sq.n) return;
    TreeRanges cut(p, ROWS, lane);
    const int64_t first = cut.first_of(s);
    const int blocks = (sq.end + 31) / 32;
    const int d = lane % D4, sl = lane / D4;
    const int h0 = (blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * heads;
    for (int h = h0; h < min(h0 + heads, p.num_heads); ++h) {
        const int kvh = h / p.group;
        const TreePieces<ROWS> pc(p, cut, first, blocks, kvh, t * p.group + (h - kvh * p.group));
        if (pc.r0 == pc.r1) continue;
        float m = kMaxSeed, l = 0.f;
        f4 o = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = pc.r0; k0 <= pc.r1; k0 += kWave) {
            const int n = min(kWave, pc.r1 + 1 - k0);
            const float2 ml = lane < n ? p.ws_ml[pc.at(k0 + lane)] : make_float2(kMaxSeed, 0.f);
            float top = fmaxf(m, ml.x);
#pragma unroll
            for (int i = 32; i > 0; i /= 2) top = fmaxf(top, shfl_xor(top, i));
            const float down = fast_exp2(m - top);
            m = top;
            const float w = fast_exp2(ml.x - m);  // (0 where there is no piece: its sum and weight are 0)
            float sum = ml.y * w;
#pragma unroll
            for (int i = 32; i > 0; i /= 2) sum += shfl_xor(sum, i);
            l = l * down + sum;
            o *= down;
#pragma unroll 4
            for (int k = sl; k < n; k += SL) {
                const float wk = shfl(w, k);
                if (sl < SL) o += *reinterpret_cast<const f4*>(p.ws_o + (pc.at(k0 + k) * D4 + d) * 4) * wk;
            }
        }
#pragma unroll
        for (int i = 1; i < SL; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = shfl(o[e], (lane + i * D4) & 63);
                o[e] += sl == 0 ? x : 0.f;
            }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t to = (int64_t)(sq.q0 + t) * p.num_heads + h;
        if (lane < D4) *reinterpret_cast<f4*>(p.out + (to * D4 + d) * 4) = o * inv;
        if (lane == 0 && p.lse) p.lse[to] = row_lse(m, l);
    }
}

template <int KV, int D, int ROWS>
hipError_t launch_tile(const TreeParams& p, hipStream_t stream) {
    using L = TreeTile<KV, D, ROWS>;
    using T = TreeDims<KV, D, L::RB, L::WR, L::ST>;
    static_assert(T::ROWS == ROWS, "tile");
    const auto kernel = tree_kernel<KV, D, L::RB, L::WR, L::ST>;
    const size_t lds = T::TABLE + (size_t)p.table_cap * (T::SCALED ? 16 : 8);
    if (lds > 64 * 1024) {
        const hipError_t e =
            hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    const int64_t grid = (int64_t)(p.ranges + 7) / 8 * 8 * p.num_kv_heads;
    kernel<<<dim3((uint32_t)grid), dim3(64 * L::WR), lds, stream>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.ranges == 1) return e;
    // Ranges per unit, where the sequences are as long as their bound: above 6
    // a wave per row (of about 8192), else a thread per 4 dims (3 pieces, 512
    // rows of 64 heads: 12.5 us against 21).
    const int64_t rows = (int64_t)p.num_seqs * p.max_nodes;
    const int64_t units = (int64_t)p.num_seqs * ((p.max_nodes * p.group + ROWS - 1) / ROWS);
    if (p.ranges <= 6 * units) {
        const dim3 grid2((uint32_t)rows, (uint32_t)((p.num_heads * (D / 4) + 255) / 256));
        tree_merge_few_kernel<ROWS, D><<<grid2, dim3(256), 0, stream>>>(p);
    } else {
        const int heads = (int)std::max<int64_t>(1, rows * p.num_heads / 8192);
        const dim3 grid2((uint32_t)rows, (uint32_t)((p.num_heads + 4 * heads - 1) / (4 * heads)));
        tree_merge_kernel<ROWS, D><<<grid2, dim3(256), 0, stream>>>(p, heads);
    }
    return hipGetLastError();
}

template <int KV, int D>
hipError_t launch_shape(const TreeParams& p, hipStream_t stream) {
    switch (tree_tile_rows(KV, D, p.max_nodes * p.group)) {
        case 16: return launch_tile<KV, D, 16>(p, stream);
        case 32: return launch_tile<KV, D, 32>(p, stream);
        case 64: return launch_tile<KV, D, 64>(p, stream);
        case 128: return launch_tile<KV, D, 128>(p, stream);
        default: return launch_tile<KV, D, 256>(p, stream);
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
    for (int t = 16; t < 256; t *= 2)
        if (rows <= t) return t;
    return 256;
}

int tree_wgs_per_cu(int kv_dtype, int head_dim, int rows) {
    const int t = tree_tile_rows(kv_dtype, head_dim, rows);
    if (t == 256) return head_dim == 128 || (head_dim == 80 && kv_dtype == VCPP_KV_I8) ? 1 : 2;
    return t <= 32 ? 4 : 2;
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
