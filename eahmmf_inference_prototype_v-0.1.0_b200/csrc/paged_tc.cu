// paged_tc.cu -- attention of chunks of new tokens over 16-bit pages with the 5th-generation tensor cores.
//
// The mathematics is paged.cu's. A block takes two tiles of 128 rows (tokens x the q heads of one kv head) of a
// sequence and walks units of 128 positions; per tile and unit
//   S = q_lo k^T + q_hi k^T   (128 x 128, tensor memory)
//   p = 2^(S c - m + 15) in two 11-bit parts, written over S
//   O = p_lo v + p_hi v       (128 x hd, tensor memory, started afresh for every unit)
// O is added to the row's sums in registers: the tensor cores cut their sums, and one chain over a long context would
// bias them (12,289 positions: up to 5.7e-6 off in one chain, 8e-7 in chains of one unit).
//
// Operands: k and v by TMA from the pages (boxes of gcd(page, 128) positions, 128-byte swizzle), k read with hd
// contiguous, v with hd contiguous as the transposed operand; q scaled and split by the softmax warps; p from tensor memory.
//
// Bound: 4 hd flops per row and position, twice because of the two parts: 2 * 2 * 2 * 128 * 128 * hd per tile and unit. Two
// tiles share every k and v tile and take turns: while one tile's scores are in the softmax the other's products run.
// 4,096 tokens over 12,289 positions, 32 q heads of 128 on 4 kv heads, 16-bit pages: 1,037 us in a burst (1,327 TFLOP/s of both
// parts), 1,200 back to back, where the power cap holds the clock at 1.52 to 1.64 GHz. 64 tokens over 2,111 positions of 32-bit
// pages: 36 us, two units a block, most of it start, q and joining.
//
// Warps: 0-3 softmax of tile 0, 4-7 of tile 1 (thread = row = tensor-memory lane), 8 loads k, 11 loads v, 9 issues q k, 10 issues
// p v (one warp for both products left the tensor cores idle a third of the time: each wait costs it some 150 cycles). 32-bit
// pools: one row tile, 0-3 softmax, 4-11 split k and v, 12 and 13 issue.
#include <cuda.h>

#include <mutex>

#include "kernels.cuh"
#include "paged.cuh"
#include "tc.cuh"

namespace eb {
namespace {

constexpr int UNIT = 128;  // positions of a unit
constexpr int MROWS = 128;
constexpr int VALID_RING = 16;  // the loads run fewer units than this ahead of the softmax

// Registers: all threads are launched with REGS; a softmax thread holds its row's hd sums beside its scores, so its warps
// take registers over from the others: 16-bit pools 2 x 128 x 208 + 128 x 88 = 384 x 168, 32-bit pools 128 x 208 + 256 x 104 +
// 128 x 96 = 512 x 128, the launch's own totals (checked before the launch).
template <int HD, bool F32>
struct Tc {
    static constexpr int NM = F32 ? 1 : 2;               // row tiles that share the k and v tiles
    static constexpr int PARTS = F32 ? 2 : 1;            // 11-bit parts of a pool element
    static constexpr int HALVES = HD / 64;               // 128-byte column blocks of an operand tile
    static constexpr int BLK = 128 * 128;                // bytes of a column block of 128 rows
    static constexpr int TILE = HALVES * BLK;            // bytes of a 128 x hd operand tile
    static constexpr int STAGE = PARTS * TILE;           // of a k or v tile in all its parts: hi, lo
    // Tiles of k and of v in shared memory. Where there is room for three in all, k has two: the next scores wait for the last
    // product p v of the other tile anyway (its p lies in the score buffer that they take), v is needed a softmax later. One
    // ring of three for both, two for v, or halves of tiles in twice as many slots measured within 3 % of it.
    static constexpr int NK = F32 ? 1 : HD == 128 ? 2 : 4, NV = F32 || HD == 128 ? 1 : 4, NST = NK + NV;
    static constexpr int Q_BYTES = NM * 2 * TILE;
    static constexpr int SMEM = 1024 + Q_BYTES + NST * STAGE + 1024;
    static constexpr uint32_t O_COL = 384;               // tensor memory: three S, one O
    static constexpr uint32_t COLS = 512;
    static constexpr int W_LOAD = 4 * NM, N_LOAD = F32 ? 8 : 1;  // first warp that brings k and v, how many do
    static constexpr int W_QK = F32 ? 12 : 9, W_PV = W_QK + 1, W_LOAD_V = 11;  // 16-bit pools: k and v have a warp each
    static constexpr int NT = F32 ? 512 : 384;
    static constexpr int REGS = F32 ? 128 : 168, REGS_SOFTMAX = 208, REGS_LOAD = F32 ? 104 : 88, REGS_ISSUE = F32 ? 96 : 88;
};
static_assert(128 * (2 * 208 + 88) == 384 * 168 && 128 * (208 + 2 * 104 + 96) == 512 * 128, "register shares");

// Bytes of a row tile's q (q_lo, then q_hi: 2 HALVES column blocks of 128 rows of 128 bytes) that a softmax warp writes. Its next q
// is in q_at's layout; before that its 32 rows of the output pass through the same bytes, in stage_at's. Nothing but the warp's own
// order keeps the two apart, so they have to lie within the rows of the warp: no other warp of the tile writes or reads there.
__host__ __device__ constexpr int q_at(int row, int ch) {  // 16-byte chunk ch (8 f16) of a row of q_lo or q_hi
    return (ch >> 3) * 128 * 128 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
}
__host__ __device__ constexpr int stage_at(int row, int c) {  // 16-byte chunk c (4 floats) of a row of the output
    return (c >> 3) * 128 * 128 + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}
template <int HD, bool F32>
constexpr bool stage_stays_in_the_rows_of_its_warp() {
    for (int row = 0; row < MROWS; row++)
        for (int c = 0; c < HD / 4; c++) {
            const int at = stage_at(row, c), block = at / Tc<HD, F32>::BLK, in = at % Tc<HD, F32>::BLK;
            if (block >= 2 * Tc<HD, F32>::HALVES || in / 128 / 32 != row / 32) return false;
        }
    for (int row = 0; row < MROWS; row++)
        for (int ch = 0; ch < HD / 8; ch++)
            if (q_at(row, ch) % Tc<HD, F32>::BLK / 128 / 32 != row / 32) return false;
    return true;
}
static_assert(stage_stays_in_the_rows_of_its_warp<64, false>() && stage_stays_in_the_rows_of_its_warp<128, false>() &&
                  stage_stays_in_the_rows_of_its_warp<64, true>() && stage_stays_in_the_rows_of_its_warp<128, true>(),
              "a warp's output passes through its own rows");
struct Bars {
    uint64_t kv_full[8], kv_empty[8], q_full[2], s_full[2][2], p_full[2], pv_done[2], s_free[3], o_free;
    uint32_t valid[VALID_RING];                     // by unit: which boxes lie in pages of the pool
    float k_back[VALID_RING], v_back[VALID_RING];   // 32-bit pools, by unit: what undoes the scale of the k (v) tile
    float wmax[2][8];
    uint32_t tmem;
    int seq;
    long long start, scan_u[16], scan_p[16];
};
static_assert(sizeof(Bars) <= 1024, "");

// Bounded wait, as mbar_wait_bounded, without its suspend hint: these waits last a few hundred cycles.
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity) {
    for (int i = 0; i < 64; i++)
        if (bar_try(bar, parity)) return true;
    const uint64_t t0 = globaltimer_ns();
    for (;;) {
        if (bar_try(bar, parity)) return true;
        if (globaltimer_ns() - t0 > WAIT_LIMIT_NS) return false;
    }
}
// Shared-memory matrix descriptors, 128-byte swizzle: rows of 128 bytes, groups of 8 rows 1024 bytes apart; lbo: distance of
// the 64-element blocks of a transposed operand. The high word is the same for every operand, so that a product costs
// one 32-bit addition for each descriptor.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
__device__ __forceinline__ void mma_smem_a(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI));
}
__device__ __forceinline__ void mma_tmem_a(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(DESC_HI));
}
#define EB_R16(r, o)                                                                                                        \
    "=r"(r[o + 0]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]),         \
        "=r"(r[o + 7]), "=r"(r[o + 8]), "=r"(r[o + 9]), "=r"(r[o + 10]), "=r"(r[o + 11]), "=r"(r[o + 12]), "=r"(r[o + 13]), \
        "=r"(r[o + 14]), "=r"(r[o + 15])
#define EB_W16(r, o)                                                                                                    \
    "r"(r[o + 0]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]),            \
        "r"(r[o + 7]), "r"(r[o + 8]), "r"(r[o + 9]), "r"(r[o + 10]), "r"(r[o + 11]), "r"(r[o + 12]), "r"(r[o + 13]),    \
        "r"(r[o + 14]), "r"(r[o + 15])
// 32 columns of this warp's 32 lanes; the wait names the registers, so that nothing uses them before it
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : EB_R16(r, 0), EB_R16(r, 16)
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
    asm volatile(""
                 : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
// 64 columns, both loads in flight together
__device__ __forceinline__ void tm_ld64(uint32_t addr, uint32_t (&r)[64]) {
#define EB_LD32(o)                                                                                                            \
    asm volatile(                                                                                                             \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"  \
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"                                                                \
        : EB_R16(r, o), EB_R16(r, o + 16)                                                                                     \
        : "r"(addr + o))
    EB_LD32(0);
    EB_LD32(32);
#undef EB_LD32
#define EB_RW8(o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
    asm volatile("tcgen05.wait::ld.sync.aligned;" : EB_RW8(0), EB_RW8(8)::"memory");
    asm volatile("" : EB_RW8(16), EB_RW8(24));
    asm volatile("" : EB_RW8(32), EB_RW8(40));
    asm volatile("" : EB_RW8(48), EB_RW8(56));
#undef EB_RW8
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        EB_W16(r, 0), EB_W16(r, 16)
        : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_box(const CUtensorMap* map, void* dst, uint64_t* bar, int x, int row, int head, int page) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(row), "r"(head), "r"(page)
        : "memory");
}

__device__ __forceinline__ float ex2(float v) {  // 2 units of 32 bits; results below 2^-126 are zero, as weights of them may be
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// two 32-bit operations in one instruction
__device__ __forceinline__ uint64_t f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ bool elect() {  // one lane of a converged warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }

// The walk of a block through its share: work in (sequence, pair of row tiles, kv head, unit) order. Shares are even in
// ticks: one for a unit and TILE_TICKS for a pair's q and output; where there are fewer than CUT_UNITS units for each block, pairs
// are cut into so many shares that every block pays for q and output, and only units count.
constexpr int TILE_TICKS = 3, CUT_UNITS = 8;
struct Pair {
    int t0, t1;                   // tokens of the pair (32-bit pools: of one row tile)
    int low_min, lim_max;         // positions that some row sees: [low_min, lim_max] and the first n_sink
    int us, uw, ue;               // their units
    __device__ __forceinline__ int n() const { return max(1, us + ue - uw); }
    __device__ __forceinline__ int unit(int i) const { return i < us ? i : uw + (i - us); }
};
__device__ __forceinline__ Pair pair_of(const PagedAttnArgs& A, const Seq& sq, int pair, int tok) {
    Pair p;
    p.t0 = pair * tok;
    p.t1 = min(sq.q, p.t0 + tok);
    const int first = sq.kv - sq.q + p.t0;
    p.lim_max = sq.kv - sq.q + p.t1 - 1;
    p.low_min = A.window > 0 ? max(first, 0) - A.window + 1 : 0;  // a row before position 0 sees nothing
    p.ue = (max(p.lim_max, -1) + UNIT) / UNIT;
    p.uw = min(max(0, p.low_min) / UNIT, p.ue);
    p.us = A.window > 0 ? min((min(A.n_sink, max(p.lim_max, -1) + 1) + UNIT - 1) / UNIT, p.uw) : 0;
    return p;
}
__device__ __forceinline__ bool tc_takes(const PagedAttnArgs& A, const Seq& sq) { return sq.q > 0 && sq.q * A.c.grp > A.rows_min; }

struct Walk {
    const PagedAttnArgs& A;
    int tok, extra, seq, pair = 0;  // tok: tokens of a pair; extra: its ticks beside its units'
    long long at, end, base;
    Seq sq;
    Pair pr;
    int kvh, u0, n_it, nu;
    __device__ Walk(const PagedAttnArgs& A_, int tok_, int extra_, int seq_, long long base_, long long at_, long long end_)
        : A(A_), tok(tok_), extra(extra_), seq(seq_), at(at_), end(end_), base(base_) {
        sq.q = 0;
    }
    __device__ bool next() {
        while (at < end) {
            if (seq >= A.c.n_seq) return false;
            sq = paged_seq(A.c, seq, false);
            if (!tc_takes(A, sq) || pair * tok >= sq.q) {
                seq++;
                pair = 0;
                continue;
            }
            pr = pair_of(A, sq, pair, tok);
            nu = pr.n();
            const int ticks = nu + extra;
            const long long w = (long long)ticks * A.c.n_kv;
            if (at >= base + w) {
                base += w;
                pair++;
                continue;
            }
            const int idx = (int)(at - base);
            kvh = idx / ticks;
            const int t0 = idx - kvh * ticks, t1 = (int)min((long long)ticks, t0 + (end - at));
            at += t1 - t0;
            u0 = max(0, t0 - extra);
            n_it = max(0, t1 - extra) - u0;
            if (n_it > 0) return true;  // else this block's share ends before the tile's first unit
        }
        return false;
    }
};

template <int N>
__device__ __forceinline__ void regs_more() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_less() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

template <int HD, bool F32>
__global__ void __launch_bounds__(Tc<HD, F32>::NT, 1) k_paged_attn_tc(PagedAttnArgs A, const __grid_constant__ CUtensorMap kmap,
                                                                      const __grid_constant__ CUtensorMap vmap, int box) {
    using C = Tc<HD, F32>;
    constexpr int TC_NT = C::NT;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sq_ = sm;                      // q: [tile][lo, hi][column block][128 rows][128 bytes]
    uint8_t* skv = sm + C::Q_BYTES;         // k, v tiles
    Bars& B = *reinterpret_cast<Bars*>(skv + C::NST * C::STAGE);
    const PagedArgs& a = A.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tpt = MROWS / a.grp;  // tokens of a row tile
    if (tid == 0) {
        for (int i = 0; i < C::NST; i++) {
            mbar_init(&B.kv_full[i], F32 ? 32 * C::N_LOAD : 1);
            mbar_init(&B.kv_empty[i], 1);
        }
        for (int m = 0; m < 2; m++) {
            mbar_init(&B.q_full[m], MROWS);
            mbar_init(&B.s_full[m][0], 2);
            mbar_init(&B.s_full[m][1], 2);
            mbar_init(&B.p_full[m], MROWS);
            mbar_init(&B.pv_done[m], 2);
        }
        mbar_init(&B.o_free, MROWS);
        for (int b = 0; b < 3; b++) mbar_init(&B.s_free[b], 1);
        mbar_fence_init();
    }
    if (warp == C::W_LOAD) tc_alloc(&B.tmem, C::COLS);
    pdl_wait();
    pdl_trigger();
    // ---- this block's share: sums over the sequences of their units and pairs
    long long units = 0, pairs = 0, mine_u = 0, mine_p = 0, upto_u = 0, upto_p = 0;  // of sequence s0 + tid; with all before it
    auto scan = [&](int s0, bool flag) {
        mine_u = mine_p = 0;
        if (s0 + tid < a.n_seq) {
            const Seq sq = paged_seq(a, s0 + tid, flag);
            if (tc_takes(A, sq))
                for (int p = 0; p * C::NM * tpt < sq.q; p++, mine_p++) mine_u += pair_of(A, sq, p, C::NM * tpt).n();
        }
        upto_u = mine_u;
        upto_p = mine_p;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, upto_u, o), p = __shfl_up_sync(0xffffffffu, upto_p, o);
            if (lane >= o) {
                upto_u += u;
                upto_p += p;
            }
        }
        __syncthreads();  // the sums of the round before are read
        if (lane == 31) {
            B.scan_u[warp] = upto_u;
            B.scan_p[warp] = upto_p;
        }
        __syncthreads();
        upto_u += units;
        upto_p += pairs;
        for (int w = 0; w < TC_NT / 32; w++) {
            if (w < warp) {
                upto_u += B.scan_u[w];
                upto_p += B.scan_p[w];
            }
            units += B.scan_u[w];
            pairs += B.scan_p[w];
        }
    };
    if (tid == 0) {
        A.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
        B.seq = a.n_seq;
        B.start = 0;
    }
    for (int s0 = 0; s0 < a.n_seq; s0 += TC_NT) scan(s0, blockIdx.x == 0);
    const int extra = units * a.n_kv >= (long long)CUT_UNITS * gridDim.x ? TILE_TICKS : 0;
    const long long total = (units + extra * pairs) * a.n_kv;
    const long long share = max(div64(total + gridDim.x - 1, gridDim.x), (long long)A.min_units);
    const long long begin = share * blockIdx.x, end = min(total, begin + share);
    units = pairs = 0;
    for (int s0 = 0; s0 < a.n_seq && begin < total && (units + extra * pairs) * a.n_kv <= begin; s0 += TC_NT) {
        if (a.n_seq > TC_NT)
            scan(s0, false);
        else
            units = total;  // scanned already: one round
        const long long to = (upto_u + extra * upto_p) * a.n_kv, from = to - (mine_u + extra * mine_p) * a.n_kv;
        if (from <= begin && begin < to) {
            B.seq = s0 + tid;
            B.start = from;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = B.tmem;
    Walk w(A, C::NM * tpt, extra, B.seq, B.start, begin, end);
    uint32_t ok_all = 1;
    (void)ok_all;
    bool ok = true;  // a bounded wait that gives up ends the walk; the other warps' own waits then give up too

    if (warp < 4 * C::NM) {
        regs_more<C::REGS_SOFTMAX>();
        // ---------------------------------------------------------------- softmax and sums of row tile mt
        const int mt = warp >> 2, r = tid & 127;
        uint8_t* q_lo = sq_ + mt * 2 * C::TILE;
        uint8_t* q_hi = q_lo + C::TILE;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t o_tm = tmem + lanes + C::O_COL;
        const int n_box = UNIT / box;
        uint32_t n_s = 0, n_pv = 0, n_valid = 0, n_buf = 0;  // uses of the barriers, units and score buffers so far
        while (ok && w.next()) {
            const int tok = w.pr.t0 + mt * tpt + r / a.grp;
            const int n_m = !F32 && w.pr.t0 + tpt < w.pr.t1 ? 2 : 1;
            if (mt >= n_m) {  // the pair has one row tile
                n_valid += w.n_it;
                n_buf += w.n_it;
                continue;
            }
            const bool row_ok = r < tpt * a.grp && tok < w.pr.t1;
            const int head = w.kvh * a.grp + r % a.grp;
            const int lim = row_ok ? w.sq.kv - w.sq.q + tok : -1;
            const int low = A.window > 0 ? max(0, max(lim, 0) - A.window + 1) : 0;
            // ---- q: every row scaled by the power of two that brings its largest element to [2^14, 2^15), then split. The low
            // parts are exact to 2^-25 of that: an element is held to 2^-22 of itself or 2^-39 of its row's largest. (One scale for a
            // warp's rows, which let a large row take the bits of the small ones beside it, was 0.7 % faster over a long prompt.) Rows come one (hd 128) or two (hd 64)
            // to a load instruction.
            float cs;
            {
                constexpr int LPR = HD / 4, RPP = 32 / LPR;
                const int el = lane % LPR, sub = lane / LPR;
                const float* mine = A.q + (size_t)(w.sq.q0 + (row_ok ? tok : w.pr.t0)) * A.ldq + (size_t)head * HD;  // lane = row
                const uint32_t rows_ok = __ballot_sync(0xffffffffu, row_ok);
                auto load = [&](int row, float4& f) {
                    const float* src =
                        reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(mine), row + sub));
                    asm volatile("ld.global.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "l"(src + 4 * el));
                };
                // of a row whose largest finite element has these bits; elements that are not finite make a NaN of the row alone
                auto scale_of = [](uint32_t mx) { return mx > 0 ? pow2f(min(max(14 - ((int)(mx >> 23) - 127), -100), 100)) : 1.f; };
                uint32_t mx_mine = 0;  // of the row of this thread
                float4 f[32 / RPP];    // all of the warp's rows in flight at once (the sums are not live yet)
#pragma unroll
                for (int i = 0; i < 32 / RPP; i++) load(i * RPP, f[i]);
#pragma unroll
                for (int i = 0; i < 32 / RPP; i++) {
                    const int ro = i * RPP + sub, row = 32 * (warp & 3) + ro;
                    const float v = fmaxf(fmaxf(fabsf(f[i].x), fabsf(f[i].y)), fmaxf(fabsf(f[i].z), fabsf(f[i].w)));
                    uint32_t mx = v < INFINITY ? __float_as_uint(v) : 0u;  // bits of values >= 0 have their order
                    if constexpr (LPR == 32) {
                        mx = __reduce_max_sync(0xffffffffu, mx);
                        if (lane == i) mx_mine = mx;
                    } else {
#pragma unroll
                        for (int o = LPR / 2; o; o >>= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        const uint32_t other = __shfl_sync(0xffffffffu, mx, (lane % RPP) * LPR);
                        if (lane / RPP == i) mx_mine = other;
                    }
                    float sc = scale_of(mx);
                    if (A.scale <= 0.f) sc = A.scale < 0.f ? -sc : 0.f;  // the running maximum is that of +c S
                    if (!((rows_ok >> ro) & 1)) f[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    const __half2 h0 = __floats2half2_rn(f[i].x * sc, f[i].y * sc), h1 = __floats2half2_rn(f[i].z * sc, f[i].w * sc);
                    const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
                    const __half2 l0 = __floats2half2_rn(fmaf(f[i].x, sc, -b0.x), fmaf(f[i].y, sc, -b0.y)),
                                  l1 = __floats2half2_rn(fmaf(f[i].z, sc, -b1.x), fmaf(f[i].w, sc, -b1.y));
                    const int ch = el >> 1;  // 16-byte chunk
                    const int at = q_at(row, ch) + (el & 1) * 8;
                    *reinterpret_cast<uint2*>(q_hi + at) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                    *reinterpret_cast<uint2*>(q_lo + at) =
                        make_uint2(*reinterpret_cast<const uint32_t*>(&l0), *reinterpret_cast<const uint32_t*>(&l1));
                }
                cs = fmaxf(fabsf(A.scale) * 1.4426950408889634f / scale_of(mx_mine), 1e-37f);  // never zero: c times -infinity
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&B.q_full[mt]);
            }
            uint64_t acc[HD / 2];
#pragma unroll
            for (int c = 0; c < HD / 2; c++) acc[c] = 0;
            float m = -INFINITY, l = 0.f, alpha = 1.f;
            n_buf += mt;
#pragma unroll 1
            for (int i = 0;; i++) {
                if (i > 0) {  // acc <- acc alpha + O of the unit before
                    ok = bar_wait(&B.pv_done[mt], n_pv++ & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const float vb = F32 ? B.v_back[(n_valid - 1) % VALID_RING] : 1.f;
                    const uint64_t al = f2(alpha, alpha), vb2 = f2(vb, vb);
#pragma unroll
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t o[32];
                        tm_ld32(o_tm + c, o);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const uint64_t u = f2(__uint_as_float(o[j]), __uint_as_float(o[j + 1]));
                            acc[(c + j) / 2] = F32 ? fma2(u, vb2, fma2(acc[(c + j) / 2], al, 0)) : fma2(acc[(c + j) / 2], al, u);
                        }
                    }
                    tc_fence_before();
                    mbar_arrive(&B.o_free);
                }
                if (i == w.n_it) break;
                const int p0 = w.pr.unit(w.u0 + i) * UNIT;
                ok = bar_wait(&B.s_full[mt][n_s & 1], (n_s >> 1) & 1);
                n_s++;
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_tm = tmem + lanes + (n_buf % 3) * UNIT, valid = B.valid[n_valid % VALID_RING];
                const float csu = F32 ? fminf(fmaxf(cs * B.k_back[n_valid % VALID_RING], 1e-37f), 1e37f) : cs;
                n_valid++;
                n_buf += n_m;
                const bool all = p0 + UNIT - 1 <= lim && (p0 >= low || p0 + UNIT <= A.n_sink) && valid == (1u << n_box) - 1;
                if (!__all_sync(0xffffffffu, all)) {  // hidden positions' scores become -infinity
#pragma unroll 1
                    for (int c = 0; c < UNIT; c += 32) {
                        const int p = p0 + c;
                        uint32_t ok32 = 0;
                        if (box >= 32)
                            ok32 = (valid >> (c / box)) & 1 ? 0xffffffffu : 0u;
                        else
                            ok32 = ((valid >> (c / 16)) & 1 ? 0xffffu : 0u) | ((valid >> (c / 16 + 1)) & 1 ? 0xffff0000u : 0u);
                        ok32 &= low_bits(lim - p + 1) & (~low_bits(low - p) | low_bits(A.n_sink - p));
                        uint32_t s[32];
                        tm_ld32(s_tm + c, s);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!((ok32 >> j) & 1)) s[j] = 0xff800000u;
                        tm_st32(s_tm + c, s);
                    }
                    tm_wait_st();
                }
                float mx = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < UNIT; c += 64) {
                    uint32_t s[64];
                    tm_ld64(s_tm + c, s);
                    float m2 = -INFINITY;
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        mx = fmaxf(mx, fmaxf(__uint_as_float(s[j]), __uint_as_float(s[j + 1])));
                        m2 = fmaxf(m2, fmaxf(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])));
                    }
                    mx = fmaxf(mx, m2);
                }
                const float mn = mx == -INFINITY ? m : fmaxf(m, mx * csu);
                alpha = mn == -INFINITY ? 1.f : ex2(m - mn);
                m = mn;
                // c S - (m - 15) in one rounding, of which c S loses none: where m itself is rounded by more than a little (from
                // 2^22 an eighth), the largest weight would miss 2^15 and overflow. Such scores are rounded first, as m was. To
                // look for them costs 0.8 % of a long prompt.
                float c1 = csu, mo = mn == -INFINITY ? 0.f : mn - 15.f;
                const bool far = mn != -INFINITY && fabsf(mn) >= 4194304.f;
                if (__any_sync(0xffffffffu, far)) {
#pragma unroll 1
                    for (int c = 0; c < UNIT; c += 32) {
                        uint32_t s[32];
                        tm_ld32(s_tm + c, s);
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (far) s[j] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(s[j]), csu), mn));
                        tm_st32(s_tm + c, s);
                    }
                    tm_wait_st();
                    if (far) {
                        c1 = 1.f;
                        mo = -15.f;
                    }
                }
                const uint64_t cs2 = f2(c1, c1), mo2 = f2(-mo, -mo);
                uint64_t ls2 = 0;
#pragma unroll 1
                for (int c = 0; c < UNIT; c += 32) {
                    uint32_t s[32], out[32];
                    tm_ld32(s_tm + c, s);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float u, v, d0, d1;
                        un2(fma2(f2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), cs2, mo2), u, v);
                        u = ex2(u);
                        v = ex2(v);
                        const uint64_t uv = f2(u, v);
                        ls2 = add2(ls2, uv);
                        const __half2 h = __floats2half2_rn(u, v);
                        const float2 b = __half22float2(h);
                        un2(add2(uv, f2(-b.x, -b.y)), d0, d1);
                        const __half2 l2 = __floats2half2_rn(d0, d1);
                        out[j / 2] = *reinterpret_cast<const uint32_t*>(&h);
                        out[16 + j / 2] = *reinterpret_cast<const uint32_t*>(&l2);
                    }
                    tm_st32(s_tm + c, out);
                }
                float ls, ls_b;
                un2(ls2, ls, ls_b);
                l = fmaf(l, alpha, ls + ls_b);
                tm_wait_st();
                tc_fence_before();
                mbar_arrive(&B.p_full[mt]);
            }
            n_buf -= mt;
            if (!ok) break;
            const bool whole = w.u0 == 0 && w.n_it == w.nu;
            if (!whole && w.u0 == 0 && tid == 0) {
                const long long tile_end = w.at + (w.nu - w.n_it);
                A.meta[blockIdx.x] = make_int4(((int)div64(tile_end - 1, share) - blockIdx.x) | (w.pr.t1 - w.pr.t0) * a.grp << 16, w.sq.q0, w.kvh,
                                                w.pr.t0 * a.grp);
            }
            // ---- the warp's rows through the bytes of their own q (which is read), so that a row leaves as one run: to the output, or
            // to this block's record (rows in (token, head) order: the two tiles' rows follow each other)
            const int rr = mt * tpt * a.grp + r;
            float* rec = A.part + ((size_t)blockIdx.x * 2 + (w.u0 == 0 ? 1 : 0)) * (256 * (HD + 2));
            float* dst = whole ? A.out + (size_t)(w.sq.q0 + (row_ok ? tok : w.pr.t0)) * A.ldo + (size_t)head * HD : rec + (size_t)rr * HD;
            if (!whole && row_ok) {
                rec[256 * HD + rr] = m;
                rec[256 * HD + 256 + rr] = l;
            }
            const float f = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
            const uint64_t ff = f2(f, f);
            uint8_t* st = q_lo + (r & ~31) * 128;  // row 0 of the warp's in every column block
#pragma unroll
            for (int c = 0; c < HD / 4; c++) {
                float4 v;
                un2(fma2(acc[2 * c], ff, 0), v.x, v.y);
                un2(fma2(acc[2 * c + 1], ff, 0), v.z, v.w);
                *reinterpret_cast<float4*>(st + stage_at(lane, c)) = v;
            }
            __syncwarp();
            {
                constexpr int LPR = HD / 4, RPP = 32 / LPR;
                const int el = lane % LPR, sub = lane / LPR;
                const uint32_t rows_ok = __ballot_sync(0xffffffffu, row_ok);
                // rows read before the first of them is written, since the stores hold later reads back: the output of a tile took
                // 2.5 instead of 3.2 us of a block that has one
                constexpr int AHEAD = 8;
#pragma unroll 1
                for (int i = 0; i < 32; i += AHEAD * RPP) {
                    float4 v[AHEAD];
                    float* d[AHEAD];
#pragma unroll
                    for (int j = 0; j < AHEAD; j++) {
                        const int row = i + j * RPP + sub;
                        d[j] = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(dst), row));
                        v[j] = *reinterpret_cast<const float4*>(st + stage_at(row, el));
                    }
#pragma unroll
                    for (int j = 0; j < AHEAD; j++)
                        if ((rows_ok >> (i + j * RPP + sub)) & 1) *reinterpret_cast<float4*>(d[j] + 4 * el) = v[j];
                }
            }
            __syncwarp();
        }
    } else if (F32 && warp < C::W_LOAD + C::N_LOAD) {
        regs_less<C::REGS_LOAD>();
        // ---------------------------------------------------------------- k and v tiles of 32-bit pools
        // Eight warps, 16 positions each (of one page): read, scaled by the power of two that brings the tile's largest element to
        // [2^14, 2^15), split in two 11-bit parts. What the parts leave out of an element is 2^-39 of the tile's largest, or 2^-22 of
        // the element itself, whichever is more: below the rounding of 32 bits for a score of elements of one size, and for the
        // columns of v that are not 2^-16 of the tile's largest or less. Positions that no row sees are not read: their rows are zero.
        constexpr int LPR = HD / 4, RPP = 32 / LPR, N = 16 / RPP;
        const int cw = warp - C::W_LOAD, el = lane % LPR, sub = lane / LPR;
        uint32_t n = 0, n_valid = 0;
        auto any = [&](int p) { return p <= w.pr.lim_max && (p >= w.pr.low_min || p < A.n_sink); };
        auto page_id = [&](int i) {  // lanes 0 .. 7: the pages of the unit's eight groups of 16 positions; -1: none that is seen
            const int p = w.pr.unit(w.u0 + i) * UNIT + 16 * (lane & 7);
            int id = -1;
            if (i < w.n_it && p <= w.pr.lim_max && (p + 15 >= w.pr.low_min || p < A.n_sink)) {
                id = a.table[(size_t)w.seq * a.table_ld + p / a.page];
                if ((unsigned)id >= (unsigned)a.n_pages) {
                    if (cw == 0 && lane < 8) paged_flag(a.status);
                    id = -2;
                }
            }
            return id;
        };
        while (ok && w.next()) {
            int ids = page_id(0);
            for (int i = 0; i < w.n_it && ok; i++) {
                const uint32_t valid = __ballot_sync(0xffffffffu, ids != -2) & 0xff;
                const int id = __shfl_sync(0xffffffffu, ids, cw), p = w.pr.unit(w.u0 + i) * UNIT + 16 * cw;
                const size_t at = (size_t)(id >= 0 ? id : 0) * a.page_stride + ((size_t)w.kvh * a.page + p % a.page) * HD + 4 * lane;
                const float* src[2] = {static_cast<const float*>(a.k) + at, static_cast<const float*>(a.v) + at};
                const bool full = id >= 0 && p + 15 <= w.pr.lim_max && (p >= w.pr.low_min || p + 16 <= A.n_sink);
                if (id >= 0)  // v's lines on their way while k is split
#pragma unroll
                    for (int r = 0; r < 16; r += 8)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(src[1] - 4 * lane + ((r + (lane >> 2)) * HD + (lane & 3) * (HD / 4))));
                ids = page_id(i + 1);
#pragma unroll 1
                for (int kv = 0; kv < 2 && ok; kv++, n++) {
                    float4 f[N];
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        f[j] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (full || (id >= 0 && any(p + j * RPP + sub)))
                            f[j] = __ldg(reinterpret_cast<const float4*>(src[kv] + (size_t)j * 128));
                    }
                    if (kv == 1) {  // and the next unit's k
                        const int idn = __shfl_sync(0xffffffffu, ids, cw);
                        if (idn >= 0) {
                            const int pn = w.pr.unit(w.u0 + i + 1) * UNIT + 16 * cw;
                            const float* s = static_cast<const float*>(a.k) + (size_t)idn * a.page_stride +
                                             ((size_t)w.kvh * a.page + pn % a.page) * HD;
#pragma unroll
                            for (int r = 0; r < 16; r += 8)
                                asm volatile("prefetch.global.L2 [%0];" ::"l"(s + (r + (lane >> 2)) * HD + (lane & 3) * (HD / 4)));
                        }
                    }
                    float mx = 0.f;
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        const float v = fmaxf(fmaxf(fabsf(f[j].x), fabsf(f[j].y)), fmaxf(fabsf(f[j].z), fabsf(f[j].w)));
                        if (v < INFINITY) mx = fmaxf(mx, v);
                    }
#pragma unroll
                    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    if (lane == 0) B.wmax[n & 1][cw] = mx;
                    asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 8; j++) mx = fmaxf(mx, B.wmax[n & 1][j]);
                    const int ex = (int)((__float_as_uint(mx) >> 23) & 255) - 127, e = min(max(14 - ex, -100), 100);
                    const float sc = mx > 0.f ? pow2f(e) : 1.f;
                    const uint32_t st = n % C::NST, use = n / C::NST;
                    if (use > 0) ok = bar_wait(&B.kv_empty[st], (use - 1) & 1);
                    // a wait that gave up is taken by all eight warps alike: the barrier above counts on them
                    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 2, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                                 : "=r"(ok_all)
                                 : "r"((uint32_t)ok)
                                 : "memory");
                    ok = ok_all != 0;
                    if (!ok) break;
                    if (cw == 0 && lane == 0) {
                        (kv ? B.v_back : B.k_back)[n_valid % VALID_RING] = mx > 0.f ? pow2f(-e) : 1.f;
                        if (kv == 0) B.valid[n_valid % VALID_RING] = valid;
                    }
                    uint8_t* hi = skv + st * C::STAGE;
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        const int row = 16 * cw + j * RPP + sub, ch = el >> 1;
                        const __half2 h0 = __floats2half2_rn(f[j].x * sc, f[j].y * sc), h1 = __floats2half2_rn(f[j].z * sc, f[j].w * sc);
                        const float2 b0 = __half22float2(h0), b1 = __half22float2(h1);
                        const __half2 l0 = __floats2half2_rn(fmaf(f[j].x, sc, -b0.x), fmaf(f[j].y, sc, -b0.y)),
                                      l1 = __floats2half2_rn(fmaf(f[j].z, sc, -b1.x), fmaf(f[j].w, sc, -b1.y));
                        const int to = (ch >> 3) * C::BLK + row * 128 + (((ch & 7) ^ (row & 7)) << 4) + (el & 1) * 8;
                        *reinterpret_cast<uint2*>(hi + to) =
                            make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                        *reinterpret_cast<uint2*>(hi + C::TILE + to) =
                            make_uint2(*reinterpret_cast<const uint32_t*>(&l0), *reinterpret_cast<const uint32_t*>(&l1));
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    mbar_arrive(&B.kv_full[st]);
                }
                n_valid++;
            }
        }
    } else {
        regs_less<C::REGS_ISSUE>();
        if (!F32 && (warp == C::W_LOAD || warp == C::W_LOAD_V)) {
        // ---------------------------------------------------------------- k and v tiles
        const bool is_v = warp == C::W_LOAD_V;
        const CUtensorMap* map = is_v ? &vmap : &kmap;
        const int n_box = UNIT / box, slot0 = is_v ? C::NK : 0, slots = is_v ? C::NV : C::NK;
        uint32_t n = 0;  // units
        while (ok && w.next()) {
            for (int i = 0; i < w.n_it && ok; i++, n++) {
                const int p = w.pr.unit(w.u0 + i) * UNIT + lane * box;
                int id = a.n_pages;  // outside the pool: the box is filled with zeros
                bool good = lane < n_box;
                if (good && p <= w.pr.lim_max && (p + box - 1 >= w.pr.low_min || p < A.n_sink)) {
                    id = a.table[(size_t)w.seq * a.table_ld + p / a.page];
                    if ((unsigned)id >= (unsigned)a.n_pages) {
                        if (!is_v) paged_flag(a.status);
                        id = a.n_pages;
                        good = false;
                    }
                }
                const uint32_t valid = __ballot_sync(0xffffffffu, good);
                if (!is_v && lane == 0) B.valid[n % VALID_RING] = valid;
                const int slot = slot0 + n % slots;
                const uint32_t use = n / slots;
                if (use > 0) ok = bar_wait(&B.kv_empty[slot], (use - 1) & 1);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(&B.kv_full[slot], C::STAGE);
                __syncwarp();
                if (lane < n_box) {
#pragma unroll
                    for (int b = 0; b < C::HALVES; b++)
                        tma_box(map, skv + slot * C::STAGE + b * C::BLK + lane * box * 128, &B.kv_full[slot], 64 * b, p % a.page, w.kvh, id);
                }
            }
        }
        // copies in flight land before the block ends
        for (uint32_t k = n > (uint32_t)slots ? n - slots : 0; k < n; k++) bar_wait(&B.kv_full[slot0 + k % slots], (k / slots) & 1);
        } else if (warp == C::W_QK) {
        // ---------------------------------------------------------------- products q k
        // Scores rotate through three buffers, so that new ones wait for the product p v that read their buffer, two
        // products before, and not for the last one of their own tile.
        constexpr uint32_t ID_S = tc_idesc_f16(128, UNIT);
        uint32_t n = 0, n_q0 = 0, n_q1 = 0, n_s0 = 0, n_s1 = 0, n_buf = 0;
        const uint32_t q_addr = __shfl_sync(0xffffffffu, smem_u32(sq_), 0), kv_addr = __shfl_sync(0xffffffffu, smem_u32(skv), 0);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        while (ok && w.next()) {
            const bool two = !F32 && w.pr.t0 + tpt < w.pr.t1;
            ok = bar_wait(&B.q_full[0], n_q0++ & 1);
            if (ok && two) ok = bar_wait(&B.q_full[1], n_q1++ & 1);
#pragma unroll 1
            for (int i = 0; i < w.n_it && ok; i++, n++) {
                const uint32_t st = n % C::NK;
#pragma unroll 1
                for (int mt = 0; mt < (two ? 2 : 1); mt++) {
                    const uint32_t b = n_buf % 3, use = n_buf / 3;
                    if (use > 0) ok = bar_wait(&B.s_free[b], (use - 1) & 1);
                    // A wait sees a phase by its parity, so none may complete twice between two looks. A tile's units take turns on two
                    // barriers: its scores may be two units ahead of its softmax, not three. With two tiles the buffer's turn sees to
                    // that, with one the product p v of the unit before the last has to be done.
                    if (ok && !two && n_buf >= 2) ok = bar_wait(&B.s_free[(n_buf - 2) % 3], ((n_buf - 2) / 3) & 1);
                    if (ok && mt == 0) ok = bar_wait(&B.kv_full[st], (n / C::NK) & 1);
                    if (!ok) break;
                    n_buf++;
                    uint64_t* full = &B.s_full[mt][(mt ? n_s1++ : n_s0++) & 1];
                    tc_fence_after();
                    const uint32_t d = tm + b * UNIT;
                    const uint32_t qd = desc_lo(q_addr + mt * 2 * C::TILE, 0), kd = desc_lo(kv_addr + st * C::STAGE, 0);
                    if (elect()) {
#pragma unroll
                        for (int part = 0; part < C::PARTS + 1; part++)  // q_lo k_hi, (q_hi k_lo,) q_hi k_hi: low parts first
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) {
                                const uint32_t off = ((k >> 2) * C::BLK + (k & 3) * 32) >> 4;
                                mma_smem_a(d, qd + (part ? C::TILE >> 4 : 0) + off, kd + (F32 && part == 1 ? C::TILE >> 4 : 0) + off, ID_S,
                                           part | k);
                            }
                        tc_commit(full);
                        mbar_arrive(full);  // what this warp saw of the loads (B.valid) is passed on
                        if (mt == 1 || !two) tc_commit(&B.kv_empty[st]);
                    }
                    __syncwarp();
                }
            }
        }
        // whatever was issued is done before the tensor memory goes back: the last k tile's release follows its products
        if (n > 0) bar_wait(&B.kv_empty[(n - 1) % C::NK], ((n - 1) / C::NK) & 1);
        } else if (warp == C::W_PV) {
        // ---------------------------------------------------------------- products p v
        // O is one buffer, read by the tile's softmax warps while the other products run.
        constexpr uint32_t ID_O = tc_idesc_f16(128, HD) | (1u << 16);
        uint32_t n = 0, n_p0 = 0, n_p1 = 0, n_buf = 0;
        const uint32_t kv_addr = __shfl_sync(0xffffffffu, smem_u32(skv), 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
        while (ok && w.next()) {
            const bool two = !F32 && w.pr.t0 + tpt < w.pr.t1;
#pragma unroll 1
            for (int i = 0; i < w.n_it && ok; i++, n++) {
                const uint32_t st = C::NK + n % C::NV;
                ok = bar_wait(&B.kv_full[st], (n / C::NV) & 1);
                if (!ok) break;
                const int p0 = w.pr.unit(w.u0 + i) * UNIT;
                if (!F32 && (p0 + UNIT - 1 > w.pr.lim_max || (p0 < w.pr.low_min && p0 + UNIT > A.n_sink))) {
                    // positions that no row sees may hold anything: their v rows become zero, as their p are
                    uint8_t* vt = skv + st * C::STAGE;
#pragma unroll 4
                    for (int j = lane >> 3; j < UNIT; j += 4) {  // 8 lanes a row
                        const int p = p0 + j;
                        if (p <= w.pr.lim_max && (p >= w.pr.low_min || p < A.n_sink)) continue;
#pragma unroll
                        for (int h = 0; h < C::HALVES; h++)
                            *reinterpret_cast<uint4*>(vt + h * C::BLK + j * 128 + 16 * (lane & 7)) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
#pragma unroll 1
                for (int mt = 0; mt < (two ? 2 : 1); mt++) {
                    if (n_buf > 0) ok = bar_wait(&B.o_free, (n_buf - 1) & 1);
                    if (ok) ok = bar_wait(&B.p_full[mt], (mt ? n_p1++ : n_p0++) & 1);
                    if (!ok) break;
                    const uint32_t b = n_buf++ % 3;
                    tc_fence_after();
                    const uint32_t vd = desc_lo(kv_addr + st * C::STAGE, C::BLK), p = tm + b * UNIT;
                    if (elect()) {
#pragma unroll
                        for (int part = 0; part < C::PARTS + 1; part++)  // low parts first
#pragma unroll
                            for (int k = 0; k < UNIT / 16; k++)
                                mma_tmem_a(tm + C::O_COL, p + 32 * (k >> 1) + (part ? 0 : 16) + 8 * (k & 1),
                                           vd + ((k * 2048) >> 4) + (F32 && part == 1 ? C::TILE >> 4 : 0), ID_O, part | k);
                        tc_commit(&B.pv_done[mt]);
                        mbar_arrive(&B.pv_done[mt]);  // passes on what this warp saw (B.v_back)
                        tc_commit(&B.s_free[b]);
                        if (mt == 1 || !two) tc_commit(&B.kv_empty[st]);
                    }
                    __syncwarp();
                }
            }
        }
        if (n > 0) bar_wait(&B.kv_empty[C::NK + (n - 1) % C::NV], ((n - 1) / C::NV) & 1);
        }
    }
    if (!ok && lane == 0 && a.status) atomicOr(a.status, (int)ST_WAIT_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == C::W_LOAD) tc_dealloc(tmem, C::COLS);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
    static EncodeFn fn = []() -> EncodeFn {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}
// A layer's pool as [page][kv head][position][hd]; a box: 64 elements (128 bytes, swizzled) of `box` positions.
bool pool_map(CUtensorMap* m, const PagedArgs& a, const void* base, int hd, int box) {
    const EncodeFn fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)a.page, (cuuint64_t)a.n_kv, (cuuint64_t)a.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)a.page * hd * 2, (cuuint64_t)a.page_stride * 2};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1}, steps[4] = {1, 1, 1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, boxes, steps,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool F32>
cudaError_t tc_go(const PagedAttnArgs& A, cudaStream_t st) {
    using C = Tc<HD, F32>;
    int box = F32 ? 16 : UNIT;
    while (A.c.page % box) box /= 2;  // gcd(page, 128): at least 16
    CUtensorMap km{}, vm{};
    if (!F32 && (!pool_map(&km, A.c, A.c.k, HD, box) || !pool_map(&vm, A.c, A.c.v, HD, box))) return cudaErrorInvalidValue;
    cudaFuncAttributes at;
    cudaError_t e = cudaFuncGetAttributes(&at, k_paged_attn_tc<HD, F32>);
    if (e != cudaSuccess || at.numRegs != C::REGS) return e != cudaSuccess ? e : cudaErrorInvalidConfiguration;
    e = smem_limit<C>(k_paged_attn_tc<HD, F32>, C::SMEM);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_paged_attn_tc<HD, F32>, dim3(A.grid), dim3(C::NT), C::SMEM, st, A, km, vm, box);
}
}  // namespace

int paged_tc_grid() { return sm_count(); }
cudaError_t launch_paged_attn_tc(int type, int hd, const PagedAttnArgs& A, cudaStream_t st) {
    if (type == T_F16) return hd == 128 ? tc_go<128, false>(A, st) : tc_go<64, false>(A, st);
    return hd == 128 ? tc_go<128, true>(A, st) : tc_go<64, true>(A, st);
}

}  // namespace eb
