// paged.cu -- the paged key/value cache on sm_100a: rotary positions with the append of new keys and values,
// attention of new tokens over the pages, and copies of whole pages.
//
// A pool holds pages [n_kv][page][hd]; a page of one kv head is one contiguous run, so 16 positions of a head
// (PAGE_MIN) are contiguous too and a warp that takes 16 of them needs one page id.
//
//   k_rope_append   one block per row of the q|k|v projection
//   k_paged_attn    rows of a few tokens against a span of positions, the whole call split evenly over the GPU
//   k_paged_merge   joins the row tiles that the split cut
//   k_pages_copy    page copies of a list of pairs, every layer, both pools
#include <algorithm>
#include <mutex>
#include <type_traits>
#include <utility>

#include "kernels.cuh"
#include "paged.cuh"

namespace eb {
namespace {

// ------------------------------------------------------------------------------------------------
// rotary positions + append
// ------------------------------------------------------------------------------------------------
// Row r of sequence s is at position p = kv - q + (r - q0). Each q and k head x: x <- x / sqrt(mean x^2 + eps) * w
// when weights are given; then for pair i < n_rot / 2 with angle p * inv_freq[i]:
//   (a, b) <- (a cos - b sin, a sin + b cos),  (a, b) = (x[i], x[i + n_rot/2]) or (x[2i], x[2i + 1]).
// The angle and what is left of it after whole turns are in 64 bits (at p = 1e5 a 32-bit product is off by 4e-3 rad), its
// sine and cosine in 32 bits, with the part of the remainder that 32 bits lose added to first order: within 2^-23. A
// sincos in 64 bits cost 1.1 us of the 8 us that a step's call took then, and a seventh of a prompt's rate.
// Bytes: 4 hd (n_head + 2 n_kv) in, 4 hd n_head + 2 hd n_kv es out per row; nothing is read twice. Bound by them: 4,273 rows of 32
// q and 4 kv heads of 128, 32-bit pages: 175 MB in 29.4 us (5.96 TB/s); 32 rows 4.8 us, a chain of dependent loads.
constexpr int AP_NT = 256;
constexpr int AP_PF = 5;  // head vectors a thread loads before it needs the row's sequence: 4,273 rows of 40 heads took 33.4 us with 4
                          // and 32.8 with 6 (registers for one block fewer), 29.4 with 5

__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__half* p, const float (&v)[4]) {  // one rounding to the pool's 11 bits
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

template <typename T, int HD>
__global__ void __launch_bounds__(AP_NT) k_rope_append(PagedArgs a, EahmmfRope rope, const float* __restrict__ qkv,
                                                       int ld, const float* __restrict__ qn,
                                                       const float* __restrict__ kn, float eps, float* __restrict__ q,
                                                       int ldq) {
    constexpr int LPH = HD / 4, HPP = AP_NT / LPH;  // lanes per head, heads per pass of the block
    __shared__ float2 cs[HD / 2];
    __shared__ __align__(16) float xs[HPP][HD];
    const int row = blockIdx.x, tid = threadIdx.x, l = tid % LPH, hp = tid / LPH;
    const uint32_t lanes = LPH == 32 ? 0xffffffffu : 0xffffu << (tid & 16);  // the lanes of this head (two heads a warp at 64)
    const int n_q = a.n_head, n_all = a.n_head + 2 * a.n_kv, half = rope.n_rot / 2;
    pdl_wait();
    pdl_trigger();
    const float* src = qkv + (size_t)row * ld + 4 * l;
    float4 pf[AP_PF];
#pragma unroll
    for (int j = 0; j < AP_PF; j++)
        if (hp + j * HPP < n_all) pf[j] = *reinterpret_cast<const float4*>(src + (size_t)(hp + j * HPP) * HD);
    const float fr = tid < half ? rope.d_inv_freq[tid] : 0.f;
    // the row's sequence: how many sequences end at or before the row
    int seq = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += AP_NT)
        seq += __syncthreads_count(s0 + tid < a.n_seq && a.cu_q[s0 + tid + 1] <= row);
    if (seq >= a.n_seq) return;  // a row behind the last sequence
    const Seq sq = paged_seq(a, seq, tid == 0);
    if (row < sq.q0 || row >= sq.q0 + sq.q) {
        if (tid == 0) paged_flag(a.status);
        return;
    }
    const int pos = sq.kv - sq.q + (row - sq.q0);
    if (pos < 0) {  // no such position: nothing to append, an empty q row
        const float z[4] = {0.f, 0.f, 0.f, 0.f};
        for (int h = hp; h < n_q; h += HPP) store4(q + (size_t)row * ldq + (size_t)h * HD + 4 * l, z);
        return;
    }
    const int id = a.table[(size_t)seq * a.table_ld + pos / a.page];
    if (tid < half) {
        const double ang = (double)pos * (double)fr, turns = rint(ang * 0.15915494309189535);
        const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, ang));  // 2 pi in two parts
        const float r = (float)rest, lo = (float)(rest - (double)r);
        float sn, co;
        sincosf(r, &sn, &co);
        cs[tid] = make_float2(fmaf(-sn, lo, co) * rope.mscale, fmaf(co, lo, sn) * rope.mscale);
    }
    const bool page_ok = (unsigned)id < (unsigned)a.n_pages;
    if (!page_ok && tid == 0) paged_flag(a.status);
    const size_t at = (size_t)(page_ok ? id : 0) * a.page_stride + (size_t)(pos % a.page) * HD + 4 * l;
    __syncthreads();
    // this lane's elements 4l .. 4l + 3 of every head: y = x * co + partner * sn (sn carries the pair's sign)
    float co[4], sn[4];
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const int e = 4 * l + c;
        const bool first = rope.style == EAHMMF_ROPE_HALF ? e < half : (e & 1) == 0;
        const int i = rope.style == EAHMMF_ROPE_HALF ? (first ? e : e - half) : e >> 1;
        const float2 r = e < rope.n_rot ? cs[i] : make_float2(1.f, 0.f);
        co[c] = r.x;
        sn[c] = first ? -r.y : r.y;
    }
    auto head = [&](int h, const float4& x4) {
        float v[4] = {x4.x, x4.y, x4.z, x4.w};
        if (h >= n_q + a.n_kv) {  // a v head, as it is
            if (page_ok) store4(static_cast<T*>(a.v) + at + (size_t)(h - n_q - a.n_kv) * a.page * HD, v);
            return;
        }
        const float* w = h < n_q ? qn : kn;
        if (w) {
            float ss = fmaf(v[0], v[0], fmaf(v[1], v[1], fmaf(v[2], v[2], v[3] * v[3])));
#pragma unroll
            for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
            const float sc = 1.0f / sqrtf(ss / (float)HD + eps);
            const float4 g = __ldg(reinterpret_cast<const float4*>(w) + l);
            v[0] = v[0] * sc * g.x;
            v[1] = v[1] * sc * g.y;
            v[2] = v[2] * sc * g.z;
            v[3] = v[3] * sc * g.w;
        }
        float y[4];
        if (rope.style == EAHMMF_ROPE_HALF) {
            store4(&xs[hp][4 * l], v);
            __syncwarp(lanes);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int e = 4 * l + c;
                y[c] = e < rope.n_rot ? xs[hp][e < half ? e + half : e - half] : 0.f;
            }
            __syncwarp(lanes);
        } else {
            y[0] = v[1];
            y[1] = v[0];
            y[2] = v[3];
            y[3] = v[2];
        }
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (4 * l + c < rope.n_rot) v[c] = fmaf(v[c], co[c], y[c] * sn[c]);
        if (h < n_q)
            store4(q + (size_t)row * ldq + (size_t)h * HD + 4 * l, v);
        else if (page_ok)
            store4(static_cast<T*>(a.k) + at + (size_t)(h - n_q) * a.page * HD, v);
    };
    const int passes = (n_all + HPP - 1) / HPP;
#pragma unroll
    for (int j = 0; j < AP_PF; j++) {
        const int h = hp + j * HPP;
        if (j < passes && h < n_all) head(h, pf[j]);
    }
    for (int j = AP_PF; j < passes; j++) {
        const int h = hp + j * HPP;
        if (h < n_all) head(h, *reinterpret_cast<const float4*>(src + (size_t)h * HD));
    }
}

// ------------------------------------------------------------------------------------------------
// page copies
// ------------------------------------------------------------------------------------------------
// The pairs travel as a kernel argument: the list is in host memory, checked there, and the call neither
// copies nor keeps anything. Bytes: each page read once and written once, in every layer, both pools: 501 pages of 64 KB in 8
// layers, 1.05 GB, in 164 us (6.4 TB/s).
constexpr int CP_NT = 256, CP_VEC = 4;  // 16-byte vectors a thread has in flight
constexpr int CP_PAIRS = 480;           // 3840 bytes of the 4 KB that every kernel's arguments may take
struct CopyList {
    int2 p[CP_PAIRS];
};
__global__ void __launch_bounds__(CP_NT) k_pages_copy(uint4* __restrict__ k, uint4* __restrict__ v, size_t layer_stride,
                                                      size_t page_stride, int vecs, const CopyList list) {
    const int2 pr = list.p[blockIdx.z];
    pdl_wait();
    pdl_trigger();
    uint4* pool = (blockIdx.y & 1) ? v : k;
    const size_t lo = (size_t)(blockIdx.y >> 1) * layer_stride;
    const uint4* s = pool + lo + (size_t)pr.x * page_stride;
    uint4* d = pool + lo + (size_t)pr.y * page_stride;
    const int i0 = blockIdx.x * CP_NT * CP_VEC + threadIdx.x;
    uint4 r[CP_VEC];
#pragma unroll
    for (int j = 0; j < CP_VEC; j++)
        if (i0 + j * CP_NT < vecs) r[j] = s[i0 + j * CP_NT];
#pragma unroll
    for (int j = 0; j < CP_VEC; j++)
        if (i0 + j * CP_NT < vecs) d[i0 + j * CP_NT] = r[j];
}

// ------------------------------------------------------------------------------------------------
// attention of a few rows per sequence
// ------------------------------------------------------------------------------------------------
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q.k_j - m), over the positions j that the row sees: j <= p, and with
// a window j > p - window or j < n_sink. One pass with the running maximum m; parts of a row's positions are
// joined by their (m, sum, o).
//
// A step reads 2 hd es bytes per position and kv head and does 4 hd flops per q head with them: it is bound by
// the reads. 2 sequences of 131,000 positions, 4 kv heads of 128, 16-bit pages: 533 MB in 88 us (6.0 TB/s), with the joining
// launch 92; 32 sequences of 300 to 4,500: 138 MB in 35 us, of which 5 before the first reads and 5 joining. 32-bit pages wait
// for the splitting below: 32 sequences of 200 to 2,050, 101 MB in 31 us. Every warp has its own positions and its own ring of tiles in shared memory, which it fills ahead by
// asynchronous 16-byte copies: no barrier between warps. A tile keeps rows of 128 bytes with exchanged 16-byte chunks
// (chunk c of row r at c ^ (r mod 8)); the sums run over hd and over positions, whose order is free, and so is the order of
// the output's columns, so a thread's operands of several instructions are one 16-byte load without bank conflicts.
//
// Numerics. Activations are 32-bit and the pools hold 11 or 24 bits. q and p are split in two parts of 11 bits
// (hi + lo: 22 bits, 2^-23 relative), which the matrix instructions multiply exactly and add in 32 bits:
//   16-bit pools   m16n8k16: (q_hi + q_lo) k and (p_hi + p_lo) v. Rows of q are first scaled by a power of two to
//                  [2^8, 2^9), p by 2^15, so that the low parts stay above the smallest half
//   32-bit pools   m16n8k8 on 11-bit parts of a 32-bit range: hi hi + lo hi + hi lo (lo lo is 2^-22 of it)
// The matrix instructions cut their running sums where an addition would round, which biases long chains: a step's
// products go to sums of their own (low parts first) and are added to the row's sums in the ordinary way.
// Up to 8 rows (STACK) the two parts of a row lie in rows g and g + 8 of one instruction: no extra work, and the
// thread that holds row g holds row g + 8 too. 16 rows take an instruction for each part.
constexpr int PA_NW = 4, PA_NT = 32 * PA_NW;
constexpr int STEP_BLOCKS = 3;  // blocks an SM holds, by registers and by the rings' shared memory: all run at once (but for 9 to 16
                                // rows over 32-bit pages with heads of 128, whose 82 KB let two run and the rest follow)
constexpr float P_SHIFT = 15.f;

template <typename T>
constexpr int pos_step() {
    return sizeof(T) == 2 ? 16 : 8;  // positions a warp takes at once
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, int bytes) {  // bytes 16, or 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t h2(__half a, __half b) {
    const __half2 v = __halves2half2(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// (x, y) as 11-bit parts in two packed registers
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half hx = __float2half_rn(x), hy = __float2half_rn(y);
    hi = h2(hx, hy);
    lo = h2(__float2half_rn(x - __half2float(hx)), __float2half_rn(y - __half2float(hy)));
}
// x as two parts of 11 bits, hi rounded and lo cut, in integer instructions: at most 2^-21 of x is left out, with either sign. An infinity or a NaN gives a NaN.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// the same of the adjacent values x, y: one subtraction for both
__device__ __forceinline__ void split2_tf32(uint32_t x, uint32_t y, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
    hi[0] = (x + 0x1000u) & 0xffffe000u;
    hi[1] = (y + 0x1000u) & 0xffffe000u;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %6};\n\t"
        "fma.rn.f32x2 a, b, c, a;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=r"(lo[0]), "=r"(lo[1])
        : "r"(x), "r"(y), "r"(hi[0]), "r"(hi[1]), "r"(0xbf800000u));  // x - hi
    lo[0] &= 0xffffe000u;
    lo[1] &= 0xffffe000u;
}
__device__ __forceinline__ float ex2(float v) {  // 2 units of 32 bits; results below 2^-126 are zero, as weights of them may be
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {  // (a, b) += (c, d) in one instruction
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a), "+f"(b)
        : "f"(c), "f"(d));
}
// Two 8 x 8 blocks of 16-bit elements below each other, twice, transposed: the right operands of two column tiles
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// Units of positions that some row of a sequence sees: sink units [0, us), then units [uw, ue).
struct Units {
    int us, uw, ue;
    __device__ __forceinline__ int n() const { return max(1, us + ue - uw); }  // 1: rows that see nothing are written too
    __device__ __forceinline__ int unit(int i) const { return i < us ? i : uw + (i - us); }
};
__device__ __forceinline__ Units units_of(const Seq& sq, int window, int n_sink, int unit) {
    Units u;
    u.ue = (sq.kv + unit - 1) / unit;
    const int low = window > 0 ? max(0, max(0, sq.kv - sq.q) - window + 1) : 0;
    u.uw = min(low / unit, u.ue);
    u.us = window > 0 ? min((min(n_sink, sq.kv) + unit - 1) / unit, u.uw) : 0;
    return u;
}

__device__ __forceinline__ bool step_takes(const PagedAttnArgs& A, const Seq& sq) {
    return sq.q > 0 && (long long)sq.q * A.c.grp <= A.rows_max;
}

template <typename T, int HD, bool STACK>
struct AttnSmem {
    static constexpr int RT = STACK ? 8 : 16;
    static constexpr int KS = sizeof(T) == 2 ? HD / 16 : HD / 8;  // k steps of a score
    static constexpr int TILE = 32 * HD;                          // bytes of a step's k (v) rows
    static constexpr int NS = HD == 128 ? 2 : 4;                  // tiles of a warp's ring: 16 KB, 64 KB a block
    uint8_t ring[PA_NW][NS][2][TILE];                             // at a tile's end the warp's sums [RT][HD + 4]
    uint4 qf[STACK ? 1 : KS * 32 * 2];                            // 16 rows: q in fragment order, hi then lo
    float m[PA_NW][RT], l[PA_NW][RT];
};

// A partial record: o [16][hd], m [16], sum [16].
__host__ __device__ constexpr int part_floats(int hd) { return 16 * hd + 32; }

// Parts of a row joined by their maxima and sums.
struct Joined {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float mj, float lj, const float4& f) {
        const float mn = fmaxf(m, mj);
        if (mn == -INFINITY) {  // nothing seen so far (a NaN sum stays one)
            l += lj;
            return;
        }
        const float a = ex2(m - mn), b = ex2(mj - mn);
        m = mn;
        l = fmaf(l, a, lj * b);
        o.x = fmaf(o.x, a, f.x * b);
        o.y = fmaf(o.y, a, f.y * b);
        o.z = fmaf(o.z, a, f.z * b);
        o.w = fmaf(o.w, a, f.w * b);
    }
};
// Four elements of row r from the records of block b and the `follow` blocks after it, from record j0 on by `step`. A record:
// o [cap][hd], m [cap], sum [cap]; block b's is its second (begun and not finished), the others' their first.
__device__ __forceinline__ void join_records(Joined& j, const float* part, int cap, int hd, int r, int c4, int b, int follow, int j0,
                                             int step) {
    constexpr int N = 4;  // in flight
    for (; j0 <= follow; j0 += N * step) {
        float mj[N], lj[N];
        float4 f[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int k = min(j0 + i * step, follow);
            const float* rec = part + ((size_t)(b + k) * 2 + (k == 0 ? 1 : 0)) * ((size_t)cap * (hd + 2));
            mj[i] = __ldcg(rec + cap * hd + r);
            lj[i] = __ldcg(rec + cap * hd + cap + r);
            f[i] = __ldcg(reinterpret_cast<const float4*>(rec) + r * (hd / 4) + c4);
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            if (j0 + i * step <= follow) j.add(mj[i], lj[i], f[i]);
    }
}
__device__ __forceinline__ void store_joined(const PagedAttnArgs& A, const Joined& j, int q0, int kvh, int row, int hd, int c4) {
    const float inv = j.l == 0.f ? 0.f : 1.f / j.l;
    const int tok = row / A.c.grp;
    *reinterpret_cast<float4*>(A.out + (size_t)(q0 + tok) * A.ldo + (size_t)(kvh * A.c.grp + row - tok * A.c.grp) * hd + 4 * c4) =
        make_float4(j.o.x * inv, j.o.y * inv, j.o.z * inv, j.o.w * inv);
}
template <typename T, int HD, bool STACK, bool WHOLE>
__global__ void __launch_bounds__(PA_NT, STEP_BLOCKS) k_paged_attn(PagedAttnArgs A) {
    constexpr bool H16 = sizeof(T) == 2;
    constexpr int STEP = pos_step<T>(), UNIT = STEP * PA_NW, RT = STACK ? 8 : 16, NR = STACK ? 1 : 2;
    constexpr int KS = AttnSmem<T, HD, STACK>::KS;  // k steps of q k
    constexpr int NT = HD / 8;                      // column tiles of p v
    constexpr int PA_NS = AttnSmem<T, HD, STACK>::NS;
    constexpr int NB = HD * (int)sizeof(T) / 128;   // 128-byte blocks of a row
    constexpr int CPL = STEP * NB * 8 / 32;         // 16-byte chunks of a step's k (v) that a lane copies
    constexpr int JT = STEP / 8;                    // score tiles of a step
    constexpr int PT = 2 * JT;                      // positions whose v rows a thread reads
    constexpr int BLK = STEP * 128;                 // bytes of a block of a tile
    extern __shared__ __align__(128) uint8_t smem_raw[];
    AttnSmem<T, HD, STACK>& S = *reinterpret_cast<AttnSmem<T, HD, STACK>*>(smem_raw);
    auto sums = [&](int w, int r) { return reinterpret_cast<float*>(S.ring[w]) + r * (HD + 4); };
    __shared__ long long s_scan[PA_NW], s_start;
    __shared__ int s_seq;
    const PagedArgs& a = A.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();

    // ---- this block's share of the call: work items in (sequence, kv head, row tile, unit) order; or, where tiles stay whole,
    // every gridDim-th (sequence, kv head) with its row tiles, which needs no sums over the sequences (a kernel of its own: as a
    // branch it took registers that the other needs, 31.1 instead of 29.7 us for 32 sequences over 32-bit pages)
    long long share = 0, begin = 0, end = 0;
    if constexpr (!WHOLE) {
        auto weight = [&](int s, bool flag) -> long long {
            const Seq sq = paged_seq(a, s, flag);
            if (!step_takes(A, sq)) return 0;
            return (long long)units_of(sq, A.window, A.n_sink, UNIT).n() * a.n_kv * ((sq.q * a.grp + RT - 1) / RT);
        };
        long long total = 0, mine = 0, upto = 0;  // of thread's sequence s0 + tid: its weight, and the sum with it
        auto scan = [&](int s0, bool flag) {
            mine = s0 + tid < a.n_seq ? weight(s0 + tid, flag) : 0;
            upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long n = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += n;
            }
            __syncthreads();  // s_scan is read
            if (lane == 31) s_scan[warp] = upto;
            __syncthreads();
            upto += total;
            for (int w = 0; w < PA_NW; w++) {
                if (w < warp) upto += s_scan[w];
                total += s_scan[w];
            }
        };
        for (int s0 = 0; s0 < a.n_seq; s0 += PA_NT) scan(s0, blockIdx.x == 0);
        const long long all = total;
        share = max(div64(all + gridDim.x - 1, gridDim.x), (long long)(A.min_units));
        begin = share * blockIdx.x;
        end = min(all, begin + share);
        if (tid == 0) A.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
        if (begin >= all) return;
        total = 0;
        for (int s0 = 0; s0 < a.n_seq && total <= begin; s0 += PA_NT) {  // the sequence that holds `begin`
            if (a.n_seq > PA_NT)
                scan(s0, false);
            else
                total = all;
            if (mine > 0 && upto - mine <= begin && begin < upto) {
                s_seq = s0 + tid;
                s_start = upto - mine;
            }
        }
        __syncthreads();
    }
    long long seq_at = WHOLE ? 0 : s_start, at = begin;
    long long pick = blockIdx.x;  // whole tiles: sequence * n_kv + kv head, and the row tile
    int seq = WHOLE ? (int)div64(pick, a.n_kv) : s_seq, kvh = (int)(pick - (long long)seq * a.n_kv), rt = 0;
    const T* kp = static_cast<const T*>(a.k);
    const T* vp = static_cast<const T*>(a.v);

    while ((WHOLE || at < end) && seq < a.n_seq) {
        const Seq sq = paged_seq(a, seq, WHOLE && kvh == 0 && rt == 0 && tid == 0);
        const Units un = units_of(sq, A.window, A.n_sink, UNIT);
        const int nu = un.n(), nrt = (sq.q * a.grp + RT - 1) / RT;
        int u0 = 0, n_it = nu;
        if constexpr (WHOLE) {
            if (rt >= nrt || !step_takes(A, sq)) {
                pick += gridDim.x;
                seq = (int)div64(pick, a.n_kv);
                kvh = (int)(pick - (long long)seq * a.n_kv);
                rt = 0;
                continue;
            }
        } else {
            const long long here = (long long)nu * nrt * a.n_kv;
            const bool takes = step_takes(A, sq);
            if (!takes || at >= seq_at + here) {
                if (takes) seq_at += here;
                seq++;
                continue;
            }
            const long long idx = at - seq_at;
            const int item = (int)div64(idx, nu);
            u0 = (int)(idx - (long long)item * nu);
            kvh = item / nrt;
            rt = item - kvh * nrt;
            n_it = (int)min((long long)(nu - u0), end - at);
        }
        // ---- the row tile: rows r0 .. of (token, q head of the group)
        const int r0 = rt * RT, n_rows = min(RT, sq.q * a.grp - r0), p_first = sq.kv - sq.q;
        const int lim_max = p_first + (r0 + n_rows - 1) / a.grp, first_pos = p_first + r0 / a.grp;
        const int low_min = A.window > 0 ? max(first_pos, 0) - A.window + 1 : 0;  // a row before position 0 sees nothing
        const int lim_min = first_pos, low_max = A.window > 0 ? max(lim_max, 0) - A.window + 1 : 0;
        auto any = [&](int j) { return j <= lim_max && (j >= low_min || j < A.n_sink); };

        // ---- k and v of a step: page ids of 32 steps at a time, one per lane, the next 32 fetched ahead
        auto fetch_ids = [&](int it) {
            const int i = it + lane;
            int id = -1;
            if (i < n_it) {
                const int p = un.unit(u0 + i) * UNIT + warp * STEP;
                if (any(p) || any(p + STEP - 1) || (p < low_min && p + STEP > low_min && low_min <= lim_max)) {
                    id = a.table[(size_t)seq * a.table_ld + p / a.page];
                    if ((unsigned)id >= (unsigned)a.n_pages) {
                        paged_flag(a.status);
                        id = -1;
                    }
                }
            }
            return id;
        };
        int ids = fetch_ids(0), ids_next = n_it > 32 ? fetch_ids(32) : -1;
        uint32_t live = 0;  // steps in the ring (bit: it mod 32) whose page is one of the pool's
        const uint32_t ring = smem_u32(S.ring[warp]);
        constexpr int RPP = 32 / (NB * 8);  // rows that a warp's copies of one instruction cover
        const uint32_t lane_at = ((lane % (NB * 8)) >> 3) * BLK + lane / (NB * 8) * 128 + (((lane & 7) ^ (lane / (NB * 8))) << 4);
        auto load = [&](int it) {  // rows of positions that no row sees become zero: 0 * NaN is NaN
            if (it < n_it) {
                if ((it & 31) == 0 && it > 0) {
                    ids = ids_next;
                    if (it + 32 < n_it) ids_next = fetch_ids(it + 32);
                }
                const int id = __shfl_sync(0xffffffffu, ids, it & 31), p = un.unit(u0 + it) * UNIT + warp * STEP;
                live = id >= 0 ? live | 1u << (it & 31) : live & ~(1u << (it & 31));
                const size_t at = (size_t)(id >= 0 ? id : 0) * a.page_stride + ((size_t)kvh * a.page + p % a.page) * HD;
                const uint8_t* ks = reinterpret_cast<const uint8_t*>(kp + at) + 16 * lane;
                const uint8_t* vs = reinterpret_cast<const uint8_t*>(vp + at) + 16 * lane;
                const uint32_t slot = ring + (it % PA_NS) * 2 * AttnSmem<T, HD, STACK>::TILE;
                // rows lane / (8 NB) + RPP j: the exchange of chunks splits into the lane's and j's part
                if (id >= 0 && p + STEP - 1 <= lim_max && (p >= low_min || p + STEP <= A.n_sink)) {
#pragma unroll
                    for (int j = 0; j < CPL; j++) {
                        const uint32_t d = (slot + lane_at + j * RPP * 128) ^ (((j * RPP) & 7) << 4);
                        cp_async16(d, ks + 512 * j);
                        cp_async16(d + AttnSmem<T, HD, STACK>::TILE, vs + 512 * j);
                    }
                } else {
#pragma unroll 2
                    for (int j = 0; j < CPL; j++) {
                        const uint32_t d = (slot + lane_at + j * RPP * 128) ^ (((j * RPP) & 7) << 4);
                        const int n = id >= 0 && any(p + lane / (NB * 8) + j * RPP) ? 16 : 0;
                        cp_async16_or_zero(d, ks + 512 * j, n);
                        cp_async16_or_zero(d + AttnSmem<T, HD, STACK>::TILE, vs + 512 * j, n);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < PA_NS - 1; i++) load(i);
        auto q_row = [&](int r) {
            const int rr = r0 + r, tok = rr / a.grp;
            return A.q + (size_t)(sq.q0 + tok) * A.ldq + (size_t)(kvh * a.grp + (rr - tok * a.grp)) * HD;
        };
        int lim[NR], low[NR];  // the positions that this thread's rows see
        float cs[NR];
        uint32_t qa[STACK ? KS : 1][4];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            const int r = g + 8 * i;
            lim[i] = r < n_rows ? p_first + (r0 + r) / a.grp : -1;
            low[i] = A.window > 0 ? max(lim[i], 0) - A.window + 1 : 0;
            const bool ok = r < n_rows;
            const float* qr = ok ? q_row(r) : nullptr;
            float x[KS * (H16 ? 4 : 2)];  // the thread's elements of the row, in k-step order
            constexpr int PER = H16 ? 4 : 2;
#pragma unroll
            for (int c = 0; c < (int)(sizeof(x) / 16); c++) {
                const int e = H16 ? 64 * (c >> 2) + 8 * (2 * t + ((c >> 1) & 1)) + 4 * (c & 1) : 32 * (c >> 1) + 4 * (2 * t + (c & 1));
                const float4 f = ok ? *reinterpret_cast<const float4*>(qr + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[4 * c] = f.x;
                x[4 * c + 1] = f.y;
                x[4 * c + 2] = f.z;
                x[4 * c + 3] = f.w;
            }
            float sc = 1.f;
            if (H16) {
                float mx = 0.f;
#pragma unroll
                for (int c = 0; c < KS * PER; c++) mx = fmaxf(mx, fabsf(x[c]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const int ex = (int)((__float_as_uint(mx) >> 23) & 255) - 127;  // mx in [2^ex, 2^(ex+1))
                if (ex < 128 && mx > 0.f) sc = pow2f(min(max(8 - ex, -100), 100));
            }
            cs[i] = A.scale * 1.4426950408889634f / sc;
            if (STACK) {
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    if (H16) {
                        split_f16(x[4 * k] * sc, x[4 * k + 1] * sc, qa[k][0], qa[k][1]);
                        split_f16(x[4 * k + 2] * sc, x[4 * k + 3] * sc, qa[k][2], qa[k][3]);
                    } else {
                        split_tf32(x[2 * k], qa[k][0], qa[k][1]);
                        split_tf32(x[2 * k + 1], qa[k][2], qa[k][3]);
                    }
                }
            } else {
                uint32_t* hi = reinterpret_cast<uint32_t*>(S.qf);
#pragma unroll
                for (int k = 0; k < KS; k++)
                    if (k % PA_NW == warp) {
                        uint32_t h0, l0, h1, l1;
                        if (H16) {
                            split_f16(x[4 * k] * sc, x[4 * k + 1] * sc, h0, l0);
                            split_f16(x[4 * k + 2] * sc, x[4 * k + 3] * sc, h1, l1);
                        } else {
                            split_tf32(x[2 * k], h0, l0);
                            split_tf32(x[2 * k + 1], h1, l1);
                        }
                        uint32_t* f = hi + ((size_t)k * 32 + lane) * 8;
                        f[i] = h0;
                        f[2 + i] = h1;
                        f[4 + i] = l0;
                        f[6 + i] = l1;
                    }
            }
        }
        if (!STACK) __syncthreads();
        float o[NT][2 * NR];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 2 * NR; i++) o[n][i] = 0.f;
        float m[NR], l[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) {
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
        for (int it = 0; it < n_it; it++) {
            asm volatile("cp.async.wait_group %0;" ::"n"(PA_NS - 2) : "memory");
            __syncwarp();  // every lane's copies have landed, and every lane is done with the tile that comes free
            load(it + PA_NS - 1);
            const uint8_t* kt = S.ring[warp][it % PA_NS][0];
            const uint8_t* vt = S.ring[warp][it % PA_NS][1];
            const int p_cur = un.unit(u0 + it) * UNIT + warp * STEP;
            const bool on = (live >> (it & 31)) & 1;
            if (!on) continue;  // warp-uniform: no row sees any of the step's positions
            float sacc[JT][4], slow[JT][4];  // the high parts' product and the rest (32-bit pools: and every other high one's)
#pragma unroll
            for (int j = 0; j < JT; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) sacc[j][i] = slow[j][i] = 0.f;
#pragma unroll
            for (int c = 0; c < KS / 2; c++) {  // a 16-byte chunk of the k rows: two k steps
                uint4 w[JT];
#pragma unroll
                for (int j = 0; j < JT; j++)
                    w[j] = *reinterpret_cast<const uint4*>(kt + (c >> 1) * BLK + (8 * j + g) * 128 + (((2 * t + (c & 1)) ^ g) << 4));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int k = 2 * c + h;
                    uint32_t ah[4], al[4];
                    if (STACK) {
#pragma unroll
                        for (int i = 0; i < 4; i++) ah[i] = qa[k][i];
                    } else {
                        const uint4 f = S.qf[(k * 32 + lane) * 2], lo4 = S.qf[(k * 32 + lane) * 2 + 1];
                        ah[0] = f.x, ah[1] = f.y, ah[2] = f.z, ah[3] = f.w;
                        al[0] = lo4.x, al[1] = lo4.y, al[2] = lo4.z, al[3] = lo4.w;
                    }
#pragma unroll
                    for (int j = 0; j < JT; j++) {
                        const uint32_t b0 = h ? w[j].z : w[j].x, b1 = h ? w[j].w : w[j].y;
                        if (H16) {
                            mma_f16(sacc[j], ah, b0, b1);
                            if (!STACK) mma_f16(slow[j], al, b0, b1);
                        } else {
                            uint32_t hi[2], lo[2];
                            split2_tf32(b0, b1, hi, lo);
                            mma_tf32(h ? slow[j] : sacc[j], ah, hi[0], hi[1]);
                            mma_tf32(slow[j], ah, lo[0], lo[1]);
                            if (!STACK) mma_tf32(slow[j], al, hi[0], hi[1]);
                        }
                    }
                }
            }
            // ---- scores of this thread's rows: positions p + 8 j + 2 t + c
            const bool plain = p_cur + STEP - 1 <= lim_min && (p_cur >= low_max || p_cur + STEP <= A.n_sink);  // all rows see all
            float sv[NR][PT];
            float mx[NR];
#pragma unroll
            for (int i = 0; i < NR; i++)
#pragma unroll
                for (int j = 0; j < PT; j++) {
                    const int e = (j & 1) + 2 * i;
                    float raw = H16 && STACK ? sacc[j >> 1][e] : sacc[j >> 1][e] + slow[j >> 1][e];
                    if (STACK) raw += H16 ? sacc[j >> 1][e + 2] : sacc[j >> 1][e + 2] + slow[j >> 1][e + 2];
                    sv[i][j] = raw * cs[i];
                }
            if (!plain) {
#pragma unroll
                for (int i = 0; i < NR; i++)
#pragma unroll
                    for (int j = 0; j < PT; j++) {
                        const int pos = p_cur + 8 * (j >> 1) + 2 * t + (j & 1);
                        if (!(pos <= lim[i] && (pos >= low[i] || pos < A.n_sink))) sv[i][j] = -INFINITY;
                    }
            }
#pragma unroll
            for (int i = 0; i < NR; i++) {
                mx[i] = sv[i][0];
#pragma unroll
                for (int j = 1; j < PT; j++) mx[i] = fmaxf(mx[i], sv[i][j]);
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                mx[i] = fmaxf(mx[i], m[i]);
            }
            bool grew = mx[0] > m[0];
            if (NR == 2) grew = grew || mx[NR - 1] > m[NR - 1];
            if (__any_sync(0xffffffffu, grew)) {
                float al[NR];
#pragma unroll
                for (int i = 0; i < NR; i++) {
                    al[i] = mx[i] == -INFINITY ? 1.f : ex2(m[i] - mx[i]);
                    l[i] *= al[i];
                    m[i] = mx[i];
                }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2 * NR; i++) o[n][i] *= al[i >> 1];
            }
            uint32_t ph[4], pl[4];
#pragma unroll
            for (int i = 0; i < NR; i++) {
                const float mo = m[i] == -INFINITY ? 0.f : __fadd_ru(m[i], -P_SHIFT);  // up: no weight passes 2^15, which halves hold
#pragma unroll
                for (int j = 0; j < PT; j++) {
                    sv[i][j] = ex2(sv[i][j] - mo);
                    l[i] += sv[i][j];
                }
                if (H16) {
#pragma unroll
                    for (int j = 0; j < JT; j++)
                        split_f16(sv[i][2 * j], sv[i][2 * j + 1], ph[2 * j + i], STACK ? ph[2 * j + 1] : pl[2 * j + i]);
                } else {
#pragma unroll
                    for (int j = 0; j < PT; j++) split_tf32(sv[i][j], ph[2 * j + i], STACK ? ph[2 * j + 1] : pl[2 * j + i]);
                }
            }
            // this step's part of the sums apart, see "Numerics"
            auto join = [&](int n, const float (&s)[4]) {
                if (STACK) {
                    float x = s[0], y = s[1];
                    add2(x, y, s[2], s[3]);
                    add2(o[n][0], o[n][1], x, y);
                } else {
                    add2(o[n][0], o[n][1], s[0], s[1]);
                    add2(o[n][2 * NR - 2], o[n][2 * NR - 1], s[2], s[3]);
                }
            };
            if (H16) {
                const uint32_t va = smem_u32(vt) + (lane & 15) * 128;  // lanes 0-15: rows of a column tile's chunk, 16-31: the next chunk
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b[4];
                    ldsm_t(b, va + (n >> 3) * BLK + ((((n & 7) + (lane >> 4)) ^ (lane & 7)) << 4));
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float s[4] = {0.f, 0.f, 0.f, 0.f};
                        if (!STACK) mma_f16(s, pl, b[2 * h], b[2 * h + 1]);
                        mma_f16(s, ph, b[2 * h], b[2 * h + 1]);
                        join(n + h, s);
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < NB; c++) {
                    uint32_t hi[2][4], lo[2][4];  // rows 2t and 2t + 1: chunk g of the block
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const uint4 w = *reinterpret_cast<const uint4*>(vt + c * BLK + (2 * t + j) * 128 + ((g ^ (2 * t + j)) << 4));
                        uint32_t h0[2], l0[2], h1[2], l1[2];
                        split2_tf32(w.x, w.y, h0, l0);
                        split2_tf32(w.z, w.w, h1, l1);
                        hi[j][0] = h0[0], hi[j][1] = h0[1], hi[j][2] = h1[0], hi[j][3] = h1[1];
                        lo[j][0] = l0[0], lo[j][1] = l0[1], lo[j][2] = l1[0], lo[j][3] = l1[1];
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float s[4] = {0.f, 0.f, 0.f, 0.f};
                        if (!STACK) mma_tf32(s, pl, hi[0][e], hi[1][e]);
                        mma_tf32(s, ph, lo[0][e], lo[1][e]);
                        mma_tf32(s, ph, hi[0][e], hi[1][e]);
                        join(4 * c + e, s);
                    }
                }
            }
        }
        __syncwarp();  // the ring is read
        // ---- the four warps' parts joined, then the output or this block's partial record
#pragma unroll
        for (int i = 0; i < NR; i++) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) {
                S.m[warp][g + 8 * i] = m[i];
                S.l[warp][g + 8 * i] = l[i];
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            // 16-bit v: columns 8 n + 2t, + 1; 32-bit v: columns 4 (2t + 8 (n / 4)) + n % 4, + 4
            const int col = H16 ? 8 * n + 2 * t : 4 * (2 * t + 8 * (n / 4)) + n % 4, next = H16 ? 1 : 4;
#pragma unroll
            for (int i = 0; i < NR; i++) {
                sums(warp, g + 8 * i)[col] = o[n][2 * i];
                sums(warp, g + 8 * i)[col + next] = o[n][2 * i + 1];
            }
        }
        __syncthreads();
        const bool whole = WHOLE || (u0 == 0 && n_it == nu);
        float* rec = A.part + ((size_t)blockIdx.x * 2 + (u0 == 0 ? 1 : 0)) * part_floats(HD);
        for (int i = tid; i < n_rows * (HD / 4); i += PA_NT) {
            const int r = i / (HD / 4), c4 = i - r * (HD / 4);
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < PA_NW; w++) M = fmaxf(M, S.m[w][r]);
            float L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < PA_NW; w++) {
                const float e = S.m[w][r] == -INFINITY ? 0.f : exp2f(S.m[w][r] - M);
                if (S.m[w][r] == -INFINITY && !(S.l[w][r] != S.l[w][r])) continue;
                const float4 f = *reinterpret_cast<const float4*>(sums(w, r) + 4 * c4);
                L = fmaf(S.l[w][r], e, L);
                acc.x = fmaf(f.x, e, acc.x);
                acc.y = fmaf(f.y, e, acc.y);
                acc.z = fmaf(f.z, e, acc.z);
                acc.w = fmaf(f.w, e, acc.w);
            }
            if (whole) {
                const float inv = L == 0.f ? 0.f : 1.f / L;
                const int rr = r0 + r, tok = rr / a.grp;
                *reinterpret_cast<float4*>(A.out + (size_t)(sq.q0 + tok) * A.ldo +
                                           (size_t)(kvh * a.grp + (rr - tok * a.grp)) * HD + 4 * c4) =
                    make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                reinterpret_cast<float4*>(rec)[r * (HD / 4) + c4] = acc;
                if (c4 == 0) {
                    rec[16 * HD + r] = M;
                    rec[16 * HD + 16 + r] = L;
                }
            }
        }
        if (!whole && u0 == 0 && tid == 0)  // the blocks after this one hold the rest of the tile
            A.meta[blockIdx.x] = make_int4(((int)div64(at + nu - 1, share) - blockIdx.x) | n_rows << 16, sq.q0, kvh, r0);
        __syncthreads();
        if constexpr (WHOLE)
            rt++;
        else
            at += n_it;
    }
}

// Joins the records of the row tiles that the split cut: block (b, y) takes rows of the tile
// that block b of the attention began and left to the blocks after it (meta: how many, with the tile's rows above bit 16;
// output row of the sequence's first token; kv head; the tile's first row). With ONE one row, its records dealt over the
// block (a long context is cut often), else a row to each group of hd / 4 threads.
constexpr int PM_NT = 256;
template <int HD, bool ONE>
__global__ void __launch_bounds__(PM_NT) k_paged_merge(PagedAttnArgs A, int cap) {
    constexpr int LN = HD / 4, G = PM_NT / LN;
    __shared__ __align__(16) float4 so[ONE ? G : 1][LN];
    __shared__ float sm[G], sl[G];
    const int b = blockIdx.x, lane = threadIdx.x % LN, grp = threadIdx.x / LN;
    const int r = ONE ? blockIdx.y : blockIdx.y * G + grp;
    pdl_wait();
    pdl_trigger();
    const int4 me = A.meta[b];
    if (me.x == 0 || r >= me.x >> 16) return;
    Joined j;
    join_records(j, A.part, cap, HD, r, lane, b, me.x & 0xffff, ONE ? grp : 0, ONE ? G : 1);
    if (ONE) {
        so[grp][lane] = j.o;
        if (lane == 0) {
            sm[grp] = j.m;
            sl[grp] = j.l;
        }
        __syncthreads();
        if (grp) return;
        j = Joined();
#pragma unroll
        for (int i = 0; i < G; i++) j.add(sm[i], sl[i], so[i][lane]);
    }
    store_joined(A, j, me.y, me.z, me.w + r, HD, lane);
}

// Up to this many positions a row tile is one block's work: cutting it would save less than joining it costs. Heads of 128, 4
// kv heads, whole and cut: one sequence over 16-bit pages 11.6 and 15.6 us at 700 positions, 13.9 and 15.4 at 900, 14.8 and 12.7
// at 1,000; over 32-bit pages 14.5 and 16.4 at 320, 17.0 and 14.5 at 380. With more tiles than blocks some blocks take two, and
// a cut pays sooner: 128 sequences over 16-bit pages 26.7 and 30.0 at 400, 33.7 and 31.6 at 500; over 32-bit pages 31.3 and
// 33.4 at 200, 39.5 and 34.9 at 256.
int whole_kv(int es, bool block_each) { return es == 2 ? (block_each ? 896 : 448) : (block_each ? 352 : 224); }
int step_grid() { return STEP_BLOCKS * sm_count(); }

template <typename T, int HD, bool STACK, bool WHOLE>
cudaError_t attn_launch(const PagedAttnArgs& A, int blocks, cudaStream_t st) {
    using Smem = AttnSmem<T, HD, STACK>;
    using Tag = std::pair<Smem, std::bool_constant<WHOLE>>;
    cudaError_t e = smem_limit<Tag>(k_paged_attn<T, HD, STACK, WHOLE>, sizeof(Smem));
    return e == cudaSuccess ? launch_pdl(k_paged_attn<T, HD, STACK, WHOLE>, dim3(blocks), dim3(PA_NT), sizeof(Smem), st, A) : e;
}
template <typename T, int HD, bool STACK>
cudaError_t attn_go(PagedAttnArgs A, int max_kv, cudaStream_t st) {
    constexpr int RT = STACK ? 8 : 16;
    A.grid = step_grid();
    A.min_units = 4;
    const long long heads = (long long)A.c.n_seq * A.c.n_kv;
    if (max_kv <= whole_kv((int)sizeof(T), heads <= A.grid))
        return attn_launch<T, HD, STACK, true>(A, (int)std::min<long long>(heads, A.grid), st);
    cudaError_t e = attn_launch<T, HD, STACK, false>(A, A.grid, st);
    if (e != cudaSuccess) return e;
    // A launch of its own joins the pieces: few tiles, each in many, with a row's pieces dealt over a block; many tiles, each in
    // two or three, with a row to each group. (The block that ends last joining them within the launch took 36.3 instead of
    // 34.7 us for 32 sequences of 300 to 4,500 positions: the fences of every piece cost more than the launch.)
    if ((long long)A.c.n_seq * A.c.n_kv * 16 <= A.grid)
        return launch_pdl(k_paged_merge<HD, true>, dim3(A.grid, RT), dim3(PM_NT), 0, st, A, 16);
    return launch_pdl(k_paged_merge<HD, false>, dim3(A.grid, (RT * HD / 4 + PM_NT - 1) / PM_NT), dim3(PM_NT), 0, st, A, 16);
}
template <typename T, int HD>
cudaError_t attn_rows(const PagedAttnArgs& A, bool stack, int max_kv, cudaStream_t st) {
    return stack ? attn_go<T, HD, true>(A, max_kv, st) : attn_go<T, HD, false>(A, max_kv, st);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
size_t step_ws_bytes(int hd) {
    return align256((size_t)step_grid() * sizeof(int4)) + align256((size_t)step_grid() * 2 * part_floats(hd) * sizeof(float));
}
size_t tc_ws_bytes(int hd) {
    return align256((size_t)paged_tc_grid() * sizeof(int4)) + (size_t)paged_tc_grid() * 2 * 256 * (hd + 2) * sizeof(float);
}
bool tc_call(int grp, int max_q) { return (long long)max_q * grp > STEP_ROWS; }

void carve(PagedAttnArgs& A, int grid, void* ws) {
    A.grid = grid;
    A.meta = static_cast<int4*>(ws);
    A.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + align256((size_t)grid * sizeof(int4)));
}
}  // namespace

size_t paged_attn_ws_bytes(int type, int hd, int grp, int max_q) {
    return step_ws_bytes(hd) + (tc_call(grp, max_q) ? tc_ws_bytes(hd) : 0);
}

cudaError_t launch_paged_attention(int type, int hd, int max_q, int max_kv, PagedAttnArgs A, void* ws, cudaStream_t st) {
    const bool tc = tc_call(A.c.grp, max_q);
    A.rows_min = 0;
    A.rows_max = 0x7fffffff;
    if (tc) {
        // sequences of more than STEP_ROWS rows as chunks; the others, if there may be any, by the step kernel
        A.rows_min = A.c.n_seq > 1 ? STEP_ROWS : 0;
        A.rows_max = A.rows_min;
        A.min_units = 1;
        carve(A, paged_tc_grid(), static_cast<uint8_t*>(ws) + step_ws_bytes(hd));
        cudaError_t e = launch_paged_attn_tc(type, hd, A, st);
        if (e != cudaSuccess) return e;
        e = hd == 128 ? launch_pdl(k_paged_merge<128, false>, dim3(A.grid, 256 / (PM_NT / 32)), dim3(PM_NT), 0, st, A, 256)
                      : launch_pdl(k_paged_merge<64, false>, dim3(A.grid, 256 / (PM_NT / 16)), dim3(PM_NT), 0, st, A, 256);
        if (e != cudaSuccess || A.c.n_seq == 1) return e;
    }
    carve(A, step_grid(), ws);
    const bool stack = (long long)max_q * A.c.grp <= 8;
    if (type == T_F16) return hd == 128 ? attn_rows<__half, 128>(A, stack, max_kv, st) : attn_rows<__half, 64>(A, stack, max_kv, st);
    return hd == 128 ? attn_rows<float, 128>(A, stack, max_kv, st) : attn_rows<float, 64>(A, stack, max_kv, st);
}

cudaError_t launch_rope_append(int type, int hd, const PagedArgs& a, const EahmmfRope& rope, const float* qkv, int ld,
                               const float* qn, const float* kn, float eps, float* q, int ldq, cudaStream_t st) {
    auto go = [&](auto kern) {
        return launch_pdl(kern, dim3(a.n_tok), dim3(AP_NT), 0, st, a, rope, qkv, ld, qn, kn, eps, q, ldq);
    };
    if (type == T_F16) return hd == 128 ? go(k_rope_append<__half, 128>) : go(k_rope_append<__half, 64>);
    return hd == 128 ? go(k_rope_append<float, 128>) : go(k_rope_append<float, 64>);
}

cudaError_t launch_pages_copy(const EahmmfPagedKv& kv, const int* pairs, int n, cudaStream_t st) {
    const size_t es = kv.type == T_F16 ? 2 : 4;
    const int vecs = (int)((size_t)kv.n_kv * kv.page * kv.hd * es / 16);
    for (int i = 0; i < n; i += CP_PAIRS) {
        const int m = std::min(CP_PAIRS, n - i);
        CopyList list;
        for (int j = 0; j < m; j++) list.p[j] = make_int2(pairs[2 * (i + j)], pairs[2 * (i + j) + 1]);
        const cudaError_t e =
            launch_pdl(k_pages_copy, dim3((vecs + CP_NT * CP_VEC - 1) / (CP_NT * CP_VEC), 2 * kv.n_layer, m), dim3(CP_NT), 0,
                       st, static_cast<uint4*>(kv.d_k), static_cast<uint4*>(kv.d_v), kv.layer_stride * es / 16,
                       kv.page_stride * es / 16, vecs, list);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace eb
