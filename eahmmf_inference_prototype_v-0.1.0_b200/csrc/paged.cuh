// paged.cuh -- launch-side declarations of the paged key/value cache (paged.cu) and the device helpers its
// kernels share: a call's sequences, their pages and the positions a row sees.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "../../include/eahmmf_b200.h"
#include "common.cuh"

namespace eb {

constexpr int PAGE_MIN = 16;      // positions per page: a multiple of this, so 16 positions never straddle pages
constexpr int PAGED_MAX_GRP = 64;  // q heads per kv head

// One layer of a cache and the sequences of a call, as the kernels take them.
struct PagedArgs {
    void* k;  // pool of the layer: page p at p * page_stride elements, [n_kv][page][hd] inside
    void* v;
    size_t page_stride;
    int n_pages, n_kv, page, n_head, grp;
    int n_seq, n_tok, table_ld;
    const int* cu_q;    // [n_seq + 1] first activation row of each sequence
    const int* kv_len;  // [n_seq] cached positions with the call's new ones
    const int* table;   // [n_seq][table_ld] page ids
    int* status;
};

__device__ __forceinline__ void paged_flag(int* status) {
    if (status) atomicOr(status, (int)ST_BAD_INDEX);
}

// a / b of non-negative values: nearly always both fit 32 bits, whose division is several times shorter
__device__ __forceinline__ long long div64(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// Sequence s of a call: its activation rows [q0, q0 + q) and kv cached positions. Lengths that do not fit the
// buffers (rows past n_tok, more positions than the table row names) are cut to what does and flagged.
struct Seq {
    int q0, q, kv;
};
__device__ __forceinline__ Seq paged_seq(const PagedArgs& a, int s, bool flag) {
    const int c0 = a.cu_q[s], c1 = a.cu_q[s + 1], n = a.kv_len[s];
    const long long cap = min((long long)a.table_ld * a.page, 0x7fff0000ll);
    Seq r;
    r.q0 = min(max(c0, 0), a.n_tok);
    r.q = min(max(c1, r.q0), a.n_tok) - r.q0;
    r.kv = n < 0 ? 0 : (long long)n > cap ? (int)cap : n;
    if (flag && (r.q0 != c0 || r.q != c1 - c0 || r.kv != n)) paged_flag(a.status);
    return r;
}

cudaError_t launch_rope_append(int type, int hd, const PagedArgs& a, const EahmmfRope& rope, const float* qkv, int ld,
                               const float* qn, const float* kn, float eps, float* q, int ldq, cudaStream_t st);

struct PagedAttnArgs {
    PagedArgs c;
    const float* q;  // [n_tok][ldq]
    float* out;      // [n_tok][ldo]
    int ldq, ldo;
    float scale;
    int window, n_sink;  // window 0: every earlier position is visible
    int grid;            // blocks of the split launch, also the records of `part`
    int min_units;       // least share of a block
    int rows_min, rows_max;  // sequences of more rows (tokens x q heads of a kv head) than rows_min go to the chunk
                             // kernel, of at most rows_max to the step kernel
    float* part;         // [grid][2] partial results
    int4* meta;          // [grid] the row tile a block began and did not finish
};
constexpr int STEP_ROWS = 16;  // rows of a sequence that the step kernel takes in one row tile
size_t paged_attn_ws_bytes(int type, int hd, int grp, int max_q);
cudaError_t launch_paged_attention(int type, int hd, int max_q, int max_kv, PagedAttnArgs a, void* ws, cudaStream_t st);

int paged_tc_grid();  // blocks of the chunk kernel
cudaError_t launch_paged_attn_tc(int type, int hd, const PagedAttnArgs& A, cudaStream_t st);

// Raises a kernel's dynamic shared-memory limit, once on each device; Tag: a type of the kernel's own.
template <typename Tag, typename Kern>
cudaError_t smem_limit(Kern k, size_t bytes) {
    constexpr int MAX_DEV = 64;
    static std::mutex mu;
    static bool done[MAX_DEV] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || dev < 0 || dev >= MAX_DEV) return e != cudaSuccess ? e : cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> g(mu);
    if (!done[dev]) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done[dev] = true;
    return e;
}

// Every sequence of the list (each named once) grows by one position; where there are not enough pages for all of them
// (ST_CAPACITY) none does, and no copy is recorded.
int pages_grow(EahmmfPages* p, const int* seqs, int n);

cudaError_t launch_pages_copy(const EahmmfPagedKv& kv, const int* pairs, int n, cudaStream_t st);

}  // namespace eb
