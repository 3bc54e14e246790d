// pages.cu -- the paged key/value cache on the host: the C entry points of its kernels (paged.cu) with their checks,
// the frequency table of rotary positions, and the bookkeeping of pages (which sequence holds which page, how many
// share it, which copies a step needs).
#include <math.h>

#include <algorithm>
#include <memory>
#include <new>
#include <vector>

#include "paged.cuh"

using namespace eb;

// ---- checks ----------------------------------------------------------------------------------------
namespace {

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_kv(const EahmmfPagedKv* kv) {
    if (!kv) return ST_BAD_ARG;
    if (kv->type != T_F32 && kv->type != T_F16) return ST_BAD_TYPE;
    if (!kv->d_k || !kv->d_v || !aligned(kv->d_k, 16) || !aligned(kv->d_v, 16) || kv->n_layer < 1 || kv->n_pages < 1 ||
        kv->n_kv < 1 || kv->n_kv > 1024 || kv->page < PAGE_MIN || kv->page > 1024 || kv->page % PAGE_MIN ||
        (kv->hd != 64 && kv->hd != 128))
        return ST_BAD_ARG;
    const size_t own = (size_t)kv->n_kv * kv->page * kv->hd;
    if (kv->page_stride < own || kv->page_stride % 8 || kv->layer_stride % 8) return ST_BAD_ARG;
    // pages of a layer beside each other, or a page's layers beside each other; never overlapping
    const bool layer_major = kv->layer_stride >= kv->page_stride * (size_t)(kv->n_pages - 1) + own;
    const bool page_major = kv->layer_stride >= own && kv->page_stride >= kv->layer_stride * (size_t)(kv->n_layer - 1) + own;
    if (kv->n_layer > 1 && !layer_major && !page_major) return ST_BAD_ARG;
    return ST_OK;
}

int check_seqs(const EahmmfPagedSeqs* s) {
    if (!s || s->n_seq < 0 || s->n_tok < 0 || s->max_q < 0 || s->max_kv < 0) return ST_BAD_ARG;
    if (s->n_seq > 0 && (!s->d_cu_q || !s->d_kv_len || !s->d_table || s->table_ld < 1)) return ST_BAD_ARG;
    return ST_OK;
}

bool heads_ok(const EahmmfPagedKv* kv, int n_head) {
    return n_head >= 1 && n_head % kv->n_kv == 0 && n_head / kv->n_kv <= PAGED_MAX_GRP;
}
bool rows_ok(const void* p, int ld, int width) { return p && aligned(p, 16) && ld >= width && ld % 4 == 0; }

PagedArgs args_of(const EahmmfPagedKv* kv, int layer, const EahmmfPagedSeqs* s, int n_head, int* status) {
    const size_t at = (size_t)layer * kv->layer_stride * (kv->type == T_F16 ? 2 : 4);
    PagedArgs a{};
    a.k = static_cast<uint8_t*>(kv->d_k) + at;
    a.v = static_cast<uint8_t*>(kv->d_v) + at;
    a.page_stride = kv->page_stride;
    a.n_pages = kv->n_pages;
    a.n_kv = kv->n_kv;
    a.page = kv->page;
    a.n_head = n_head;
    a.grp = n_head / kv->n_kv;
    a.n_seq = s->n_seq;
    a.n_tok = s->n_tok;
    a.table_ld = s->table_ld;
    a.cu_q = s->d_cu_q;
    a.kv_len = s->d_kv_len;
    a.table = s->d_table;
    a.status = status;
    return a;
}

}  // namespace

// ---- kernels ---------------------------------------------------------------------------------------
extern "C" int eahmmf_cuda_rope_append(const EahmmfPagedKv* kv, int layer, const EahmmfPagedSeqs* seqs,
                                       const EahmmfRope* rope, int n_head, const float* d_qkv, int ld,
                                       const float* d_qnorm, const float* d_knorm, float eps, float* d_q, int ldq,
                                       void* stream, int* d_status) {
    int rc = check_kv(kv);
    if (rc == ST_OK) rc = check_seqs(seqs);
    if (rc != ST_OK) return rc;
    if (layer < 0 || layer >= kv->n_layer || !heads_ok(kv, n_head) || !rope || !rope->d_inv_freq ||
        (rope->style != EAHMMF_ROPE_HALF && rope->style != EAHMMF_ROPE_INTERLEAVED) || rope->n_rot < 2 ||
        rope->n_rot > kv->hd || rope->n_rot % 2 || !(eps >= 0.f) || !aligned(d_qnorm, 16) || !aligned(d_knorm, 16))
        return ST_BAD_ARG;
    if (seqs->n_seq == 0 || seqs->n_tok == 0) return ST_OK;
    if (!rows_ok(d_qkv, ld, (n_head + 2 * kv->n_kv) * kv->hd) || !rows_ok(d_q, ldq, n_head * kv->hd)) return ST_BAD_ARG;
    return launch_rope_append(kv->type, kv->hd, args_of(kv, layer, seqs, n_head, d_status), *rope, d_qkv, ld, d_qnorm,
                              d_knorm, eps, d_q, ldq, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess
               ? ST_OK
               : ST_CUDA;
}

extern "C" size_t eahmmf_cuda_paged_attention_workspace_bytes(const EahmmfPagedKv* kv, const EahmmfPagedSeqs* seqs,
                                                              int n_head) {
    if (check_kv(kv) != ST_OK || check_seqs(seqs) != ST_OK || !heads_ok(kv, n_head)) return 0;
    return paged_attn_ws_bytes(kv->type, kv->hd, n_head / kv->n_kv, seqs->max_q);
}

extern "C" int eahmmf_cuda_paged_attention(const EahmmfPagedKv* kv, int layer, const EahmmfPagedSeqs* seqs, int n_head,
                                           const float* d_q, int ldq, float scale, int window, int n_sink, float* d_out,
                                           int ldo, void* d_workspace, size_t workspace_bytes, void* stream,
                                           int* d_status) {
    int rc = check_kv(kv);
    if (rc == ST_OK) rc = check_seqs(seqs);
    if (rc != ST_OK) return rc;
    if (layer < 0 || layer >= kv->n_layer || !heads_ok(kv, n_head) || window < 0 || n_sink < 0 || !(fabsf(scale) < INFINITY))
        return ST_BAD_ARG;
    if (seqs->n_seq == 0 || seqs->n_tok == 0) return ST_OK;
    if (!rows_ok(d_q, ldq, n_head * kv->hd) || !rows_ok(d_out, ldo, n_head * kv->hd) || !d_workspace ||
        !aligned(d_workspace, 256))
        return ST_BAD_ARG;
    if (workspace_bytes < eahmmf_cuda_paged_attention_workspace_bytes(kv, seqs, n_head)) return ST_CAPACITY;
    PagedAttnArgs A{};
    A.c = args_of(kv, layer, seqs, n_head, d_status);
    A.q = d_q;
    A.ldq = ldq;
    A.out = d_out;
    A.ldo = ldo;
    A.scale = scale;
    A.window = window;
    A.n_sink = n_sink;
    return launch_paged_attention(kv->type, kv->hd, seqs->max_q, seqs->max_kv, A, d_workspace,
                                  reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess
               ? ST_OK
               : ST_CUDA;
}

extern "C" int eahmmf_cuda_pages_copy(const EahmmfPagedKv* kv, const int* pairs, int n, void* stream) {
    const int rc = check_kv(kv);
    if (rc != ST_OK) return rc;
    if (n < 0 || (n > 0 && !pairs) || kv->n_layer > 32767) return ST_BAD_ARG;
    if (n == 0) return ST_OK;
    std::vector<int> to, from;
    try {
        to.resize(n);
        from.resize(n);
    } catch (const std::bad_alloc&) {
        return ST_CAPACITY;
    }
    for (int i = 0; i < n; i++) {
        from[i] = pairs[2 * i];
        to[i] = pairs[2 * i + 1];
        if (from[i] < 0 || from[i] >= kv->n_pages || to[i] < 0 || to[i] >= kv->n_pages) return ST_BAD_INDEX;
    }
    std::sort(to.begin(), to.end());
    std::sort(from.begin(), from.end());
    for (int i = 0, j = 0; i < n; i++) {  // no page written twice, none read and written
        if (i && to[i] == to[i - 1]) return ST_BAD_ARG;
        while (j < n && from[j] < to[i]) j++;
        if (j < n && from[j] == to[i]) return ST_BAD_ARG;
    }
    return launch_pages_copy(*kv, pairs, n, reinterpret_cast<cudaStream_t>(stream)) == cudaSuccess ? ST_OK : ST_CUDA;
}

// ---- rotary frequencies ----------------------------------------------------------------------------
extern "C" int eahmmf_rope_inv_freq(int scaling, int n_rot, double base, double factor, int ctx_orig, double beta_fast,
                                    double beta_slow, float* inv_freq, float* mscale) {
    if (!inv_freq || n_rot < 2 || n_rot % 2 || !(base > 1.0) || !std::isfinite(base) || scaling < EAHMMF_ROPE_PLAIN ||
        scaling > EAHMMF_ROPE_YARN)
        return ST_BAD_ARG;
    if (scaling != EAHMMF_ROPE_PLAIN && !(factor >= 1.0 && std::isfinite(factor))) return ST_BAD_ARG;
    if (scaling == EAHMMF_ROPE_NTK && n_rot < 4) return ST_BAD_ARG;
    if (scaling == EAHMMF_ROPE_YARN && (ctx_orig < 1 || !(beta_slow > 0.0) || !(beta_fast > beta_slow) || !std::isfinite(beta_fast)))
        return ST_BAD_ARG;
    if (scaling == EAHMMF_ROPE_NTK) base *= pow(factor, (double)n_rot / (n_rot - 2));
    // the pair whose wave turns `turns` times over ctx_orig: base^(2i / n_rot) = ctx_orig / (2 pi turns)
    auto pair_of = [&](double turns) { return n_rot * log(ctx_orig / (turns * 2.0 * M_PI)) / (2.0 * log(base)); };
    double lo = 0.0, hi = 0.0;
    if (scaling == EAHMMF_ROPE_YARN) {
        lo = std::max(0.0, floor(pair_of(beta_fast)));
        hi = std::min(n_rot - 1.0, ceil(pair_of(beta_slow)));
        if (hi <= lo) lo = hi - 0.001;  // every pair past hi (a short ctx_orig), or none of them up to lo
    }
    for (int i = 0; i < n_rot / 2; i++) {
        double f = pow(base, -2.0 * i / n_rot);
        if (scaling == EAHMMF_ROPE_LINEAR) f /= factor;
        if (scaling == EAHMMF_ROPE_YARN) {
            const double ramp = std::min(1.0, std::max(0.0, (i - lo) / (hi - lo)));  // 0 keeps, 1 divides
            f = f * (1.0 - ramp) + f / factor * ramp;
        }
        inv_freq[i] = (float)f;
    }
    if (mscale) *mscale = scaling == EAHMMF_ROPE_YARN ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
    return ST_OK;
}

// ---- pages on the host -----------------------------------------------------------------------------
// A page is free, held by one sequence, or shared (refs > 1). Sharing pages cover whole pages of a common prefix and
// at most one part-filled page; a sequence that grows into a shared part-filled page gets a copy of it first. Copies are
// recorded as (from, to) until the caller takes them. A page that loses its last holder while copies are recorded is
// handed out again only after they are taken, so no recorded copy reads or writes a page twice.
struct EahmmfPages {
    int n_pages, page, n_seq, max_pages;
    std::vector<int> refs;              // of each page
    std::vector<int> len;               // positions of each sequence
    std::vector<std::vector<int>> ids;  // page ids of each sequence (-1: given back by slide)
    std::vector<int> pairs;             // recorded copies
    std::vector<uint8_t> held;          // pages freed since the first recorded copy
    std::vector<int> src_of;            // recorded source of a page that a recorded copy fills, or -1
    int n_free = 0, low = 0;            // free pages; no free page lies below `low`

    bool recorded() const { return !pairs.empty(); }
    int take() {  // the lowest free page
        for (; low < n_pages; low++)
            if (refs[low] == 0 && !held[low]) {
                refs[low] = 1;
                n_free--;
                return low++;
            }
        return -1;
    }
    void drop(int id) {
        if (id < 0 || --refs[id] > 0) return;
        if (recorded()) {
            held[id] = 1;
        } else {
            n_free++;
            low = std::min(low, id);
        }
    }
    void record(int from, int to) {
        const int s = src_of[from] >= 0 ? src_of[from] : from;  // a page not yet filled: read what fills it
        pairs.push_back(s);
        pairs.push_back(to);
        src_of[to] = s;
    }
};

extern "C" EahmmfPages* eahmmf_pages_create(int n_pages, int page, int n_seq, int max_pages) {
    if (n_pages < 1 || page < PAGE_MIN || page > 1024 || page % PAGE_MIN || n_seq < 1 || max_pages < 1 ||
        (long long)max_pages * page > 0x7fffffffLL)
        return nullptr;
    try {
        std::unique_ptr<EahmmfPages> p(new EahmmfPages());
        std::vector<std::vector<int>> ids(n_seq);
        p->n_pages = p->n_free = n_pages;
        p->page = page;
        p->n_seq = n_seq;
        p->max_pages = max_pages;
        p->refs.assign(n_pages, 0);
        p->held.assign(n_pages, 0);
        p->src_of.assign(n_pages, -1);
        p->pairs.reserve(2 * (size_t)n_pages);
        p->len.assign(n_seq, 0);
        for (auto& v : ids) v.reserve(std::min(max_pages, 64));
        p->ids.swap(ids);
        return p.release();
    } catch (const std::bad_alloc&) {
        return nullptr;
    }
}
extern "C" void eahmmf_pages_destroy(EahmmfPages* p) { delete p; }

static bool seq_ok(const EahmmfPages* p, int s) { return p && s >= 0 && s < p->n_seq; }

extern "C" int eahmmf_pages_extend(EahmmfPages* p, int seq, int len) {
    if (!seq_ok(p, seq) || len < p->len[seq]) return ST_BAD_ARG;
    std::vector<int>& v = p->ids[seq];
    const int want = (int)(((long long)len + p->page - 1) / p->page), have = (int)v.size();
    if (want > p->max_pages) return ST_CAPACITY;
    // the part-filled last page is written when the sequence grows: not while another sequence holds it
    const int last = p->len[seq] % p->page ? p->len[seq] / p->page : -1;
    const bool copy = len > p->len[seq] && last >= 0 && v[last] >= 0 && p->refs[v[last]] > 1;
    if (want - have + (copy ? 1 : 0) > p->n_free) return ST_CAPACITY;
    try {
        v.reserve(want);
    } catch (const std::bad_alloc&) {
        return ST_CAPACITY;
    }
    if (copy) {
        const int to = p->take();
        p->record(v[last], to);
        p->refs[v[last]]--;
        v[last] = to;
    }
    while ((int)v.size() < want) v.push_back(p->take());
    p->len[seq] = len;
    return ST_OK;
}

int eb::pages_grow(EahmmfPages* p, const int* seqs, int n) {
    int want = 0;
    for (int i = 0; i < n; i++) {
        if (!seq_ok(p, seqs[i])) return ST_BAD_ARG;
        const std::vector<int>& v = p->ids[seqs[i]];
        const int at = p->len[seqs[i]] / p->page;
        if (p->len[seqs[i]] % p->page == 0) {
            if (at + 1 > p->max_pages) return ST_CAPACITY;
            want++;
        } else if (v[at] >= 0) {  // a copy, unless the rows before left this one the last holder
            int holders = p->refs[v[at]];
            for (int j = 0; j < i; j++) {
                const int other = p->len[seqs[j]];
                if (other % p->page && p->ids[seqs[j]][other / p->page] == v[at]) holders--;
            }
            want += holders > 1;
        }
    }
    if (want > p->n_free) return ST_CAPACITY;
    try {
        for (int i = 0; i < n; i++) p->ids[seqs[i]].reserve(p->len[seqs[i]] / p->page + 1);
    } catch (const std::bad_alloc&) {
        return ST_CAPACITY;
    }
    for (int i = 0; i < n; i++) eahmmf_pages_extend(p, seqs[i], p->len[seqs[i]] + 1);  // which finds its pages and its room
    return ST_OK;
}

extern "C" int eahmmf_pages_fork(EahmmfPages* p, int src, int dst) {
    if (!seq_ok(p, src) || !seq_ok(p, dst) || src == dst || !p->ids[dst].empty() || p->len[dst]) return ST_BAD_ARG;
    try {
        p->ids[dst] = p->ids[src];
    } catch (const std::bad_alloc&) {
        return ST_CAPACITY;
    }
    for (int id : p->ids[dst])
        if (id >= 0) p->refs[id]++;
    p->len[dst] = p->len[src];
    return ST_OK;
}

extern "C" int eahmmf_pages_truncate(EahmmfPages* p, int seq, int len) {
    if (!seq_ok(p, seq) || len < 0 || len > p->len[seq]) return ST_BAD_ARG;
    const int want = (int)(((long long)len + p->page - 1) / p->page);
    std::vector<int>& v = p->ids[seq];
    if (len % p->page && v[want - 1] < 0) return ST_BAD_ARG;  // it would grow into a page that slide gave back
    while ((int)v.size() > want) {
        p->drop(v.back());
        v.pop_back();
    }
    p->len[seq] = len;
    return ST_OK;
}

extern "C" int eahmmf_pages_slide(EahmmfPages* p, int seq, int first_pos, int n_sink) {
    if (!seq_ok(p, seq) || first_pos < 0 || n_sink < 0) return ST_BAD_ARG;
    std::vector<int>& v = p->ids[seq];
    const long long keep = ((long long)n_sink + p->page - 1) / p->page, to = std::min<long long>(first_pos, p->len[seq]) / p->page;
    for (long long i = keep; i < to; i++) {
        p->drop(v[i]);
        v[i] = -1;
    }
    return ST_OK;
}

extern "C" int eahmmf_pages_compact(EahmmfPages* p) {
    if (!p || p->recorded()) return ST_BAD_ARG;  // pages still waiting to be filled do not move
    std::vector<int> at;
    try {
        at.assign(p->n_pages, -1);
    } catch (const std::bad_alloc&) {
        return ST_CAPACITY;
    }
    const int used = p->n_pages - p->n_free;  // they end as pages 0 .. used - 1
    int to = 0;
    for (int from = used; from < p->n_pages; from++) {
        if (!p->refs[from]) continue;
        while (p->refs[to]) to++;
        p->refs[to] = p->refs[from];
        p->refs[from] = 0;
        at[from] = to;
        p->record(from, to);
        p->held[from] = 1;  // not free until the copies are taken
    }
    for (auto& v : p->ids)
        for (int& id : v)
            if (id >= 0 && at[id] >= 0) id = at[id];
    p->n_free = 0;
    for (int i = 0; i < p->n_pages; i++)
        if (!p->refs[i] && !p->held[i]) p->n_free++;
    p->low = 0;
    return ST_OK;
}

extern "C" int eahmmf_pages_take_copies(EahmmfPages* p, int* pairs, int cap) {
    if (!p || cap < 0 || (cap > 0 && !pairs)) return -1;
    const int n = (int)(p->pairs.size() / 2);
    if (n > cap) return n;  // nothing taken: call again with room for n
    std::copy(p->pairs.begin(), p->pairs.end(), pairs);
    p->pairs.clear();
    std::fill(p->src_of.begin(), p->src_of.end(), -1);
    for (int i = 0; i < p->n_pages; i++)
        if (p->held[i]) {
            p->held[i] = 0;
            p->n_free++;
            p->low = std::min(p->low, i);
        }
    return n;
}

extern "C" int eahmmf_pages_table(const EahmmfPages* p, int* table, int ld, int* len) {
    if (!p || !table) return ST_BAD_ARG;
    for (int s = 0; s < p->n_seq; s++) {
        if ((int)p->ids[s].size() > ld) return ST_CAPACITY;
    }
    for (int s = 0; s < p->n_seq; s++) {
        int* row = table + (size_t)s * ld;
        std::copy(p->ids[s].begin(), p->ids[s].end(), row);
        std::fill(row + p->ids[s].size(), row + ld, -1);
        if (len) len[s] = p->len[s];
    }
    return ST_OK;
}

extern "C" int eahmmf_pages_free_count(const EahmmfPages* p) { return p ? p->n_free : 0; }
extern "C" int eahmmf_pages_refs(const EahmmfPages* p, int id) { return p && id >= 0 && id < p->n_pages ? p->refs[id] : -1; }
