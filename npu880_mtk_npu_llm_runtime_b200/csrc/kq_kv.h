// kq_kv.h -- index arithmetic of the paged key-value cache and the checks of the attention calls.
//
// Plain C++ without CUDA calls: the kernels and the host use the same functions, and a host
// compiler can check them alone.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

#include "../../include/kq.h"

#ifdef __CUDACC__
#define KQ_HD __host__ __device__ __forceinline__
#else
#define KQ_HD inline
#endif

namespace kq {

// The cache as the kernels take it.
struct KvView {
    uint16_t *k, *v;
    const int32_t *table;
    int n_pages, page_shift, kv_heads, head_dim, n_seqs, table_stride;
};

// Positions of a sequence that the table reaches.
KQ_HD long long kv_reach(const KvView &c) { return (long long)c.table_stride << c.page_shift; }

// A sequence's length, held to what the table reaches (bad: it was not).  Positions are int32.
KQ_HD int kv_length(const KvView &c, int len, bool &bad) {
    const long long reach = kv_reach(c);
    if (len < 0) {
        bad = true;
        return 0;
    }
    if (len > reach) {
        bad = true;
        return (int)reach;
    }
    return len;
}

KQ_HD bool kv_page_ok(const KvView &c, int page) { return page >= 0 && page < c.n_pages; }

// Element offset of row `slot` of key head `head` in `page`: 64 bits, a cache may pass 2^31 values.
KQ_HD long long kv_row(const KvView &c, int page, int head, int slot) {
    return ((((long long)page * c.kv_heads + head) << c.page_shift) + slot) * c.head_dim;
}

// The keys that position p sees, of a sequence of `len` keys: [0, kept) and [lo, hi).
struct KvSpan {
    int kept, lo, hi;
};
KQ_HD KvSpan kv_span(int p, int len, int window, int sinks) {
    KvSpan s;
    s.hi = p + 1 < len ? p + 1 : len;
    if (s.hi < 0) s.hi = 0;
    s.lo = (window > 0 && p + 1 > window) ? p + 1 - window : 0;
    if (s.lo > s.hi) s.lo = s.hi;
    s.kept = sinks < s.lo ? sinks : s.lo;
    return s;
}
KQ_HD bool kv_sees(const KvSpan &s, int j) { return j < s.hi && (j >= s.lo || j < s.kept); }
KQ_HD int kv_count(const KvSpan &s) { return s.hi - s.lo + s.kept; }
// the e-th of them (0 <= e < kv_count)
KQ_HD int kv_nth(const KvSpan &s, int e) { return e < s.kept ? e : e - s.kept + s.lo; }

// The keys in blocks of B positions (a power of two, aligned): blocks [0, n_kept) and [first, end).
struct KvBlocks {
    int n_kept, first, count;
};
KQ_HD KvBlocks kv_blocks(int kept, int lo, int hi, int B) {
    KvBlocks b;
    if (hi <= lo && kept <= 0) {
        b.n_kept = b.first = b.count = 0;
        return b;
    }
    b.first = lo / B;
    const int end = (hi + B - 1) / B;
    const int nk = (kept + B - 1) / B;
    b.n_kept = nk < b.first ? nk : b.first;
    b.count = b.n_kept + (end - b.first);
    return b;
}
KQ_HD int kv_block(const KvBlocks &b, int i) { return i < b.n_kept ? i : i - b.n_kept + b.first; }

// Rows of sequence s: [begin, begin + n), from q_start held to [0, M] (bad: it was not, or decreases)
struct KvRows {
    int begin, n;
};
KQ_HD KvRows kv_rows(int start, int end, int M, bool &bad) {
    KvRows r;
    r.begin = start;
    r.n = end - start;
    if (start < 0 || end > M || end < start) {
        bad = true;
        r.begin = 0;
        r.n = 0;
    }
    return r;
}

// The same where ranges overlap because q_start falls in between: rows before `limit` (the furthest end of the
// sequences before s, each taken for itself) are another sequence's, so a range that begins there has none.
// What is left is disjoint, M rows in all at most.
KQ_HD KvRows kv_rows_behind(int start, int end, int M, int limit, bool &bad) {
    KvRows r = kv_rows(start, end, M, bad);
    if (r.n > 0 && r.begin < limit) {
        bad = true;
        r.begin = 0;
        r.n = 0;
    }
    return r;
}

// Total units cut into `parts` contiguous shares that differ by one at most.
struct Shares {
    long long q;          // total / parts
    unsigned r, parts;    // total % parts
    float inv;            // about parts / total
    KQ_HD Shares() {}
    KQ_HD Shares(long long total, int n) : parts((unsigned)n) {
        if (total < 0xffffffffll) {  // 32-bit division where it will do
            q = (unsigned)total / parts;
        } else {
            q = total / n;
        }
        r = (unsigned)(total - q * n);
        inv = (float)n / (float)total;
    }
    KQ_HD long long begin(int c) const { return q * c + (r * (unsigned)c) / parts; }
    KQ_HD int of(long long u) const {
        int c = (int)((float)u * inv) < (int)parts - 1 ? (int)((float)u * inv) : (int)parts - 1;
        while (c + 1 < (int)parts && begin(c + 1) <= u) ++c;
        while (c > 0 && begin(c) > u) --c;
        return c;
    }
};

// ------------------------------------------------------------------ checks (host)

inline bool kv_aligned(const void *p, size_t n) { return ((uintptr_t)p % n) == 0; }

// KQ_OK, or a status and why.
inline int check_head_dim(int d, const char **why) {
    if (d == 64 || d == 128 || d == 256) return KQ_OK;
    *why = "head_dim must be 64, 128 or 256";
    return KQ_ERR_SHAPE;
}

inline int check_cache(const kq_kv_cache *c, const char **why) {
    *why = "";
    if (!c || !c->k || !c->v || !c->page_table) {
        *why = "the cache, its pages or its page table is NULL";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (!kv_aligned(c->k, 16) || !kv_aligned(c->v, 16) || !kv_aligned(c->page_table, 4)) {
        *why = "cache pages must be 16-byte aligned, the page table 4-byte";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (int r = check_head_dim(c->head_dim, why)) return r;
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) {
        *why = "page_size must be a power of two from 16 to 256";
        return KQ_ERR_SHAPE;
    }
    if (c->kv_heads < 1 || c->kv_heads > KQ_MAX_HEADS || c->n_pages < 1 || c->n_seqs < 1 || c->n_seqs > KQ_MAX_SEQS ||
        c->table_stride < 1) {
        *why = "kv_heads, n_pages, n_seqs or table_stride out of range";
        return KQ_ERR_SHAPE;
    }
    if ((long long)c->table_stride * c->page_size > 0x40000000ll) {
        *why = "a sequence may reach 2^30 positions at most";
        return KQ_ERR_SHAPE;
    }
    if ((long long)c->n_seqs * c->table_stride * c->page_size > (1ll << 34)) {
        *why = "the table may reach 2^34 positions at most";
        return KQ_ERR_SHAPE;
    }
    return KQ_OK;
}

inline int check_rope(const kq_rope *r, int head_dim, const char **why) {
    *why = "";
    if (!r || r->rot_dim == 0) return KQ_OK;
    if (r->rot_dim < 0 || r->rot_dim % 16 || r->rot_dim > head_dim) {
        *why = "rot_dim must be a multiple of 16 up to head_dim";
        return KQ_ERR_SHAPE;
    }
    if (r->style != KQ_ROPE_HALF && r->style != KQ_ROPE_ADJACENT) {
        *why = "rope style must be KQ_ROPE_HALF or KQ_ROPE_ADJACENT";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    return KQ_OK;
}

inline int check_rows(int M, const char **why) {
    if (M >= 0 && M <= KQ_MAX_M) return KQ_OK;
    *why = "M out of range";
    return KQ_ERR_SHAPE;
}

// rows of `heads` heads at p
inline int check_head_rows(const void *p, size_t stride, int heads, int head_dim, const char **why) {
    if (!p) {
        *why = "rows are NULL";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (heads < 1 || heads > KQ_MAX_HEADS) {
        *why = "heads out of range";
        return KQ_ERR_SHAPE;
    }
    if (stride < (size_t)heads * (size_t)head_dim || stride % 8 || stride > ((size_t)1 << 38)) {
        *why = "a row stride must be at least heads * head_dim and a multiple of 8";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (!kv_aligned(p, 16)) {
        *why = "rows must be 16-byte aligned";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    return KQ_OK;
}

// a kq_heads: `to` says whether out has to be given (1) or NULL (0)
inline int check_heads(const kq_heads *h, int head_dim, int to, const char **why) {
    *why = "";
    if (!h) {
        *why = "heads are NULL";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (int r = check_head_rows(h->in, h->in_stride, h->heads, head_dim, why)) return r;
    if (to) {
        if (int r = check_head_rows(h->out, h->out_stride, h->heads, head_dim, why)) return r;
    } else if (h->out) {
        *why = "keys and values go to the cache: out must be NULL";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (h->gamma && !kv_aligned(h->gamma, 16)) {
        *why = "gamma must be 16-byte aligned";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    return KQ_OK;
}

inline int check_append(const kq_kv_cache *c, const kq_rope *rope, int M, const int32_t *seq, const int32_t *pos,
                        const kq_heads *q, const kq_heads *k, const kq_heads *v, const char **why) {
    if (int r = check_cache(c, why)) return r;
    if (int r = check_rope(rope, c->head_dim, why)) return r;
    if (int r = check_rows(M, why)) return r;
    if (M == 0) return KQ_OK;  // nothing to do: the rows may be NULL
    if (q)
        if (int r = check_heads(q, c->head_dim, 1, why)) return r;
    if (int r = check_heads(k, c->head_dim, 0, why)) return r;
    if (int r = check_heads(v, c->head_dim, 0, why)) return r;
    if (v->gamma) {
        *why = "values are not normed: v->gamma must be NULL";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (k->heads != c->kv_heads || v->heads != c->kv_heads) {
        *why = "k and v must have the cache's kv_heads";
        return KQ_ERR_SHAPE;
    }
    if (!seq || !pos || !kv_aligned(seq, 4) || !kv_aligned(pos, 4)) {
        *why = "sequences or positions are NULL or not 4-byte aligned";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    return KQ_OK;
}

inline int check_attn(const kq_kv_cache *c, const kq_attn *a, bool prefill, const char **why) {
    if (int r = check_cache(c, why)) return r;
    if (!a || !a->kv_len || (prefill && !a->q_start) || !kv_aligned(a->kv_len, 4) || (prefill && !kv_aligned(a->q_start, 4))) {
        *why = "the attention's description or its lengths are NULL or not 4-byte aligned";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (int r = check_rows(a->M, why)) return r;
    if (!prefill && a->M != c->n_seqs) {
        *why = "decode takes one row per sequence: M must equal n_seqs";
        return KQ_ERR_SHAPE;
    }
    if (a->M == 0) return KQ_OK;  // nothing to do: the rows may be NULL
    if (int r = check_head_rows(a->q, a->q_stride, a->heads, c->head_dim, why)) return r;
    if (int r = check_head_rows(a->out, a->out_stride, a->heads, c->head_dim, why)) return r;
    if (a->q == a->out) {
        *why = "out may not overlap q";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    if (a->heads % c->kv_heads || a->heads / c->kv_heads > KQ_MAX_GROUP) {
        *why = "heads must be a multiple of kv_heads, at most KQ_MAX_GROUP times it";
        return KQ_ERR_SHAPE;
    }
    if (a->window < 0 || a->sinks < 0 || (a->window == 0 && a->sinks != 0)) {
        *why = "window and sinks must not be negative, and sinks needs a window";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    // (256 products of fp16's largest values stay below fp32's with it, so no finite score is lost)
    if (!(a->scale >= 0.0f) || a->scale > 1e24f) {
        *why = "scale must be 0 or a positive number up to 1e24";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    return KQ_OK;
}

// ---- what a call writes may not lie over what it reads

// n rows of `width` bytes, `stride` bytes apart (stride >= width, or n = 1).
struct Rows {
    const void *at;
    size_t stride, width;
    int n;
};

// Do two sets of rows share a byte?  (Rows of one set between rows of the other do not.)
inline bool rows_overlap(const Rows &a, const Rows &b) {
    if (!a.n || !b.n || !a.at || !b.at) return false;
    const long long at = (long long)(uintptr_t)a.at, bt = (long long)(uintptr_t)b.at;
    const long long as = (long long)a.stride, bs = (long long)b.stride, aw = (long long)a.width, bw = (long long)b.width;
    if (at + (a.n - 1) * as + aw <= bt || bt + (b.n - 1) * bs + bw <= at) return false;
    if (a.n == 1 || b.n == 1 || as != bs) {
        // both in the order of their addresses
        for (int i = 0, j = 0; i < a.n && j < b.n;) {
            const long long x = at + i * as, y = bt + j * bs;
            if (x + aw <= y) ++i;
            else if (y + bw <= x) ++j;
            else return true;
        }
        return false;
    }
    // one stride: row i of a and row i + t of b overlap, for every i, when -bw < d + t s < aw
    const long long s = as, d = bt - at, least = 1 - bw - d;
    long long t = least / s + (least % s > 0);  // the smallest t of the first
    if (t < 1 - a.n) t = 1 - a.n;
    return t < b.n && d + t * s < aw;
}

inline Rows rows_of(const uint16_t *p, size_t stride, int heads, int head_dim, int M) {
    return Rows{p, stride * 2, (size_t)heads * head_dim * 2, M};
}
inline Rows pages_of(const kq_kv_cache *c, const uint16_t *p) {
    return Rows{p, 0, (size_t)c->n_pages * c->kv_heads * c->page_size * c->head_dim * 2, 1};
}

// The rows of a norm, rotation or append call, checked one by one before.
inline int check_heads_apart(const kq_kv_cache *c, int head_dim, int M, const kq_heads *q, const kq_heads *k,
                             const kq_heads *v, const char **why) {
    *why = "";
    const kq_heads *h[3] = {q, k, v};
    for (int i = 0; i < 3; ++i) {
        if (!h[i] || !h[i]->out) continue;
        const Rows out = rows_of(h[i]->out, h[i]->out_stride, h[i]->heads, head_dim, M);
        for (int j = 0; j < 3; ++j) {
            if (!h[j]) continue;
            const bool in_place = i == j && h[i]->in == h[i]->out && (M == 1 || h[i]->in_stride == h[i]->out_stride);
            if (!in_place && rows_overlap(out, rows_of(h[j]->in, h[j]->in_stride, h[j]->heads, head_dim, M))) {
                *why = "out must be the rows themselves or lie apart from all rows that the call reads";
                return KQ_ERR_INVALID_ARGUMENT;
            }
            if (j < i && h[j]->out && rows_overlap(out, rows_of(h[j]->out, h[j]->out_stride, h[j]->heads, head_dim, M))) {
                *why = "two sets of heads go to the same place";
                return KQ_ERR_INVALID_ARGUMENT;
            }
        }
    }
    if (!c) return KQ_OK;
    if (rows_overlap(pages_of(c, c->k), pages_of(c, c->v))) {
        *why = "the cache's keys and values lie over each other";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    for (const uint16_t *pages : {c->k, c->v})
        for (int i = 0; i < 3; ++i)
            if (h[i] && (rows_overlap(pages_of(c, pages), rows_of(h[i]->in, h[i]->in_stride, h[i]->heads, head_dim, M)) ||
                         rows_overlap(pages_of(c, pages), rows_of(h[i]->out, h[i]->out_stride, h[i]->heads, head_dim, M)))) {
                *why = "rows lie in the cache's pages";
                return KQ_ERR_INVALID_ARGUMENT;
            }
    return KQ_OK;
}

// The output of an attention call, checked before.
inline int check_attn_apart(const kq_kv_cache *c, const kq_attn *a, const char **why) {
    *why = "";
    const Rows out = rows_of(a->out, a->out_stride, a->heads, c->head_dim, a->M);
    if (rows_overlap(out, rows_of(a->q, a->q_stride, a->heads, c->head_dim, a->M)) || rows_overlap(out, pages_of(c, c->k)) ||
        rows_overlap(out, pages_of(c, c->v))) {
        *why = "out may not overlap q or the cache";
        return KQ_ERR_INVALID_ARGUMENT;
    }
    return KQ_OK;
}

}  // namespace kq
