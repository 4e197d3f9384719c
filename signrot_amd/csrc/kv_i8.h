// The paged int8 KV cache: codes with one fp32 scale for each block of 16
// tokens and head.
//   data  i8  [pages, L, 2, H, page, 128]   (K at 0, V at 1)
//   scale f32 [pages, L, 2, H, page / 16]
// value = code * scale; codes lie in [-127, 127].  Request b owns pages
// indices[indptr[b] .. indptr[b + 1]); its length is
// (pages - 1) * page + last[b], the page table of the int4 cache.
#pragma once

#include "common.h"

constexpr int kI8Block = 16;   // tokens that share a scale (one MFMA tile of keys)
constexpr int kI8D = 128;

struct PagedI8 {
    int8_t *data;
    float *scale;
    const int32_t *indptr, *indices, *last;
    int64_t pages, n_indices;      // bounds of the pool and of `indices`
    int64_t L, layer;
    int H, page, bpp;              // bpp = page / 16
};

// The table entries are read from device memory, so the host cannot check
// them: a length never exceeds the pages that the request has in the table,
// and a page outside the pool is one that is not there (-1).
struct I8Request {
    int64_t first;    // of `indices`
    int64_t len;
};

SRQ_DEV I8Request i8_request(const PagedI8 &p, int64_t b) {
    int64_t p0 = p.indptr[b], p1 = p.indptr[b + 1];
    if (p0 < 0) p0 = 0;
    if (p1 > p.n_indices) p1 = p.n_indices;
    int64_t last = p.last[b];
    last = last < 0 ? 0 : (last > p.page ? p.page : last);
    const int64_t np = p1 - p0;
    return {p0, np > 0 ? (np - 1) * p.page + last : 0};
}

// New tokens [s, s + n) of request b in a tensor of `rows` rows; one per
// request without an index.
SRQ_DEV void i8_new_rows(const int32_t *new_indptr, int64_t b, int64_t rows, int64_t &s,
                         int64_t &n) {
    if (!new_indptr) {
        s = b;
        n = 1;
        return;
    }
    s = new_indptr[b];
    int64_t e = new_indptr[b + 1];
    s = s < 0 ? 0 : s;
    e = e > rows ? rows : e;
    n = e > s ? e - s : 0;
}

SRQ_DEV int64_t i8_page(const PagedI8 &p, int64_t first, int64_t block) {
    const int64_t pg = p.indices[first + (uint32_t)block / (uint32_t)p.bpp];
    return pg >= 0 && pg < p.pages ? pg : -1;
}

// row of `data` (128 codes each) and index of `scale` of a block of K; V is
// H * page rows and H * bpp scales further
SRQ_DEV int64_t i8_scale_index(const PagedI8 &p, int64_t pg, int head, uint32_t in_page) {
    return ((pg * p.L + p.layer) * 2 * p.H + head) * p.bpp + in_page;
}

// Host-side checks that every entry point of this cache makes.
static inline int i8_check(const char *name, const void *data, const void *scale,
                           const int32_t *indptr, const int32_t *indices, const int32_t *last,
                           int64_t pages, int64_t n_indices, int64_t batch, int64_t L,
                           int64_t layer, int64_t H, int64_t page, int64_t D, PagedI8 &p) {
    SRQ_CHECK_ARG(D == kI8D, "%s: head_dim=%lld, only 128 is supported", name, (long long)D);
    SRQ_CHECK_ARG(page > 0 && page % kI8Block == 0 && page <= (1 << 20),
                  "%s: page_size=%lld must be a multiple of 16", name, (long long)page);
    SRQ_CHECK_ARG(L > 0 && layer >= 0 && layer < L, "%s: layer_idx=%lld outside [0, %lld)", name,
                  (long long)layer, (long long)L);
    SRQ_CHECK_ARG(H > 0 && H <= 4096, "%s: bad number of KV heads", name);
    SRQ_CHECK_ARG(batch >= 0 && batch <= 65535, "%s: batch=%lld outside [0, 65535]", name,
                  (long long)batch);
    SRQ_CHECK_ARG(pages >= 0 && n_indices >= 0 && n_indices <= 0x7fffffff, "%s: negative size",
                  name);
    if (batch == 0) return SRQ_OK;
    SRQ_CHECK_ARG(pages > 0, "%s: the cache holds no pages", name);
    // (a tile of keys past the longest request still counts in 32 bits)
    SRQ_CHECK_ARG(n_indices <= (int64_t)(0x7fffffff - 64) / page,
                  "%s: table x page_size >= 2^31 tokens", name);
    SRQ_CHECK_ARG(data && scale && indptr && last && (indices || n_indices == 0),
                  "%s: null pointer", name);
    SRQ_CHECK_ARG(srq_aligned(data, 16) && srq_aligned(scale, 4),
                  "%s: kv_data must be 16-byte aligned", name);
    p.data = (int8_t *)data;
    p.scale = (float *)scale;
    p.indptr = indptr;
    p.indices = indices;
    p.last = last;
    p.pages = pages;
    p.n_indices = n_indices;
    p.L = L;
    p.layer = layer;
    p.H = (int)H;
    p.page = (int)page;
    p.bpp = (int)(page / kI8Block);
    return SRQ_OK;
}
