// What the kernels over a cache in pages share: where a batch's sequences, rows and pages are.
#pragma once

#include "rows_meet.h"
#include "scan.cuh"

struct pg_batch {
    const int32_t *row_start, *kv_len, *pages;
    int64_t page_stride;
    int n_seq, n_row, max_new, max_kv, n_page, page_log2;
};

struct pg_seq { int row0, n_new, kv; bool ok; };

// Sequence s as the device arrays have it.  ok: it takes part -- it has new tokens, and every index that follows from its entries is one the launch was sized
// for.  Entries that are not raise the error flag.
static __device__ __forceinline__ pg_seq pg_checked(const pg_batch &b, int row0, int row1, int kv, int *err) {
    pg_seq q;
    q.row0 = row0; q.n_new = row1 - row0; q.kv = kv;
    const bool sound = row0 >= 0 && row1 >= row0 && row1 <= b.n_row && q.n_new <= b.max_new && kv >= 0 && kv <= b.max_kv && (int64_t)kv <= (b.page_stride << b.page_log2);
    if (!sound && err) *err = 1;
    q.ok = sound && q.n_new > 0;
    return q;
}
// An entry of an array that no kernel of the call writes, at an index that is the same for the whole wave: read through the scalar cache
static __device__ __forceinline__ int32_t pg_entry(const int32_t *p, int64_t i) { return *(const __attribute__((address_space(4))) int32_t *)(p + i); }
static __device__ __forceinline__ pg_seq pg_sequence(const pg_batch &b, int s, int *err) {
    return pg_checked(b, b.row_start[s], b.row_start[s + 1], b.kv_len[s], err);
}

// Host side: a tensor of rows of `hd` elements that the kernels take (alignment and strides as the header has them)
static inline bool pg_rows_ok(const spy_hip_tensor *t, int64_t hd, int64_t n_head, int64_t n_row) {
    return t->data && ((uintptr_t)t->data & 15) == 0 && t->ne[0] == hd && t->ne[1] == n_head && t->ne[2] == n_row && t->ne[3] == 1 && t->nb[0] == spy_type_size(t->type) &&
           t->nb[1] > 0 && t->nb[2] > 0 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0;
}

// Batch and pages of a call: 0, or the code that it is refused with.  page_dim: the dimension of the page tensor that counts positions (K 1, V^T 0).
static inline int pg_check_batch(const spy_hip_paged_batch *b) {
    SPY_CHECK_ARG(b && b->n_seq > 0 && b->n_seq <= (1 << 20) && b->max_new > 0 && b->max_kv > 0 && b->max_new <= (1 << 24) && b->max_kv <= (1 << 30) && b->page_stride > 0 &&
                  b->page_stride <= (1 << 30));
    SPY_CHECK_ARG(b->row_start && b->kv_len && b->pages && (((uintptr_t)b->row_start | (uintptr_t)b->kv_len | (uintptr_t)b->pages) & 3) == 0);
    return 0;
}
static inline int pg_check_pages(const spy_hip_tensor *t, int page_dim) {
    SPY_CHECK_ARG(t->data && ((uintptr_t)t->data & 15) == 0 && t->ne[2] > 0 && t->ne[3] > 0 && t->ne[3] < (1ll << 31) && t->nb[0] == 2);
    for (int i = 1; i < 4; i++) SPY_CHECK_ARG(t->nb[i] > 0 && t->nb[i] % 16 == 0);
    SPY_CHECK_ARG(t->nb[1] <= (1 << 20) && t->nb[3] < (1ll << 32));         // offsets inside a page are 32-bit numbers, and so is a page's size
    const int64_t ps = t->ne[page_dim], hd = t->ne[1 - page_dim];
    if (t->type != SPY_HIP_F16 || (hd != 64 && hd != 128 && hd != 256) || ps < 16 || ps > 1024 || (ps & (ps - 1))) return SPY_HIP_EUNSUPPORTED;
    return 0;
}
static inline int pg_log2(int64_t v) { int n = 0; while ((1ll << n) < v) n++; return n; }
