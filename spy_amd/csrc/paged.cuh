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

// Sequences in groups: those of one begin with the same tokens
struct pg_groups {
    const int32_t *seq_start, *length;     // sequences seq_start[g] .. seq_start[g + 1] - 1 have their first length[g] tokens in common
    int n_group, max_rows, max_common;
};
// Rows and keys that belong together: a sequence's, of the pages of sequence s, from position `from` on
struct pg_span : pg_seq { int s, from; };

// Group of sequences s0 .. s1 - 1 with `length` tokens in common, as a sequence of their rows and that many cached tokens
static __device__ __forceinline__ pg_span pg_group(const pg_batch &b, const pg_groups &g, int s0, int s1, int length, int *err) {
    pg_span q;
    q.s = s0; q.from = 0; q.kv = length; q.row0 = 0; q.n_new = 0;
    bool sound = s0 >= 0 && s1 >= s0 && s1 <= b.n_seq && length >= 0 && length <= g.max_common && (int64_t)length <= (b.page_stride << b.page_log2);
    if (sound) {
        q.row0 = b.row_start[s0];
        const int row1 = b.row_start[s1];
        q.n_new = row1 - q.row0;
        sound = q.row0 >= 0 && row1 >= q.row0 && row1 <= b.n_row && q.n_new <= g.max_rows;
    }
    if (!sound && err) *err = 1;
    q.ok = sound && q.n_new > 0;
    return q;
}
// Sequence s with what its group has not in common, by every lane of a wave alike.  A sequence of a group takes part where the group does and its new tokens are behind what the group has
// in common; one of none as ever.
static __device__ __forceinline__ pg_span pg_own(const pg_batch &b, const pg_groups &g, int s, int *err, pg_span *its_group = nullptr) {
    const int lane = threadIdx.x & 63;
    pg_span q;
    if (its_group) its_group->ok = false;
    (pg_seq &)q = pg_sequence(b, s, err);
    q.s = s; q.from = 0;
    for (int base = 0; base < g.n_group; base += 64) {
        const int i = min(base + lane, g.n_group - 1), s0 = g.seq_start[i], s1 = g.seq_start[i + 1], length = g.length[i];
        const unsigned long long past = __ballot(base + lane < g.n_group && s1 > s);
        if (!past) continue;
        const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
        if (__builtin_amdgcn_readlane(s0, at) > s) break;
        const pg_span all = pg_group(b, g, __builtin_amdgcn_readlane(s0, at), __builtin_amdgcn_readlane(s1, at), __builtin_amdgcn_readlane(length, at), err);
        if (its_group) *its_group = all;
        q.from = all.kv;
        if (q.ok && !(all.ok && all.kv <= max(q.kv - q.n_new, 0) && all.row0 <= q.row0 && q.row0 + q.n_new <= all.row0 + all.n_new)) {
            q.ok = false;
            if (err) *err = 1;
        }
        break;
    }
    return q;
}
static __device__ __forceinline__ pg_span pg_span_of(const pg_batch &b, const pg_groups &g, int which, bool common, int *err) {
    if (common) return pg_group(b, g, g.seq_start[which], g.seq_start[which + 1], g.length[which], err);
    return pg_own(b, g, which, err);
}

// Sequence of row r, by every lane of a wave: the first s with row_start[s + 1] > r.  64 sequences per round, their entries requested together.
static __device__ __forceinline__ int row_sequence(const pg_batch &b, int r, int lane, int &row1, int &kv) {
    for (int base = 0; base < b.n_seq; base += 64) {
        const int s = base + lane;
        const int end = s < b.n_seq ? b.row_start[s + 1] : 0x7fffffff, len = s < b.n_seq ? b.kv_len[s] : 0;
        const unsigned long long past = __ballot(s < b.n_seq && end > r);
        if (past) {
            const int at = __ffsll(past) - 1;
            row1 = __shfl(end, at, SPY_WAVE);
            kv = __shfl(len, at, SPY_WAVE);
            return base + at;
        }
    }
    return -1;
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
// Pages in 8 bits, and the scales beside them: one to 32 elements of a row (K: dimension 0 of the scales counts them; V^T: dimension 1)
static inline int pg_check_pages_q8(const spy_hip_tensor *t, int page_dim) {
    if (t->type != SPY_HIP_I8) return SPY_HIP_EUNSUPPORTED;
    SPY_CHECK_ARG(t->data && ((uintptr_t)t->data & 15) == 0 && t->ne[2] > 0 && t->ne[3] > 0 && t->ne[3] < (1ll << 31) && t->nb[0] == 1);
    for (int i = 1; i < 4; i++) SPY_CHECK_ARG(t->nb[i] > 0 && t->nb[i] % 16 == 0);
    SPY_CHECK_ARG(t->nb[1] <= (1 << 20) && t->nb[3] < (1ll << 32));
    const int64_t ps = t->ne[page_dim], hd = t->ne[1 - page_dim];
    if ((hd != 64 && hd != 128 && hd != 256) || ps < 16 || ps > 1024 || (ps & (ps - 1))) return SPY_HIP_EUNSUPPORTED;
    return 0;
}
static inline int pg_check_scales(const spy_hip_tensor *t, const spy_hip_tensor *pages, int page_dim) {
    if (t->type != SPY_HIP_F16) return SPY_HIP_EUNSUPPORTED;
    const int64_t blocks = pages->ne[1 - page_dim] / 32;
    SPY_CHECK_ARG(t->data && ((uintptr_t)t->data & 15) == 0 && t->ne[page_dim] == pages->ne[page_dim] && t->ne[1 - page_dim] == blocks && t->ne[2] == pages->ne[2] && t->ne[3] == pages->ne[3]);
    SPY_CHECK_ARG(t->nb[0] == 2 && t->nb[1] > 0 && (page_dim == 1 ? t->nb[1] == 2 * blocks : t->nb[1] % 16 == 0) && t->nb[1] <= (1 << 20));
    SPY_CHECK_ARG(t->nb[2] > 0 && t->nb[2] % 16 == 0 && t->nb[3] > 0 && t->nb[3] % 16 == 0 && t->nb[3] < (1ll << 32));
    return 0;
}
static inline int pg_log2(int64_t v) { int n = 0; while ((1ll << n) < v) n++; return n; }
