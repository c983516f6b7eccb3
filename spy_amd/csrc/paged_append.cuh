// What the two kernels that store new tokens into a cache in pages share: their arguments, the sequence of a row, a row's angles, and the checks of a call.
#pragma once

#include "paged.cuh"

int *spy_hip_err_flag_ptr();

#define PA_THREADS 256

struct append_args {
    const uint8_t *q, *k, *v;                     // rows of hd elements; strides in bytes: of a head, of a row
    uint8_t *qo, *kp, *vp;
    int64_t q_h, q_t, k_h, k_t, v_h, v_t, qo_h, qo_t;
    int64_t kp_p, kp_h, kp_g, vp_d, vp_h, vp_g;   // K pages: position, head, page; V^T pages: dimension, head, page
    pg_batch b;
    int H, G, hd, mode, nd;                       // H: 0 without q
    double turn0, turn1;                          // log2 of revolutions per position of pair i: turn0 + i * turn1
    float mscale;
    int *err;
};

// 8 elements of a row as floats
template <bool F16IN> static __device__ __forceinline__ void load8(const uint8_t *p, float (&x)[8]) {
    if constexpr (F16IN) {
        const uint4 w = *(const uint4 *)p;
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = h2f((uint16_t)(v[i] & 0xFFFFu)); x[2 * i + 1] = h2f((uint16_t)(v[i] >> 16)); }
    } else {
        const float4 a = *(const float4 *)p, b = *(const float4 *)(p + 16);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
}
static __device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = (uint32_t)f2h(x[2 * i]) | ((uint32_t)f2h(x[2 * i + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// cos and sin of the pairs of R rows, whose positions are in s_pos, to s_cs
template <int R> static __device__ __forceinline__ void append_angles(const append_args &a, const int *s_pos, float2 (*s_cs)[128]) {
    const int npair = a.nd / 2;
    for (int i = threadIdx.x; i < R * npair; i += PA_THREADS) {
        const int r = i / npair, p = i - r * npair;
        const double turns = (double)s_pos[r] * exp2(a.turn0 + p * a.turn1);
        const float x = (float)(turns - rint(turns));
        float sn, cs;
        sincospif(2.0f * x, &sn, &cs);
        s_cs[r][p] = make_float2(cs * a.mscale, sn * a.mscale);
    }
}
// Where row `tile` * R + wave goes, by its wave: to s_pos its position, or INT32_MIN where it takes no part, and to s_page its page, or -1
template <int R> static __device__ __forceinline__ void append_place(const append_args &a, int tile, int *s_pos, int *s_page) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = tile * R + wave;
    int row1 = 0, kv = 0, pos = -1, page = -1;
    const int s = r < a.b.n_row ? row_sequence(a.b, r, lane, row1, kv) : -1;
    bool takes = false;
    if (s >= 0) {
        const pg_seq q = pg_checked(a.b, a.b.row_start[s], row1, kv, a.err);
        takes = q.ok && r >= q.row0;
        pos = kv - (row1 - r);
        if (takes && pos >= 0) page = a.b.pages[s * a.b.page_stride + (pos >> a.b.page_log2)];
        if (takes && (page < 0 || page >= a.b.n_page)) { page = -1; if (a.err) *a.err = 1; }
    }
    if (lane == 0) { s_pos[wave] = takes ? pos : INT32_MIN; s_page[wave] = page; }
}
// Tile `tile` of 64 positions (a multiple of 64 on) of the sequences one after the other, by every wave: its sequence, and its number there
static __device__ __forceinline__ int append_tile(const append_args &a, int tile, int &first) {
    const int lane = threadIdx.x & 63;
    for (int base = 0, left = tile; base < a.b.n_seq; base += 64) {
        int n = 0, f = 0;
        if (base + lane < a.b.n_seq) {
            const pg_seq q = pg_sequence(a.b, base + lane, a.err);
            f = max(q.kv - q.n_new, 0) >> 6;
            n = q.ok && q.kv > 0 ? ((q.kv - 1) >> 6) - f + 1 : 0;
        }
        const int sum = (int)wave_scan((uint32_t)n);
        const unsigned long long past = __ballot(sum > left);
        if (past) {
            const int at = __ffsll(past) - 1;
            first = __shfl(f, at, SPY_WAVE) + left - __shfl(sum - n, at, SPY_WAVE);
            return base + at;
        }
        left -= __shfl(sum, 63, SPY_WAVE);
    }
    return -1;
}

// Rows, batch and rotation of a call: 0 and `a` without what it says of the pages' memory, or the code that the call is refused with.  The pages have been checked, each kind by itself.
static inline int append_check(append_args &a, const spy_hip_tensor *q, const spy_hip_tensor *k, const spy_hip_tensor *v, const spy_hip_paged_batch *batch, const spy_hip_rope_param *rope,
                               const spy_hip_tensor *q_out, const spy_hip_tensor *k_pages, const spy_hip_tensor *v_pages) {
    if ((k->type != SPY_HIP_F32 && k->type != SPY_HIP_F16) || v->type != k->type || (q && (q->type != k->type || q_out->type != SPY_HIP_F16))) return SPY_HIP_EUNSUPPORTED;
    const int64_t hd = k_pages->ne[0], ps = k_pages->ne[1], G = k_pages->ne[2], n_row = k->ne[2], H = q ? q->ne[1] : 0;
    SPY_CHECK_ARG(v_pages->ne[0] == ps && v_pages->ne[1] == hd && v_pages->ne[2] == G && v_pages->ne[3] == k_pages->ne[3]);
    SPY_CHECK_ARG(n_row > 0 && n_row < (1 << 28) && G <= 65535 && H <= 65535 && pg_rows_ok(k, hd, G, n_row) && pg_rows_ok(v, hd, G, n_row));
    SPY_CHECK_ARG(!q || (H > 0 && H % G == 0 && pg_rows_ok(q, hd, H, n_row) && pg_rows_ok(q_out, hd, H, n_row)));
    a.mode = rope ? rope->mode : -1;
    a.nd = 16; a.turn0 = a.turn1 = 0; a.mscale = 1.0f;
    if (a.mode != -1) {
        if ((a.mode != 0 && a.mode != 2) || rope->extend_factor != 0.0f || rope->xpos_base != 0.0f) return SPY_HIP_EUNSUPPORTED;
        SPY_CHECK_ARG(rope->num_dim > 0 && rope->num_dim % 16 == 0 && rope->num_dim <= hd && rope->freq_base > 0.0f && rope->freq_scale > 0.0f && rope->freq_base <= 3.4e38f && rope->freq_scale <= 3.4e38f);
        a.nd = rope->num_dim;
        a.turn1 = -2.0 * log2((double)rope->freq_base) / rope->num_dim;
        a.turn0 = log2((double)rope->freq_scale) - 2.6514961294723187980432933;             // log2(2 pi)
        a.mscale = rope->attention_factor;
    }
    SPY_CHECK_ARG(!q || (!pg_rows_meet(q_out, q) && !pg_rows_meet(q_out, k) && !pg_rows_meet(q_out, v)));
    a.q = q ? (const uint8_t *)q->data : nullptr; a.k = (const uint8_t *)k->data; a.v = (const uint8_t *)v->data;
    a.qo = q ? (uint8_t *)q_out->data : nullptr;
    a.q_h = q ? q->nb[1] : 0; a.q_t = q ? q->nb[2] : 0; a.qo_h = q ? q_out->nb[1] : 0; a.qo_t = q ? q_out->nb[2] : 0;
    a.k_h = k->nb[1]; a.k_t = k->nb[2]; a.v_h = v->nb[1]; a.v_t = v->nb[2];
    a.b.row_start = batch->row_start; a.b.kv_len = batch->kv_len; a.b.pages = batch->pages; a.b.page_stride = batch->page_stride;
    a.b.n_seq = batch->n_seq; a.b.n_row = (int)n_row; a.b.max_new = batch->max_new; a.b.max_kv = batch->max_kv; a.b.n_page = (int)k_pages->ne[3]; a.b.page_log2 = pg_log2(ps);
    a.H = (int)H; a.G = (int)G; a.hd = (int)hd; a.err = spy_hip_err_flag_ptr();
    return 0;
}
