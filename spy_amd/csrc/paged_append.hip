// New tokens of a batch of sequences into a cache in pages, with the position rotation on the way: what Rope, the fp16 rounding and the two cache copies of the
// LLaMA graph do for one sequence (non-linear.cpp:270-371; view.cpp:83-227; attention.cpp:180-265 in the Spy tree), for the whole batch in one launch.
//
// Pair i of a token at position p turns by p * f_i, f_i = freq_scale * freq_base^(-2i / num_dim).  The turn is taken in revolutions and reduced to [-1/2, 1/2] in
// 64 bits (at position 10^6 a 32-bit angle is off by up to 0.03), sine and cosine of what is left in 32.  They are worked out once per row and workgroup and kept in LDS.
//
// Bound by memory, or a launch: 2048 rows of 32 + 2 x 32 heads, 128 wide, F32, 31.9 us, which is 4.7 TB/s as a copy has; a row 5 us, of which the kernel is 3.6.
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

// One workgroup: R rows by `per` heads (of q, then k, then -- VROWS -- v), a thread on two groups of 8 elements, 8u .. and half + 8u .. of a region of the row: the
// rotated elements, and those behind them.  In mode 2 the two groups are the two elements of 8 pairs, in mode 0 four pairs each.
template <bool F16IN, int R, bool VROWS>
static __device__ __forceinline__ void append_rows(const append_args &a, int tile, int head0, int per) {
    __shared__ float2 s_cs[R][128];
    __shared__ int s_pos[R], s_page[R];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int heads = min(per, a.H + a.G * (VROWS ? 2 : 1) - head0), U = a.hd / 16, ulog = a.hd == 64 ? 2 : a.hd == 128 ? 3 : 4, npair = a.nd / 2;
    if (wave < R) {                                            // where the rows go
        const int r = tile * R + wave;
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
    // entries that are wrong but belong to no row: one workgroup's idle wave looks at all (with tiles of V every workgroup that finds none does)
    if (VROWS && blockIdx.x == 0 && wave == R)
        for (int i = lane; i < a.b.n_seq; i += 64) pg_sequence(a.b, i, a.err);
    __syncthreads();
    if (a.mode >= 0) {
        for (int i = tid; i < R * npair; i += PA_THREADS) {
            const int r = i / npair, p = i - r * npair;
            const double turns = (double)s_pos[r] * exp2(a.turn0 + p * a.turn1);
            const float x = (float)(turns - rint(turns));
            float sn, cs;
            sincospif(2.0f * x, &sn, &cs);
            s_cs[r][p] = make_float2(cs * a.mscale, sn * a.mscale);
        }
        __syncthreads();
    }
    for (int i = tid; i < R * heads * U; i += PA_THREADS) {
        const int u = i & (U - 1), rh = i >> ulog, r = R == 1 ? 0 : rh / heads, head = head0 + (R == 1 ? rh : rh - r * heads);
        const int64_t row = (int64_t)tile * R + r;
        if (s_pos[r] == INT32_MIN) continue;
        const bool is_q = head < a.H, is_v = head >= a.H + a.G;
        const int h = is_q ? head : is_v ? head - a.H - a.G : head - a.H;
        const uint8_t *src = is_q ? a.q + row * a.q_t + h * a.q_h : is_v ? a.v + row * a.v_t + h * a.v_h : a.k + row * a.k_t + h * a.k_h;
        const int turned = a.mode < 0 || is_v ? 0 : a.nd;
        const bool rot = 16 * u < turned;
        const int half = (rot ? turned : a.hd - turned) / 2, lo = rot ? 8 * u : turned + 8 * u - turned / 2, hi = lo + half;
        float x[8], y[8];
        const int es = F16IN ? 2 : 4;
        load8<F16IN>(src + lo * es, x);
        load8<F16IN>(src + hi * es, y);
        if (rot) {
            if (a.mode == 2) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float2 t = s_cs[r][lo + j];
                    const float p = x[j] * t.x - y[j] * t.y, q = x[j] * t.y + y[j] * t.x;
                    x[j] = p; y[j] = q;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 t = s_cs[r][lo / 2 + j], w = s_cs[r][hi / 2 + j];
                    const float p = x[2 * j] * t.x - x[2 * j + 1] * t.y, q = x[2 * j] * t.y + x[2 * j + 1] * t.x;
                    const float c = y[2 * j] * w.x - y[2 * j + 1] * w.y, d = y[2 * j] * w.y + y[2 * j + 1] * w.x;
                    x[2 * j] = p; x[2 * j + 1] = q; y[2 * j] = c; y[2 * j + 1] = d;
                }
            }
        }
        const int page = s_page[r], at = s_pos[r] & ((1 << a.b.page_log2) - 1);
        if (is_q) {
            uint8_t *o = a.qo + row * a.qo_t + h * a.qo_h;
            *(uint4 *)(o + lo * 2) = pack8(x);
            *(uint4 *)(o + hi * 2) = pack8(y);
        } else if (page < 0) {
            continue;
        } else if (!is_v) {
            uint8_t *o = a.kp + page * a.kp_g + h * a.kp_h + at * a.kp_p;
            *(uint4 *)(o + lo * 2) = pack8(x);
            *(uint4 *)(o + hi * 2) = pack8(y);
        } else {
            uint8_t *o = a.vp + page * a.vp_g + h * a.vp_h + at * 2;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                *(uint16_t *)(o + (lo + j) * a.vp_d) = f2h(x[j]);
                *(uint16_t *)(o + (hi + j) * a.vp_d) = f2h(y[j]);
            }
        }
    }
}

// One workgroup: the new ones among 64 positions (a multiple of 64 on) of one sequence, one head of V, turned around in LDS so that a dimension's positions are stored together
#define PA_VT 66
template <bool F16IN> static __device__ __forceinline__ void append_v_tile(const append_args &a, int tile, int h) {
    __shared__ uint16_t s_v[256 * PA_VT];
    const int tid = threadIdx.x, lane = tid & 63;
    // every wave finds the tile's sequence: tiles of the sequences one after the other, 64 sequences per round
    int s = -1, first = 0;
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
            s = base + at;
            first = __shfl(f, at, SPY_WAVE) + left - __shfl(sum - n, at, SPY_WAVE);
            break;
        }
        left -= __shfl(sum, 63, SPY_WAVE);
    }
    if (s < 0) return;
    const pg_seq q = pg_sequence(a.b, s, a.err);
    const int p0 = first * 64, from = max(p0, max(q.kv - q.n_new, 0)), to = min(p0 + 64, q.kv), G8 = a.hd / 8;
    for (int i = tid; i < 64 * G8; i += PA_THREADS) {
        const int g = i & (G8 - 1), j = i / G8, p = p0 + j;
        if (p < from || p >= to) continue;
        float x[8];
        load8<F16IN>(a.v + (int64_t)(q.row0 + q.n_new - q.kv + p) * a.v_t + h * a.v_h + g * 8 * (F16IN ? 2 : 4), x);
#pragma unroll
        for (int e = 0; e < 8; e++) s_v[(g * 8 + e) * PA_VT + j] = f2h(x[e]);
    }
    __syncthreads();
    for (int i = tid; i < 8 * a.hd; i += PA_THREADS) {
        const int j = (i & 7) * 8, d = i >> 3, p = p0 + j;
        if (p + 8 <= from || p >= to) continue;
        const int page = a.b.pages[s * a.b.page_stride + (p >> a.b.page_log2)];      // a group of 8 lies in one page
        if (page < 0 || page >= a.b.n_page) { if (a.err) *a.err = 1; continue; }
        uint8_t *o = a.vp + page * a.vp_g + h * a.vp_h + d * a.vp_d + (p & ((1 << a.b.page_log2) - 1)) * 2;
        if (p >= from && p + 8 <= to) {
            const uint32_t *w = (const uint32_t *)(s_v + d * PA_VT + j);
            *(uint4 *)o = make_uint4(w[0], w[1], w[2], w[3]);
        } else
            for (int e = 0; e < 8; e++)
                if (p + e >= from && p + e < to) ((uint16_t *)o)[e] = s_v[d * PA_VT + j + e];
    }
}

template <bool F16IN, int R, bool VROWS>
__global__ __launch_bounds__(PA_THREADS) void append_kernel(append_args a, int row_blocks, int chunks, int per) {
    if ((int)blockIdx.x < row_blocks) append_rows<F16IN, R, VROWS>(a, blockIdx.x / chunks, (blockIdx.x % chunks) * per, per);
    else if constexpr (!VROWS) {
        const int i = blockIdx.x - row_blocks;
        append_v_tile<F16IN>(a, i / a.G, i % a.G);
    }
}

extern "C" int spy_hip_paged_append(void *stream, const spy_hip_tensor *q, const spy_hip_tensor *k, const spy_hip_tensor *v, const spy_hip_paged_batch *batch,
                                    const spy_hip_rope_param *rope, const spy_hip_tensor *q_out, const spy_hip_tensor *k_pages, const spy_hip_tensor *v_pages) {
    SPY_CHECK_ARG(k && v && k_pages && v_pages && (q != nullptr) == (q_out != nullptr));
    int rc = pg_check_batch(batch);
    if (!rc) rc = pg_check_pages(k_pages, 1);
    if (!rc) rc = pg_check_pages(v_pages, 0);
    if (rc) return rc;
    if ((k->type != SPY_HIP_F32 && k->type != SPY_HIP_F16) || v->type != k->type || (q && (q->type != k->type || q_out->type != SPY_HIP_F16))) return SPY_HIP_EUNSUPPORTED;
    const int64_t hd = k_pages->ne[0], ps = k_pages->ne[1], G = k_pages->ne[2], n_row = k->ne[2], H = q ? q->ne[1] : 0;
    SPY_CHECK_ARG(v_pages->ne[0] == ps && v_pages->ne[1] == hd && v_pages->ne[2] == G && v_pages->ne[3] == k_pages->ne[3]);
    SPY_CHECK_ARG(n_row > 0 && n_row < (1 << 28) && G <= 65535 && H <= 65535 && pg_rows_ok(k, hd, G, n_row) && pg_rows_ok(v, hd, G, n_row));
    SPY_CHECK_ARG(!q || (H > 0 && H % G == 0 && pg_rows_ok(q, hd, H, n_row) && pg_rows_ok(q_out, hd, H, n_row)));
    append_args a;
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
    a.qo = q ? (uint8_t *)q_out->data : nullptr; a.kp = (uint8_t *)k_pages->data; a.vp = (uint8_t *)v_pages->data;
    a.q_h = q ? q->nb[1] : 0; a.q_t = q ? q->nb[2] : 0; a.qo_h = q ? q_out->nb[1] : 0; a.qo_t = q ? q_out->nb[2] : 0;
    a.k_h = k->nb[1]; a.k_t = k->nb[2]; a.v_h = v->nb[1]; a.v_t = v->nb[2];
    a.kp_p = k_pages->nb[1]; a.kp_h = k_pages->nb[2]; a.kp_g = k_pages->nb[3];
    a.vp_d = v_pages->nb[1]; a.vp_h = v_pages->nb[2]; a.vp_g = v_pages->nb[3];
    a.b.row_start = batch->row_start; a.b.kv_len = batch->kv_len; a.b.pages = batch->pages; a.b.page_stride = batch->page_stride;
    a.b.n_seq = batch->n_seq; a.b.n_row = (int)n_row; a.b.max_new = batch->max_new; a.b.max_kv = batch->max_kv; a.b.n_page = (int)k_pages->ne[3]; a.b.page_log2 = pg_log2(ps);
    a.H = (int)H; a.G = (int)G; a.hd = (int)hd; a.err = spy_hip_err_flag_ptr();
    // V in tiles of 64 positions, rows four at a time, or a row per workgroup (128-wide, 32 heads): 16 sequences of 6 tokens each 9.5 and 9.0 us, of 8 9.7 and 10.4, of 256
    // 70 and 223; one sequence of 64 tokens 8.8 and 6.7 us, of 256 11.4 and 12.3.  Sequences of few tokens fill no tile.
    const bool f16 = k->type == SPY_HIP_F16, tiles = batch->max_new >= 8 && n_row >= 128;
    const int64_t heads = H + G * (tiles ? 1 : 2), per = tiles ? heads : PA_THREADS / (hd / 16), chunks = (heads + per - 1) / per;
    const int64_t row_blocks = (tiles ? (n_row + 3) / 4 : n_row) * chunks, blocks = row_blocks + (tiles ? (n_row / 64 + 2 * (int64_t)batch->n_seq) * G : 0);
    SPY_CHECK_ARG(blocks * PA_THREADS < (1ll << 32));                       // threads of a launch
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks), block(PA_THREADS);
    if (tiles) {
        if (f16) append_kernel<true, 4, false><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
        else append_kernel<false, 4, false><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
    } else {
        if (f16) append_kernel<true, 1, true><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
        else append_kernel<false, 1, true><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
    }
    return SPY_LAUNCH_RC();
}
