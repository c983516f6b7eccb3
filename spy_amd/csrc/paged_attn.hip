// Attention of a batch's new tokens over a cache in pages: MatMul(K, q) -> Softmax(mask, scale) -> MatMul(V^T, P) of the LLaMA graph (attention.cpp:25-302 in the
// Spy tree), per sequence and head, in one pass over the keys.
//
// For a query row i and the keys j that it sees: x_j = scale * q_i.K_j, out_i = sum_j e^(x_j - m) V_j / sum_j e^(x_j - m) for any m.  A wave walks its keys 32 at a
// time with a running m (the largest x so far), l (the sum of the exponentials) and o (the weighted sum of V); when m grows, l and o are scaled to the new one.
// Waves, and workgroups that share a row's keys, add up their (m, l, o) the same way.
//
// Scores are taken as S^T = K Q^T: the accumulator layout of the matrix instruction then has one query per lane, so that a row's maximum and sum are in-lane but for
// two steps between the four lanes that share a query, and -- with the rows of K dealt to the instruction's rows in the right order -- a lane's own probabilities
// are what the next instruction, O^T = V^T P^T, wants from it.  P never leaves the registers; V^T pages give its other operand as 16 contiguous bytes.
#include "paged.cuh"

int *spy_hip_err_flag_ptr();

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct attn_args {
    const uint8_t *q, *kp, *vp;
    uint8_t *out;
    int64_t q_h, q_t, o_h, o_t;
    int64_t kp_p, kp_h, kp_g, vp_d, vp_h, vp_g;
    pg_batch b;
    int G, group;                        // K/V heads, query heads to one
    float c;                             // scale * log2(e)
    int causal, window;                  // window: 0 or how many positions back
    int tiles, split;                    // tiles of 16 rows per sequence and K/V head; key tiles (of 32) per workgroup
    int n_split;
    float *part;                         // (o, m, l) of the workgroups that share rows
    int *err;
};

static __device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// over the four lanes l, l ^ 16, l ^ 32, l ^ 48
template <class Op> static __device__ __forceinline__ float quad_reduce(float v, Op op) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(h[0]), __uint_as_float(h[1]));
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
static __device__ __forceinline__ v8h halves(uint4 w) { return __builtin_bit_cast(v8h, w); }
// whether any of the eight fp16 values is an infinity or NaN
static __device__ __forceinline__ bool unbounded(uint4 w) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) any |= (v[i] & 0x7C00u) == 0x7C00u || (v[i] & 0x7C000000u) == 0x7C000000u;
    return any;
}
// the values of positions j with bit j set, 0 for the others and -- bounded -- for infinities and NaN
static __device__ __forceinline__ uint4 only(uint4 w, uint32_t mask, bool bounded) {
    uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (!(mask >> (2 * i) & 1) || (bounded && (v[i] & 0x7C00u) == 0x7C00u)) v[i] &= 0xFFFF0000u;
        if (!(mask >> (2 * i + 1) & 1) || (bounded && (v[i] & 0x7C000000u) == 0x7C000000u)) v[i] &= 0x0000FFFFu;
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// ---- 16 rows per workgroup: single tokens, and a few of them -------------------------------------------------------------------------
// A row is a new token and one of the query heads that share the K/V head: with a group of heads, or several new tokens, the keys are read once for all of them.
// Bound by the bytes of K and V.  The four waves take every fourth tile of 32 keys, straight from memory into the registers of the matrix instruction: nothing is
// shared between waves before the end.
template <int D, bool F32OUT>
__global__ __launch_bounds__(256) void attn_few_kernel(attn_args a) {
    constexpr int KS = D / 32, DT = D / 16, HALF = D < 128 ? D : 128;
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ __attribute__((aligned(16))) float s_o[4][16][HALF + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, quarter = lane >> 4;
    const int unit = blockIdx.x, piece = blockIdx.y;
    const int s = unit / (a.tiles * a.G), rest = unit - s * a.tiles * a.G, tile = rest / a.G, head = rest - tile * a.G;
    const pg_seq sq = pg_sequence(a.b, s, a.err);
    if (!sq.ok) return;
    const int rows = sq.n_new * a.group, r0 = tile * 16;
    if (r0 >= rows) return;
    const int r = min(r0 + n, rows - 1), token = r / a.group, hq = head * a.group + (r - token * a.group);
    const int past = sq.kv - sq.n_new;                                     // position of token 0; negative where the cache holds less than the new tokens
    // keys that a token t sees: lo(t) <= j < hi(t)
    auto hi_of = [&](int t) { return a.causal ? max(past + t + 1, 0) : sq.kv; };
    auto lo_of = [&](int t) { return a.window > 0 ? max(past + t - a.window + 1, 0) : 0; };
    const int t_first = r0 / a.group, t_last = min(r0 + 15, rows - 1) / a.group;
    const int hi = hi_of(token), lo = lo_of(token), hi_all = hi_of(t_first), lo_all = lo_of(t_last);          // all rows see lo_all .. hi_all - 1
    const int begin = lo_of(t_first) & ~31, end = hi_of(t_last);                                            // some row sees a key in begin .. end - 1
    const int n_tile = max((end - begin + 31) >> 5, 0);
    if (piece > 0 && piece * a.split >= n_tile) return;
    const int stop = min((piece + 1) * a.split, n_tile);
    const bool whole = n_tile <= a.split;

    const uint8_t *qrow = a.q + (int64_t)(sq.row0 + token) * a.q_t + (int64_t)hq * a.q_h;
    v8h fq[KS];
#pragma unroll
    for (int k = 0; k < KS; k++) fq[k] = halves(*(const uint4 *)(qrow + (32 * k + 8 * quarter) * 2));
    const int32_t *table = a.b.pages + (int64_t)s * a.b.page_stride;
    const int pmask = (1 << a.b.page_log2) - 1, last = (sq.kv - 1) >> a.b.page_log2;

    float m = -INFINITY, l = 0.0f;
    v4f o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = v4f{0, 0, 0, 0};
    for (int kt = piece * a.split + wave; kt < stop; kt += 4) {
        const int kb = begin + 32 * kt;
        // instruction row i of score tile t is key 8 (i / 4) + 4 t + i % 4: a lane's scores are then of keys 8 quarter + 4 t + 0 .. 3
        const int kk = kb + 8 * (n >> 2) + (n & 3), vk = kb + 8 * quarter;
        int kpage = table[min(kk >> a.b.page_log2, last)], vpage = table[min(vk >> a.b.page_log2, last)];
        const bool kbad = kpage < 0 || kpage >= a.b.n_page, vbad = vpage < 0 || vpage >= a.b.n_page;
        if (kbad) kpage = 0;
        if (vbad) vpage = 0;
        const uint8_t *kr = a.kp + kpage * a.kp_g + head * a.kp_h + (kk & pmask) * a.kp_p + quarter * 16;
        const uint8_t *vr = a.vp + vpage * a.vp_g + head * a.vp_h + (vk & pmask) * 2 + n * a.vp_d;
        uint4 fk[2][KS], fv[DT];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < KS; k++) fk[t][k] = *(const uint4 *)(kr + t * 4 * a.kp_p + k * 64);
#pragma unroll
        for (int d = 0; d < DT; d++) fv[d] = *(const uint4 *)(vr + 16 * d * a.vp_d);
        v4f x[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            x[t] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; k++) x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(fk[t][k]), fq[k], x[t], 0, 0, 0);
        }
        float e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = x[j >> 2][j & 3] * a.c;
        uint32_t seen = 0xFF;                                              // bit j: this lane's query sees key 8 quarter + j
        const bool masked = __any(kb + 32 > hi_all || kb < lo_all || vbad);
        bool fix = false;
        if (masked) {
            seen = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) seen |= (uint32_t)(vk + j >= lo && vk + j < hi && !vbad) << j;
#pragma unroll
            for (int j = 0; j < 8; j++) e[j] = seen >> j & 1 ? e[j] : -INFINITY;
            if (vbad && vk < end && vk + 8 > lo_of(t_first) && a.err) *a.err = 1;     // (a page before the window may be gone)
            // positions behind the cache's last one hold anything: their V is taken as 0.  Infinities and NaN among the others, which some rows may see and
            // others not, go the long way round
            uint32_t there = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) there |= (uint32_t)(vk + j < end && !vbad) << j;
            bool any = false;
#pragma unroll
            for (int d = 0; d < DT; d++) { fv[d] = only(fv[d], there, false); any |= unbounded(fv[d]); }
            fix = __any(any);
            if (fix)
#pragma unroll
                for (int d = 0; d < DT; d++) fv[d] = only(fv[d], 0xFF, true);
        }
        float top = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
        top = fmaxf(m, quad_reduce(top, [](float p, float q) { return fmaxf(p, q); }));
        const float base = top == -INFINITY ? 0.0f : top, shrink = exp2_(m - base);
        m = top;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) { e[j] = exp2_(e[j] - base); sum += e[j]; }
        l = l * shrink + sum;
        v8h p, p2;
#pragma unroll
        for (int j = 0; j < 8; j++) { p[j] = (_Float16)e[j]; if (F32OUT) p2[j] = (_Float16)(e[j] - (float)p[j]); }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            o[d] *= shrink;
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(fv[d]), p, o[d], 0, 0, 0);
            if (F32OUT) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(fv[d]), p2, o[d], 0, 0, 0);
        }
        if (fix) {
            for (int j = 0; j < 32; j++) {                                 // key kb + j, held by the lanes of quarter j / 8
                const int from = n + 16 * (j >> 3), key = kb + j;
                float pj = 0.0f;
                uint32_t sj = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) if (i == (j & 7)) pj = e[i];
                pj = __shfl(pj, from, SPY_WAVE);
                sj = (uint32_t)__shfl((int)seen, from, SPY_WAVE) >> (j & 7) & 1;
                if (key >= end || !sj) continue;
                const int page = table[key >> a.b.page_log2];              // in range: the key is seen
                const uint8_t *v = a.vp + page * a.vp_g + head * a.vp_h + (key & pmask) * 2;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint16_t b = *(const uint16_t *)(v + (16 * d + 4 * quarter + i) * a.vp_d);
                        if ((b & 0x7C00u) == 0x7C00u) o[d][i] += pj * h2f(b);
                    }
            }
        }
    }
    l = quad_reduce(l, [](float p, float q) { return p + q; });
    if (quarter == 0) { s_m[wave][n] = m; s_l[wave][n] = l; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) top = fmaxf(top, s_m[w][n]);
    const float shrink = exp2_(m - (top == -INFINITY ? 0.0f : top));
    float *part = a.part + (int64_t)((int64_t)unit * a.n_split + piece) * 16 * (D + 2);
#pragma unroll
    for (int h = 0; h < D / HALF; h++) {
        if (h) __syncthreads();
#pragma unroll
        for (int d = 0; d < HALF / 16; d++) {
            const v4f v = o[h * (HALF / 16) + d] * shrink;
            *(v4f *)&s_o[wave][n][16 * d + 4 * quarter] = v;
        }
        __syncthreads();
        for (int i = tid; i < 16 * (HALF / 4); i += 256) {
            const int row = i / (HALF / 4), d = (i - row * (HALF / 4)) * 4;
            v4f v = v4f{0, 0, 0, 0};
            float mx = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; w++) { v += *(const v4f *)&s_o[w][row][d]; mx = fmaxf(mx, s_m[w][row]); }
            const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int w = 0; w < 4; w++) sum += s_l[w][row] * exp2_(s_m[w][row] - base);
            if (r0 + row >= rows) continue;
            const int dd = h * HALF + d;
            if (whole) {
                const int t = (r0 + row) / a.group, hh = head * a.group + (r0 + row - t * a.group);
                uint8_t *dst = a.out + (int64_t)(sq.row0 + t) * a.o_t + (int64_t)hh * a.o_h;
                const bool none = mx == -INFINITY && sum == 0.0f;          // sees no key
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = none ? 0.0f : v[k] / sum;
                if (F32OUT) *(v4f *)(dst + dd * 4) = v;
                else *(uint2 *)(dst + dd * 2) = make_uint2(f2h(v[0]) | (uint32_t)f2h(v[1]) << 16, f2h(v[2]) | (uint32_t)f2h(v[3]) << 16);
            } else {
                *(v4f *)(part + row * D + dd) = v;
                if (dd == 0) { part[16 * D + row] = mx; part[16 * D + 16 + row] = sum; }
            }
        }
    }
}

// The rows whose keys several workgroups shared
template <int D, bool F32OUT>
__global__ __launch_bounds__(256) void attn_join_kernel(attn_args a) {
    const int unit = blockIdx.x, s = unit / (a.tiles * a.G), rest = unit - s * a.tiles * a.G, tile = rest / a.G, head = rest - tile * a.G;
    const pg_seq sq = pg_sequence(a.b, s, nullptr);
    if (!sq.ok) return;
    const int rows = sq.n_new * a.group, r0 = tile * 16;
    if (r0 >= rows) return;
    const int past = sq.kv - sq.n_new, t_first = r0 / a.group, t_last = min(r0 + 15, rows - 1) / a.group;
    const int begin = (a.window > 0 ? max(past + t_first - a.window + 1, 0) : 0) & ~31, end = a.causal ? max(past + t_last + 1, 0) : sq.kv;
    const int n_tile = max((end - begin + 31) >> 5, 0), pieces = (n_tile + a.split - 1) / a.split;
    if (pieces <= 1) return;
    const float *part = a.part + (int64_t)unit * a.n_split * 16 * (D + 2);
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
        const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
        if (r0 + row >= rows) continue;
        float mx = -INFINITY, sum = 0.0f;
        for (int p = 0; p < pieces; p++) mx = fmaxf(mx, part[(int64_t)p * 16 * (D + 2) + 16 * D + row]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        v4f v = v4f{0, 0, 0, 0};
        for (int p = 0; p < pieces; p++) {
            const float *q = part + (int64_t)p * 16 * (D + 2);
            const float w = exp2_(q[16 * D + row] - base);
            sum += w * q[16 * D + 16 + row];
            v += w * *(const v4f *)(q + row * D + d);
        }
        const int t = (r0 + row) / a.group, hh = head * a.group + (r0 + row - t * a.group);
        uint8_t *dst = a.out + (int64_t)(sq.row0 + t) * a.o_t + (int64_t)hh * a.o_h;
        const bool none = mx == -INFINITY && sum == 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = none ? 0.0f : v[k] / sum;
        if (F32OUT) *(v4f *)(dst + d * 4) = v;
        else *(uint2 *)(dst + d * 2) = make_uint2(f2h(v[0]) | (uint32_t)f2h(v[1]) << 16, f2h(v[2]) | (uint32_t)f2h(v[3]) << 16);
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
struct attn_plan { int64_t tiles, units, split, n_split; size_t scratch; };
static int attn_make_plan(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *b, attn_plan &p) {
    SPY_CHECK_ARG(q && k_pages && q->ne[1] > 0 && q->ne[1] <= 65535);
    int rc = pg_check_batch(b);
    if (!rc) rc = pg_check_pages(k_pages, 1);
    if (rc) return rc;
    const int64_t G = k_pages->ne[2], H = q->ne[1], hd = k_pages->ne[0];
    SPY_CHECK_ARG(G <= 65535 && H % G == 0);
    const int64_t group = H / G;
    p.tiles = ((int64_t)b->max_new * group + 15) / 16;
    p.units = (int64_t)b->n_seq * p.tiles * G;
    SPY_CHECK_ARG(p.units < (1ll << 30));
    // Keys are shared out in pieces of one size, so that long sequences of a ragged batch take more workgroups: as many as fill the card twice over, 256 keys at least
    const int64_t key_tiles = ((int64_t)b->max_kv + 31) / 32 + 1, want = (2 * (int64_t)spy_num_cu() + p.units - 1) / p.units;
    p.split = (key_tiles + want - 1) / want;
    if (p.split < 8) p.split = 8;
    p.n_split = (key_tiles + p.split - 1) / p.split;
    if (p.n_split > 65535) { p.n_split = 65535; p.split = (key_tiles + 65534) / 65535; }
    p.scratch = p.n_split > 1 ? (size_t)(p.units * p.n_split * 16 * (hd + 2) * 4) : 0;
    return 0;
}

extern "C" size_t spy_hip_paged_attention_scratch_size(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *batch) {
    attn_plan p;
    return attn_make_plan(q, k_pages, batch, p) ? 0 : p.scratch;
}

template <int D, bool F32OUT> static int attn_launch(const attn_args &a, const attn_plan &p, hipStream_t st) {
    attn_few_kernel<D, F32OUT><<<dim3((unsigned)p.units, (unsigned)p.n_split), dim3(256), 0, st>>>(a);
    int rc = SPY_LAUNCH_RC();
    if (rc || p.n_split == 1) return rc;
    attn_join_kernel<D, F32OUT><<<dim3((unsigned)p.units), dim3(256), 0, st>>>(a);
    return SPY_LAUNCH_RC();
}

extern "C" int spy_hip_paged_attention(void *stream, const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_tensor *v_pages, const spy_hip_tensor *out,
                                       const spy_hip_paged_batch *batch, float scale, int32_t causal, int32_t window, void *scratch, size_t scratch_bytes) {
    SPY_CHECK_ARG(q && k_pages && v_pages && out);
    attn_plan p;
    int rc = attn_make_plan(q, k_pages, batch, p);
    if (!rc) rc = pg_check_pages(v_pages, 0);
    if (rc) return rc;
    if (q->type != SPY_HIP_F16 || (out->type != SPY_HIP_F32 && out->type != SPY_HIP_F16)) return SPY_HIP_EUNSUPPORTED;
    const int64_t hd = k_pages->ne[0], ps = k_pages->ne[1], G = k_pages->ne[2], n_row = q->ne[2], H = q->ne[1];
    SPY_CHECK_ARG(v_pages->ne[0] == ps && v_pages->ne[1] == hd && v_pages->ne[2] == G && v_pages->ne[3] == k_pages->ne[3]);
    SPY_CHECK_ARG(n_row > 0 && n_row < (1 << 28) && pg_rows_ok(q, hd, H, n_row) && pg_rows_ok(out, hd, H, n_row) && window >= 0 && scale - scale == 0.0f);
    if (p.scratch) {
        if (scratch_bytes < p.scratch) return SPY_HIP_ENOSPACE;
        SPY_CHECK_ARG(scratch && ((uintptr_t)scratch & 255) == 0);
    }
    attn_args a;
    a.q = (const uint8_t *)q->data; a.kp = (const uint8_t *)k_pages->data; a.vp = (const uint8_t *)v_pages->data; a.out = (uint8_t *)out->data;
    a.q_h = q->nb[1]; a.q_t = q->nb[2]; a.o_h = out->nb[1]; a.o_t = out->nb[2];
    a.kp_p = k_pages->nb[1]; a.kp_h = k_pages->nb[2]; a.kp_g = k_pages->nb[3];
    a.vp_d = v_pages->nb[1]; a.vp_h = v_pages->nb[2]; a.vp_g = v_pages->nb[3];
    a.b.row_start = batch->row_start; a.b.kv_len = batch->kv_len; a.b.pages = batch->pages; a.b.page_stride = batch->page_stride;
    a.b.n_seq = batch->n_seq; a.b.n_row = (int)n_row; a.b.max_new = batch->max_new; a.b.max_kv = batch->max_kv; a.b.n_page = (int)k_pages->ne[3]; a.b.page_log2 = pg_log2(ps);
    a.G = (int)G; a.group = (int)(H / G); a.c = scale * 1.44269504088896341f; a.causal = causal != 0; a.window = window > (1 << 30) ? 0 : window;
    a.tiles = (int)p.tiles; a.split = (int)p.split; a.n_split = (int)p.n_split; a.part = (float *)scratch; a.err = spy_hip_err_flag_ptr();
    hipStream_t st = (hipStream_t)stream;
    const bool f32 = out->type == SPY_HIP_F32;
    if (hd == 64) return f32 ? attn_launch<64, true>(a, p, st) : attn_launch<64, false>(a, p, st);
    if (hd == 128) return f32 ? attn_launch<128, true>(a, p, st) : attn_launch<128, false>(a, p, st);
    return f32 ? attn_launch<256, true>(a, p, st) : attn_launch<256, false>(a, p, st);
}
