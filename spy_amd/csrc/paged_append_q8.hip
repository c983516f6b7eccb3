// New tokens of a batch into a cache in pages of 8 bits: what paged_append.hip does, and K (rotated) and V as blocks of 32 elements of a row, as Q8_0 has them
// (Quantizator<FP32,Q8_0>, vec_convert.h:178-261 in the Spy tree): with m the largest magnitude, d = m / 127 as fp16 and q = x * (127 / m) to the nearest whole number, halves to even.
// A block with an infinity or NaN, or whose d has no fp16 value, gets d = NaN: it reads back as NaN, as fp16 pages would hold infinities.
// The whole numbers and the scales lie in planes of their own, so that both are read in whole aligned pieces: a block of 34 bytes is not.
// A block's maximum is taken by the four lanes that hold it.  One launch, rows and tiles of V as in paged_append.hip: V^T by tiles of 64 positions through LDS, so that 16 positions of a dimension are stored
// together (from 8 new tokens a sequence and 128 rows on), else byte by byte.  Bound by memory: 2048 tokens of 32 heads each, F32, with q: 30.7 us, 4.4 TB/s (F16: 25 us, 3.4 TB/s); a single token 4.3 us, a launch.
#include "paged_append.cuh"

struct append_q8_args : append_args {
    uint8_t *ks, *vs;
    int64_t ks_h, ks_g, vs_b, vs_h, vs_g;         // K scales: head, page; V scales: block, head, page
};

static __device__ __forceinline__ float q8_larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }       // NaN if either is
// over the four lanes whose numbers differ in the last two bits
static __device__ __forceinline__ float q8_of_four(float v) {
    v = q8_larger(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));
    return q8_larger(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));
}
// 8 elements of a lane, whose block the lanes of a group of four share: its scale, and to w the whole numbers, four to a word
static __device__ __forceinline__ uint16_t q8_block(const float (&x)[8], uint32_t (&w)[2]) {
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) top = q8_larger(top, fabsf(x[j]));
    top = q8_of_four(top);
    const float d = top / 127.0f, inv = top > 1e-36f ? 127.0f / top : 0.0f;       // (below that 127 / top has no value, and d none but 0)
#pragma unroll
    for (int i = 0; i < 2; i++) {
        w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w[i] |= ((uint32_t)(int)fminf(fmaxf(rintf(x[4 * i + j] * inv), -127.0f), 127.0f) & 0xFFu) << (8 * j);
    }
    return d < 65520.0f ? f2h(d) : (uint16_t)0x7E00u;                            // 65520 and more round to infinity
}

// 8 elements from `at` on of a row of which the first a.nd turn, as floats, turned.  cs: the row's angles.  In mode 2 an element's partner is nd / 2 away: read as well.
template <bool F16IN> static __device__ __forceinline__ void turned8(const append_args &a, const uint8_t *row, int at, const float2 *cs, float (&x)[8]) {
    constexpr int ES = F16IN ? 2 : 4;
    load8<F16IN>(row + at * ES, x);
    if (a.mode < 0 || at >= a.nd) return;
    if (a.mode == 0) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 t = cs[at / 2 + j];
            const float u = x[2 * j] * t.x - x[2 * j + 1] * t.y, v = x[2 * j] * t.y + x[2 * j + 1] * t.x;
            x[2 * j] = u; x[2 * j + 1] = v;
        }
    } else {
        const int half = a.nd / 2;
        const bool second = at >= half;
        float y[8];
        load8<F16IN>(row + (second ? at - half : at + half) * ES, y);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float2 t = cs[(second ? at - half : at) + j];
            x[j] = second ? y[j] * t.y + x[j] * t.x : x[j] * t.x - y[j] * t.y;
        }
    }
}

// One workgroup: R rows by `per` heads (of q, then k, then -- VROWS -- v), a thread on 8 elements of one
template <bool F16IN, int R, bool VROWS> static __device__ __forceinline__ void append_q8_rows(const append_q8_args &a, int tile, int head0, int per) {
    __shared__ float2 s_cs[R][128];
    __shared__ int s_pos[R], s_page[R];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int heads = min(per, a.H + a.G * (VROWS ? 2 : 1) - head0), U = a.hd / 8, ulog = a.hd == 64 ? 3 : a.hd == 128 ? 4 : 5;
    if (wave < R) append_place<R>(a, tile, s_pos, s_page);
    // entries that are wrong but belong to no row: one workgroup's idle wave looks at all (with tiles of V every workgroup that finds none does)
    if (VROWS && blockIdx.x == 0 && wave == R)
        for (int i = tid & 63; i < a.b.n_seq; i += 64) pg_sequence(a.b, i, a.err);
    __syncthreads();
    if (a.mode >= 0) {
        append_angles<R>(a, s_pos, s_cs);
        __syncthreads();
    }
    for (int i = tid; i < R * heads * U; i += PA_THREADS) {
        const int u = i & (U - 1), rh = i >> ulog, r = R == 1 ? 0 : rh / heads, head = head0 + (R == 1 ? rh : rh - r * heads);
        const int64_t row = (int64_t)tile * R + r;
        if (s_pos[r] == INT32_MIN) continue;
        const bool is_q = head < a.H, is_v = head >= a.H + a.G;
        const int h = is_q ? head : is_v ? head - a.H - a.G : head - a.H;
        float x[8];
        if (is_v) load8<F16IN>(a.v + row * a.v_t + h * a.v_h + u * 8 * (F16IN ? 2 : 4), x);
        else turned8<F16IN>(a, is_q ? a.q + row * a.q_t + h * a.q_h : a.k + row * a.k_t + h * a.k_h, 8 * u, s_cs[r], x);
        if (is_q) {
            *(uint4 *)(a.qo + row * a.qo_t + h * a.qo_h + u * 16) = pack8(x);
            continue;
        }
        uint32_t w[2];
        const uint16_t d = q8_block(x, w);                     // (a block's four lanes are of one head: all here)
        const int page = s_page[r], at = s_pos[r] & ((1 << a.b.page_log2) - 1);
        if (page < 0) continue;
        if (!is_v) {
            *(uint2 *)(a.kp + page * a.kp_g + h * a.kp_h + at * a.kp_p + u * 8) = make_uint2(w[0], w[1]);
            if ((u & 3) == 0) *(uint16_t *)(a.ks + page * a.ks_g + h * a.ks_h + at * (a.hd / 16) + (u >> 2) * 2) = d;
        } else {
            uint8_t *o = a.vp + page * a.vp_g + h * a.vp_h + 8 * u * a.vp_d + at;
#pragma unroll
            for (int j = 0; j < 8; j++) o[j * a.vp_d] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
            if ((u & 3) == 0) *(uint16_t *)(a.vs + page * a.vs_g + h * a.vs_h + (u >> 2) * a.vs_b + at * 2) = d;
        }
    }
}

// One workgroup: the new ones among 64 positions (a multiple of 64 on) of one sequence, one head of V, turned around in LDS so that a dimension's positions are stored together
#define PA_VB 68
template <bool F16IN> static __device__ __forceinline__ void append_q8_v_tile(const append_q8_args &a, int tile, int h) {
    __shared__ __attribute__((aligned(16))) uint8_t s_v[256 * PA_VB];
    __shared__ __attribute__((aligned(16))) uint16_t s_d[8][64];
    const int tid = threadIdx.x;
    int first = 0;
    const int s = append_tile(a, tile, first);
    if (s < 0) return;
    const pg_seq q = pg_sequence(a.b, s, a.err);
    const int p0 = first * 64, from = max(p0, max(q.kv - q.n_new, 0)), to = min(p0 + 64, q.kv), G8 = a.hd / 8;
    // four positions by 8 elements: the bytes of four positions are one word
    for (int i = tid; i < 16 * G8; i += PA_THREADS) {
        const int g = i & (G8 - 1), j = i / G8 * 4;
        uint32_t w[4][2];
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const int p = p0 + j + n;
            w[n][0] = w[n][1] = 0;
            if (p < from || p >= to) continue;
            float x[8];
            load8<F16IN>(a.v + (int64_t)(q.row0 + q.n_new - q.kv + p) * a.v_t + h * a.v_h + g * 8 * (F16IN ? 2 : 4), x);
            const uint16_t d = q8_block(x, w[n]);
            if ((g & 3) == 0) s_d[g >> 2][j + n] = d;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int by = 8 * (e & 3), k = e >> 2;
            *(uint32_t *)(s_v + (g * 8 + e) * PA_VB + j) = (w[0][k] >> by & 0xFFu) | (w[1][k] >> by & 0xFFu) << 8 | (w[2][k] >> by & 0xFFu) << 16 | (w[3][k] >> by & 0xFFu) << 24;
        }
    }
    __syncthreads();
    const int pmask = (1 << a.b.page_log2) - 1;
    for (int i = tid; i < 4 * (a.hd + a.hd / 32); i += PA_THREADS) {
        const int j = (i & 3) * 16, d = i >> 2, p = p0 + j;
        if (p + 16 <= from || p >= to) continue;
        const int page = a.b.pages[s * a.b.page_stride + (p >> a.b.page_log2)];      // a group of 16 lies in one page
        if (page < 0 || page >= a.b.n_page) { if (a.err) *a.err = 1; continue; }
        const bool all = p >= from && p + 16 <= to;
        if (d < a.hd) {
            uint8_t *o = a.vp + page * a.vp_g + h * a.vp_h + d * a.vp_d + (p & pmask);
            const uint32_t *w = (const uint32_t *)(s_v + d * PA_VB + j);
            if (all) *(uint4 *)o = make_uint4(w[0], w[1], w[2], w[3]);
            else
                for (int e = 0; e < 16; e++)
                    if (p + e >= from && p + e < to) o[e] = s_v[d * PA_VB + j + e];
        } else {
            uint16_t *o = (uint16_t *)(a.vs + page * a.vs_g + h * a.vs_h + (d - a.hd) * a.vs_b + (p & pmask) * 2);
            const uint4 *w = (const uint4 *)&s_d[d - a.hd][j];
            if (all) { ((uint4 *)o)[0] = w[0]; ((uint4 *)o)[1] = w[1]; }
            else
                for (int e = 0; e < 16; e++)
                    if (p + e >= from && p + e < to) o[e] = s_d[d - a.hd][j + e];
        }
    }
}

template <bool F16IN, int R, bool VROWS>
__global__ __launch_bounds__(PA_THREADS) void append_q8_kernel(append_q8_args a, int row_blocks, int chunks, int per) {
    if ((int)blockIdx.x < row_blocks) append_q8_rows<F16IN, R, VROWS>(a, blockIdx.x / chunks, (blockIdx.x % chunks) * per, per);
    else if constexpr (!VROWS) {
        const int i = blockIdx.x - row_blocks;
        append_q8_v_tile<F16IN>(a, i / a.G, i % a.G);
    }
}

extern "C" int spy_hip_paged_append_q8(void *stream, const spy_hip_tensor *q, const spy_hip_tensor *k, const spy_hip_tensor *v, const spy_hip_paged_batch *batch, const spy_hip_rope_param *rope,
                                       const spy_hip_tensor *q_out, const spy_hip_tensor *k_pages, const spy_hip_tensor *k_scales, const spy_hip_tensor *v_pages, const spy_hip_tensor *v_scales) {
    SPY_CHECK_ARG(k && v && k_pages && k_scales && v_pages && v_scales && (q != nullptr) == (q_out != nullptr));
    int rc = pg_check_batch(batch);
    if (!rc) rc = pg_check_pages_q8(k_pages, 1);
    if (!rc) rc = pg_check_pages_q8(v_pages, 0);
    if (!rc) rc = pg_check_scales(k_scales, k_pages, 1);
    if (!rc) rc = pg_check_scales(v_scales, v_pages, 0);
    if (rc) return rc;
    const int64_t hd = k_pages->ne[0], G = k_pages->ne[2], n_row = k->ne[2], H = q ? q->ne[1] : 0;
    append_q8_args a;
    rc = append_check(a, q, k, v, batch, rope, q_out, k_pages, v_pages);
    if (rc) return rc;
    a.kp = (uint8_t *)k_pages->data; a.vp = (uint8_t *)v_pages->data; a.ks = (uint8_t *)k_scales->data; a.vs = (uint8_t *)v_scales->data;
    a.kp_p = k_pages->nb[1]; a.kp_h = k_pages->nb[2]; a.kp_g = k_pages->nb[3]; a.ks_h = k_scales->nb[2]; a.ks_g = k_scales->nb[3];
    a.vp_d = v_pages->nb[1]; a.vp_h = v_pages->nb[2]; a.vp_g = v_pages->nb[3]; a.vs_b = v_scales->nb[1]; a.vs_h = v_scales->nb[2]; a.vs_g = v_scales->nb[3];
    const bool f16 = k->type == SPY_HIP_F16, tiles = batch->max_new >= 8 && n_row >= 128;
    // Rows of four: heads shared out so that there are four workgroups to a compute unit (2048 rows of 64 heads: 37.6 us by all heads, 30.4 by 32, 31.2 by 16), 8 at least
    const int64_t heads = H + G * (tiles ? 1 : 2), enough = heads * ((n_row + 3) / 4) / (4 * spy_num_cu());
    const int64_t per = !tiles ? PA_THREADS / (hd / 8) : enough < 8 ? 8 : enough < heads ? enough : heads, chunks = (heads + per - 1) / per;
    const int64_t row_blocks = (tiles ? (n_row + 3) / 4 : n_row) * chunks, blocks = row_blocks + (tiles ? (n_row / 64 + 2 * (int64_t)batch->n_seq) * G : 0);
    SPY_CHECK_ARG(blocks * PA_THREADS < (1ll << 32));                       // threads of a launch
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)blocks), block(PA_THREADS);
    if (tiles) {
        if (f16) append_q8_kernel<true, 4, false><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
        else append_q8_kernel<false, 4, false><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
    } else {
        if (f16) append_q8_kernel<true, 1, true><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
        else append_q8_kernel<false, 1, true><<<grid, block, 0, st>>>(a, (int)row_blocks, (int)chunks, (int)per);
    }
    return SPY_LAUNCH_RC();
}
