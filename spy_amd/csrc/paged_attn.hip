// Attention over pages of fp16: the kernels of paged_attn.cuh as they are, and the join of the rows whose keys several workgroups shared.
#include "paged_attn.cuh"

// ---- the rows whose keys several workgroups shared: 16 rows per workgroup ---------------------------------------------------------------
// Latency, and what the first launch wrote: a wave has the (m, l) of four rows, a lane one workgroup's; eight pieces of o are requested at a time, the first before (m, l) are
// there.  Measured: one request of 4096 keys (17 pieces) 4.5 us, 512 tokens on 7680 (two pieces, 17 MB) 8.
template <int D, bool F32OUT, int TILE> static __device__ __forceinline__ void join_rows(const attn_args &a, const row_tile &rt, const pg_seq &sq, int head, int sub, int pieces, const float *part) {
    __shared__ float s_w[16][64], s_sum[16];
    constexpr int64_t STEP = TILE * (D + 2);
    constexpr int ITEMS = 16 * (D / 4) / 256;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = min(16, rt.n_row - 16 * sub);
    if (rows <= 0) return;
    v4f v[ITEMS], x[ITEMS][8];
    const auto request = [&](int p) {                                      // the first eight of o from piece p on, for every item of the thread
#pragma unroll
        for (int k = 0; k < ITEMS; k++) {
            const int i = threadIdx.x + 256 * k, row = i / (D / 4), d = (i % (D / 4)) * 4;
            if (row >= rows) continue;
#pragma unroll
            for (int j = 0; j < 8; j++) x[k][j] = *(const v4f *)(part + min(p + j, pieces - 1) * STEP + (16 * sub + row) * D + d);
        }
    };
    float m0[4], l0[4], top[4], sum[4];                                    // m and l of the first 64 pieces, all asked for before the first is waited for
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float *q = part + min(lane, pieces - 1) * STEP + TILE * D + 16 * sub + min(4 * wave + i, rows - 1);
        m0[i] = q[0]; l0[i] = q[TILE];
    }
    request(0);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = 4 * wave + i;
        sum[i] = 0.0f;
        top[i] = m0[i];                                                    // (a lane past the pieces has the last one's)
        for (int p = 64 + lane; p < pieces; p += 64) top[i] = fmaxf(top[i], part[p * STEP + TILE * D + 16 * sub + min(row, rows - 1)]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) top[i] = wave_max(top[i]);
#pragma unroll
    for (int k = 0; k < ITEMS; k++) v[k] = v4f{0, 0, 0, 0};
    for (int base = 0; base < pieces; base += 64) {
        const int n = min(64, pieces - base);
        if (base) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = 4 * wave + i;
            if (row >= rows) continue;
            float w = 0.0f;
            if (lane < n) {
                const float *q = part + (base + lane) * STEP + TILE * D + 16 * sub + row;
                w = above_0(exp2_((base ? q[0] : m0[i]) - (top[i] == -INFINITY ? 0.0f : top[i])));
                sum[i] += w * (base ? q[TILE] : l0[i]);
            }
            s_w[row][lane] = w;
        }
        __syncthreads();
        for (int p = 0; p < n; p += 8) {
            if (base + p) request(base + p);
#pragma unroll
            for (int k = 0; k < ITEMS; k++) {
                const int row = (threadIdx.x + 256 * k) / (D / 4);
                if (row >= rows) continue;
#pragma unroll
                for (int j = 0; j < 8; j++) if (p + j < n) v[k] += s_w[row][p + j] * x[k][j];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float all = wave_sum(sum[i]);
        if (lane == 0) s_sum[4 * wave + i] = top[i] == -INFINITY && all == 0.0f ? 0.0f : all;      // 0: sees no key
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const int i = threadIdx.x + 256 * k, row = i / (D / 4), d = (i % (D / 4)) * 4;
        if (row >= rows) continue;
        const int r = rt.r0 + 16 * sub + row, t = r / a.group, hh = head * a.group + (r - t * a.group);
        uint8_t *dst = a.out + (int64_t)(sq.row0 + t) * a.o_t + (int64_t)hh * a.o_h;
        const float all = s_sum[row];
#pragma unroll
        for (int j = 0; j < 4; j++) v[k][j] = all == 0.0f ? 0.0f : v[k][j] / all;
        if (F32OUT) *(v4f *)(dst + d * 4) = v[k];
        else *(uint2 *)(dst + d * 2) = make_uint2(f2h(v[k][0]) | (uint32_t)f2h(v[k][1]) << 16, f2h(v[k][2]) | (uint32_t)f2h(v[k][3]) << 16);
    }
}
template <int D, bool F32OUT> __global__ __launch_bounds__(256) void attn_join_kernel(attn_args a, int few_units) {
    if ((int)blockIdx.x < few_units) {
        const int unit = blockIdx.x, s = unit / a.G, head = unit - s * a.G;
        const pg_seq sq = pg_sequence(a.b, s, nullptr);
        if (!sq.ok) return;
        const row_tile rt(a, sq, 0, 16);
        if (rt.rows > a.few) return;
        const int n_tile = max((rt.end() - (rt.lo_any() & ~31) + 31) >> 5, 0), pieces = (n_tile + a.few_split - 1) / a.few_split;
        if (pieces > 1) join_rows<D, F32OUT, 16>(a, rt, sq, head, 0, pieces, a.few_part + (int64_t)unit * a.few_pieces * 16 * (D + 2));
        return;
    }
    const int b = blockIdx.x - few_units, unit = b / (CHUNK_ROWS / 16), sub = b % (CHUNK_ROWS / 16), head = unit % a.G;
    int tile, count;
    pg_seq sq;
    const int s = find_tile(a, unit / a.G, tile, count, sq);
    if (s < 0) return;
    const row_tile rt(a, sq, count - 1 - tile, CHUNK_ROWS);
    const int n_tile = max((rt.end() - (rt.lo_any() & ~63) + 63) >> 6, 0), pieces = (n_tile + a.chunk_split - 1) / a.chunk_split;
    if (pieces > 1) join_rows<D, F32OUT, CHUNK_ROWS>(a, rt, sq, head, sub, pieces, a.chunk_part + (int64_t)unit * a.chunk_pieces * CHUNK_ROWS * (D + 2));
}

template <int D, bool F32OUT> __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_few_kernel(attn_args a) {
    __shared__ few_shared<D, 4> sh;
    attn_few<D, F32OUT, 4>(a, sh, blockIdx.x);
}
// Both kinds of sequences in one launch, the chunks first: they take longest, and the single tokens' reads of memory run beside their products
template <int D, bool F32OUT> __global__ __launch_bounds__(256 * chunk_groups(D)) void attn_mixed_kernel(attn_args a) {
    __shared__ union { few_shared<D, 4 * chunk_groups(D)> few; chunk_shared<D> chunk; } sh;
    if ((int)blockIdx.x < a.chunk_blocks) attn_chunk<D, F32OUT>(a, sh.chunk, blockIdx.x);
    else attn_few<D, F32OUT, 4 * chunk_groups(D)>(a, sh.few, blockIdx.x - a.chunk_blocks);
}

int spy_attn_join(const attn_args &a, const attn_plan &p, int64_t hd, bool f32, hipStream_t st) {
    if (!p.scratch) return 0;
    const int64_t few = p.few_pieces > 1 ? p.few_units : 0, chunk = p.chunk_pieces > 1 ? p.chunk_units * (CHUNK_ROWS / 16) : 0;
    const auto go = [&](auto kernel) { kernel<<<dim3((unsigned)(few + chunk)), dim3(256), 0, st>>>(a, (int)few); };
    if (hd == 64) go(f32 ? attn_join_kernel<64, true> : attn_join_kernel<64, false>);
    else if (hd == 128) go(f32 ? attn_join_kernel<128, true> : attn_join_kernel<128, false>);
    else go(f32 ? attn_join_kernel<256, true> : attn_join_kernel<256, false>);
    return SPY_LAUNCH_RC();
}

extern "C" size_t spy_hip_paged_attention_scratch_size(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *batch) {
    attn_plan p;
    return attn_make_plan(q, k_pages, batch, false, p) ? 0 : p.scratch;
}

template <int D, bool F32OUT> static int attn_launch(const attn_args &a, const attn_plan &p, hipStream_t st) {
    if (a.chunk_blocks) attn_mixed_kernel<D, F32OUT><<<dim3((unsigned)(a.chunk_blocks + a.few_blocks)), dim3(256 * chunk_groups(D)), 0, st>>>(a);
    else attn_few_kernel<D, F32OUT><<<dim3((unsigned)a.few_blocks), dim3(256), 0, st>>>(a);
    const int rc = SPY_LAUNCH_RC();
    return rc ? rc : spy_attn_join(a, p, D, F32OUT, st);
}

extern "C" int spy_hip_paged_attention(void *stream, const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_tensor *v_pages, const spy_hip_tensor *out,
                                       const spy_hip_paged_batch *batch, float scale, int32_t causal, int32_t window, void *scratch, size_t scratch_bytes) {
    SPY_CHECK_ARG(q && k_pages && v_pages && out);
    attn_plan p;
    attn_args a;
    int rc = attn_make_plan(q, k_pages, batch, false, p);
    if (!rc) rc = attn_check(q, k_pages, nullptr, v_pages, nullptr, out, batch, scale, causal, window, p.scratch, scratch, scratch_bytes, a);
    if (rc) return rc;
    attn_use_plan(p, scratch, a);
    hipStream_t st = (hipStream_t)stream;
    const int64_t hd = k_pages->ne[0];
    const bool f32 = out->type == SPY_HIP_F32;
    if (hd == 64) return f32 ? attn_launch<64, true>(a, p, st) : attn_launch<64, false>(a, p, st);
    if (hd == 128) return f32 ? attn_launch<128, true>(a, p, st) : attn_launch<128, false>(a, p, st);
    return f32 ? attn_launch<256, true>(a, p, st) : attn_launch<256, false>(a, p, st);
}
