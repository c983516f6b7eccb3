// Attention of sequences that begin alike: the plan of a call, and the launch that adds up its pieces (the first launch: paged_shared.cuh).
#include "paged_shared.cuh"

// A row and head of the output: D / 4 lanes, the heads of a wave of one row.  PARTS: so many waves of the workgroup share the pieces of the same heads.  Latency, and what the first launch wrote:
// up to eight pieces of o (two by a wave alone) are requested at a time, the first before the weights are worked out.  A wave for four times the heads took
// 16 us instead of 15 for 965 rows.
template <int D, bool F32OUT, int PARTS> __global__ __launch_bounds__(256) void attn_shared_join_kernel(attn_more a, int waves) {
    constexpr int L = D / 4, HEADS = 64 / L, AHEAD = PARTS == 1 ? 2 : L / PARTS < 8 ? L / PARTS : 8;        // lanes to a head, heads to a wave, pieces requested at a time
    static_assert(L % (PARTS * AHEAD) == 0);                               // whole turns for the weights that the lanes of a head have
    __shared__ v4f s_v[4][64];
    const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % PARTS, wave = __builtin_amdgcn_readfirstlane((blockIdx.x * 4 + (threadIdx.x >> 6)) / PARTS), lane = threadIdx.x & 63;
    const int n_head = a.G * a.group, row = wave / waves, h = (wave - row * waves) * HEADS + lane / L, at = lane % L, hq = min(h, n_head - 1);
    int n_common = 0, n = 0;
    if (row < a.b.n_row) {
        int row1, kv;
        const int s = row_sequence(a.b, row, lane, row1, kv);
        if (s >= 0) {
            pg_span all;
            const pg_span sq = pg_own(a.b, a.groups, s, nullptr, &all);
            // pieces of the keys in common, and of the row's own: as the first launch shares them out
            const auto pieces_of = [&](const row_tile &rt, bool few, int few_split, int chunk_split) {
                const int n_tile = few ? (rt.end() - (rt.lo_any() & ~31) + 31) >> 5 : (rt.end() - (rt.lo_any() & ~63) + 63) >> 6, split = few ? few_split : chunk_split;
                return n_tile > 0 ? (n_tile + split - 1) / split : 0;
            };
            if (sq.ok && row >= sq.row0) {
                if (all.ok) {
                    const bool few = all.n_new * a.group <= a.few;
                    n_common = pieces_of(row_tile(a, all, 0, few ? 16 : CHUNK_ROWS, true), few, a.common.few_split, a.common.chunk_split);
                }
                const bool few = sq.n_new * a.group <= a.few;
                const int r = (row - sq.row0) * a.group + hq % a.group;
                n = n_common + pieces_of(row_tile(a, sq, few ? 0 : r / CHUNK_ROWS, few ? 16 : CHUNK_ROWS, false), few, a.few_split, a.chunk_split);
            } else n = -1;
        } else n = -1;
    } else n = -1;                                                         // left alone
    const int64_t first = ((int64_t)min(row, a.b.n_row - 1) * n_head + hq) * a.slots;
    const auto slot = [&](int p) { p = max(min(p, n - 1), 0); return first + (p < n_common ? p : a.own_slot + p - n_common); };
    const auto piece = [&](int i) { return part + PARTS * i; };            // the wave's i-th
    // (heads of a wave may have different numbers of pieces: loops end for all of them together)
    v4f x[AHEAD];
    const auto request = [&](int i) {
#pragma unroll
        for (int j = 0; j < AHEAD; j++) if (piece(i + j) < n) x[j] = *(const v4f *)(a.part_o + slot(piece(i + j)) * D + 4 * at);
    };
    v4f v = {0, 0, 0, 0};
    float top = -INFINITY, sum = 0.0f;
    if (__any(n > 0)) {
        float2 ml = *(const float2 *)(a.part_ml + 2 * slot(at));
        request(0);
        for (int p = at; __any(p < n); p += L) if (p < n) top = fmaxf(top, p == at ? ml.x : a.part_ml[2 * slot(p)]);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, SPY_WAVE));
        const float base = top == -INFINITY ? 0.0f : top;
        for (int p0 = 0; __any(p0 < n); p0 += L) {                         // pieces p0 .. p0 + L - 1, a lane the weight of one
            if (p0) ml = *(const float2 *)(a.part_ml + 2 * slot(p0 + at));
            const float w = p0 + at < n ? above_0(exp2_(ml.x - base)) : 0.0f;      // (infinities stay: what is not above 2^-126 of a larger part adds nothing)
            sum += p0 + at < n ? w * ml.y : 0.0f;
            for (int i = p0 / PARTS; i < (p0 + L) / PARTS && __any(piece(i) < n); i += AHEAD) {
                if (i) request(i);
#pragma unroll
                for (int j = 0; j < AHEAD; j++) {
                    const float wj = __shfl(w, lane - at + (piece(i + j) - p0) % L, SPY_WAVE);
                    if (piece(i + j) < n) v += wj * x[j];
                }
            }
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, SPY_WAVE);
    }
    if constexpr (PARTS > 1) {
        s_v[threadIdx.x >> 6][lane] = v;
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int p = 1; p < PARTS; p++) v += s_v[(threadIdx.x >> 6) + p][lane];
    }
    if (h >= n_head || n < 0) return;
    const bool none = top == -INFINITY && sum == 0.0f;                     // sees no key
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = none ? 0.0f : v[k] / sum;
    uint8_t *dst = a.out + (int64_t)row * a.o_t + (int64_t)hq * a.o_h;
    if (F32OUT) *(v4f *)(dst + at * 16) = v;
    else *(uint2 *)(dst + at * 8) = make_uint2(f2h(v[0]) | (uint32_t)f2h(v[1]) << 16, f2h(v[2]) | (uint32_t)f2h(v[3]) << 16);
}

template <int D, bool F32OUT> static int attn_shared_join(const attn_more &a, hipStream_t st) {
    const int heads = 256 / D, waves = (a.G * a.group + heads - 1) / heads;        // heads of a wave; waves of a row
    const int64_t all = (int64_t)a.b.n_row * waves;
    // Pieces that a row may be expected to have: those of chunks where the batch may bring them.  32 rows of 32 heads with 30 pieces each 14.5 us by a wave, 6.6 by four; 965 rows with two 16 and 42.
    const int pieces = (a.common.chunk_blocks ? a.common.chunk_pieces : a.common.few_pieces) + (a.chunk_blocks ? a.chunk_pieces : a.few_pieces);
    if (pieces > 8 && all <= 4096) attn_shared_join_kernel<D, F32OUT, 4><<<dim3((unsigned)all), dim3(256), 0, st>>>(a, waves);
    else attn_shared_join_kernel<D, F32OUT, 1><<<dim3((unsigned)((all + 3) / 4)), dim3(256), 0, st>>>(a, waves);
    return SPY_LAUNCH_RC();
}

// Own keys much as attn_make_plan shares them out; those in common the same way, with groups for sequences.  Chunks: a workgroup to a compute unit (one term of a probability in all: 64 requests behind four prompts of 8000 tokens, 32 behind one of
// 20000 in 8 bits, and 965 rows behind 2000: 63, 43 and 86 us; two workgroups 72, 51 and 91: more pieces to write and to join); few rows three (61.0 us for the first; six: 63.1).
struct shared_plan { attn_plan own, common; int64_t slots, own_slot; size_t ml_bytes, scratch; };
static int attn_make_shared_plan(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *b, const spy_hip_paged_prefix *x, shared_plan &p) {
    SPY_CHECK_ARG(q && k_pages && q->ne[1] > 0 && q->ne[1] <= 65535 && q->ne[2] > 0 && q->ne[2] < (1 << 28));
    int rc = pg_check_batch(b);
    if (!rc) rc = k_pages->type == SPY_HIP_I8 ? pg_check_pages_q8(k_pages, 1) : pg_check_pages(k_pages, 1);
    if (rc) return rc;
    SPY_CHECK_ARG(x && x->n_group > 0 && x->n_group <= (1 << 20) && x->max_rows > 0 && x->max_rows <= (1 << 28) && x->max_prefix > 0 && x->max_prefix <= (1 << 30));
    SPY_CHECK_ARG(x->seq_start && x->length && (((uintptr_t)x->seq_start | (uintptr_t)x->length) & 3) == 0);
    const int64_t G = k_pages->ne[2], H = q->ne[1], hd = k_pages->ne[0], n_row = q->ne[2];
    SPY_CHECK_ARG(G <= 65535 && H % G == 0);
    const int64_t group = H / G, cu = spy_num_cu();
    // Every row has places for the pieces of either kind of tile: those of few rows, of which there may be many, are no more than take 128 MB, or four
    // (2048 rows of 32 heads on up to 30000 keys: 0.27 GB of scratch instead of 1.6; a chunk of 2048 tokens and eight single ones behind 4000, 32 heads to 8: 270 us instead of 280)
    const int64_t fit = (128ll << 20) / (n_row * H * hd * 4), room = fit < 4 ? 4 : fit;
    const auto share = [&](attn_plan &a, int64_t count, int64_t rows, int64_t keys) {
        const int64_t most = (rows < n_row ? rows : n_row) * group, tiles = ((keys + 31) / 32 + 1);
        a.few = FEW_ROWS;
        a.few_units = count * G;
        attn_share(a.few_units, tiles, 3 * cu, 8, a.few_split, a.few_pieces);
        if (a.few_pieces > room) {
            a.few_split = ((tiles + room - 1) / room + 3) / 4 * 4;
            a.few_pieces = (tiles + a.few_split - 1) / a.few_split;
        }
        a.chunk_tiles = a.chunk_units = 0; a.chunk_split = a.chunk_pieces = 1;
        if (most <= FEW_ROWS) return;
        const int64_t each = (most + CHUNK_ROWS - 1) / CHUNK_ROWS, all = n_row * group / CHUNK_ROWS + count;
        a.chunk_tiles = each * count < all ? each * count : all;
        a.chunk_units = a.chunk_tiles * G;
        const int64_t key_tiles = (keys + 63) / 64 + (&a == &p.own), n = (cu + a.chunk_units - 1) / a.chunk_units;
        a.chunk_split = n == 1 ? key_tiles : (key_tiles + n - 1) / n;
        if (a.chunk_split < 8) a.chunk_split = 8;
        a.chunk_pieces = (key_tiles + a.chunk_split - 1) / a.chunk_split;
    };
    share(p.own, b->n_seq, b->max_new, b->max_kv);
    share(p.common, x->n_group, x->max_rows, x->max_prefix);
    const auto most = [](int64_t u, int64_t v) { return u > v ? u : v; };
    p.own_slot = most(p.common.few_pieces, p.common.chunk_pieces);
    p.slots = p.own_slot + most(p.own.few_pieces, p.own.chunk_pieces);
    const auto threads = [&](int64_t blocks) { return blocks * 256 < (1ll << 32); };
    SPY_CHECK_ARG(threads(p.own.few_units * p.own.few_pieces + p.own.chunk_units * p.own.chunk_pieces + p.common.few_units * p.common.few_pieces + p.common.chunk_units * p.common.chunk_pieces));
    SPY_CHECK_ARG(n_row * (H + 3) * hd < (1ll << 32) && n_row * H < (1ll << 31));              // ... and of the second
    p.ml_bytes = ((size_t)(n_row * H * p.slots) * 8 + 255) / 256 * 256;
    p.scratch = p.ml_bytes + (size_t)(n_row * H * p.slots * hd) * 4;
    return 0;
}

extern "C" size_t spy_hip_paged_attention_shared_scratch_size(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *batch, const spy_hip_paged_prefix *prefix) {
    shared_plan p;
    return attn_make_shared_plan(q, k_pages, batch, prefix, p) ? 0 : p.scratch;
}

extern "C" int spy_hip_paged_attention_shared(void *stream, const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_tensor *k_scales, const spy_hip_tensor *v_pages,
                                              const spy_hip_tensor *v_scales, const spy_hip_tensor *out, const spy_hip_paged_batch *batch, const spy_hip_paged_prefix *prefix, float scale, void *scratch,
                                              size_t scratch_bytes) {
    SPY_CHECK_ARG(q && k_pages && v_pages && out);
    SPY_CHECK_ARG((k_pages->type == SPY_HIP_I8) == (k_scales != nullptr) && (k_scales != nullptr) == (v_scales != nullptr));
    shared_plan p;
    attn_more a = {};
    int rc = attn_make_shared_plan(q, k_pages, batch, prefix, p);
    if (!rc) rc = attn_check(q, k_pages, k_scales, v_pages, v_scales, out, batch, scale, 1, 0, p.scratch, scratch, scratch_bytes, a);
    if (rc) return rc;
    attn_use_plan(p.own, nullptr, a);
    attn_use_scales(k_scales, v_scales, a);
    a.few_part = a.chunk_part = nullptr;
    a.groups.seq_start = prefix->seq_start; a.groups.length = prefix->length;
    a.groups.n_group = prefix->n_group; a.groups.max_rows = prefix->max_rows; a.groups.max_common = prefix->max_prefix;
    a.common.few_split = (int)p.common.few_split; a.common.few_pieces = (int)p.common.few_pieces; a.common.few_blocks = (int)(p.common.few_units * p.common.few_pieces);
    a.common.chunk_tiles = (int)p.common.chunk_tiles; a.common.chunk_split = (int)p.common.chunk_split; a.common.chunk_pieces = (int)p.common.chunk_pieces;
    a.common.chunk_blocks = (int)(p.common.chunk_units * p.common.chunk_pieces);
    a.part_ml = (float *)scratch; a.part_o = (float *)((uint8_t *)scratch + p.ml_bytes);
    a.slots = (int)p.slots; a.own_slot = (int)p.own_slot;
    hipStream_t st = (hipStream_t)stream;
    const int64_t hd = k_pages->ne[0];
    const bool f32 = out->type == SPY_HIP_F32;
    const bool two = f32 || (int64_t)batch->max_new * a.group <= a.few;    // (no sequence of many rows: two terms for all)
    rc = k_scales ? spy_attn_shared_q8(a, hd, two, st) : attn_shared_launch<ATTN_SHARED>(a, hd, two, st);
    if (rc) return rc;
    if (hd == 64) return f32 ? attn_shared_join<64, true>(a, st) : attn_shared_join<64, false>(a, st);
    if (hd == 128) return f32 ? attn_shared_join<128, true>(a, st) : attn_shared_join<128, false>(a, st);
    return f32 ? attn_shared_join<256, true>(a, st) : attn_shared_join<256, false>(a, st);
}
