// Tiles of 16 rows over pages of 8 bits: attn_few of paged_attn.cuh with fp16(d * q) for the elements of K and V, the same sums in the same order.
//
// A tile of 32 keys goes from memory to LDS as it lies there, by 16 bytes a lane of rows that follow each other, and from LDS to the operands of the matrix instruction: an operand takes 8 bytes from
// each of 16 rows, and loads of such pieces from memory, which the vector cache takes a few bytes at a time (744 lookups a tile), took as long as all else (64 requests of up to 8000 tokens, 32 heads to 8, 128 wide:
// 171 us; by way of LDS 144).  Each wave has a tile of its own and waits for no other before the end; the next tile's K is requested when this one's is read, its V when this one's is.
// Bound by memory, 4.65 TB/s there; one request of 4096 tokens and 32 heads 15.7 us with the second launch, of which 11 are the chain from lengths to the last sum.  With two whole tiles for a wave, 16.2 and
// 143 us, and 256 wide, where only one wave has room on a SIMD then, 177 us for 32 requests instead of 154 (64 wide, 24 heads to 8: 82.7 and 79.4).
#pragma once

#include "paged_attn.cuh"

template <int D, int WAVES> struct few_q8_shared {
    static constexpr int K = 32 * D, V = 32 * D, KD = 2 * D, DS = 4 * D;                              // bytes: rows of K, [half of the keys][dimension] of V^T; scales: of K, of both
    union {
        __attribute__((aligned(1024))) uint8_t tile[WAVES][K + V + 2 * DS];                           // (the scales: this tile's and the next one's)
        few_shared<D, WAVES> end;
    };
};

template <int N> static __device__ __forceinline__ void landed_but() { asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory"); }

template <int D, bool F32OUT, int WAVES, int MODE> static __device__ __forceinline__ void attn_few_q8(const attn_more &a, few_q8_shared<D, WAVES> &sh, int block, bool common = false) {
    constexpr bool SHARED = MODE & ATTN_SHARED;
    constexpr int KS = D / 32, DT = D / 16, NI = D / 32;                   // steps of the scores, output tiles, requests for K (and for V) of a tile
    typedef few_q8_shared<D, WAVES> lay;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, quarter = lane >> 4;
    int n_unit = a.b.n_seq, split = a.few_split;
    if constexpr (SHARED) if (common) { n_unit = a.groups.n_group; split = a.common.few_split; }
    const int units = n_unit * a.G, piece = block / units, unit = block - piece * units, which = unit / a.G, head = unit - which * a.G;
    const auto sq = [&] {
        if constexpr (SHARED) return pg_span_of(a.b, a.groups, which, common, a.err);
        else return pg_sequence(a.b, which, a.err);
    }();
    if (!sq.ok) return;
    const row_tile rt = [&] {
        if constexpr (SHARED) return row_tile(a, sq, 0, 16, common);
        else return row_tile(a, sq, 0, 16);
    }();
    int s = which;                                                         // whose pages
    if constexpr (SHARED) s = sq.s;
    if (rt.rows > a.few) return;
    const int rows = rt.rows, r = min(n, rows - 1), token = r / a.group, hq = head * a.group + (r - token * a.group);
    const int hi = rt.hi(token), lo = rt.lo(token), hi_all = alone(rt.hi_all()), lo_all = alone(rt.lo_all()), begin = alone(rt.lo_any() & ~31), end = alone(rt.end());
    const int n_tile = max((end - begin + 31) >> 5, 0);
    if ((SHARED || piece > 0) && piece * split >= n_tile) return;
    const int stop = alone(min((piece + 1) * split, n_tile)), first = alone(piece * split + wave);
    const bool whole = !SHARED && n_tile <= split;

    const uint8_t *qrow = a.q + (int64_t)(sq.row0 + token) * a.q_t + (int64_t)hq * a.q_h;
    v8h fq[KS];
#pragma unroll
    for (int k = 0; k < KS; k++) fq[k] = halves(*(const uint4 *)(qrow + (32 * k + 8 * quarter) * 2));
    const int32_t *table = alone(a.b.pages + (int64_t)s * a.b.page_stride);
    const int plog = alone(a.b.page_log2), pmask = alone((1 << plog) - 1), last = alone((sq.kv - 1) >> plog), any_from = alone(rt.lo_any());
    const uint32_t n_page = alone((uint32_t)a.b.n_page), kp_p = alone((uint32_t)a.kp_p), kp_g = alone((uint32_t)a.kp_g), vp_d = alone((uint32_t)a.vp_d), vp_g = alone((uint32_t)a.vp_g), vs_b = alone((uint32_t)a.vs_b);
    const uint32_t ks_g = alone((uint32_t)a.ks_g), vs_g = alone((uint32_t)a.vs_g);
    const uint8_t *const kp = alone(a.kp + (int64_t)head * a.kp_h), *const vp = alone(a.vp + (int64_t)head * a.vp_h), *const ks = alone(a.ks + (int64_t)head * a.ks_h),
                  *const vs = alone(a.vs + (int64_t)head * a.vs_h);
    int *const err = alone(a.err);
    const float c = a.c;
    struct page_pair { uint32_t first, second; };                          // of the tile's two groups of 16 keys
    const auto pages_of = [&](int kt) {
        const int kb = begin + 32 * min(kt, stop - 1);
        return page_pair{(uint32_t)pg_entry(table, min(kb >> plog, last)), (uint32_t)pg_entry(table, min((kb + 16) >> plog, last))};
    };

    // A row of K in LDS has its 16-byte pieces at their index xor swizzle(row), so that the 16 rows of an operand lie in different banks (they are keys 8 (i / 4) + 4 t + i % 4)
    const auto swizzle = [](int row) { return D == 256 ? (row & 3) | row >> 3 << 2 : D == 128 ? (row >> 1 & 1) | row >> 3 << 1 : row >> 3; };
    const uint32_t lds = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)sh.tile[wave]);
    uint32_t koff[NI];                                                     // request i: 1024 / D rows, one after the other; from the first of the group of 16 on
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int row = i * (1024 / D) + lane / (D / 16);
        koff[i] = (row & 15) * kp_p + (((lane % (D / 16)) ^ swizzle(row)) * 16);
    }
    const uint32_t voff = lane * vp_d;                                     // request i: 64 dimensions of 16 keys
    // scales: the first D / 8 lanes have K's, which lie together for the 16 keys of a group, the next V's, 8 keys a lane; `d_second`: of the second group of 16 keys
    const bool d_v = lane >= D / 8;
    const int d_j = d_v ? lane - D / 8 : lane;
    const bool d_second = d_v ? d_j & 2 : 16 * d_j >= D;
    const uint32_t d_unit = d_v ? 2 : D / 16, d_step = d_v ? vs_g : ks_g;  // bytes of a position, of a page
    const uint8_t *const d_base = d_v ? vs + (uint64_t)(d_j >> 2) * vs_b + (d_j & 1) * 16 + (d_second ? 16 & pmask : 0) * 2 : ks + 16 * d_j % D + (d_second ? 16 & pmask : 0) * (D / 16);
    const auto present = [&](uint32_t page) { return uniform(page < n_page ? page : 0); };
    const auto ask_k = [&](int kt, page_pair g, uint32_t buf) {            // K, and the scales to the buffer `buf` bytes behind the first
        const int kb = begin + 32 * kt;
        const uint32_t pg[2] = {present(g.first), present(g.second)};
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int q = i * (1024 / D) / 16;                             // group of 16 keys
            to_lds(uniform(kp + (uint64_t)pg[q] * kp_g + (uint64_t)((kb + 16 * q) & pmask) * kp_p), koff[i], uniform(lds + i * 1024), 1);
        }
        if (lane < D / 4) to_lds(d_base + (uint64_t)(d_second ? pg[1] : pg[0]) * d_step + (kb & pmask) * d_unit, uniform(lds + buf + lay::K + lay::V), 1);
    };
    const auto ask_v = [&](int kt, page_pair g) {
        const int kb = begin + 32 * kt;
        const uint32_t pg[2] = {present(g.first), present(g.second)};
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int q = i / (D / 64), d = i % (D / 64) * 64;
            to_lds(uniform(vp + (uint64_t)pg[q] * vp_g + ((kb + 16 * q) & pmask) + (uint64_t)d * vp_d), voff, uniform(lds + lay::K + i * 1024), 1);
        }
    };
    constexpr int ASKED_K = NI + 1, ASKED_V = NI;

    const auto v_values = [&](int kt, page_pair g, int d) {                // as they lie in memory, for the walk that counts what is not finite
        const uint32_t page = quarter & 2 ? g.second : g.first;
        const int at = (begin + 32 * kt + 8 * quarter) & pmask;
        const uint64_t p = page < n_page ? page : 0;
        return dequantized(*(const uint2 *)(vp + p * vp_g + (uint64_t)(16 * d + n) * vp_d + at), *(const v8h *)(vs + p * vs_g + (uint64_t)(d >> 1) * vs_b + at * 2));
    };

    float m, l;
    v4f o[DT];
    bool unbounded = false;
    uint32_t large = 0;
    // Values are bounded by their scales where these are below 512: in tiles that a mask, a missing page or the end of the cache touches, the scales of positions that the cache has not are taken as 0,
    // and where others are larger, infinite or NaN (to `large`), all is done once more, `careful`ly, by the values themselves.
    const auto walk = [&](auto careful_) {
        constexpr bool CAREFUL = careful_;
        m = -INFINITY; l = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = v4f{0, 0, 0, 0};
        page_pair pg = {0, 0};
        if (first < stop) {
            pg = pages_of(first);
            ask_k(first, pg, 0);
            ask_v(first, pg);
        }
        uint32_t buf = 0;
        for (int kt = first; kt < stop; kt += WAVES) {
            const page_pair next = pages_of(kt + WAVES);
            const int kb = begin + 32 * kt, vk = kb + 8 * quarter;
            const bool vbad = (quarter & 2 ? pg.second : pg.first) >= n_page;
            const bool more = kt + WAVES < stop;
            landed_but<ASKED_V>();                                         // K is there, V need not be
            const uint8_t *const tile = sh.tile[wave], *const scales = tile + lay::K + lay::V + buf;
            const int row = 8 * (n >> 2) + (n & 3);
            const uint8_t *const krow = tile + row * D + (quarter & 1) * 8, *const vcol = tile + lay::K + (quarter >> 1) * (16 * D) + n * 16 + (quarter & 1) * 8;
            const int kpiece = ((quarter >> 1) ^ swizzle(row)) * 16;
            typedef uint32_t k_scales __attribute__((ext_vector_type(KS / 2)));
            k_scales dk[2];
            uint4 dv[D / 32];
#pragma unroll
            for (int t = 0; t < 2; t++) dk[t] = *(const k_scales *)(scales + (row + 4 * t) * (D / 16));
            const auto k_piece = [&](int t, int k) { return dequantized(*(const uint2 *)(krow + 4 * t * D + (kpiece ^ k * 32)), all_of(dk[t][k / 2] >> (16 * (k & 1)))); };
            const auto v_piece = [&](int d) { return bits(dequantized(*(const uint2 *)(vcol + 256 * d), halves(dv[d / 2]))); };
            v4f x[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int t = 0; t < 2; t++) x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k_piece(t, k), fq[k], x[t], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < D / 32; d++) dv[d] = *(const uint4 *)(scales + lay::KD + d * 64 + quarter * 16);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // K is not read any more
            if (more) ask_k(kt + WAVES, next, buf ^ lay::DS);
            float e[8];                                                    // of this lane's query and keys vk ..
#pragma unroll
            for (int j = 0; j < 8; j++) e[j] = x[j >> 2][j & 3] * c;
            const bool masked = __any(kb + 32 > hi_all || kb < lo_all || vbad);
            const int there = vbad ? 0 : end - vk;                         // positions of this lane's eight that the cache has, for this tile's rows
            if (masked) {
#pragma unroll
                for (int j = 0; j < 8; j++) e[j] = vk + j >= lo && vk + j < hi && !vbad ? e[j] : -INFINITY;
                if (vbad && vk < end && vk + 8 > any_from && err) *err = 1;         // (a page before the window may be gone)
                if constexpr (!CAREFUL) {
                    const uint4 keep = first_of(make_uint4(~0u, ~0u, ~0u, ~0u), there);
#pragma unroll
                    for (int d = 0; d < D / 32; d++) {
                        dv[d] = make_uint4(dv[d].x & keep.x, dv[d].y & keep.y, dv[d].z & keep.z, dv[d].w & keep.w);
                        large |= (dv[d].x & dv[d].x << 1) | (dv[d].y & dv[d].y << 1) | (dv[d].z & dv[d].z << 1) | (dv[d].w & dv[d].w << 1);      // bit 14 of a half: 512 and more, infinite, NaN
                    }
                }
            }
            float top = e[0];
#pragma unroll
            for (int j = 1; j < 8; j++) top = fmaxf(top, e[j]);
            top = quad_reduce(top, [](float p, float q) { return fmaxf(p, q); });
            top = fmaxf(m, top - (fabsf(top) < 1e7f ? 15.0f : 7.0f));
            const float base = top == -INFINITY ? 0.0f : top, shrink = exp2_(m - base);
            m = top;
            float sum = 0.0f;
            v8h p, p2;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = exp2_(e[j] - base);
                sum += e[j];
                p[j] = (_Float16)e[j];
                p2[j] = (_Float16)(e[j] - (float)p[j]);
            }
            l = l * shrink + sum;
            if (more) landed_but<ASKED_K>();                               // V
            else landed_but<0>();
#pragma unroll
            for (int d = 0; d < DT; d++) {
                uint4 w = v_piece(d);
                if (CAREFUL && masked) w = bounded(first_of(w, there), unbounded);
                o[d] *= shrink;
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(w), p, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(w), p2, o[d], 0, 0, 0);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");             // nor V
            if (more) ask_v(kt + WAVES, next);
            buf ^= lay::DS;
            pg = next;
        }
    };
#pragma unroll
    for (int k = 0; k < KS; k++) asm volatile("" :: "v"(fq[k]));           // waited for here: in the loop the wait would be for the tiles ahead as well
    walk(std::false_type{});
    if (__any(large & 0x40004000u)) walk(std::true_type{});
    float most = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) most = larger(most, o[d][i]);
    if (__any(unbounded || !finite(most))) {
#pragma unroll
        for (int d = 0; d < DT; d++) {
#pragma unroll
            for (int i = 0; i < 4; i++) o[d][i] = finite(o[d][i]) ? o[d][i] : 0.0f;       // (of a row with a score of NaN or +inf: l is NaN)
#pragma nounroll
            for (int kind = 0; kind < 3; kind++) {
                v4f n_seen = {0, 0, 0, 0};
#pragma nounroll
                for (int kt = first; kt < stop; kt += WAVES) {
                    const page_pair g = pages_of(kt);
                    const int vk = begin + 32 * kt + 8 * quarter;
                    const bool vbad = (quarter & 2 ? g.second : g.first) >= n_page;
                    const uint4 w = first_of(bits(v_values(kt, g, d)), vbad ? 0 : end - vk);
                    uint32_t seen = 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) seen |= (uint32_t)(vk + j >= lo && vk + j < hi && !vbad) << j;
                    n_seen = __builtin_amdgcn_mfma_f32_16x16x32_f16(of_kind(w, kind), ones(seen), n_seen, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) if (n_seen[i] != 0.0f) o[d][i] += kind_value(kind);
            }
        }
    }
    __syncthreads();                                                       // the tiles are done with
    few_end<D, F32OUT, WAVES, MODE>(a, sh.end, sq, rows, head, unit, piece, whole, common, m, l, o);
}
