// Attention of a batch's new tokens over a cache in pages: MatMul(K, q) -> Softmax(mask, scale) -> MatMul(V^T, P) of the LLaMA graph (attention.cpp:25-302 in the
// Spy tree), per sequence and head, in one pass over the keys.
//
// For a query row i and the keys j that it sees: x_j = scale * q_i.K_j, out_i = sum_j e^(x_j - m) V_j / sum_j e^(x_j - m) for any m.  A wave walks its keys 32 at a
// time with a running m, l (the sum of the exponentials) and o (the weighted sum of V); when m grows, l and o are scaled to the new one.
// Waves, and workgroups that share a row's keys, add up their (m, l, o) the same way.
// Exponentials enter the product as fp16, or as two of them, which has whole precision from 2^-14 (the second one of a pair: where it is above that) up to 2^16.  So m lies below
// the largest x (in powers of two; 10 to 15): the exponentials go up to 2^15, and what a small one is off by, half a step of 2^-24, is 2^-35 of the largest at most.  (Beyond
// 10^7 a float's neighbours are 1 and more apart; from 7 below, m stays within 15 of the largest x however the difference rounds.)
// One fp16 term is taken for F16 outputs of many rows alone, where the second costs time: its 2^-11 of a probability is what the output is rounded by (512 tokens on 7680: 2.9e-4 of
// the outputs instead of 2.1e-4, 88 us instead of 112).
//
// Scores are taken as S^T = K Q^T: the accumulator layout of the matrix instruction then has one query per lane, so that a row's maximum and sum are in-lane but for
// two steps between the four lanes that share a query, and -- with the rows of K dealt to the instruction's rows in the right order -- a lane's own probabilities
// are what the next instruction, O^T = V^T P^T, wants from it.  P never leaves the registers; V^T pages give its other operand as 16 contiguous bytes.
#pragma once

#include "paged.cuh"

#include <type_traits>

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
    // Sequences of up to `few` rows: one tile of 16 per sequence and K/V head, key tiles (of 32) per workgroup, workgroups that share a row's keys at most.  The others:
    // tiles of CHUNK_ROWS rows over all sequences, key tiles (of 64).
    int few, few_split, few_pieces, few_blocks;
    int chunk_tiles, chunk_split, chunk_pieces, chunk_blocks;
    float *few_part, *chunk_part;        // (o, m, l) of the workgroups that share rows
    int *err;
};

#define CHUNK_ROWS 128

// Variants of the kernels beside the plain one: pages in 8 bits, and sequences in groups that begin alike
enum { ATTN_PLAIN = 0, ATTN_Q8 = 1, ATTN_SHARED = 2 };
struct attn_shares { int few_split, few_pieces, few_blocks, chunk_tiles, chunk_split, chunk_pieces, chunk_blocks; };
struct attn_more : attn_args {
    const uint8_t *ks, *vs;              // scales of the pages; strides in bytes: K, head and page; V, block, head and page
    int64_t ks_h, ks_g, vs_b, vs_h, vs_g;
    // Groups: what their sequences have in common is attended to by all their rows together, as one sequence would, and the rest by each sequence as ever.  `common`: how the keys
    // in common are shared out; the fields of attn_args are for the rest.  Every row leaves (o, m, l) of its pieces behind: those in common first, `slots` for a row and head in all.
    pg_groups groups;
    attn_shares common;
    float *part_o, *part_ml;
    int slots, own_slot;
};
template <int MODE> using attn_args_of = std::conditional_t<MODE == ATTN_PLAIN, attn_args, attn_more>;

// Rows of a tile: the query rows are (new token, query head of the group) pairs, token by token.  Which keys they see: a token t those in lo(t) .. hi(t) - 1.
struct row_tile {
    int rows, r0, n_row;                 // of the sequence and K/V head; first of the tile; in the tile
    int past;                            // position of the sequence's token 0; negative where the cache holds less than the new tokens
    int group, kv, causal, window, from; // from: no row sees a key before it
    __device__ __forceinline__ row_tile(const attn_args &a, const pg_seq &q, int tile, int per) {
        rows = q.n_new * a.group; r0 = tile * per; n_row = min(per, rows - r0);
        past = q.kv - q.n_new; group = a.group; kv = q.kv; causal = a.causal; window = a.window; from = 0;
    }
    __device__ __forceinline__ row_tile(const attn_more &a, const pg_span &q, int tile, int per, bool common) : row_tile((const attn_args &)a, q, tile, per) {
        causal = !common; window = 0; from = q.from;
    }
    __device__ __forceinline__ int hi(int t) const { return causal ? max(past + t + 1, 0) : kv; }
    __device__ __forceinline__ int lo(int t) const { return window > 0 ? max(past + t - window + 1, 0) : from; }
    __device__ __forceinline__ int first() const { return r0 / group; }
    __device__ __forceinline__ int last() const { return (r0 + n_row - 1) / group; }
    __device__ __forceinline__ int hi_all() const { return hi(first()); }           // every row sees lo_all .. hi_all - 1
    __device__ __forceinline__ int lo_all() const { return lo(last()); }
    __device__ __forceinline__ int end() const { return hi(last()); }               // no row sees a key outside lo_any .. end - 1
    __device__ __forceinline__ int lo_any() const { return lo(first()); }
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
// Eight whole numbers of 8 bits times their scales, each product rounded once.  b + 128 as the low bits of 1024 + b + 128, from which 1152 is taken: exact.
static __device__ __forceinline__ v8h dequantized(uint2 w, v8h d) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const uint32_t a = w.x ^ 0x80808080u, b = w.y ^ 0x80808080u;
    const uint32_t v[4] = {__builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u),
                           __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
    v8h r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const v2h x = (__builtin_bit_cast(v2h, v[i]) - (v2h){(_Float16)1152, (_Float16)1152}) * (v2h){d[2 * i], d[2 * i + 1]};
        r[2 * i] = x[0]; r[2 * i + 1] = x[1];
    }
    return r;
}
static __device__ __forceinline__ v8h all_of(uint32_t half) {                    // the low half, eight times
    const uint32_t d = __builtin_amdgcn_perm(half, half, 0x01000100u);
    return halves(make_uint4(d, d, d, d));
}
static __device__ __forceinline__ uint4 bits(v8h v) { return __builtin_bit_cast(uint4, v); }
// the first n of eight fp16 values (n <= 0: none), the others 0
static __device__ __forceinline__ uint4 first_of(uint4 w, int n) {
    uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] &= n >= 2 * i + 2 ? 0xFFFFFFFFu : n == 2 * i + 1 ? 0xFFFFu : 0u;
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// infinities and NaN among eight fp16 values taken as 0; any: whether there were some
static __device__ __forceinline__ uint4 bounded(uint4 w, bool &any) {
    uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool lo = (v[i] & 0x7C00u) == 0x7C00u, hi = (v[i] & 0x7C000000u) == 0x7C000000u;
        any |= lo | hi;
        v[i] = lo ? v[i] & 0xFFFF0000u : v[i];
        v[i] = hi ? v[i] & 0x0000FFFFu : v[i];
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}
// Where V holds infinities or NaN at positions that some rows of a tile see and others do not, a probability of 0 would not keep them out of the others' outputs (0 times
// either is NaN), so the product takes 0 in their place there; and where all rows see them, what it makes of them depends on how a probability was rounded.  So where any
// were taken out, or an output is not finite, which of +inf, -inf and NaN a row sees in which dimension is counted after all, in one more walk over V, by the matrix
// instruction over indicators: w's elements that are of kind 0, 1, 2 as 1, the others as 0.
static __device__ __forceinline__ v8h of_kind(uint4 w, int kind) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t out = 0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t b = v[i] >> (16 * h) & 0xFFFFu;
            const bool is = kind == 2 ? (b & 0x7FFFu) > 0x7C00u : b == (kind ? 0xFC00u : 0x7C00u);
            out |= is ? 0x3C00u << (16 * h) : 0u;
        }
        r[i] = out;
    }
    return halves(make_uint4(r[0], r[1], r[2], r[3]));
}
// 1 for bit j set, 0 else
static __device__ __forceinline__ v8h ones(uint32_t bits) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = (bits >> (2 * i) & 1 ? 0x3C00u : 0u) | (bits >> (2 * i + 1) & 1 ? 0x3C000000u : 0u);
    return halves(make_uint4(r[0], r[1], r[2], r[3]));
}
static __device__ __forceinline__ float kind_value(int kind) { return kind == 2 ? NAN : kind ? -INFINITY : INFINITY; }
static __device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }
static __device__ __forceinline__ float larger(float top, float x) { return __builtin_elementwise_maximum(top, fabsf(x)); }       // NaN if either is; two of them are one instruction
// A factor from one m to another that leaves infinities infinite: what is not above 2^-126 of a larger part adds nothing to it, as with 0
static __device__ __forceinline__ float above_0(float f) { return fmaxf(f, 0x1p-126f); }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes per lane from memory to LDS, in lane order from byte `lds` (uniform) on; base uniform, or an address per lane.  Written as instructions so that the compiler does
// not wait for them at the next LDS read; landed() does.
// A base that a vector instruction has written may be read five instructions later: the compiler does not look into these.
// `there` 0: not requested.  (The branch is written out as well: as one of the compiler's it would part the instructions on either side into blocks of their own.)
static __device__ __forceinline__ void to_lds(const void *base, uint32_t off, uint32_t lds, uint32_t there) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 1\n\ts_cmp_eq_u32 %3, 0\n\ts_cbranch_scc1 .Lno%=\n\tglobal_load_lds_dwordx4 %1, %2\n.Lno%=:" :: "s"(lds), "v"(off), "s"(base), "s"(there) : "memory", "m0", "scc");
}
static __device__ __forceinline__ void to_lds(const void *addr, uint32_t lds, uint32_t there) {
    asm volatile("s_mov_b32 m0, %0\n\ts_cmp_eq_u32 %2, 0\n\ts_cbranch_scc1 .Lno%=\n\tglobal_load_lds_dwordx4 %1, off\n.Lno%=:" :: "s"(lds), "v"(addr), "s"(there) : "memory", "m0", "scc");
}
#pragma clang diagnostic pop
static __device__ __forceinline__ const uint8_t *uniform(const uint8_t *p) {
    const uint64_t v = (uint64_t)p;
    return (const uint8_t *)((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v));
}
static __device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
// Arguments are loaded sixteen registers at a time; where they live through the loop over the keys, the compiler runs out of scalar registers, keeps whole groups of
// sixteen in lanes of a vector register and moves all of one back for each value it needs: 158 of 378 vector instructions per tile.  So the loop's values are scalars
// of their own, and what is wanted after it is loaded again then (from the kernel's arguments, of which this struct is the first).
template <class Args> static __device__ __forceinline__ const __attribute__((address_space(4))) Args *args_again() {
    const __attribute__((address_space(4))) Args *p = (const __attribute__((address_space(4))) Args *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}
static __device__ __forceinline__ uint32_t alone(uint32_t v) {
    uint32_t r;
    asm volatile("s_mov_b32 %0, %1" : "=s"(r) : "s"(uniform(v)));
    return r;
}
static __device__ __forceinline__ int alone(int v) { return (int)alone((uint32_t)v); }
template <class T> static __device__ __forceinline__ T *alone(T *p) {
    const uint8_t *r;
    asm volatile("s_mov_b64 %0, %1" : "=s"(r) : "s"(uniform((const uint8_t *)p)));
    return (T *)r;
}
static __device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- 16 rows per workgroup: single tokens, and a few of them -------------------------------------------------------------------------
// A row is a new token and one of the query heads that share the K/V head: with a group of heads, or several new tokens, the keys are read once for all of them.
// Bound by the bytes of K and V.  The waves take tiles of 32 keys in turn, straight from memory into the registers of the matrix instruction: nothing is shared
// between waves before the end.  Measured: 64 requests of up to 4096 cached tokens (32 heads to 8, 128 wide, pages of 16) 125 us, 5.1 TB/s; 8 of up to 30000 (64 heads to 8)
// 135 us, 4.9 TB/s; one of 4096 (32 heads) 14 us, 4.8 TB/s, and 4.4 us for the join; 32 of up to 4096 (16 heads to 8, 256 wide, F32 outputs) 140 us, 4.7 TB/s.
template <int D, int WAVES> struct few_shared {
    static constexpr int HALF = D < 128 ? D : 128;
    float m[WAVES][16], l[WAVES][16];
    __attribute__((aligned(16))) float o[WAVES][16][HALF + 4];
};
// The waves' (m, l, o) to one: the output, or (o, m, l) of the piece
template <int D, bool F32OUT, int WAVES, int MODE, class Seq> static __device__ __forceinline__ void few_end(const attn_args_of<MODE> &a, few_shared<D, WAVES> &sh, const Seq &sq, int rows, int head, int unit,
                                                                                                             int piece, bool whole, bool common, float m, float l, v4f (&o)[D / 16]) {
    constexpr bool SHARED = MODE & ATTN_SHARED;
    constexpr int HALF = few_shared<D, WAVES>::HALF;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, quarter = lane >> 4;
    l = quad_reduce(l, [](float p, float q) { return p + q; });
    if (quarter == 0) { sh.m[wave][n] = m; sh.l[wave][n] = l; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; w++) top = fmaxf(top, sh.m[w][n]);
    const float shrink = above_0(exp2_(m - (top == -INFINITY ? 0.0f : top)));
    float *part = nullptr;
    if constexpr (!SHARED) part = a.few_part + ((int64_t)unit * a.few_pieces + piece) * 16 * (D + 2);
#pragma unroll
    for (int h = 0; h < D / HALF; h++) {
        if (h) __syncthreads();
#pragma unroll
        for (int d = 0; d < HALF / 16; d++) {
            const v4f v = o[h * (HALF / 16) + d] * shrink;
            *(v4f *)&sh.o[wave][n][16 * d + 4 * quarter] = v;
        }
        __syncthreads();
        for (int i = tid; i < 16 * (HALF / 4); i += 64 * WAVES) {
            const int row = i / (HALF / 4), d = (i - row * (HALF / 4)) * 4;
            v4f v = v4f{0, 0, 0, 0};
            float mx = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) { v += *(const v4f *)&sh.o[w][row][d]; mx = fmaxf(mx, sh.m[w][row]); }
            const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int w = 0; w < WAVES; w++) sum += sh.l[w][row] * exp2_(sh.m[w][row] - base);
            if (row >= rows) continue;
            const int dd = h * HALF + d;
            const int t = row / a.group, hh = head * a.group + (row - t * a.group);
            if constexpr (SHARED) {
                const int64_t at = ((int64_t)(sq.row0 + t) * (a.G * a.group) + hh) * a.slots + (common ? 0 : a.own_slot) + piece;
                *(v4f *)(a.part_o + at * D + dd) = v;
                if (dd == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(mx, sum);
            } else if (whole) {
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

// MODE: see above.  common: the block is one of the keys that the sequences of a group have in common (the groups stand for sequences then)
template <int D, bool F32OUT, int WAVES, int MODE = ATTN_PLAIN> static __device__ __forceinline__ void attn_few(const attn_args_of<MODE> &a, few_shared<D, WAVES> &sh, int block, bool common = false) {
    constexpr bool SHARED = MODE & ATTN_SHARED;
    constexpr int KS = D / 32, DT = D / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, quarter = lane >> 4;
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
    const int hi = rt.hi(token), lo = rt.lo(token), hi_all = rt.hi_all(), lo_all = rt.lo_all(), begin = rt.lo_any() & ~31, end = rt.end();
    const int n_tile = max((end - begin + 31) >> 5, 0);
    if ((SHARED || piece > 0) && piece * split >= n_tile) return;
    const int stop = min((piece + 1) * split, n_tile);
    const bool whole = !SHARED && n_tile <= split;

    const uint8_t *qrow = a.q + (int64_t)(sq.row0 + token) * a.q_t + (int64_t)hq * a.q_h;
    v8h fq[KS];
#pragma unroll
    for (int k = 0; k < KS; k++) fq[k] = halves(*(const uint4 *)(qrow + (32 * k + 8 * quarter) * 2));
    const int32_t *table = a.b.pages + (int64_t)s * a.b.page_stride;
    const int plog = a.b.page_log2, pmask = (1 << plog) - 1, last = (sq.kv - 1) >> plog;

    // Instruction row i of score tile t is key 8 (i / 4) + 4 t + i % 4: a lane's scores are then of keys 8 quarter + 4 t + 0 .. 3, as the product wants them.
    const uint8_t *kbase = a.kp + (int64_t)head * a.kp_h + (int64_t)(n & 3) * a.kp_p + quarter * 16, *vbase = a.vp + (int64_t)head * a.vp_h + (int64_t)n * a.vp_d;
    struct page_pair { int first, second; };                               // of the tile's two groups of 16 keys
    const auto pages_of = [&](int kt) {
        const int kb = begin + 32 * min(kt, stop - 1);
        return page_pair{pg_entry(table, min(kb >> plog, last)), pg_entry(table, min((kb + 16) >> plog, last))};
    };
    const auto missing = [&](int page) { return (uint32_t)page >= (uint32_t)a.b.n_page; };
    const auto place = [&](page_pair g, int q, int64_t step) {             // keys 8 q ..: their page
        const int page = q & 2 ? g.second : g.first;
        return (int64_t)(missing(page) ? 0 : page) * step;
    };
    uint4 fk[2][KS], fv[DT];
    const auto load_k = [&](int kt, page_pair g) {
        const uint8_t *kr = kbase + place(g, n >> 2, a.kp_g) + (int64_t)((begin + 32 * kt + 8 * (n >> 2)) & pmask) * a.kp_p;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int k = 0; k < KS; k++) fk[t][k] = *(const uint4 *)(kr + 4 * t * a.kp_p + k * 64);
    };
    const auto v_row = [&](int kt, page_pair g) { return vbase + place(g, quarter, a.vp_g) + (int64_t)((begin + 32 * kt + 8 * quarter) & pmask) * 2; };
    const auto load_v = [&](const uint8_t *vr) {
#pragma unroll
        for (int d = 0; d < DT; d++) fv[d] = *(const uint4 *)(vr + 16 * d * a.vp_d);
    };

    float m = -INFINITY, l = 0.0f;
    v4f o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = v4f{0, 0, 0, 0};
    bool unbounded = false;
    // K of the next tile is requested when this one's scores are done with the registers, V^T when the product is: memory always has a tile of each wave to fetch
    const int first = piece * split + wave;
    page_pair pg = {0, 0}, pg1 = {0, 0};
    if (first < stop) {
        pg = pages_of(first);
        pg1 = pages_of(first + WAVES);
        load_k(first, pg);
        load_v(v_row(first, pg));
    }
    for (int kt = first; kt < stop; kt += WAVES) {
        const page_pair pg2 = pages_of(kt + 2 * WAVES);
        const int kb = begin + 32 * kt, vk = kb + 8 * quarter;
        const bool vbad = missing(quarter & 2 ? pg.second : pg.first);
        v4f x[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            x[t] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < KS; k++) x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(fk[t][k]), fq[k], x[t], 0, 0, 0);
        }
        if (kt + WAVES < stop) load_k(kt + WAVES, pg1);
        float e[8];                                                        // of this lane's query and keys vk ..
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = x[j >> 2][j & 3] * a.c;
        const bool masked = __any(kb + 32 > hi_all || kb < lo_all || vbad);
        const int there = vbad ? 0 : end - vk;                             // positions of this lane's eight that the cache has, for this tile's rows
        if (masked) {
#pragma unroll
            for (int j = 0; j < 8; j++) e[j] = vk + j >= lo && vk + j < hi && !vbad ? e[j] : -INFINITY;
            if (vbad && vk < end && vk + 8 > rt.lo_any() && a.err) *a.err = 1;     // (a page before the window may be gone)
            // what lies behind the cache's last position is taken as 0, and so are infinities and NaN, which some rows may see and others not
#pragma unroll
            for (int d = 0; d < DT; d++) fv[d] = bounded(first_of(fv[d], there), unbounded);
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
            p2[j] = (_Float16)(e[j] - (float)p[j]);                        // (for F16 outputs as well: the second product takes no time beside the keys' arrival)
        }
        l = l * shrink + sum;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            o[d] *= shrink;
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(fv[d]), p, o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(fv[d]), p2, o[d], 0, 0, 0);
        }
        if (kt + WAVES < stop) load_v(v_row(kt + WAVES, pg1));
        pg = pg1; pg1 = pg2;
    }
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
                    const bool vbad = missing(quarter & 2 ? g.second : g.first);
                    const uint4 w = first_of(*(const uint4 *)(v_row(kt, g) + 16 * d * a.vp_d), vbad ? 0 : end - vk);
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
    few_end<D, F32OUT, WAVES, MODE>(a, sh, sq, rows, head, unit, piece, whole, common, m, l, o);
}

// ---- CHUNK_ROWS rows per workgroup: chunks of a prompt --------------------------------------------------------------------------------
// Bound by the matrix cores and the vector instructions of the softmax together: 64 keys by 32 rows take a wave (D = 128) 32 matrix instructions of 33 cycles, and some 200
// vector instructions of 4.7, 32 of them exponentials of 11; two waves of a SIMD need 4400 of the 5200 cycles that a step takes, since the step's barrier puts both into
// the same phase, where they want the same units.  Measured (128 wide, 32 heads): a prompt of 2048 tokens 55 us, 628 TFLOP/s of what its rows see, with F32 outputs (half as
// many matrix instructions again) 67; 512 tokens on 7680 87.5 us, 761 TFLOP/s, F32 112; 13 us of the former are spent outside the loop, by two workgroups one after the
// other.  16 heads of 256, 512 tokens on 3584: 64.5 us, F32 75.8.  Tried and not kept (where this had 57 and 91 us): the next tile's scores computed beside this one's
// exponentials in one instruction stream (58 and 91), a barrier for each group by itself (59 and 98), wave priorities (no difference).
// Four waves have 32 rows each; a second group of four has the same rows and every other tile of keys, so that a SIMD always has a second wave, to the end of a long row
// of keys, and the groups exchange halves of (m, l, o) at the end (one group of 256 rows would leave the short rows of a prompt's triangle without a second wave).
// (256-wide heads: one group, one wave per SIMD with 500 of its 512 registers in use.)  The 64 keys' K and V^T of a group lie in LDS,
// requested straight from memory one tile ahead into the other of two buffers.  An LDS row is a row of the matrix instruction's operand (K: instruction row i of 32 is key
// 16 (i / 16) + 8 (i / 4 % 2) + 4 (i / 8 % 2) + i % 4, so that a lane's scores are those of 8 keys that follow each other, as the product wants its
// probabilities); its 16-byte pieces are stored at their index xor a number of the row, so that the lanes of a read meet different banks.
typedef float v16f __attribute__((ext_vector_type(16)));

template <int D> static __device__ __forceinline__ int swizzle_k(int row) { return D == 64 ? (row >> 1 & 3) | (((row ^ row >> 3) & 1) << 2) : row & 15; }
static __device__ __forceinline__ int swizzle_v(int row) { return (row >> 1 & 3) | (((row ^ row >> 3) & 1) << 2); }

// over the two lanes l, l ^ 32
template <class Op> static __device__ __forceinline__ float pair_reduce(float v, Op op) {
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(h[0]), __uint_as_float(h[1]));
}

// Tile `left` of the sequences of many rows, one after the other: its sequence and its number there.  64 sequences per round; every lane the same.
static __device__ __forceinline__ int find_tile(const attn_args &a, int left, int &tile, int &count, pg_seq &sq) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < a.b.n_seq; base += 64) {
        int n = 0;
        pg_seq q = {0, 0, 0, false};
        if (base + lane < a.b.n_seq) {
            q = pg_sequence(a.b, base + lane, a.err);
            const int rows = q.ok ? q.n_new * a.group : 0;
            n = rows > a.few ? (rows + CHUNK_ROWS - 1) / CHUNK_ROWS : 0;
        }
        const int sum = (int)wave_scan((uint32_t)n);
        const unsigned long long past = __ballot(sum > left);
        if (past) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
            tile = left - __builtin_amdgcn_readlane(sum - n, at);
            count = __builtin_amdgcn_readlane(n, at);
            sq = {__builtin_amdgcn_readlane(q.row0, at), __builtin_amdgcn_readlane(q.n_new, at), __builtin_amdgcn_readlane(q.kv, at), true};
            return base + at;
        }
        left -= __builtin_amdgcn_readlane(sum, 63);
    }
    return -1;
}

// ... of what the sequences of groups have in common, or of their own keys
struct span_tile { pg_span sq; int tile, count; };
static __device__ __forceinline__ bool find_span(const attn_more &a, bool common, int left, span_tile &found) {
    pg_span &sq = found.sq;
    int &tile = found.tile, &count = found.count;
    if (!common) {
        const int s = find_tile(a, left, tile, count, sq);
        if (s >= 0) sq = pg_own(a.b, a.groups, s, a.err);
        return s >= 0 && sq.ok;
    }
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < a.groups.n_group; base += 64) {
        int n = 0;
        pg_span q = {};
        if (base + lane < a.groups.n_group) {
            const int g = base + lane;
            q = pg_group(a.b, a.groups, a.groups.seq_start[g], a.groups.seq_start[g + 1], a.groups.length[g], a.err);
            const int rows = q.ok ? q.n_new * a.group : 0;
            n = rows > a.few ? (rows + CHUNK_ROWS - 1) / CHUNK_ROWS : 0;
        }
        const int sum = (int)wave_scan((uint32_t)n);
        const unsigned long long past = __ballot(sum > left);
        if (past) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
            tile = left - __builtin_amdgcn_readlane(sum - n, at);
            count = __builtin_amdgcn_readlane(n, at);
            sq.row0 = __builtin_amdgcn_readlane(q.row0, at); sq.n_new = __builtin_amdgcn_readlane(q.n_new, at); sq.kv = __builtin_amdgcn_readlane(q.kv, at);
            sq.s = __builtin_amdgcn_readlane(q.s, at); sq.from = 0; sq.ok = true;
            return true;
        }
        left -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

static constexpr __host__ __device__ int chunk_groups(int D) { return D == 256 ? 1 : 2; }
template <int D> struct chunk_group { __attribute__((aligned(1024))) uint8_t k[2][64 * D * 2], v[2][64 * D * 2]; };
template <int D, int GROUPS = chunk_groups(D)> struct chunk_shared { chunk_group<D> group[GROUPS]; int unbounded; };
template <int D, int GROUPS = chunk_groups(D)> struct chunk_shared_q8 : chunk_shared<D, GROUPS> { __attribute__((aligned(16))) uint8_t scales[4 * GROUPS][D * 4]; };      // of V^T, a wave's own copy

// Q8: a tile's whole numbers come to registers two tiles ahead and go to LDS as fp16 values one tile ahead, beside the matrix instructions of the scores, which leave the vector units time for it (512 tokens on 7680, 32 heads
// to 8, 128 wide: 106 us; beside the products of their own tile 110 to 113).  The registers that takes are those of operands asked for ahead, half as many as with fp16 pages: as many, 256-wide heads keep 48 registers in memory
// (512 tokens on 3584, 16 heads to 8: 99 us instead of 84), and 128-wide ones are no faster (106.8).
// found: (sequences in groups) the block's tile
template <int D, bool F32OUT, int MODE = ATTN_PLAIN, int GROUPS = chunk_groups(D), class Shared = chunk_shared<D>> static __device__ __forceinline__ void attn_chunk(const attn_args_of<MODE> &a, Shared &shared, int block, bool common = false, const span_tile &found = {}) {
    constexpr bool Q8 = MODE & ATTN_Q8, SHARED = MODE & ATTN_SHARED;
    constexpr int ES = Q8 ? 1 : 2;                                         // bytes of an element in the pages
    constexpr int KS = D / 16, DT = D / 32, NI = D / 32;                   // steps of the scores, output tiles, requests of a wave for K (and for V) per tile
    constexpr int KC = D / 8, KR = 64 / KC;                                // 16-byte pieces of a K row, K rows per request
    static_assert(2 * KS == 4 * NI && 4 * DT == 4 * NI);                   // a request beside every fourth product, and every fourth step of the second product
    const int tid = threadIdx.x, lane = tid & 63, wave8 = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wave8 & 3, group = wave8 >> 2, n = lane & 31, half = lane >> 5;
    chunk_group<D> &sh = shared.group[group];
    // heads fastest: a head's tiles run on one XCD where the number of heads is a multiple of 8, and share its L2
    int per = a.chunk_tiles * a.G, split = a.chunk_split;
    if constexpr (SHARED) if (common) { per = a.common.chunk_tiles * a.G; split = a.common.chunk_split; }
    const int piece = block / per, unit = block - piece * per, head = unit % a.G;
    int tile, count, s;
    std::conditional_t<SHARED, pg_span, pg_seq> sq;
    if constexpr (SHARED) {
        sq = found.sq; tile = found.tile; count = found.count;
        s = sq.s;
    } else {
        s = find_tile(a, unit / a.G, tile, count, sq);
        if (s < 0) return;
    }
    tile = count - 1 - tile;                                               // late tiles, which see most keys, first
    const row_tile rt = [&] {
        if constexpr (SHARED) return row_tile(a, sq, tile, CHUNK_ROWS, common);
        else return row_tile(a, sq, tile, CHUNK_ROWS);
    }();
    const int lo_any = alone(rt.lo_any()), begin = lo_any & ~63, end = alone(rt.end()), n_tile = max((end - begin + 63) >> 6, 0);
    const int from = alone(piece * split), stop = alone(min(from + split, n_tile));
    if ((SHARED || piece > 0) && from >= n_tile) return;
    const bool whole = !SHARED && alone((int)(n_tile <= split));
    const int r = min(rt.r0 + wave * 32 + n, rt.rows - 1), token = r / a.group, hq = head * a.group + (r - token * a.group);
    const int hi = rt.hi(token), lo = rt.lo(token), hi_all = alone(rt.hi_all()), lo_all = alone(rt.lo_all());
    const int n_row = alone(rt.n_row), row0 = alone(sq.row0);
    const bool idle = wave * 32 >= n_row;                                  // waves without rows fetch, and compute nothing

    const int32_t *table = alone(a.b.pages + (int64_t)s * a.b.page_stride);
    const int plog = alone(a.b.page_log2), pmask = alone((1 << plog) - 1), last = alone(max(sq.kv - 1, 0) >> plog), n_page = alone(a.b.n_page);
    const uint32_t lds_k = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)sh.k[0] + wave * 1024),
                   lds_v = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)sh.v[0] + wave * 1024);

    // K request i of a wave: LDS rows KR (4 i + wave) .., which are keys of one group of 16.  V request: V^T rows 8 (4 i + wave) .., lane's piece: keys 8 vc .. of the tile.
    // Offsets inside a page are 32-bit numbers.
    const uint32_t kp_p = alone((uint32_t)a.kp_p), vp_d = alone((uint32_t)a.vp_d), kp_g = alone((uint32_t)a.kp_g), vp_g = alone((uint32_t)a.vp_g);
    uint32_t koff[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        const int row = KR * (4 * i + wave) + lane / KC;
        koff[i] = (8 * (row >> 2 & 1) + 4 * (row >> 3 & 1) + (row & 3)) * kp_p + (((lane % KC) ^ swizzle_k<D>(row)) * 8 * ES);
    }
    const int vrow = 8 * wave + (lane >> 3), vc = (lane & 7) ^ swizzle_v(vrow);
    const uint8_t *kbase = alone(a.kp + head * a.kp_h), *vbase = alone(a.vp + head * a.vp_h);
    int *const err = alone(a.err);
    // Pages of the tiles' groups of 16 keys: 64 groups, which are 16 tiles, in the lanes of a register, and bit g of `gone`: group g's is not there
    const auto entries_of = [&](int tile) __attribute__((always_inline)) { return ((const __attribute__((address_space(1))) int32_t *)table)[min((begin + 64 * (from + (tile & ~15)) + 16 * lane) >> plog, last)]; };
    uint64_t gone = 0;
    int entries = 0;
    const auto take_entries = [&](int fetched) __attribute__((always_inline)) {
        const bool absent = (uint32_t)fetched >= (uint32_t)n_page;
        gone = __ballot(absent);
        entries = absent ? 0 : fetched;
    };
    const int first_pages = entries_of(0);                                 // asked for before the queries, which are waited for later
    const float c = fabsf(a.c);
    v8h fq[KS];
    {
        const uint8_t *qrow = a.q + (int64_t)(sq.row0 + token) * a.q_t + (int64_t)hq * a.q_h;
        const uint32_t flip = a.c < 0.0f ? 0x80008000u : 0u;               // a negative scale: -q, so that the largest product is the largest score
#pragma unroll
        for (int k = 0; k < KS; k++) {
            uint4 w = *(const uint4 *)(qrow + (16 * k + 8 * half) * 2);
            w.x ^= flip; w.y ^= flip; w.z ^= flip; w.w ^= flip;
            fq[k] = halves(w);
        }
    }
    typedef int group_pages __attribute__((ext_vector_type(4)));           // (a struct's members, chosen from by the lane, would be put into memory)
    const auto pages_of = [&](int tile) __attribute__((always_inline)) {
        const int g = 4 * tile & 63;
        return group_pages{__builtin_amdgcn_readlane(entries, g), __builtin_amdgcn_readlane(entries, g + 1), __builtin_amdgcn_readlane(entries, g + 2), __builtin_amdgcn_readlane(entries, g + 3)};
    };
    const auto gone_of = [&](int tile) __attribute__((always_inline)) { return (int)(gone >> (4 * tile & 63)) & 15; };
    // Request i of NI; buf: bytes of the buffer behind the first
    const auto ask_k = [&](int kb, group_pages g, uint32_t buf, uint32_t there, int i) __attribute__((always_inline)) {
        const int q = D == 128 ? i : D == 256 ? i >> 1 : 2 * i + (wave >> 1);
        const uint32_t page = q & 2 ? (q & 1 ? g.w : g.z) : (q & 1 ? g.y : g.x);
        to_lds(uniform(kbase + (uint64_t)page * kp_g + ((kb + 16 * q) & pmask) * kp_p), koff[i], uniform(lds_k + buf + i * 4096), there);
    };
    const auto v_source = [&](int kb, group_pages g) __attribute__((always_inline)) {
        const uint32_t mine = vc & 4 ? (vc & 2 ? g.w : g.z) : (vc & 2 ? g.y : g.x);
        return vbase + (uint64_t)mine * vp_g + (((kb + 8 * vc) & pmask) * ES + vrow * vp_d);
    };
    const auto there_is = [&](int kt) {                                    // a tile kt
        uint32_t yes;
        // written out: the compiler drops the builtin, and then keeps the number in a vector register.  The register that it reads may not be written by the instruction before.
        asm("s_nop 1\n\tv_readfirstlane_b32 %0, %1" : "=s"(yes) : "v"((kt - stop) >> 31));
        return yes;
    };
    // Q8: a tile's pieces of this wave, those that the requests of a tile of fp16 would bring
    uint2 raw_k[Q8 ? NI : 1], raw_v[Q8 ? NI : 1];
    uint32_t raw_d[Q8 ? NI : 1];
    const uint8_t *ks = nullptr, *vs = nullptr;
    uint32_t ks_g = 0, vs_g = 0, vs_at = 0, lds_d = 0;
    if constexpr (Q8) {
        ks = alone(a.ks + head * a.ks_h); vs = alone(a.vs + head * a.vs_h);
        ks_g = alone((uint32_t)a.ks_g); vs_g = alone((uint32_t)a.vs_g);
        vs_at = (uint32_t)(lane >> 3) * (uint32_t)a.vs_b;                  // lane's piece of the scales: block lane / 8, keys 8 (lane % 8) .. of the tile
        lds_d = uniform((uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)shared.scales[wave8]);
    }
    const auto ask_raw = [&](int kb, group_pages g) __attribute__((always_inline)) {
        if constexpr (Q8) {
            if (lane < D / 4) {
                const uint32_t mine = lane & 4 ? (lane & 2 ? g.w : g.z) : (lane & 2 ? g.y : g.x);
                to_lds(vs + (uint64_t)mine * vs_g + vs_at + ((kb + 8 * (lane & 7)) & pmask) * 2, lds_d, 1);
            }
            const uint8_t *const source = v_source(kb, g);
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int q = D == 128 ? i : D == 256 ? i >> 1 : 2 * i + (wave >> 1), row = KR * (4 * i + wave) + lane / KC;
                const uint32_t page = q & 2 ? (q & 1 ? g.w : g.z) : (q & 1 ? g.y : g.x);
                const int key = 8 * (row >> 2 & 1) + 4 * (row >> 3 & 1) + (row & 3), at = (kb + 16 * q) & pmask;
                raw_k[i] = *(const uint2 *)(uniform(kbase + (uint64_t)page * kp_g + at * kp_p) + koff[i]);
                raw_d[i] = *(const uint16_t *)(uniform(ks + (uint64_t)page * ks_g + at * (D / 16)) + (key * (D / 16) + (((lane % KC) ^ swizzle_k<D>(row)) >> 2) * 2));
                raw_v[i] = *(const uint2 *)(source + i * 32 * vp_d);
            }
        }
    };
    const auto ask_v = [&](const uint8_t *source, uint32_t buf, uint32_t there, int i) __attribute__((always_inline)) { to_lds(source + i * 32 * vp_d, uniform(lds_v + buf + i * 4096), there); };

    float m = -INFINITY, l = 0.0f;
    int far = 0;                                                           // some |m| of the wave is past 10^7
    v16f o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = v16f{0};
    constexpr uint32_t BUF = 64 * D * 2;                                   // bytes of one buffer
    uint32_t k_at = n * (2 * D) + (half ^ swizzle_k<D>(n)) * 16, v_at = n * 128 + (half ^ swizzle_v(n)) * 16;     // this lane's pieces in LDS
    // Q8: piece j of this wave's, of the tile in the registers, as fp16 to LDS (where there is no such tile, what is in them, to where nobody reads)
    const auto unpack_piece = [&](int j, int to) __attribute__((always_inline)) {
        if constexpr (Q8) {
            const int i = j < NI ? j : j - NI;
            const uint4 v = j < NI ? bits(dequantized(raw_k[i], all_of(raw_d[i]))) : bits(dequantized(raw_v[i], *(const v8h *)(shared.scales[wave8] + (8 * i + vc) * 16)));
            *(uint4 *)((j < NI ? sh.k[to] : sh.v[to]) + (4 * i + wave) * 1024 + lane * 16) = v;
        }
    };
    const auto compute = [&](int kt, int buf, int bad, bool masked, group_pages next) {
        const int kb = begin + 64 * kt;
        const uint32_t more = there_is(kt + GROUPS);
        // LDS answers after some 130 cycles, four times what an instruction that waits for it takes: operands are asked for in order, well before their use, and the
        // barriers between keep the compiler from moving the requests back to where they are used
        if constexpr (Q8) landed();                                        // the next tile's numbers and scales
        asm volatile("" : "+v"(k_at), "+v"(v_at));                         // (addresses once more for every tile: the compiler would keep all of them, in registers that it has not)
        const auto v_piece = [&](int d, int k) { return *(const uint4 *)(sh.v[buf] + d * 4096 + (v_at ^ k * 32)); };
        v16f x[2] = {{0}, {0}};
        constexpr int WB = Q8 ? 1 : 2;                                     // steps of V that are asked for ahead
        uint4 w[WB][DT];
        {
            constexpr int AHEAD = Q8 ? 4 : KS < 8 ? KS : 8;
            v8h fk[AHEAD];
            const auto k_piece = [&](int i) { return *(const v8h *)(sh.k[buf] + (i / KS) * 64 * D + (k_at ^ (i % KS) * 32)); };
#pragma unroll
            for (int i = 0; i < AHEAD; i++) fk[i] = k_piece(i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 2 * KS; i++) {
                x[i / KS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fk[i % AHEAD], fq[i % KS], x[i / KS], 0, 0, 0);
                if (i + AHEAD < 2 * KS) fk[i % AHEAD] = k_piece(i + AHEAD);
                else if (i + AHEAD < 2 * KS + WB * DT) w[(i + AHEAD - 2 * KS) / DT][(i + AHEAD - 2 * KS) % DT] = v_piece((i + AHEAD - 2 * KS) % DT, (i + AHEAD - 2 * KS) / DT);
                if (!Q8 && i % 4 == 0) ask_k(kb + 64 * GROUPS, next, (buf ^ 1) * BUF, more, i / 4);        // the next tile's, one at a time: all at once, they take 1000 cycles to issue
                if (Q8 && i % 2 == 1) unpack_piece(i / 2, buf ^ 1);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = AHEAD; i < WB * DT; i++) w[i / DT][i % DT] = v_piece(i % DT, i / DT);
        }
        if constexpr (Q8) if (kt + 2 * GROUPS < stop) ask_raw(kb + 128 * GROUPS, next);
        // register 8 s + j of tile t: key 32 t + 16 s + 8 half + j.  This lane's query sees register i's where lies(i, first) holds, first: the register 0's from lo on
        const int mine = kb + 8 * half;
        const uint32_t span = max(hi - lo, 0);
        const auto sees = [&](int i, int first) { return (uint32_t)(first + 16 * (i >> 3) + (i & 7)) < (bad >> (i >> 3) & 1 ? 0u : span); };
        if (masked) {
#pragma unroll
            for (int i = 0; i < 32; i++) x[i >> 4][i & 15] = sees(i, mine - lo) ? x[i >> 4][i & 15] : -INFINITY;
        }
        float top = x[0][0];
#pragma unroll
        for (int i = 1; i < 32; i++) top = fmaxf(top, x[i >> 4][i & 15]);
        top = pair_reduce(top, [](float p, float q) { return fmaxf(p, q); }) * c;
        // m starts 10 below the largest x and stays until one lies 15 above it, so that o is seldom scaled (from 12 below: 86.8 and 86.0 us for 512 tokens on 7680, from 7 85.7)
        if (__any(top - m > 15.0f)) {
            const float next = fmaxf(m, top - (fabsf(top) < 1e7f ? 10.0f : 7.0f)), shrink = exp2_(m - (next == -INFINITY ? 0.0f : next));
            m = next;
            l *= shrink;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= shrink;
            far = __any(fabsf(m) > 1e7f && m > -INFINITY) ? 1 : far;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        // m is a rounded x: where the rounding alone may be more than what fp16 has above 2^15, the others are rounded the same way
        float factor = c;
        if (far) {
            factor = 1.0f;
#pragma unroll
            for (int i = 0; i < 32; i++) x[i >> 4][i & 15] *= c;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            const float e = exp2_(fmaf(x[i >> 4][i & 15], factor, -base));
            x[i >> 4][i & 15] = e;
            if (F32OUT) sum += e;
        }
        l += sum;
        const uint8_t *const v_from = Q8 ? nullptr : v_source(kb + 64 * GROUPS, next);
        const auto probs = [&](int k, v8h &p, v8h &p2) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float e = x[k >> 1][8 * (k & 1) + j];
                p[j] = (_Float16)e;
                if (F32OUT) p2[j] = (_Float16)(e - (float)p[j]);
            }
        };
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v8h p, p2;
            probs(k, p, p2);
            if (!F32OUT) {                                                 // the sum of what the product takes, two at a time
                typedef _Float16 v2h __attribute__((ext_vector_type(2)));
                const v2h one = {1, 1};
#pragma unroll
                for (int j = 0; j < 4; j++) l = __builtin_amdgcn_fdot2((v2h){p[2 * j], p[2 * j + 1]}, one, l, false);
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(halves(w[k % WB][d]), p, o[d], 0, 0, 0);
                if (F32OUT) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(halves(w[k % WB][d]), p2, o[d], 0, 0, 0);
                if (k + WB < 4) w[k % WB][d] = v_piece(d, k + WB);
                if (!Q8 && (k * DT + d) % 4 == 0) ask_v(v_from, (buf ^ 1) * BUF, more, (k * DT + d) / 4);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // The pieces of V^T that this wave requested: as in attn_few, positions behind the cache's last one hold anything and are taken as 0, and infinities and NaN, which some
    // rows may see and others not, as well
    const auto bound_v = [&](int kt, int buf, int bad) {
        const int there = bad >> (vc >> 1) & 1 ? 0 : end - (begin + 64 * kt + 8 * vc);
        bool any = false;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            uint4 *const v = (uint4 *)(sh.v[buf] + (4 * i + wave) * 1024 + lane * 16);
            *v = bounded(first_of(*v, there), any);
        }
        if (any) shared.unbounded = 1;
    };
    const int steps = (max(stop - from, 0) + GROUPS - 1) / GROUPS;
    if (steps) {
        int kt = from + group, i = 0, fetched = 0;               // (tiles are numbered from `from` on where their pages are looked up)
        take_entries(first_pages);
        int bad = gone_of(group);
        int bad_next = 0;                                        // (Q8)
        if constexpr (Q8) {
            if (kt < stop) {
                ask_raw(begin + 64 * kt, pages_of(group));
                landed();
#pragma unroll
                for (int j = 0; j < 2 * NI; j++) unpack_piece(j, 0);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (kt + GROUPS < stop) ask_raw(begin + 64 * (kt + GROUPS), pages_of(group + GROUPS));
            }
            bad_next = gone_of(group + GROUPS);
        } else {
            const group_pages now = pages_of(group);
            const uint8_t *const v_from = v_source(begin + 64 * kt, now);
#pragma unroll
            for (int j = 0; j < NI; j++) ask_k(begin + 64 * kt, now, 0, there_is(kt), j);
#pragma unroll
            for (int j = 0; j < NI; j++) ask_v(v_from, 0, there_is(kt), j);
        }
        if (tid == 0) shared.unbounded = 0;
        __syncthreads();
        const auto step = [&](auto idle_) __attribute__((always_inline)) { // one tile; true: it was the last
            const int buf = i & 1, kb = begin + 64 * kt;
            const bool masked = kt < stop && (kb + 64 > hi_all || kb < lo_all || bad);
            if constexpr (!Q8) landed();                                   // what this wave requested of this tile is in LDS ...
            if (masked) bound_v(kt, buf, bad);
            __syncthreads();                                               // ... and all of it, and nobody reads the other buffer any more
            const int ahead = kt - from + (Q8 ? 2 : 1) * GROUPS;
            if ((ahead & 15) == group) take_entries(fetched);
            if ((ahead + GROUPS & 15) == group) fetched = entries_of(ahead + GROUPS);
            const group_pages next = pages_of(ahead);
            if (kt < stop && bad && err) {
                int wanted = 0;                                            // groups with a position that some row sees (a page before the window may be gone)
#pragma unroll
                for (int g = 0; g < 4; g++) wanted |= (kb + 16 * g < end && kb + 16 * g + 16 > lo_any) << g;
                if (bad & wanted) *err = 1;
            }
            if constexpr (idle_ && Q8) {
                landed();
#pragma unroll
                for (int j = 0; j < 2 * NI; j++) unpack_piece(j, buf ^ 1);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (kt + 2 * GROUPS < stop) ask_raw(kb + 128 * GROUPS, next);
            } else if constexpr (idle_) {
                const uint8_t *const v_from = v_source(kb + 64 * GROUPS, next);
#pragma unroll
                for (int j = 0; j < NI; j++) ask_k(kb + 64 * GROUPS, next, (buf ^ 1) * BUF, there_is(kt + GROUPS), j);
#pragma unroll
                for (int j = 0; j < NI; j++) ask_v(v_from, (buf ^ 1) * BUF, there_is(kt + GROUPS), j);
            } else if (!idle_ && kt < stop) compute(kt, buf, bad, masked, next);
            if constexpr (Q8) { bad = bad_next; bad_next = gone_of(ahead); }
            else bad = gone_of(ahead);
            kt += GROUPS;
            return ++i == steps;
        };
        // (a loop of their own for waves without rows: a branch around the products in one loop for both costs registers)
        if (idle) while (!step(std::true_type{})) {}
        else while (!step(std::false_type{})) {}
        __syncthreads();
        float most[2] = {0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int j = 0; j < 16; j++) most[j & 1] = larger(most[j & 1], o[d][j]);
        if (__any(shared.unbounded || !finite(larger(most[0], most[1])))) {
#pragma unroll
            for (int d = 0; d < DT; d++) {
#pragma unroll
                for (int j = 0; j < 16; j++) o[d][j] = finite(o[d][j]) ? o[d][j] : 0.0f;
#pragma nounroll
                for (int kind = 0; kind < 3; kind++) {
                    v16f n_seen = {0};
#pragma nounroll
                    for (int at = begin + 64 * (from + group) + 8 * half, k = 0; at < begin + 64 * stop; at += ++k & 3 ? 16 : 64 * GROUPS - 48) {   // (the tiles of this wave, 16 keys at a time)
                        const int page = table[min(at >> plog, last)], there = (uint32_t)page >= (uint32_t)n_page ? 0 : end - at;
                        const uint64_t from_page = there == 0 ? 0 : page;
                        uint4 w;
                        if constexpr (Q8) w = bits(dequantized(*(const uint2 *)(vbase + from_page * vp_g + (uint32_t)(32 * d + n) * vp_d + (at & pmask)), *(const v8h *)(vs + from_page * vs_g + d * a.vs_b + (at & pmask) * 2)));
                        else w = *(const uint4 *)(vbase + from_page * vp_g + (uint32_t)(32 * d + n) * vp_d + (at & pmask) * 2);
                        uint32_t seen = 0;
#pragma unroll
                        for (int j = 0; j < 8; j++) seen |= (uint32_t)(at + j >= lo && at + j < hi && there > 0) << j;
                        n_seen = __builtin_amdgcn_mfma_f32_32x32x16_f16(of_kind(first_of(w, there), kind), ones(seen), n_seen, 0, 0, 0);
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) if (n_seen[j] != 0.0f) o[d][j] += kind_value(kind);
                }
            }
        }
    }
    constexpr int HAVE = DT / GROUPS;                                      // output tiles that this wave has in the end, from `d0` on
    const int d0 = group * HAVE;
    if constexpr (GROUPS == 2) {                                           // each group takes one half of the output from the other
        static_assert(sizeof(chunk_shared<D, GROUPS>) >= 8 * (16 * HAVE + 2) * 256);
        const auto share = [&](int g) { return (float *)&shared + (4 * g + wave) * (16 * HAVE + 2) * 64 + lane; };
        float *const give = share(group);
        const float *const take = share(1 - group);
        __syncthreads();
        give[0] = m;
        give[64] = l;
#pragma unroll
        for (int d = 0; d < HAVE; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                give[(16 * d + i + 2) * 64] = group ? o[d][i] : o[HAVE + d][i];
                o[d][i] = group ? o[HAVE + d][i] : o[d][i];
            }
        __syncthreads();
        const float m2 = take[0], top = fmaxf(m, m2), base = top == -INFINITY ? 0.0f : top, f = above_0(exp2_(m - base)), f2 = above_0(exp2_(m2 - base));
        m = top;
        l = l * f + take[64] * f2;
#pragma unroll
        for (int d = 0; d < HAVE; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = o[d][i] * f + take[(16 * d + i + 2) * 64] * f2;
    }
    l = pair_reduce(l, [](float p, float q) { return p + q; });
    const int row = wave * 32 + n;
    if (row >= n_row) return;
    const auto late = args_again<attn_args_of<MODE>>();
    if constexpr (SHARED) {
        const int64_t at = ((int64_t)(row0 + token) * (late->G * late->group) + hq) * late->slots + (common ? 0 : late->own_slot) + piece;
#pragma unroll
        for (int d = 0; d < HAVE; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(float4 *)(late->part_o + at * D + 32 * (d0 + d) + 8 * i + 4 * half) = make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
        if (half == 0 && group == 0) *(float2 *)(late->part_ml + at * 2) = make_float2(m, l);
    } else if (whole) {
        uint8_t *dst = late->out + (int64_t)(row0 + token) * late->o_t + (int64_t)hq * late->o_h;
        const float f = m == -INFINITY && l == 0.0f ? 0.0f : 1.0f / l;     // 0: sees no key
#pragma unroll
        for (int d = 0; d < HAVE; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = 32 * (d0 + d) + 8 * i + 4 * half;
                const float v0 = o[d][4 * i] * f, v1 = o[d][4 * i + 1] * f, v2 = o[d][4 * i + 2] * f, v3 = o[d][4 * i + 3] * f;
                if (F32OUT) *(float4 *)(dst + at * 4) = make_float4(v0, v1, v2, v3);
                else *(uint2 *)(dst + at * 2) = make_uint2(f2h(v0) | (uint32_t)f2h(v1) << 16, f2h(v2) | (uint32_t)f2h(v3) << 16);
            }
    } else {
        float *part = late->chunk_part + ((int64_t)unit * late->chunk_pieces + piece) * CHUNK_ROWS * (D + 2);
#pragma unroll
        for (int d = 0; d < HAVE; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(float4 *)(part + row * D + 32 * (d0 + d) + 8 * i + 4 * half) = make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
        if (half == 0 && group == 0) { part[CHUNK_ROWS * D + row] = m; part[CHUNK_ROWS * D + CHUNK_ROWS + row] = l; }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------
// Rows of a sequence that go by a tile of 16, the rest by tiles of 128 (128-wide, 32 heads; by tiles of 16, of which a sequence may have had several then, and of 128): 17 rows on
// 4096 keys 29.6 and 25.2 us, 64 rows 46.5 and 26.7; eight sequences of 17 rows 145 and 105; only one short sequence is faster by tiles of 16 (17 rows on 500 keys: 14.4 and 17.4).
#define FEW_ROWS 16        // one tile
struct attn_plan { int64_t few, few_units, few_split, few_pieces, chunk_tiles, chunk_units, chunk_split, chunk_pieces; size_t few_bytes, scratch; };
// `units` tiles by heads and `key_tiles` tiles of keys: key tiles per workgroup so that `want` workgroups get work, `least` of them at least
static void attn_share(int64_t units, int64_t key_tiles, int64_t want, int64_t least, int64_t &split, int64_t &pieces) {
    const int64_t n = (want + units - 1) / units;
    split = n == 1 ? key_tiles : ((key_tiles + n - 1) / n + 2) / 4 * 4;    // four waves' worth
    if (split < least) split = least;
    pieces = (key_tiles + split - 1) / split;
}
static int attn_make_plan(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *b, bool q8, attn_plan &p) {
    SPY_CHECK_ARG(q && k_pages && q->ne[1] > 0 && q->ne[1] <= 65535 && q->ne[2] > 0 && q->ne[2] < (1 << 28));
    int rc = pg_check_batch(b);
    if (!rc) rc = q8 ? pg_check_pages_q8(k_pages, 1) : pg_check_pages(k_pages, 1);
    if (rc) return rc;
    const int64_t G = k_pages->ne[2], H = q->ne[1], hd = k_pages->ne[0];
    SPY_CHECK_ARG(G <= 65535 && H % G == 0);
    const int64_t group = H / G, most = (int64_t)b->max_new * group, cu = spy_num_cu();
    SPY_CHECK_ARG(most < (1ll << 30));
    // Keys are shared out in pieces of one size, so that long sequences of a ragged batch take more workgroups.  Few rows: 256 keys at least (one request of 4096 keys,
    // 32 heads: 18.0 us, 19.6 with 128 keys), else for six workgroups per compute unit (8 requests of up to 30000: 141 us, 148 with two, 150 with three).
    p.few = most > FEW_ROWS && b->n_seq == 1 ? 0 : FEW_ROWS;              // a single sequence that may bring many rows goes one way whatever it brings: no empty launches
    p.few_units = p.few ? (int64_t)b->n_seq * G : 0;
    p.few_split = 1; p.few_pieces = 0;
    if (p.few) attn_share(p.few_units, ((int64_t)b->max_kv + 31) / 32 + 1, 6 * cu, 8, p.few_split, p.few_pieces);
    p.chunk_tiles = p.chunk_units = 0; p.chunk_split = p.chunk_pieces = 1;
    if (most > p.few) {
        const int64_t each = (most + CHUNK_ROWS - 1) / CHUNK_ROWS, all = q->ne[2] * group / CHUNK_ROWS + b->n_seq;
        p.chunk_tiles = each * b->n_seq < all ? each * b->n_seq : all;
        p.chunk_units = p.chunk_tiles * G;
        // one workgroup per compute unit fits (512 tokens on 7680: 87 us, 95 with two per unit, 119 with four; eight sequences of 17 rows 105, 125 and 139), 512 keys at least
        attn_share(p.chunk_units, ((int64_t)b->max_kv + 63) / 64 + 1, cu, 8, p.chunk_split, p.chunk_pieces);
    }
    // threads of a launch are a number of 32 bits
    SPY_CHECK_ARG((p.few_units * p.few_pieces + p.chunk_units * p.chunk_pieces) * (p.chunk_units ? 256 * chunk_groups((int)hd) : 256) < (1ll << 32) && (p.few_units + p.chunk_units * (CHUNK_ROWS / 16)) * 256 < (1ll << 32));
    p.few_bytes = p.few_pieces > 1 ? (size_t)(p.few_units * p.few_pieces * 16 * (hd + 2) * 4) : 0;
    p.scratch = p.few_bytes + (p.chunk_pieces > 1 ? (size_t)(p.chunk_units * p.chunk_pieces * CHUNK_ROWS * (hd + 2) * 4) : 0);
    return 0;
}


// What a call of any of the variants is refused for, given its plan, and what attn_args has of it but for the scratch.  Pages in 8 bits: k_scales and v_scales.
static int attn_check(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_tensor *k_scales, const spy_hip_tensor *v_pages, const spy_hip_tensor *v_scales,
                      const spy_hip_tensor *out, const spy_hip_paged_batch *batch, float scale, int32_t causal, int32_t window, size_t need, const void *scratch, size_t scratch_bytes, attn_args &a) {
    int rc = k_scales ? pg_check_pages_q8(v_pages, 0) : pg_check_pages(v_pages, 0);
    if (!rc && k_scales) rc = pg_check_scales(k_scales, k_pages, 1);
    if (!rc && k_scales) rc = pg_check_scales(v_scales, v_pages, 0);
    if (rc) return rc;
    if (q->type != SPY_HIP_F16 || (out->type != SPY_HIP_F32 && out->type != SPY_HIP_F16)) return SPY_HIP_EUNSUPPORTED;
    const int64_t hd = k_pages->ne[0], ps = k_pages->ne[1], G = k_pages->ne[2], n_row = q->ne[2], H = q->ne[1];
    SPY_CHECK_ARG(v_pages->ne[0] == ps && v_pages->ne[1] == hd && v_pages->ne[2] == G && v_pages->ne[3] == k_pages->ne[3]);
    SPY_CHECK_ARG(pg_rows_ok(q, hd, H, n_row) && pg_rows_ok(out, hd, H, n_row) && window >= 0 && fabsf(scale) >= 1e-37f && fabsf(scale) <= 1e24f);
    if (need) {
        if (scratch_bytes < need) return SPY_HIP_ENOSPACE;
        SPY_CHECK_ARG(scratch && ((uintptr_t)scratch & 255) == 0);
    }
    SPY_CHECK_ARG(!pg_rows_meet(out, q));
    a.q = (const uint8_t *)q->data; a.kp = (const uint8_t *)k_pages->data; a.vp = (const uint8_t *)v_pages->data; a.out = (uint8_t *)out->data;
    a.q_h = q->nb[1]; a.q_t = q->nb[2]; a.o_h = out->nb[1]; a.o_t = out->nb[2];
    a.kp_p = k_pages->nb[1]; a.kp_h = k_pages->nb[2]; a.kp_g = k_pages->nb[3];
    a.vp_d = v_pages->nb[1]; a.vp_h = v_pages->nb[2]; a.vp_g = v_pages->nb[3];
    a.b.row_start = batch->row_start; a.b.kv_len = batch->kv_len; a.b.pages = batch->pages; a.b.page_stride = batch->page_stride;
    a.b.n_seq = batch->n_seq; a.b.n_row = (int)n_row; a.b.max_new = batch->max_new; a.b.max_kv = batch->max_kv; a.b.n_page = (int)k_pages->ne[3]; a.b.page_log2 = pg_log2(ps);
    a.G = (int)G; a.group = (int)(H / G); a.c = scale * 1.44269504088896341f; a.causal = causal != 0; a.window = window > (1 << 30) ? 0 : window;
    a.err = spy_hip_err_flag_ptr();
    return 0;
}
static inline void attn_use_plan(const attn_plan &p, void *scratch, attn_args &a) {
    a.few = (int)p.few; a.few_split = (int)p.few_split; a.few_pieces = (int)p.few_pieces; a.few_blocks = (int)(p.few_units * p.few_pieces);
    a.chunk_tiles = (int)p.chunk_tiles; a.chunk_split = (int)p.chunk_split; a.chunk_pieces = (int)p.chunk_pieces; a.chunk_blocks = (int)(p.chunk_units * p.chunk_pieces);
    a.few_part = (float *)scratch; a.chunk_part = (float *)((uint8_t *)scratch + p.few_bytes);
}
static inline void attn_use_scales(const spy_hip_tensor *k_scales, const spy_hip_tensor *v_scales, attn_more &a) {
    a.ks = a.vs = nullptr; a.ks_h = a.ks_g = a.vs_b = a.vs_h = a.vs_g = 0;
    if (!k_scales) return;
    a.ks = (const uint8_t *)k_scales->data; a.ks_h = k_scales->nb[2]; a.ks_g = k_scales->nb[3];
    a.vs = (const uint8_t *)v_scales->data; a.vs_b = v_scales->nb[1]; a.vs_h = v_scales->nb[2]; a.vs_g = v_scales->nb[3];
}
// The second launch of a plan that has one (paged_attn.hip)
int spy_attn_join(const attn_args &a, const attn_plan &p, int64_t hd, bool f32, hipStream_t st);
