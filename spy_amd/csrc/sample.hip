// A token drawn from each row of logits: temperature, top-k, top-p and min-p, by given random numbers.  Beside the greedy argmax (ops.hip).
//
// What the settings keep is in every case the first so many tokens of one ranking (logit descending, then index ascending), so the kept set is known by its last
// member.  With the rank word X = (descending order word of the logit) << 32 | index, all X different, that is one 64-bit number, and the strictest setting the
// smallest of them.  Nothing is sorted but a list of up to SM_LIST tokens in LDS, which holds the place where a setting cuts:
//   top-k of up to SM_FAST: the k-th largest of the 1024 threads' own maxima is not above the k-th largest logit, so the tokens from it on (k to 2 k of them) hold
//     the k first; everything else happens in the list;
//   else: a histogram of the tokens over their distance to the maximum, with a count and a sum of weights in every bin, says in which bin a setting cuts; the bin's
//     tokens make the list, through finer histograms of X where they are too many.
// Weights are integers, multiples of 2^-44 of the largest: sums of them are the same in any order, and exact.
// One workgroup per row, which keeps the first 32768 logits in LDS.
#include "common.cuh"

#define SM_THREADS 1024
#define SM_BINS 1024           // one per thread
#define SM_LIST 1024           // tokens that are ranked in LDS
#define SM_FAST 512            // largest top_k that is looked for among the threads' maxima
#define SM_BITS 44             // weights: multiples of 2^-44; 2^18 of them fit 64 bits
#define SM_VOCAB (1 << 18)
#define SM_HELD 2048           // logits of a wave's part of the row that lie in LDS

typedef unsigned long long u64;
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

struct sample_args {
    const uint8_t *logits;
    int64_t stride;
    int n, part, held;                 // vocabulary; a wave's part of a row (a multiple of 256), and how much of it lies in LDS
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
};

// ascending with descending logit; -0 counts as 0 (NaN and -inf have no rank: whoever asks leaves them out)
static __device__ __forceinline__ uint32_t order_word(float l) {
    const uint32_t u = __float_as_uint(l == 0.0f ? 0.0f : l);
    return u & 0x80000000u ? u : 0x7FFFFFFFu - u;
}
static __device__ __forceinline__ u64 rank_word(float l, int i) { return (u64)order_word(l) << 32 | (uint32_t)i; }
static __device__ __forceinline__ float logit_of(u64 x) {
    const uint32_t o = (uint32_t)(x >> 32);
    return __uint_as_float(o & 0x80000000u ? o : 0x7FFFFFFFu - o);
}

// e^((l - max) / T) = 2^-y as a multiple of 2^-44, y = (max - l) log2(e) / T.  log2(e) / T in two floats: a rounded one alone would shift all weights of the same
// distance the same way.  The exponential is good to an ulp.
struct weigher {
    float top, c, c_lo;
    __device__ __forceinline__ float far(float l) const {                         // of a logit above -inf
        const float d = fminf(top - l, 3.4e38f);
        return fmaf(d, c, d * c_lo);
    }
    static __device__ __forceinline__ u64 at(float y) {
        const float e = __builtin_amdgcn_exp2f(-y) * 4096.0f;                     // 2^12 and 2^32: 44 bits
        const uint32_t h = (uint32_t)e;
        return (u64)h << 32 | (uint32_t)((e - (float)h) * 4294967296.0f);
    }
    __device__ __forceinline__ u64 operator()(float l) const { return at(far(l)); }
};

struct sample_shared {
    u64 mass[SM_BINS];
    uint32_t count[SM_BINS];
    u64 x[SM_LIST], w[SM_LIST];
    u64 wave_a[16], wave_min[16], wave_max[16];
    uint32_t wave_b[16];
    float wave_f[16], wave_g[16];
    u64 pick, pick_mass;
    uint32_t pick_count, n_list;
    int bin;
};

static __device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, SPY_WAVE);
    return v;
}
// Inclusive sums over the threads of (a, b)
static __device__ __forceinline__ void block_scan(sample_shared &s, u64 &a, uint32_t &b) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 va = __shfl_up(a, o, SPY_WAVE);
        const uint32_t vb = __shfl_up(b, o, SPY_WAVE);
        if (lane >= o) { a += va; b += vb; }
    }
    __syncthreads();
    if (lane == 63) { s.wave_a[wave] = a; s.wave_b[wave] = b; }
    __syncthreads();
    for (int w = 0; w < wave; w++) { a += s.wave_a[w]; b += s.wave_b[w]; }
}
// The bin (one per thread: a weights, b tokens) where the running sum -- by_mass -- or count first reaches what is wanted, and both before it.  SM_BINS: none does.
static __device__ __forceinline__ int find_bin(sample_shared &s, u64 a, uint32_t b, bool by_mass, u64 want, uint32_t &count_before, u64 &mass_before, u64 *all = nullptr) {
    const int t = threadIdx.x;
    const u64 a0 = a;
    const uint32_t b0 = b;
    if (t == 0) s.bin = SM_BINS;
    block_scan(s, a, b);
    const bool here = by_mass ? a >= want && a - a0 < want : b >= want && b - b0 < want;
    if (here) { s.bin = t; s.pick_mass = a - a0; s.pick_count = b - b0; }         // one thread: the sums do not descend
    if (t == SM_THREADS - 1) s.pick = a;
    __syncthreads();
    const int bin = s.bin;
    count_before = s.pick_count; mass_before = s.pick_mass;
    if (all) *all = s.pick;
    __syncthreads();
    return bin;
}

// The row: wave w has the logits part * w .. , the first `held` of them in LDS.
struct sample_row {
    const float *g;
    f4 *lds;                           // this wave's
    int n, begin, end, held;
    bool infinite;                     // the largest logit is +inf: +inf counts as 0 and every other one as -inf
    __device__ __forceinline__ f4 clean(f4 v) const {                             // NaN: never drawn, as -inf
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = v[e] >= -INFINITY ? v[e] : -INFINITY;
        if (infinite)
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = v[e] == INFINITY ? 0.0f : -INFINITY;
        return v;
    }
    __device__ __forceinline__ f4 fetch(int i) const {                            // logits i .. i + 3, -inf behind the row
        if (i + 4 <= n) return clean(*(const f4u *)(g + i));
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = i + e < n ? g[i + e] : -INFINITY;
        return clean(v);
    }
    // f(four logits, index of the first) over the part's logits from `from` on, in memory: four requests at a time
    template <class F> __device__ __forceinline__ void stream(int from, F f) const {
        int i = from + 4 * ((int)threadIdx.x & 63);
        for (const int full = end - 1024; i - 4 * ((int)threadIdx.x & 63) <= full; i += 1024) {
            f4 v[4];
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = *(const f4u *)(g + i + 256 * j);
#pragma unroll
            for (int j = 0; j < 4; j++) f(clean(v[j]), i + 256 * j);
        }
        for (; i < end; i += 256) f(fetch(i), i);
    }
    // f(logit, index) of the wave's part, four indices in a row per lane; -inf past the end of the row
    template <class F> __device__ __forceinline__ void each(F f) const {
        const int lane = threadIdx.x & 63, groups = held / 4;
        f4 next = lds[lane];
        for (int i = lane; i < groups; i += 64) {
            const f4 v = next;
            next = lds[i + 64 < groups ? i + 64 : lane];
#pragma unroll
            for (int e = 0; e < 4; e++) f(v[e], begin + 4 * i + e);
        }
        stream(begin + held, [&](f4 v, int i) {
#pragma unroll
            for (int e = 0; e < 4; e++) f(v[e], i + e);
        });
    }
};

// Tokens for which `in` holds, into the list; returns their number, which may be more than the list has room for (it is incomplete then).
template <class In> static __device__ __forceinline__ uint32_t collect(sample_shared &s, const sample_row &row, const weigher &weigh, In in) {
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    row.each([&](float v, int i) {
        const bool take = in(v, i);
        const unsigned long long who = __ballot(take);
        if (who) {
            uint32_t base = 0;
            if ((threadIdx.x & 63) == 0) base = atomicAdd(&s.n_list, (uint32_t)__popcll(who));
            base = __builtin_amdgcn_readfirstlane(base) + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
            if (take && base < SM_LIST) { s.x[base] = rank_word(v, i); s.w[base] = weigh(v); }
        }
    });
    __syncthreads();
    const uint32_t m = s.n_list;
    __syncthreads();
    return m;
}
// Least and greatest of the threads' x
static __device__ __forceinline__ void block_range(sample_shared &s, u64 &least, u64 &most) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const u64 a = __shfl_xor(least, o, SPY_WAVE), b = __shfl_xor(most, o, SPY_WAVE);
        least = a < least ? a : least;
        most = b > most ? b : most;
    }
    if (lane == 0) { s.wave_min[wave] = least; s.wave_max[wave] = most; }
    __syncthreads();
    for (int w = 0; w < 16; w++) { least = s.wave_min[w] < least ? s.wave_min[w] : least; most = s.wave_max[w] > most ? s.wave_max[w] : most; }
    __syncthreads();
}
static __device__ __forceinline__ int bin_shift(u64 least, u64 most) { return max(0, 64 - __clzll((long long)(most - least)) - 10); }        // 1024 bins from least to most

// The list by rank: s.x and s.w in order, s.mass[r] the weights up to rank r.  Tokens are dealt to bins of X between its ends, of which most hold one or none.
static __device__ __forceinline__ void rank_list(sample_shared &s, uint32_t m) {
    const uint32_t t = threadIdx.x;
    const u64 x = t < m ? s.x[t] : 0, w = t < m ? s.w[t] : 0;
    u64 least = t < m ? x : ~0ull, most = x;
    s.count[t] = 0;
    block_range(s, least, most);
    const int shift = bin_shift(least, most), bin = t < m ? (int)((x - least) >> shift) : 0;
    uint32_t at = 0;
    if (t < m) at = atomicAdd(&s.count[bin], 1u);
    __syncthreads();
    u64 none = 0;
    const uint32_t mine = s.count[t];
    uint32_t sum = mine;
    block_scan(s, none, sum);
    __syncthreads();
    s.count[t] = sum - mine;                                                      // first place of bin t
    __syncthreads();
    const uint32_t from = s.count[bin], to = bin + 1 < SM_BINS ? s.count[bin + 1] : m;
    if (t < m) s.x[from + at] = x;
    __syncthreads();
    uint32_t rank = from;
    if (t < m) for (uint32_t i = from; i < to; i++) rank += s.x[i] < x;
    __syncthreads();
    if (t < m) { s.x[rank] = x; s.w[rank] = w; }
    __syncthreads();
    u64 upto = t < m ? s.w[t] : 0;
    uint32_t zero = 0;
    block_scan(s, upto, zero);
    s.mass[t] = upto;
    __syncthreads();
}
// Rank in the ordered list at which the weights first add up to `want` (they do), by every thread
static __device__ __forceinline__ uint32_t rank_of_mass(sample_shared &s, uint32_t m, u64 want) {
    const uint32_t t = threadIdx.x;
    if (t < m && s.mass[t] >= want && (t == 0 || s.mass[t - 1] < want)) s.pick_count = t;
    __syncthreads();
    const uint32_t r = s.pick_count;
    __syncthreads();
    return r;
}
static __device__ __forceinline__ u64 share_of(float p, u64 all) {                // the least whole number >= 1 that is not below p * all, at most all
    const double d = (double)fmaxf(p, 0.0f) * (double)all;
    u64 want = (u64)d;
    want += (double)want < d;
    return want < 1 ? 1 : want > all ? all : want;
}
static __device__ __forceinline__ u64 draw_at(float u, u64 total) {               // the running sum that the drawn token is the first to reach: floor(u * total) + 1
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    const u64 u64s = u >= 5.421010862427522e-20f ? (u64)((double)u * 18446744073709551616.0) : 0;
    return __umul64hi(u64s, total) + 1;
}

// Rank word of the last token kept by a setting that keeps the first tokens up to a count, or up to a sum of weights (reached by those of `in`).
// upto: the weights from `before` on, up to the found token's.
template <class In>
static __device__ __forceinline__ u64 find_last(sample_shared &s, const sample_row &row, const weigher &weigh, In in, bool by_mass, u64 want, u64 before, u64 &upto) {
    const int t = threadIdx.x;
    u64 lo = 0, hi = ~0ull;
    uint32_t m;
    while ((m = collect(s, row, weigh, [&](float v, int i) { if (!in(v)) return false; const u64 x = rank_word(v, i); return x >= lo && x <= hi; })) > SM_LIST) {
        // finer bins between the least and the greatest rank word there are
        u64 least = ~0ull, most = 0;
        row.each([&](float v, int i) {
            const u64 x = rank_word(v, i);
            if (in(v) && x >= lo && x <= hi) { least = x < least ? x : least; most = x > most ? x : most; }
        });
        s.mass[t] = 0; s.count[t] = 0;
        block_range(s, least, most);
        const int shift = bin_shift(least, most);
        row.each([&](float v, int i) {
            const u64 x = rank_word(v, i);
            if (in(v) && x >= least && x <= most) {
                const int b = (int)((x - least) >> shift);
                atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.mass[b], weigh(v));
            }
        });
        __syncthreads();
        uint32_t cb;
        u64 mb;
        const int bin = find_bin(s, s.mass[t], s.count[t], by_mass, want, cb, mb);
        want -= by_mass ? mb : cb;
        before += mb;
        lo = least + ((u64)bin << shift);
        hi = lo + ((1ull << shift) - 1);
    }
    rank_list(s, m);
    const uint32_t r = by_mass ? rank_of_mass(s, m, want) : (uint32_t)want - 1;
    const u64 x = s.x[r];
    upto = before + s.mass[r];
    __syncthreads();
    return x;
}

__global__ __launch_bounds__(SM_THREADS) void sample_kernel(sample_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    sample_shared &s = *(sample_shared *)smem;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = blockIdx.x;
    sample_row row;
    row.g = (const float *)(a.logits + r * a.stride);
    row.n = a.n; row.begin = wave * a.part; row.end = min(row.begin + a.part, a.n); row.held = a.held;
    f4 *const held = (f4 *)(smem + sizeof(sample_shared));
    row.lds = held + wave * (a.held / 4);
    const float temp = a.temperature ? a.temperature[r] : 1.0f, p = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f, u = a.uniform[r];
    const int k = a.top_k ? a.top_k[r] : 0;

    row.infinite = false;

    float own = -INFINITY;                                                        // this thread's maximum
    const auto take = [&](f4 v, int i) {                                          // i: group of four of the part
        row.lds[i] = v;
        own = fmaxf(own, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])));
    };
    if (row.begin + a.held <= a.n) {
        int i = lane;
        for (; i - lane + 512 <= a.held / 4; i += 512) {                          // eight requests at a time
            f4 v[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = *(const f4u *)(row.g + row.begin + 4 * (i + 64 * j));
#pragma unroll
            for (int j = 0; j < 8; j++) take(row.clean(v[j]), i + 64 * j);
        }
        for (; i < a.held / 4; i += 64) take(row.fetch(row.begin + 4 * i), i);
    } else
        for (int i = lane; i < a.held / 4; i += 64) take(row.fetch(row.begin + 4 * i), i);
    row.stream(row.begin + a.held, [&](f4 v, int) { own = fmaxf(own, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))); });
    float top = wave_max(own), low = -wave_max(own > -INFINITY ? -own : -INFINITY);
    if (lane == 0) { s.wave_f[wave] = top; s.wave_g[wave] = low; }
    s.count[t] = 0; s.mass[t] = 0;
    __syncthreads();
    for (int w = 0; w < 16; w++) { top = fmaxf(top, s.wave_f[w]); low = fminf(low, s.wave_g[w]); }
    if (top == -INFINITY) {
        if (t == 0) { a.tokens[r] = -1; if (a.probs) a.probs[r] = 0.0f; }
        return;
    }
    if (top == INFINITY) {
        row.infinite = true;
        for (int i = lane; i < a.held / 4; i += 64) row.lds[i] = row.clean(row.lds[i]);
        own = own == INFINITY ? 0.0f : -INFINITY;
        top = low = 0.0f;
    }
    if (!(temp > 0.0f)) {
        if (t == 0) s.bin = 0x7FFFFFFF;
        __syncthreads();
        if (own == top) {
            int first = 0x7FFFFFFF;
            row.each([&](float v, int i) { if (v == top) first = min(first, i); });
            atomicMin(&s.bin, first);
        }
        __syncthreads();
        if (t == 0) { a.tokens[r] = s.bin; if (a.probs) a.probs[r] = 1.0f; }
        return;
    }
    weigher weigh;
    const double c = 1.4426950408889634074 / (double)temp;
    weigh.top = top; weigh.c = (float)c; weigh.c_lo = (float)(c - (double)weigh.c);
    if (!(weigh.c <= 3.4e38f)) { weigh.c = 3.4e38f; weigh.c_lo = 0.0f; }          // a temperature next to 0
    const bool by_rank = k > 0 && k < a.n, by_mass = p < 1.0f;
    u64 last = ~0ull;                                                             // rank word of the last token kept
    if (mp > 0.0f && temp < INFINITY) {
        // w >= mp as a limit of the logit, in 64 bits, rounded up to a float
        const double limit = (double)top + (double)temp * log((double)mp);
        float f = (float)limit;
        if ((double)f < limit) f = nextafterf(f, INFINITY);
        last = (u64)order_word(fminf(f, top)) << 32 | 0xFFFFFFFFu;
    }
    uint32_t cb;
    u64 mb;
    if (by_rank && k <= SM_FAST) {
        // a bin of the threads' maxima, between the least and the greatest, by which k of them are counted
        const float scale = top > low ? (SM_BINS - 1) / (top - low) : 0.0f;
        const auto near = [&](float v) { return (int)fminf((top - v) * scale, (float)SM_BINS); };
        if (own > -INFINITY) atomicAdd(&s.count[min(near(own), SM_BINS - 1)], 1u);
        __syncthreads();
        const int bin = find_bin(s, 0, s.count[t], false, (u64)k, cb, mb);       // SM_BINS: fewer threads than k have a logit, all tokens make the list
        const uint32_t m = collect(s, row, weigh, [&](float v, int) { return v > -INFINITY && near(v) <= bin; });
        if (m <= SM_LIST) {
            rank_list(s, m);
            uint32_t keep = min((uint32_t)k, m);
            if (by_mass) keep = min(keep, rank_of_mass(s, m, share_of(p, s.mass[keep - 1])) + 1);
            if (t == 0) s.pick_count = 0;
            __syncthreads();
            // those that min_p leaves: the first ones too
            const unsigned long long who = __ballot((uint32_t)t < keep && s.x[t] <= last);
            if (lane == 0 && who) atomicAdd(&s.pick_count, (uint32_t)__popcll(who));
            __syncthreads();
            keep = s.pick_count;
            const u64 total = s.mass[keep - 1], want = draw_at(u, total);
            const bool mine = (uint32_t)t < keep;
            const u64 x = mine ? s.x[t] : 0, w = mine ? s.w[t] : 0;
            const uint32_t index = (uint32_t)x;
            // in order of index: weights by range of the index, then inside one of the ranges
            const int range = (int)((u64)index * SM_BINS / (uint32_t)a.n);
            __syncthreads();
            s.mass[t] = 0;
            if (t == 0) s.n_list = 0;
            __syncthreads();
            if (mine) atomicAdd(&s.mass[range], w);
            __syncthreads();
            const int in = find_bin(s, s.mass[t], 0, true, want, cb, mb);
            if (mine && range == in) { const uint32_t at = atomicAdd(&s.n_list, 1u); s.x[at] = index; s.w[at] = w; }
            __syncthreads();
            if (mine && range == in) {
                u64 upto = mb + w;
                for (uint32_t i = 0; i < s.n_list; i++) if (s.x[i] < index) upto += s.w[i];
                if (upto >= want && upto - w < want) { a.tokens[r] = (int)index; if (a.probs) a.probs[r] = (float)((double)w / (double)total); }
            }
            return;
        }
        s.count[t] = 0;
        __syncthreads();
    }
    if (by_rank || by_mass) {
        const auto bin_at = [&](float y) { return (int)fminf(y * 32.0f, (float)(SM_BINS - 1)); };
        row.each([&](float v, int) {
            if (!(v > -INFINITY)) return;
            const float y = weigh.far(v);
            const int b = bin_at(y);
            if (by_rank) atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], weigh.at(y));
        });
        __syncthreads();
        const u64 mass = s.mass[t];
        const uint32_t count = s.count[t];
        u64 upto;
        int bin = find_bin(s, mass, count, false, (u64)k, cb, mb, &upto);
        if (by_rank && bin < SM_BINS) {                                           // (not: k or fewer tokens have a logit above -inf)
            const u64 x = find_last(s, row, weigh, [&](float v) { return v > -INFINITY && bin_at(weigh.far(v)) == bin; }, false, (u64)k - cb, mb, upto);
            last = x < last ? x : last;
        }
        if (by_mass) {
            const u64 want = share_of(p, upto);
            bin = find_bin(s, mass, count, true, want, cb, mb);
            u64 unused;
            const u64 x = find_last(s, row, weigh, [&](float v) { return v > -INFINITY && bin_at(weigh.far(v)) == bin; }, true, want - mb, mb, unused);
            last = x < last ? x : last;
        }
    }
    // The kept weights of each wave's part of the row, then inside the part that the random number falls into, by threads
    const auto weight = [&](float v, int i) -> u64 { return v > -INFINITY && rank_word(v, i) <= last ? weigh(v) : 0; };
    u64 sum = 0;
    row.each([&](float v, int i) { sum += weight(v, i); });
    sum = wave_sum_u64(sum);
    if (lane == 0) s.wave_min[wave] = sum;
    __syncthreads();
    u64 total = 0;
    for (int w = 0; w < 16; w++) total += s.wave_min[w];
    u64 want = draw_at(u, total);
    int part = 0;
    while (part < 15 && want > s.wave_min[part]) want -= s.wave_min[part++];
    const int each = (a.part / 4 + SM_THREADS - 1) / SM_THREADS;                  // groups of four per thread
    const auto group = [&](int i) {                                               // of the part
        return 4 * i < a.held ? held[part * (a.held / 4) + i] : 4 * i < a.part && part * a.part + 4 * i < a.n ? row.fetch(part * a.part + 4 * i) : f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    };
    u64 here = 0;
    for (int j = 0; j < each; j++) {
        const f4 v = group(t * each + j);
#pragma unroll
        for (int e = 0; e < 4; e++) here += weight(v[e], part * a.part + 4 * (t * each + j) + e);
    }
    u64 run = here;
    uint32_t zero = 0;
    block_scan(s, run, zero);
    if (run >= want && run - here < want) {
        u64 upto = run - here;
        for (int j = 0; j < each; j++) {
            const f4 v = group(t * each + j);
            for (int e = 0; e < 4; e++) {
                const int i = part * a.part + 4 * (t * each + j) + e;
                const u64 w = weight(v[e], i);
                upto += w;
                if (upto >= want && upto - w < want) { a.tokens[r] = i; if (a.probs) a.probs[r] = (float)((double)w / (double)total); }
            }
        }
    }
}

extern "C" size_t spy_hip_sample_scratch_size(const spy_hip_tensor *logits) {
    (void)logits;
    return 0;
}

extern "C" int spy_hip_sample(void *stream, const spy_hip_tensor *logits, const spy_hip_sample_param *param, int32_t *tokens, float *probs, void *scratch, size_t scratch_bytes) {
    (void)scratch; (void)scratch_bytes;
    SPY_CHECK_ARG(logits && param && tokens && logits->data && param->uniform);
    if (logits->type != SPY_HIP_F32) return SPY_HIP_EUNSUPPORTED;
    const int64_t n = logits->ne[0], n_row = logits->ne[1];
    SPY_CHECK_ARG(n > 0 && n <= SM_VOCAB && n_row > 0 && n_row < (1ll << 31) && logits->ne[2] == 1 && logits->ne[3] == 1 && logits->nb[0] == 4 && logits->nb[1] % 4 == 0);
    SPY_CHECK_ARG((((uintptr_t)logits->data | (uintptr_t)tokens | (uintptr_t)probs | (uintptr_t)param->temperature | (uintptr_t)param->top_k | (uintptr_t)param->top_p |
                    (uintptr_t)param->min_p | (uintptr_t)param->uniform) & 3) == 0);
    sample_args a;
    a.logits = (const uint8_t *)logits->data; a.stride = logits->nb[1]; a.n = (int)n;
    a.part = (int)((n + 4095) / 4096 * 256); a.held = a.part < SM_HELD ? a.part : SM_HELD;
    a.temperature = param->temperature; a.top_p = param->top_p; a.min_p = param->min_p; a.uniform = param->uniform; a.top_k = param->top_k;
    a.tokens = tokens; a.probs = probs;
    const size_t lds = sizeof(sample_shared) + (size_t)16 * a.held * 4;
    const int rc = spy_raise_lds_limit((const void *)sample_kernel, lds);
    if (rc) return rc;
    sample_kernel<<<dim3((unsigned)n_row), dim3(SM_THREADS), lds, (hipStream_t)stream>>>(a);
    return SPY_LAUNCH_RC();
}
