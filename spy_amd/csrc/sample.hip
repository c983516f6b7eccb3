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
// One workgroup per row, which keeps 32768 logits in LDS at a time.  Measured for one row of 32000, and 64 in brackets: greedy 5.5 us (6.1), temperature alone 9.9 (10.6), top_k 40
// with top_p and min_p 10.2 (11.6), top_k 500 with top_p 17 (18), top_p alone 21 (24), top_k 5000 24 (26), with top_p 28 (30): latency, up to some forty barriers with a
// few dependent LDS accesses between them, and the slowest row of a batch decides; 256 rows of 100003 with top_p alone 81 us: vector instructions, since a weight of every logit is worked out for the sums by
// distance and once more for the sums by part (the memory's share, 103 MB at a copy's rate, is 22 us).
#include "scan.cuh"

#define SM_THREADS 1024
#define SM_BINS 1024           // one per thread
#define SM_LIST 1024           // tokens that are ranked in LDS
#define SM_FAST 512            // largest top_k that is looked for among the threads' maxima: twice as many fill the list (64 rows of 32000, by the maxima and by the histogram: top_k 40 11.0 and 26.4 us, 512 18.5 and 27.5)
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
    int range_log2;                    // a token's index by this many bits less is below SM_BINS
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
// distance the same way.  max - l and y are rounded to 2^-24 of themselves, which moves the weight by up to y ln 2 * 2^-23; the exponential is good to an ulp.  (The distance in
// two floats and y with its remainder would take off the former: 94 us instead of 82 for 256 rows of 100003, 28.3 instead of 23.9 for 64 of 32000.)
struct weigher {
    float top, unit, c, c_lo, cap;     // top and distances in units of 1 / unit; cap: distances from here on count as this one, y as 1e20 at most: products beyond a float would have either sign
    __device__ __forceinline__ float far(float l) const {                         // -inf: as good as infinitely far
        const float d = fminf(fmaf(-l, unit, top), cap);
        return fmaf(d, c, d * c_lo);
    }
    static __device__ __forceinline__ u64 at(float y) {
        const float e = __builtin_amdgcn_exp2f(-y) * 4096.0f;                     // 2^12 and 2^32: 44 bits
        return (u64)(uint32_t)e << 32 | (uint32_t)(__builtin_amdgcn_fractf(e) * 4294967296.0f);
    }
    __device__ __forceinline__ u64 operator()(float l) const { return at(far(l)); }
};

struct __attribute__((aligned(16))) sample_shared {      // (the logits lie behind it, read 16 bytes at a time)
    u64 mass[SM_BINS];
    uint32_t count[SM_BINS];
    u64 x[SM_LIST], w[SM_LIST];
    u64 wave_sum[16], part[16], least[16], most[16];
    float wave_f[16], wave_g[16];
    u64 pick;
    uint32_t pick_count, n_list;
    int bin;
};

static __device__ __forceinline__ uint32_t of_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
static __device__ __forceinline__ u64 of_lane(u64 v, int lane) { return (u64)of_lane((uint32_t)(v >> 32), lane) << 32 | of_lane((uint32_t)v, lane); }
// Inclusive sum over the threads, and the sum of all.  Two calls have a barrier between them.
template <class T> static __device__ __forceinline__ T block_scan(sample_shared &s, T v, T &all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v);
    if (lane == 63) s.wave_sum[wave] = v;
    __syncthreads();
    const T sums = row_scan((T)s.wave_sum[lane & 15]);
    all = of_lane(sums, 15);
    return wave ? v + of_lane(sums, wave - 1) : v;
}
// The bin (one per thread, v: its weights or its tokens) where the running sum first reaches `want`, and the sum before it.  SM_BINS: none does.
template <class T> static __device__ __forceinline__ int find_bin(sample_shared &s, T v, T want, T &before, T &all) {
    const int t = threadIdx.x;
    if (t == 0) s.bin = SM_BINS;
    const T upto = block_scan(s, v, all);
    if (upto >= want && upto - v < want) { s.bin = t; s.pick = upto - v; }        // one thread: the sums do not descend
    __syncthreads();
    const int bin = s.bin;
    before = (T)s.pick;
    __syncthreads();
    return bin;
}

// The row: wave w has the logits part * w .. , a piece of `held` of them in LDS at a time -- all of them up to 32768, else the piece that it looked at last.
struct sample_row {
    const float *g;
    f4 *lds;                           // this wave's
    int n, begin, part, held;          // part and held: multiples of 256
    int here;                          // the piece in LDS
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
        f4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = i + e < n ? g[i + e] : -INFINITY;
        return clean(v);
    }
    __device__ __forceinline__ int blocks(int piece) const { return min(held, part - piece * held) >> 8; }       // of 256 logits
    // A piece to LDS, all its requests at once.  What reaches over the end of the row is requested from where the row's last four logits are, and put right afterwards.
    __device__ __forceinline__ void load(int piece) {
        const int lane = threadIdx.x & 63, from = begin + piece * held, number = blocks(piece);
        f4 v[SM_HELD / 256];
#pragma unroll
        for (int j = 0; j < SM_HELD / 256; j++) if (j < number && n >= 4) v[j] = *(const f4u *)(g + min(from + 4 * (lane + 64 * j), n - 4));
#pragma unroll
        for (int j = 0; j < SM_HELD / 256; j++) if (j < number && n >= 4) lds[lane + 64 * j] = clean(v[j]);
        if (from + 256 * number > n)
#pragma nounroll
            for (int j = max(0, (n - from) >> 8); j < number; j++) lds[lane + 64 * j] = fetch(from + 4 * (lane + 64 * j));
        here = piece;
    }
    // f(four logits, index of the first) of the wave's part, by all lanes of the wave; -inf past the end of the row.  The piece in LDS first.
    template <class F> __device__ __forceinline__ void groups(F f) {
        const int lane = threadIdx.x & 63, last = (part - 1) / held, first = here;
#pragma nounroll
        for (int k = 0; k <= last; k++) {
            const int piece = k == 0 ? first : k <= first ? k - 1 : k;
            if (piece != here) load(piece);
            const int number = blocks(piece), from = begin + piece * held + 4 * lane;
            f4 next = lds[lane];
#pragma nounroll
            for (int j = 0; j < number; j++) {
                const f4 v = next;
                if (j + 1 < number) next = lds[lane + 64 * (j + 1)];
                f(v, from + 256 * j);
            }
        }
    }
    // f(logit, index)
    template <class F> __device__ __forceinline__ void each(F f) {
        groups([&](f4 v, int i) {
#pragma unroll
            for (int e = 0; e < 4; e++) f(v[e], i + e);
        });
    }
};

// Called by every lane of a wave: the token to the list where `take` holds.  n_list counts them all, also those that the list has no room for.
static __device__ __forceinline__ void append(sample_shared &s, bool take, float v, int i, const weigher &weigh) {
    const unsigned long long who = __ballot(take);
    if (!who) return;
    uint32_t base = 0;
    if ((threadIdx.x & 63) == 0) base = atomicAdd(&s.n_list, (uint32_t)__popcll(who));
    base = __builtin_amdgcn_readfirstlane(base) + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    if (take && base < SM_LIST) { s.x[base] = rank_word(v, i); s.w[base] = weigh(v); }
}
// The list by rank: s.x and s.w in order, s.mass[r] the weights up to rank r.  bin_of: a bin for a logit of the list, ascending with the rank; most hold one or none.
template <class Bin> static __device__ __forceinline__ void rank_list(sample_shared &s, uint32_t m, Bin bin_of) {
    const uint32_t t = threadIdx.x;
    const u64 x = t < m ? s.x[t] : 0, w = t < m ? s.w[t] : 0;
    const int bin = t < m ? bin_of(x) : 0;
    s.count[t] = 0;
    __syncthreads();
    uint32_t at = 0, all;
    if (t < m) at = atomicAdd(&s.count[bin], 1u);
    __syncthreads();
    const uint32_t mine = s.count[t], upto = block_scan(s, mine, all);
    s.count[t] = upto - mine;                                                     // first place of bin t
    __syncthreads();
    const uint32_t from = s.count[bin], to = bin + 1 < SM_BINS ? s.count[bin + 1] : m;
    if (t < m) s.x[from + at] = x;
    __syncthreads();
    uint32_t rank = from;
    if (t < m && to - from > 1) for (uint32_t i = from; i < to; i++) rank += s.x[i] < x;
    __syncthreads();
    if (t < m) { s.x[rank] = x; s.w[rank] = w; }
    __syncthreads();
    u64 total;
    s.mass[t] = block_scan(s, t < m ? s.w[t] : 0ull, total);
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

// The draw from a list of up to 128 tokens that has all that top_k leaves, by one wave: two tokens a lane, ranked by comparing each with all.
static __device__ __forceinline__ void draw_from_few(const sample_args &a, sample_shared &s, int r, uint32_t m, int k, bool by_mass, float p, u64 last, float u) {
    const uint32_t lane = threadIdx.x & 63, q = lane + 64;
    u64 x0 = lane < m ? s.x[lane] : ~0ull, x1 = q < m ? s.x[q] : ~0ull, w0 = lane < m ? s.w[lane] : 0, w1 = q < m ? s.w[q] : 0;
    uint32_t r0 = 0, r1 = 0;
    for (uint32_t j = 0; j < m; j++) { const u64 x = s.x[j]; r0 += x < x0; r1 += x < x1; }
    // in rank order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    if (lane < m) { s.x[r0] = x0; s.w[r0] = w0; }
    if (q < m) { s.x[r1] = x1; s.w[r1] = w1; }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    x0 = lane < m ? s.x[lane] : ~0ull; x1 = q < m ? s.x[q] : ~0ull; w0 = lane < m ? s.w[lane] : 0; w1 = q < m ? s.w[q] : 0;
    const u64 upto0 = wave_scan(w0), upto1 = of_lane(upto0, 63) + wave_scan(w1);
    const auto upto = [&](uint32_t rank) { return rank < 64 ? of_lane(upto0, rank) : of_lane(upto1, rank - 64); };
    const auto number = [&](bool in0, bool in1) { return (uint32_t)__popcll(__ballot(in0)) + (uint32_t)__popcll(__ballot(in1)); };
    uint32_t keep = min((uint32_t)k, m);
    if (by_mass) {
        const u64 want = share_of(p, upto(keep - 1));
        keep = min(keep, number(upto0 < want, upto1 < want) + 1);
    }
    keep = min(keep, number(lane < m && x0 <= last, q < m && x1 <= last));
    const u64 total = upto(keep - 1), want = draw_at(u, total);
    // in order of index: the first with a running sum that reaches `want`
    u64 sum0 = 0, sum1 = 0;
    for (uint32_t j = 0; j < keep; j++) {
        const uint32_t index = (uint32_t)s.x[j];
        const u64 w = s.w[j];
        sum0 += index <= (uint32_t)x0 ? w : 0;
        sum1 += index <= (uint32_t)x1 ? w : 0;
    }
    if (lane < keep && sum0 >= want && sum0 - w0 < want) { a.tokens[r] = (int)(uint32_t)x0; if (a.probs) a.probs[r] = (float)((double)w0 / (double)total); }
    if (q < keep && sum1 >= want && sum1 - w1 < want) { a.tokens[r] = (int)(uint32_t)x1; if (a.probs) a.probs[r] = (float)((double)w1 / (double)total); }
}

// More tokens than the list has room for in a bin of the distances (`in`): those of them whose rank words are in lo .. hi, a narrower range at every turn, until the
// list has room.  Finds where a running count or sum reaches `want`, which it leaves as what is wanted of the list; before: the weights before the list, added up.
template <class In> static __device__ __forceinline__ uint32_t narrow(sample_shared &s, sample_row &row, const weigher &weigh, In in, bool by_mass, u64 &want, u64 &before, u64 &lo, int &fine) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    u64 hi = ~0ull;
    lo = 0;
    for (;;) {
        u64 least = ~0ull, most = 0;
        row.each([&](float v, int i) {
            const u64 x = rank_word(v, i);
            if (in(v) && x >= lo && x <= hi) { least = x < least ? x : least; most = x > most ? x : most; }
        });
        s.mass[t] = 0; s.count[t] = 0;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const u64 a = __shfl_xor(least, o, SPY_WAVE), b = __shfl_xor(most, o, SPY_WAVE);
            least = a < least ? a : least;
            most = b > most ? b : most;
        }
        if (lane == 0) { s.least[wave] = least; s.most[wave] = most; }
        __syncthreads();
        for (int w = 0; w < 16; w++) { least = s.least[w] < least ? s.least[w] : least; most = s.most[w] > most ? s.most[w] : most; }
        const int shift = max(0, 64 - __clzll((long long)(most - least)) - 10);
        row.each([&](float v, int i) {
            const u64 x = rank_word(v, i);
            if (in(v) && x >= least && x <= most) {
                const int b = (int)((x - least) >> shift);
                atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.mass[b], weigh(v));
            }
        });
        __syncthreads();
        u64 sum, all;
        // (the last bin where none reaches it, which only logits that are written meanwhile can bring about: the range gets narrower all the same)
        const int bin = min(find_bin(s, by_mass ? s.mass[t] : (u64)s.count[t], want, sum, all), SM_BINS - 1);
        const u64 upto = block_scan(s, s.mass[t], all);
        if (t == bin) s.pick = upto - s.mass[t];
        __syncthreads();
        before += s.pick;
        want -= sum;
        const uint32_t m = s.count[bin];
        __syncthreads();
        lo = least + ((u64)bin << shift);
        hi = lo + ((1ull << shift) - 1);
        if (m > SM_LIST) continue;
        fine = max(0, shift - 10);
        row.each([&](float v, int i) { const u64 x = rank_word(v, i); append(s, in(v) && x >= lo && x <= hi, v, i, weigh); });
        __syncthreads();
        if (t == 0) s.n_list = 0;
        return m;
    }
}

__global__ __launch_bounds__(SM_THREADS) void sample_kernel(sample_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    sample_shared &s = *(sample_shared *)smem;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), r = blockIdx.x;
    sample_row row;
    row.g = (const float *)(a.logits + r * a.stride);
    row.n = a.n; row.begin = wave * a.part; row.part = a.part; row.held = a.held;
    f4 *const held = (f4 *)(smem + sizeof(sample_shared));
    row.lds = held + wave * (a.held / 4);
    const float temp = a.temperature ? a.temperature[r] : 1.0f, p = a.top_p ? a.top_p[r] : 1.0f, mp = a.min_p && a.min_p[r] > 0.0f ? fminf(a.min_p[r], 1.0f) : 0.0f, u = a.uniform[r];
    const int k = a.top_k ? a.top_k[r] : 0;

    row.infinite = false;

    float own = -INFINITY;                                                        // this thread's maximum
    row.load(0);
    row.groups([&](f4 v, int) { own = fmaxf(own, fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))); });
    float top = wave_max(own), low = -wave_max(own > -INFINITY ? -own : -INFINITY);
    if (lane == 0) { s.wave_f[wave] = top; s.wave_g[wave] = low; }
    s.count[t] = 0; s.mass[t] = 0;
    if (t == 0) s.n_list = 0;
    __syncthreads();
    for (int w = 0; w < 16; w++) { top = fmaxf(top, s.wave_f[w]); low = fminf(low, s.wave_g[w]); }
    if (top == -INFINITY) {
        if (t == 0) { a.tokens[r] = -1; if (a.probs) a.probs[r] = 0.0f; }
        return;
    }
    if (top == INFINITY) {
        row.infinite = true;
        row.load(row.here);
        own = own == INFINITY ? 0.0f : -INFINITY;
        top = low = 0.0f;
    }
    if (!(temp > 0.0f)) {
        if (t == 0) s.bin = 0x7FFFFFFF;
        __syncthreads();
        if (__any(own == top)) {
            int first = 0x7FFFFFFF;
            row.each([&](float v, int i) { if (v == top) first = min(first, i); });
            if (own == top) atomicMin(&s.bin, first);
        }
        __syncthreads();
        if (t == 0) { a.tokens[r] = s.bin; if (a.probs) a.probs[r] = 1.0f; }
        return;
    }
    weigher weigh;
    // Beside a large temperature distances past the largest float count: they are taken in units of 2^64, which loses logits that are nothing beside it
    weigh.unit = temp > 1e18f ? 0x1p-64f : 1.0f;
    const double c = 1.4426950408889634074 / ((double)temp * (double)weigh.unit);
    weigh.top = top * weigh.unit; weigh.c = (float)c; weigh.c_lo = (float)(c - (double)weigh.c);
    if (!(weigh.c <= 3.4e38f)) { weigh.c = 3.4e38f; weigh.c_lo = 0.0f; }          // a temperature next to 0
    weigh.cap = weigh.c > 1e-18f ? 1e20f / weigh.c : 3.4e38f;
    const bool by_rank = k > 0 && k < a.n, by_mass = p < 1.0f;
    u64 last = ~0ull;                                                             // rank word of the last token kept
    if (mp > 0.0f && temp < INFINITY) {
        // w >= mp as a limit of the logit, in 64 bits, rounded up to a float
        const double limit = (double)top + (double)temp * log((double)mp);
        float f = (float)limit;
        if ((double)f < limit) f = nextafterf(f, INFINITY);
        last = (u64)order_word(fminf(f, top)) << 32 | 0xFFFFFFFFu;
    }
    if (by_rank && k <= SM_FAST) {
        // a bin of the threads' maxima, between the least and the greatest, by which k of them are counted
        const float scale = top > low ? (SM_BINS - 1) / (top - low) : 0.0f;
        const auto near = [&](float v) { return (int)fminf((top - v) * scale, (float)(SM_BINS - 1)); };
        if (own > -INFINITY) atomicAdd(&s.count[near(own)], 1u);
        __syncthreads();
        uint32_t some, number;
        const int bin = find_bin(s, s.count[t], (uint32_t)k, some, number);
        // the least of those k or more maxima.  Fewer threads than k have a logit above -inf: all those tokens
        float limit = own > -INFINITY && near(own) <= bin ? own : INFINITY;
        limit = bin == SM_BINS ? -3.4028235e38f : -wave_max(-limit);
        if (lane == 0) s.wave_g[wave] = limit;
        __syncthreads();
        for (int w = 0; w < 16; w++) limit = fminf(limit, s.wave_g[w]);
        row.groups([&](f4 v, int i) {
            if (!__any(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= limit)) return;
#pragma unroll
            for (int e = 0; e < 4; e++) append(s, v[e] >= limit, v[e], i + e, weigh);
        });
        __syncthreads();
        const uint32_t m = s.n_list;
        if (m <= 128) {
            if (wave == 0) draw_from_few(a, s, r, m, k, by_mass, p, last, u);
            return;
        }
        __syncthreads();
        if (t == 0) s.n_list = 0;
        if (m <= SM_LIST) {
            const float fine = scale * (float)SM_BINS / (float)(bin + 1);
            rank_list(s, m, [&](u64 x) { return (int)fminf((top - logit_of(x)) * fine, (float)(SM_BINS - 1)); });
            uint32_t keep = min((uint32_t)k, m);
            if (by_mass) keep = min(keep, rank_of_mass(s, m, share_of(p, s.mass[keep - 1])) + 1);
            // those that min_p leaves: the first ones too
            if ((uint32_t)t < keep && s.x[t] <= last && ((uint32_t)t + 1 == keep || s.x[t + 1] > last)) s.pick_count = t + 1;
            __syncthreads();
            keep = s.pick_count;
            const u64 total = s.mass[keep - 1], want = draw_at(u, total);
            const bool mine = (uint32_t)t < keep;
            const u64 x = mine ? s.x[t] : 0, w = mine ? s.w[t] : 0;
            const uint32_t index = (uint32_t)x;
            // in order of index: weights by range of the index, then inside one of the ranges
            const int range = (int)(index >> a.range_log2);
            __syncthreads();
            s.mass[t] = 0;
            __syncthreads();
            if (mine) atomicAdd(&s.mass[range], w);
            __syncthreads();
            u64 before, all;
            const int in = find_bin(s, s.mass[t], want, before, all);
            if (mine && range == in) { const uint32_t at = atomicAdd(&s.n_list, 1u); s.x[at] = index; s.w[at] = w; }
            __syncthreads();
            if (mine && range == in) {
                u64 upto = before + w;
                for (uint32_t i = 0; i < s.n_list; i++) if (s.x[i] < index) upto += s.w[i];
                if (upto >= want && upto - w < want) { a.tokens[r] = (int)index; if (a.probs) a.probs[r] = (float)((double)w / (double)total); }
            }
            return;
        }
        __syncthreads();
        s.count[t] = 0;
        __syncthreads();
    }
    bool summed = false;                                                          // the kept weights of this wave's part are in s.part
    const bool flat = weigh.c == 0.0f;                                            // an infinite temperature: -inf is not far away by itself
    if (by_rank || by_mass) {
        const float reach = (float)(SM_BINS - 1) / 32.0f;                         // distances from here on have one bin together
        u64 tail = 0;
        uint32_t n_tail = 0;
        const bool look = by_rank || flat;                                        // (else -inf adds 0, and nothing is counted)
        row.each([&](float v, int) {
            const bool there = (!look) | (v > -INFINITY);
            const float y = weigh.far(v);
            const u64 w = weigh.at(y);
            if ((y < reach) & there) {
                const int b = (int)(y * 32.0f);
                if (by_rank) atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.mass[b], w);
            } else if (there) { tail += w; n_tail++; }
        });
        n_tail = of_lane(wave_scan(n_tail), 63);                                  // (one addition per wave: the same place for all)
        tail = of_lane(wave_scan(tail), 63);
        if (lane == 0 && n_tail) { atomicAdd(&s.count[SM_BINS - 1], n_tail); atomicAdd(&s.mass[SM_BINS - 1], tail); }
        __syncthreads();
        const u64 mass = s.mass[t], count = s.count[t];
        u64 upto;
        const u64 mass_upto = block_scan(s, mass, upto);
        __syncthreads();
#pragma nounroll
        for (int which = by_rank ? 0 : 1; which < (by_mass ? 2 : 1); which++) {   // 0: top_k, 1: top_p
            u64 want = which ? share_of(p, upto) : (u64)k, before, all;
            const int bin = find_bin(s, which ? mass : count, want, before, all);
            if (bin == SM_BINS) continue;                                         // k or fewer tokens have a logit above -inf
            want -= before;
            if (t == bin) s.pick = mass_upto - mass;
            __syncthreads();
            before = s.pick;
            // the bin's tokens, and beside them for top_p, which is the last to cut, the weights of the parts in the bins before it, as far as the others leave them
            const float near = bin * (1.0f / 32.0f), upper = bin == SM_BINS - 1 ? NAN : (bin + 1) * (1.0f / 32.0f);
            const auto in = [&](float v) { const float y = weigh.far(v); return y >= near && !(y >= upper) && v > -INFINITY; };
            const float last_l = last == ~0ull ? -INFINITY : logit_of(last);
            const int last_i = (int)(uint32_t)min(last & 0xFFFFFFFFull, 0x7FFFFFFFull);
            u64 sum = 0;
            row.groups([&](f4 v, int i) {
                float y[4];
                bool there[4], any = false;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    y[e] = weigh.far(v[e]);
                    if (flat) y[e] = v[e] > -INFINITY ? y[e] : INFINITY;
                    there[e] = (y[e] >= near) & !(y[e] >= upper) & (v[e] > -INFINITY);
                    any |= there[e];
                }
                if (__any(any))
#pragma unroll
                    for (int e = 0; e < 4; e++) append(s, there[e], v[e], i + e, weigh);
                if (which) {
                    bool some = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool before_it = (y[e] < near) & ((v[e] > last_l) | ((v[e] == last_l) & (i + e <= last_i)));
                        y[e] = before_it ? y[e] : INFINITY;
                        some |= before_it;
                    }
                    if (__any(some))
#pragma unroll
                        for (int e = 0; e < 4; e++) sum += weigh.at(y[e]);
                }
            });
            sum = of_lane(wave_scan(sum), 63);
            if (lane == 0) s.part[wave] = sum;
            __syncthreads();
            uint32_t m = s.n_list;
            __syncthreads();
            if (t == 0) s.n_list = 0;
            const bool listed = m <= SM_LIST;
            u64 lo = 0;
            int fine = 0;
            if (!listed) { __syncthreads(); m = narrow(s, row, weigh, in, which == 1, want, before, lo, fine); }
            rank_list(s, m, [&](u64 x) {
                return listed ? (int)fminf((weigh.far(logit_of(x)) * 32.0f - (float)bin) * (float)SM_BINS, (float)(SM_BINS - 1)) : (int)((x - lo) >> fine);
            });
            const uint32_t rank = which ? rank_of_mass(s, m, want) : (uint32_t)want - 1;
            const u64 x = s.x[rank];
            upto = before + s.mass[rank];
            last = x < last ? x : last;
            if (which && listed) {
                if ((uint32_t)t < m && s.x[t] <= last) atomicAdd(&s.part[(uint32_t)s.x[t] / (uint32_t)a.part], s.w[t]);
                summed = true;
            }
            __syncthreads();
        }
    }
    // The kept weights of each wave's part of the row, then inside the part that the random number falls into, by threads
    const bool all_kept = last == ~0ull;
    const float last_l = all_kept ? -INFINITY : logit_of(last);
    const int last_i = (int)(uint32_t)min(last & 0xFFFFFFFFull, 0x7FFFFFFFull);
    const auto kept = [&](float v, int i) { return (v > -INFINITY) & ((v > last_l) | ((v == last_l) & (i <= last_i))); };
    const auto weight = [&](float v, int i) { return weigh.at(kept(v, i) ? weigh.far(v) : INFINITY); };
    if (!summed) {
        u64 sum = 0;
        if (all_kept && !flat) row.each([&](float v, int) { sum += weigh(v); });  // (-inf adds 0)
        else
            row.groups([&](f4 v, int i) {
                bool in[4], some = false;
#pragma unroll
                for (int e = 0; e < 4; e++) { in[e] = kept(v[e], i + e); some |= in[e]; }
                if (!__any(some)) return;
#pragma unroll
                for (int e = 0; e < 4; e++) sum += weigh.at(in[e] ? weigh.far(v[e]) : INFINITY);
            });
        sum = of_lane(wave_scan(sum), 63);
        if (lane == 0) s.part[wave] = sum;
    }
    __syncthreads();
    const u64 sums = row_scan(s.part[lane & 15]), total = of_lane(sums, 15), want_all = draw_at(u, total);
    const int part = max(__ffsll(__ballot(sums >= want_all)) - 1, 0);              // the first of the row's 16 lanes
    const u64 want = want_all - (part ? of_lane(sums, part - 1) : 0);
    const int each = (a.part / 4 + SM_THREADS - 1) / SM_THREADS;                  // groups of four per thread
    const auto group = [&](int i) {                                               // of the part
        return a.held == a.part && 4 * i < a.held ? held[part * (a.held / 4) + i] : 4 * i < a.part ? row.fetch(part * a.part + 4 * i) : f4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    };
    u64 here = 0, whole;
#pragma nounroll
    for (int j = 0; j < each; j++) {
        const f4 v = group(t * each + j);
#pragma unroll
        for (int e = 0; e < 4; e++) here += weight(v[e], part * a.part + 4 * (t * each + j) + e);
    }
    const u64 run = block_scan(s, here, whole);
    if (run >= want && run - here < want) {
        u64 upto = run - here;
#pragma nounroll
        for (int j = 0; j < each; j++) {
            const f4 v = group(t * each + j);
#pragma unroll
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
    SPY_CHECK_ARG(n > 0 && n <= SM_VOCAB && n_row > 0 && n_row * SM_THREADS < (1ll << 32) && logits->ne[2] == 1 && logits->ne[3] == 1 && logits->nb[0] == 4 && logits->nb[1] % 4 == 0);
    SPY_CHECK_ARG((((uintptr_t)logits->data | (uintptr_t)tokens | (uintptr_t)probs | (uintptr_t)param->temperature | (uintptr_t)param->top_k | (uintptr_t)param->top_p |
                    (uintptr_t)param->min_p | (uintptr_t)param->uniform) & 3) == 0);
    sample_args a;
    a.logits = (const uint8_t *)logits->data; a.stride = logits->nb[1]; a.n = (int)n;
    a.part = (int)((n + 4095) / 4096 * 256); a.held = a.part < SM_HELD ? a.part : SM_HELD;
    a.range_log2 = 0;
    while ((n - 1) >> a.range_log2 >= SM_BINS) a.range_log2++;
    a.temperature = param->temperature; a.top_p = param->top_p; a.min_p = param->min_p; a.uniform = param->uniform; a.top_k = param->top_k;
    a.tokens = tokens; a.probs = probs;
    const size_t lds = sizeof(sample_shared) + (size_t)16 * a.held * 4;
    const int rc = spy_raise_lds_limit((const void *)sample_kernel, lds);
    if (rc) return rc;
    sample_kernel<<<dim3((unsigned)n_row), dim3(SM_THREADS), lds, (hipStream_t)stream>>>(a);
    return SPY_LAUNCH_RC();
}
