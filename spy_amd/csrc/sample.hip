// A token drawn from each row of logits: temperature, top-k, top-p and min-p, by given random numbers.  Beside the greedy argmax (ops.hip).
//
// What the settings keep is in every case the first so many tokens of one ranking (logit descending, then index ascending), so the kept set is known by its last
// member.  With the rank word X = (descending order word of the logit) << 32 | index, all X different, that is one 64-bit number, and the strictest setting the
// smallest of them.  No sorting: a histogram of the tokens over their distance to the maximum, with a count and a sum of weights in every bin, says in which bin a
// setting cuts; the tokens of that bin are ranked in LDS, through finer histograms of X first where they are too many.
// Weights are integers, multiples of 2^-44 of the largest: sums of them are the same in any order, and exact.
#include "common.cuh"

#define SM_THREADS 1024
#define SM_BINS 1024           // one per thread
#define SM_LIST 1024           // tokens that are ranked in LDS
#define SM_BITS 44             // weights: multiples of 2^-44; n < 2^19 of them fit 64 bits

typedef unsigned long long u64;

struct sample_args {
    const uint8_t *logits;
    int64_t stride;
    int n;
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

// e^((l - max) / T) as a multiple of 2^-44.  y = (max - l) log2(e) / T with the product's rounding made good; 2^-y = 2^(f - k), k whole, 0 <= f < 1; the 24 bits of
// 2^f are shifted to their place.
struct weigher {
    float top, c, c_lo;
    __device__ __forceinline__ float far(float l) const { return l == top ? 0.0f : (top - l) * c; }          // distance in halvings, for the bins
    __device__ __forceinline__ u64 operator()(float l) const {
        if (l == top) return 1ull << SM_BITS;
        const float d = top - l, y = d * c;
        if (!(y < 64.0f)) return 0;
        const float k = ceilf(y), f = (k - y) - (fmaf(d, c, -y) + d * c_lo);
        const float e = __builtin_amdgcn_exp2f(f);                                // within an ulp of [1, 2]
        const uint32_t b = __float_as_uint(e);
        const u64 mant = (u64)((b & 0x7FFFFFu) | 0x800000u) << (SM_BITS - 23);
        const int shift = (int)k - ((int)(b >> 23) - 127);
        return shift > 63 ? 0 : mant >> max(shift, 0);
    }
};

static __device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, SPY_WAVE);
    return v;
}

struct sample_shared {
    u64 mass[SM_BINS];
    uint32_t count[SM_BINS];
    u64 x[SM_LIST], w[SM_LIST];
    u64 wave_a[16];
    uint32_t wave_b[16];
    float wave_f[16];
    u64 pick, pick_mass;
    uint32_t pick_count, n_list;
    int bin;
};

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

// The bin where a running count or a running sum first reaches what is wanted (by_mass: the sum), and both before it.  s.count, s.mass: the bins.
static __device__ __forceinline__ void find_bin(sample_shared &s, bool by_mass, u64 want, int &bin, uint32_t &count_before, u64 &mass_before) {
    const int t = threadIdx.x;
    u64 a = s.mass[t];
    uint32_t b = s.count[t];
    const u64 a0 = a;
    const uint32_t b0 = b;
    block_scan(s, a, b);
    if (t == 0) s.bin = SM_BINS;
    __syncthreads();
    const bool here = by_mass ? a >= want && (a - a0 < want) : b >= want && b - b0 < want;
    if (here) { s.bin = t; s.pick_mass = a - a0; s.pick_count = b - b0; }         // one thread: the sums do not descend
    __syncthreads();
    bin = s.bin; count_before = s.pick_count; mass_before = s.pick_mass;
    __syncthreads();
}

// Rank word of the last token kept by a setting that keeps the first tokens up to a count, or up to a sum of weights (want >= 1, reached by all tokens together).
// `in`: the tokens that have not been told apart yet; count and mass before them come off `want`.  mass_upto: weights of all tokens up to the found one, from
// `before` on.
template <class In>
static __device__ u64 find_last(const sample_args &a, sample_shared &s, const float *l, const weigher &weigh, In in, bool by_mass, u64 want, uint32_t n_in, u64 before, u64 &mass_upto) {
    const int t = threadIdx.x;
    u64 lo = 0, hi = ~0ull;
    while (n_in > SM_LIST) {
        // finer bins between the least and the greatest rank word there are
        u64 least = ~0ull, most = 0;
        for (int i = t; i < a.n; i += SM_THREADS) {
            const float v = l[i];
            const u64 x = rank_word(v, i);
            if (in(v) && x >= lo && x <= hi) { least = x < least ? x : least; most = x > most ? x : most; }
        }
        s.mass[t] = 0; s.count[t] = 0;
        if (t == 0) { s.x[0] = ~0ull; s.x[1] = 0; }
        __syncthreads();
        atomicMin(&s.x[0], least);
        atomicMax(&s.x[1], most);
        __syncthreads();
        least = s.x[0]; most = s.x[1];
        const int shift = max(0, 64 - __clzll((long long)(most - least)) - 10);
        for (int i = t; i < a.n; i += SM_THREADS) {
            const float v = l[i];
            const u64 x = rank_word(v, i);
            if (in(v) && x >= least && x <= most) {
                const int b = (int)((x - least) >> shift);
                atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.mass[b], weigh(v));
            }
        }
        __syncthreads();
        int bin;
        uint32_t cb;
        u64 mb;
        find_bin(s, by_mass, want, bin, cb, mb);
        n_in = s.count[bin];
        want -= by_mass ? mb : cb;
        before += mb;
        lo = least + ((u64)bin << shift);
        hi = lo + ((1ull << shift) - 1);
        __syncthreads();
    }
    // the tokens left, by rank
    if (t == 0) s.n_list = 0;
    __syncthreads();
    for (int i = t; i < a.n; i += SM_THREADS) {
        const float v = l[i];
        const u64 x = rank_word(v, i);
        if (in(v) && x >= lo && x <= hi) { const uint32_t k = atomicAdd(&s.n_list, 1u); s.x[k] = x; s.w[k] = weigh(v); }
    }
    __syncthreads();
    const int m = s.n_list;
    if (t < m) {
        const u64 x = s.x[t];
        uint32_t rank = 0;
        u64 sum = 0;
        for (int k = 0; k < m; k++) { const bool upto = s.x[k] <= x; rank += upto; sum += upto ? s.w[k] : 0; }
        const u64 w = s.w[t];
        if (by_mass ? sum >= want && sum - w < want : rank == want) { s.pick = x; s.pick_mass = sum; }
    }
    __syncthreads();
    const u64 x = s.pick;
    mass_upto = before + s.pick_mass;
    __syncthreads();
    return x;
}

__global__ __launch_bounds__(SM_THREADS) void sample_kernel(sample_args a) {
    __shared__ sample_shared s;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
    const float *l = (const float *)(a.logits + row * a.stride);
    const float temp = a.temperature ? a.temperature[row] : 1.0f;
    float top = -INFINITY;
    for (int i = t; i < a.n; i += SM_THREADS) top = fmaxf(top, l[i]);           // NaN never wins
    top = wave_max(top);
    if (lane == 0) s.wave_f[wave] = top;
    __syncthreads();
    for (int w = 0; w < 16; w++) top = fmaxf(top, s.wave_f[w]);
    if (top == -INFINITY) {
        if (t == 0) { a.tokens[row] = -1; if (a.probs) a.probs[row] = 0.0f; }
        return;
    }
    if (!(temp > 0.0f)) {
        if (t == 0) s.bin = 0x7FFFFFFF;
        __syncthreads();
        int first = 0x7FFFFFFF;
        for (int i = t; i < a.n; i += SM_THREADS) if (l[i] == top) { first = i; break; }
        if (first != 0x7FFFFFFF) atomicMin(&s.bin, first);
        __syncthreads();
        if (t == 0) { a.tokens[row] = s.bin; if (a.probs) a.probs[row] = 1.0f; }
        return;
    }
    weigher weigh;
    const double c = 1.4426950408889634074 / (double)temp;
    weigh.top = top; weigh.c = (float)c; weigh.c_lo = (float)(c - (double)weigh.c);
    if (!(weigh.c <= 3.4e38f)) { weigh.c = 3.4e38f; weigh.c_lo = 0.0f; }          // a temperature next to 0
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, mp = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
    const bool by_rank = k > 0 && k < a.n, by_mass = p < 1.0f;
    u64 last = ~0ull;                                                             // rank word of the last token kept
    if (mp > 0.0f && temp < INFINITY) {
        // w >= mp as a limit of the logit, in 64 bits, rounded up to a float
        const double limit = (double)top + (double)temp * log((double)mp);
        float f = (float)limit;
        if ((double)f < limit) f = nextafterf(f, INFINITY);
        last = (u64)order_word(fminf(f, top)) << 32 | 0xFFFFFFFFu;
    }
    if (by_rank || by_mass) {
        s.mass[t] = 0; s.count[t] = 0;
        __syncthreads();
        const auto bin_of = [&](float v) { return (int)fminf(weigh.far(v) * 32.0f, (float)(SM_BINS - 1)); };
        for (int i = t; i < a.n; i += SM_THREADS) {
            const float v = l[i];
            if (!(v > -INFINITY)) continue;
            const int b = bin_of(v);
            atomicAdd(&s.count[b], 1u);
            atomicAdd(&s.mass[b], weigh(v));
        }
        __syncthreads();
        u64 all = s.mass[t];
        uint32_t number = s.count[t];
        block_scan(s, all, number);
        __syncthreads();
        if (t == SM_BINS - 1) { s.pick_mass = all; s.pick_count = number; }
        __syncthreads();
        all = s.pick_mass; number = s.pick_count;
        __syncthreads();
        int bin;
        uint32_t cb;
        u64 mb, upto = all;
        const u64 first_mass = s.mass[t];
        const uint32_t first_count = s.count[t];
        if (by_rank && (uint32_t)k < number) {
            find_bin(s, false, (u64)k, bin, cb, mb);
            const uint32_t n_in = s.count[bin];
            __syncthreads();
            const u64 x = find_last(a, s, l, weigh, [&](float v) { return v > -INFINITY && bin_of(v) == bin; }, false, (u64)k - cb, n_in, mb, upto);
            last = x < last ? x : last;
        }
        if (by_mass) {
            s.mass[t] = first_mass; s.count[t] = first_count;
            __syncthreads();
            // the sum that the kept tokens have to reach: the least whole number that is not below p * upto
            const double want_d = (double)fmaxf(p, 0.0f) * (double)upto;
            u64 want = (u64)want_d;
            want += (double)want < want_d;
            if (want < 1) want = 1;
            if (want > upto) want = upto;
            find_bin(s, true, want, bin, cb, mb);
            const uint32_t n_in = s.count[bin];
            __syncthreads();
            u64 unused;
            const u64 x = find_last(a, s, l, weigh, [&](float v) { return v > -INFINITY && bin_of(v) == bin; }, true, want - mb, n_in, mb, unused);
            last = x < last ? x : last;
        }
    }
    // The kept weights by ranges of the index, then inside the range that the random number falls into
    const int span = ((a.n + SM_THREADS - 1) / SM_THREADS + 63) & ~63;            // whole waves of tokens
    const auto weight = [&](int i) -> u64 {
        const float v = l[i];
        return v > -INFINITY && rank_word(v, i) <= last ? weigh(v) : 0;
    };
    const int n_span = (a.n + span - 1) / span;
    for (int g = wave; g < SM_BINS; g += 16) {
        u64 sum = 0;
        if (g < n_span) for (int i = g * span + lane; i < min((g + 1) * span, a.n); i += 64) sum += weight(i);
        sum = wave_sum_u64(sum);
        if (lane == 0) { s.mass[g] = sum; s.count[g] = 0; }
    }
    __syncthreads();
    u64 total = s.mass[t];
    uint32_t zero = 0;
    block_scan(s, total, zero);
    __syncthreads();
    if (t == SM_BINS - 1) s.pick_mass = total;
    __syncthreads();
    total = s.pick_mass;
    __syncthreads();
    // first token whose running sum exceeds u * total, u in [0, 1) as a multiple of 2^-64
    float u = a.uniform[row];
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    const u64 u64s = u >= 5.421010862427522e-20f ? (u64)((double)u * 18446744073709551616.0) : 0;
    const u64 want = __umul64hi(u64s, total) + 1;                                 // running sum >= floor(u * total) + 1
    int bin;
    uint32_t cb;
    u64 mb;
    find_bin(s, true, want, bin, cb, mb);
    if (wave == 0) {
        u64 left = want - mb;
        for (int base = bin * span; ; base += 64) {
            const int i = base + lane;
            const u64 w = i < min((bin + 1) * span, a.n) ? weight(i) : 0;
            u64 sum = w;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) { const u64 v = __shfl_up(sum, o, SPY_WAVE); if (lane >= o) sum += v; }
            const unsigned long long past = __ballot(sum >= left);
            if (past) {
                if (lane == __ffsll(past) - 1) {
                    a.tokens[row] = i;
                    if (a.probs) a.probs[row] = (float)((double)w / (double)total);
                }
                break;
            }
            left -= __shfl(sum, 63, SPY_WAVE);
            if (base + 64 >= min((bin + 1) * span, a.n)) break;                   // (not reached: the range holds the sum)
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
    SPY_CHECK_ARG(n > 0 && n < (1 << 19) && n_row > 0 && n_row < (1ll << 31) && logits->ne[2] == 1 && logits->ne[3] == 1 && logits->nb[0] == 4 && logits->nb[1] % 4 == 0);
    SPY_CHECK_ARG((((uintptr_t)logits->data | (uintptr_t)tokens | (uintptr_t)probs | (uintptr_t)param->temperature | (uintptr_t)param->top_k | (uintptr_t)param->top_p |
                    (uintptr_t)param->min_p | (uintptr_t)param->uniform) & 3) == 0);
    sample_args a;
    a.logits = (const uint8_t *)logits->data; a.stride = logits->nb[1]; a.n = (int)n;
    a.temperature = param->temperature; a.top_p = param->top_p; a.min_p = param->min_p; a.uniform = param->uniform; a.top_k = param->top_k;
    a.tokens = tokens; a.probs = probs;
    sample_kernel<<<dim3((unsigned)n_row), dim3(SM_THREADS), 0, (hipStream_t)stream>>>(a);
    return SPY_LAUNCH_RC();
}
