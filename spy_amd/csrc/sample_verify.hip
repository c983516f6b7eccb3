// Drafted tokens against what the target model would have drawn (sample.cuh has the distributions): token d of row i is taken where a_i q_i(d) < p_i(d), p the target's and q the
// draft's distribution and a_i a given random number; the first that is not taken is replaced by one drawn from max(p_i - q_i, 0), and behind the last one that is taken one is drawn from p.
// Tokens that come out are distributed as the target's alone: min(p, q) of d is what the draft proposes and is taken, and max(p - q, 0) is what p has beyond that.
//
// First launch: a workgroup for each row and distribution finds what the settings leave -- the last rank word, the sum of the weights and d's own (sample_row_of<true>), and the tokens themselves where
// they are 1024 at most.  Second launch: four workgroups for each request find the row where its drafts end and draw there, one of them alone where it has those tokens.  p and q are weights over
// their sums, in 64 bits; p - q is held as a multiple of 2^-60 (itself off by 2^-50 of the larger of them, verify_share.h), so that sums of it are exact in any order, and what comes out is the same each time.
//
// Latency and vector instructions: the first launch reads each row once from memory (verify of 32 requests with 1 to 6 rows of 32000 and a drafter's: 37.6 us, 24.6 of them here), and where top_p alone is set it
// works out every weight: 160 rows of 100003 by as many workgroups 55 us, 12 for the reads, 24 for the weights (20 instructions a token beside an addition in LDS), 17 for the bin's tokens.  The
// second is a chain of dependent reads (one request: 6 us) and, where more tokens are left, one pass over the row: 18 us for 64 requests of 100003.  One request with 5 rows of 32000: 21 us in all.  Taking the
// weights of tokens that are not left as well took 102 us for the large case; three launches, the parts' sums one of their own, 0.3 to 0.8 more than two.
#include "launch_index.h"
#include "paged.cuh"
#include "sample.cuh"
#include "verify_share.h"

int *spy_hip_err_flag_ptr();

struct verify_args {
    sample_args target, draft;
    const int32_t *drafted, *row_start;
    const float *accept;
    int n_seq, n_row;
    int32_t *tokens, *accepted;
    float *probs;
    sample_cut *cuts;                    // of the target's rows, then of the draft's
    u64 *kept;                           // of the target's rows: SM_KEPT each
    u64 *sums;                           // of the requests: VF_PARTS each
    int32_t *arrived;                    // of the requests: workgroups that have added up their parts
    int32_t *owner;                      // of the target's rows: the request that it was looked at for, or -1
    int *err;
};

__global__ __launch_bounds__(SM_THREADS) void verify_cut_kernel(verify_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int side = (int)blockIdx.x >= a.n_row, r = blockIdx.x - side * a.n_row, lane = threadIdx.x & 63;
    for (int64_t i = launch_first(blockIdx.x, SM_THREADS, threadIdx.x); i < a.n_seq; i += launch_step(gridDim.x, SM_THREADS)) a.arrived[i] = 0;
    // The row's request: the first that ends behind it, looked for from the first one on, so that one that begins before the end of another in front of it has none of that one's rows, whatever lies between.
    // 64 at a time: of 1024 requests of two rows (vocabulary of 12) it takes nothing beside the rows' work, 185 us in all; of 65536 it is most of 49 ms.
    int row0 = -1, row1 = -1, owner = -1;
    for (int base = 0; base < a.n_seq; base += 64) {
        const int s = min(base + lane, a.n_seq - 1), from = a.row_start[s], to = a.row_start[s + 1];
        const unsigned long long past = __ballot(base + lane < a.n_seq && to > r);
        if (!past) continue;
        const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
        row0 = __builtin_amdgcn_readlane(from, at);
        row1 = __builtin_amdgcn_readlane(to, at);
        owner = row0 >= 0 && r >= row0 && row1 <= a.n_row ? base + at : -1;
        break;
    }
    if (!side && threadIdx.x == 0) a.owner[r] = owner;
    if (owner < 0 || (side && r == row1 - 1)) return;
    const int d = r < row1 - 1 ? a.drafted[r] : -1;
    sample_row_of<true>(side ? a.draft : a.target, smem, r, d, a.cuts + side * (int64_t)a.n_row + r, side ? nullptr : a.kept + (int64_t)r * SM_KEPT);
}

// What settings leave of a row
struct verify_left {
    weigher weigh;
    float last_l;
    int last_i;
    bool infinite;
    __device__ __forceinline__ verify_left(float temp, const sample_cut &c) {
        const u64 last = c.last;
        weigh = weigher_of(temp > 0.0f ? temp : 1.0f, c.top);                     // (the only token left of a greedy row has the largest logit: any temperature)
        last_l = last == ~0ull ? -INFINITY : logit_of(last);
        last_i = (int)(uint32_t)min(last & 0xFFFFFFFFull, 0x7FFFFFFFull);
        infinite = c.infinite;
    }
    __device__ __forceinline__ float clean(float v) const { return infinite ? (v == INFINITY ? 0.0f : -INFINITY) : v; }          // (a NaN is never left)
    __device__ __forceinline__ bool has(float v, int i) const { return (v > -INFINITY) & ((v > last_l) | ((v == last_l) & (i <= last_i))); }
};
static __device__ __forceinline__ double share_of_all(u64 w, u64 all) { return all ? (double)w / (double)all : 0.0; }
static __device__ __forceinline__ double verify_p(const verify_args &a, int64_t r) { return share_of_all(a.cuts[r].weight, a.cuts[r].total); }

// Weights of the tokens of row `stop`, where a request's drafts end: of p - q, or -- as_p -- of p
struct verify_weights {
    verify_left p, q;
    const float *gp, *gq;
    int n, drafted;
    bool beyond_q, as_p;
    double one_p, one_q;
    __device__ __forceinline__ verify_weights(const verify_args &a, int stop, bool at_end, int drafted_, float temp_p, const sample_cut &cut_p, float temp_q, const sample_cut &cut_q) : p(temp_p, cut_p), q(temp_q, cut_q) {
        beyond_q = !at_end && a.draft.logits;
        as_p = at_end;
        gp = (const float *)(a.target.logits + stop * a.target.stride);
        gq = beyond_q ? (const float *)(a.draft.logits + stop * a.draft.stride) : gp;
        n = a.target.n;
        drafted = at_end ? -1 : drafted_;
        one_p = 1.0 / (double)cut_p.total;
        one_q = beyond_q && cut_q.total ? 1.0 / (double)cut_q.total : 0.0;
    }
    // of a token that p has, with the logits v (as p.clean() has it) and l
    __device__ __forceinline__ u64 operator()(float v, float l, int i) const {
        const u64 w = p.weigh(v);
        if (as_p) return w;
        if (!beyond_q) return i == drafted ? 0 : w;
        l = q.clean(l);
        return verify_more(w, one_p, q.has(l, i) ? q.weigh(l) : 0, one_q);
    }
    // By a wave: f(weight, token, its logit; 0, 0, 0 where there is none) for the tokens from .. to - 1 that p has, in order of index, a token a lane.  They are looked for first, 256 at a time, in `list`:
    // a weight takes some hundred instructions, and few tokens of many have one.
    template <class F> __device__ __forceinline__ void each(int from, int to, uint2 *list, F f) const {
        const int lane = threadIdx.x & 63;
        float x[4], ahead[4];
#pragma unroll
        for (int j = 0; j < 4; j++) ahead[j] = gp[min(from + 64 * j + lane, n - 1)];
        for (int base = from; base < to; base += 256) {
#pragma unroll
            for (int j = 0; j < 4; j++) { x[j] = ahead[j]; ahead[j] = gp[min(base + 256 + 64 * j + lane, n - 1)]; }
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int i = base + 64 * j + lane;
                const float v = p.clean(x[j]);
                const unsigned long long who = __ballot(i < to && p.has(v, i));
                if (i < to && p.has(v, i)) list[m + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = make_uint2((uint32_t)i, __float_as_uint(v));
                m += (uint32_t)__popcll(who);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
            for (uint32_t k = 0; k < m; k += 64) {
                const bool there = k + lane < m;
                const uint2 e = there ? list[k + lane] : make_uint2(0, 0);
                const float l = beyond_q && there ? gq[e.x] : 0.0f;
                f(there ? (*this)(__uint_as_float(e.y), l, (int)e.x) : 0, (int)e.x, __uint_as_float(e.y));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
            __builtin_amdgcn_wave_barrier();
        }
    }
    __device__ __forceinline__ u64 sum(int from, int to, uint2 *list) const {     // by a wave, to every lane
        u64 all = 0;
        each(from, to, list, [&](u64 w, int, float) { all += w; });
        return of_lane(wave_scan(all), 63);
    }
};
#define VF_PARTS 64
#define VF_BLOCKS (VF_PARTS / 16)
static __device__ __forceinline__ void verify_part(int n, int part, int &from, int &to) {
    const int size = (n + VF_PARTS - 1) / VF_PARTS;
    from = min(part * size, n); to = min(from + size, n);
}

// Four workgroups to a request.  Each finds where its drafts end.  Where the tokens that are left of that row are known, the first one draws; else each wave adds up the weights of a part of the row, and the
// workgroup that is done last draws (a.arrived: zeroed by the launch before).
__global__ __launch_bounds__(SM_THREADS) void verify_draw_kernel(verify_args a) {
    __shared__ sample_shared s;
    __shared__ uint2 s_list[16][256];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), request = blockIdx.x / VF_BLOCKS, block = blockIdx.x % VF_BLOCKS;
    const int row0 = a.row_start[request], row1 = a.row_start[request + 1];
    if (row0 < 0 || row1 < row0 || row1 > a.n_row) { if (a.err) *a.err = 1; return; }
    if (row0 == row1) return;
    const int owner = a.owner[min(row0 + lane, row1 - 1)];                        // (asked for here, looked at below)
    int stop = row1 - 1;
    for (int base = row0; base < row1 - 1; base += 64) {
        const int r = min(base + lane, row1 - 2);
        const float u = a.accept[r] > 0.0f ? fminf(a.accept[r], 0.99999994f) : 0.0f;
        const double p = verify_p(a, r), q = a.draft.logits ? verify_p(a, (int64_t)a.n_row + r) : 1.0;        // (no distribution: the draft is certain)
        const unsigned long long not_taken = __ballot(!((double)u * q < p));
        if (not_taken) { stop = min(base + __ffsll(not_taken) - 1, row1 - 2); break; }
    }
    stop = __builtin_amdgcn_readfirstlane(stop);
    // rows that one of the requests before it goes further than are that one's
    bool taken = __any(owner != request);
    for (int base = row0 + 64; base < row1; base += 64) taken |= __any(a.owner[min(base + lane, row1 - 1)] != request);
    if (taken) { if (a.err) *a.err = 1; return; }
    // all that the draw wants of the row, requested together
    const bool at_end = stop == row1 - 1;
    const sample_cut cut_p = a.cuts[stop], cut_q = a.cuts[(at_end || !a.draft.logits ? 0 : (int64_t)a.n_row) + stop];
    const float temp_p = a.target.temperature ? a.target.temperature[stop] : 1.0f, temp_q = a.draft.temperature ? a.draft.temperature[stop] : 1.0f, u = a.target.uniform[stop];
    const int drafted = a.drafted[stop];
    const u64 x = a.kept[(int64_t)stop * SM_KEPT + t], c_total = cut_p.total;     // (whatever lies there, where there are fewer)
    const uint32_t n_kept = cut_p.n_kept;
    const bool many = c_total && n_kept > SM_KEPT;
    if (block && !many) return;
    verify_weights weights(a, stop, at_end, drafted, temp_p, cut_p, temp_q, cut_q);
    if (many) {
        int from, to;
        verify_part(weights.n, 16 * block + wave, from, to);
        const u64 sum = weights.sum(from, to, s_list[wave]);
        if (lane == 0) s.part[wave] = sum;
        __syncthreads();
        // One wave stores the sums of all and counts the workgroup: a release waits for its own wave's stores, and a barrier for nobody's
        if (wave == 0) {
            if (lane < 16) __hip_atomic_store(a.sums + (int64_t)request * VF_PARTS + 16 * block + lane, s.part[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (lane == 0) s.bin = __hip_atomic_fetch_add(a.arrived + request, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (s.bin != VF_BLOCKS - 1) return;
    }
    for (int r = row0 + t; r < row1; r += SM_THREADS) {
        if (r == stop) continue;
        a.tokens[r] = r < stop ? a.drafted[r] : -1;
        if (a.probs) a.probs[r] = r < stop ? (float)verify_p(a, r) : 0.0f;
    }
    if (t == 0) {
        a.accepted[request] = stop - row0;
        if (!c_total) { a.tokens[stop] = -1; if (a.probs) a.probs[stop] = 0.0f; }
    }
    if (!c_total) return;                                                         // a row without a logit above -inf
    const auto drawn = [&](int i, float v) { a.tokens[stop] = i; if (a.probs) a.probs[stop] = (float)share_of_all(weights.p.weigh(v), c_total); };
    if (n_kept <= SM_KEPT) {
        // one token a thread
        const bool there = (uint32_t)t < n_kept;
        const float v = there ? logit_of(x) : -INFINITY;
        const int i = there ? (int)(uint32_t)x : 0, range = i >> a.target.range_log2;
        const float l = there && weights.beyond_q ? weights.gq[i] : 0.0f;
        s.mass[t] = 0;
        if (t == 0) s.n_list = 0;
        u64 w, total, before, all;
        for (;;) {
            w = there ? weights(v, l, i) : 0;
            block_scan(s, w, total);
            if (weights.as_p || total) break;
            weights.as_p = true;                                                  // p and q are the same but for their roundings
            __syncthreads();
        }
        const u64 want = draw_at(u, total);
        // in order of index: weights by range of the index, then inside one of the ranges
        if (w) atomicAdd(&s.mass[range], w);
        __syncthreads();
        const int in = find_bin(s, s.mass[t], want, before, all);
        const bool mine = w && range == in;
        if (mine) { const uint32_t k = atomicAdd(&s.n_list, 1u); s.x[k] = (uint32_t)i; s.w[k] = w; }
        __syncthreads();
        if (mine) {
            u64 upto = before + w;
            for (uint32_t j = 0; j < s.n_list; j++) if (s.x[j] < (uint32_t)i) upto += s.w[j];
            if (upto >= want && upto - w < want) drawn(i, v);
        }
        return;
    }
    u64 sums = wave_scan(__hip_atomic_load(a.sums + (int64_t)request * VF_PARTS + lane, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    if (!weights.as_p && !of_lane(sums, 63)) {
        weights.as_p = true;                                                      // as above: the sums once more, four parts by each wave
        for (int k = 0; k < VF_PARTS / 16; k++) {
            int from, to;
            verify_part(weights.n, 16 * k + wave, from, to);
            const u64 sum = weights.sum(from, to, s_list[wave]);
            if (lane == 0) s.mass[16 * k + wave] = sum;
        }
        __syncthreads();
        sums = wave_scan(s.mass[lane]);
    }
    // the part that the random number falls into, a sixteenth of it by each wave, then a token a lane
    const u64 want_all = draw_at(u, of_lane(sums, 63));
    const int part = max(__ffsll(__ballot(sums >= want_all)) - 1, 0);
    u64 want = want_all - (part ? of_lane(sums, part - 1) : 0);
    int from, to;
    verify_part(weights.n, part, from, to);
    const int size = (to - from + 15) / 16, begin = min(from + wave * size, to), end = min(begin + size, to);
    const u64 sum = weights.sum(begin, end, s_list[wave]);
    if (lane == 0) s.part[wave] = sum;
    __syncthreads();
    const u64 parts = row_scan(s.part[lane & 15]);
    if (wave != max(__ffsll(__ballot(parts >= want)) - 1, 0)) return;
    want -= wave ? of_lane(parts, wave - 1) : 0;
    u64 before = 0;
    weights.each(begin, end, s_list[wave], [&](u64 w, int i, float v) {
        const u64 upto = before + wave_scan(w);
        if (w && upto >= want && upto - w < want) drawn(i, v);
        before = of_lane(upto, 63);
    });
}

static inline size_t verify_cuts(int64_t n_row) { return ((size_t)n_row * 2 * sizeof(sample_cut) + 255) / 256 * 256; }
static inline size_t verify_scratch(int64_t n_row, int64_t n_seq) { return verify_cuts(n_row) + (size_t)n_row * (SM_KEPT * 8 + 4) + (size_t)n_seq * (VF_PARTS * 8 + 4); }
extern "C" size_t spy_hip_sample_verify_scratch_size(const spy_hip_tensor *logits, int32_t n_seq) {
    return logits && n_seq > 0 && logits->ne[1] > 0 && logits->ne[1] < (1 << 22) ? verify_scratch(logits->ne[1], n_seq) : 0;
}

extern "C" int spy_hip_sample_verify(void *stream, const spy_hip_tensor *logits, const spy_hip_sample_param *param, const spy_hip_tensor *draft_logits, const spy_hip_sample_param *draft_param,
                                     const int32_t *drafted, const int32_t *row_start, int32_t n_seq, const float *accept, int32_t *tokens, int32_t *accepted, float *probs, void *scratch,
                                     size_t scratch_bytes) {
    SPY_CHECK_ARG(logits && param && logits->data && param->uniform && drafted && row_start && accept && tokens && accepted && n_seq > 0 && n_seq <= (1 << 20));
    SPY_CHECK_ARG((((uintptr_t)drafted | (uintptr_t)row_start | (uintptr_t)accept | (uintptr_t)tokens | (uintptr_t)accepted | (uintptr_t)probs) & 3) == 0);
    const spy_hip_sample_param none = {};
    if (!draft_param) draft_param = &none;
    int rc = sample_check(logits, param);
    if (!rc && draft_logits) rc = sample_check(draft_logits, draft_param);
    if (rc) return rc;
    SPY_CHECK_ARG(!draft_logits || (draft_logits->data && draft_logits->ne[0] == logits->ne[0] && draft_logits->ne[1] == logits->ne[1]));
    const int64_t n_row = logits->ne[1], blocks = n_row * (draft_logits ? 2 : 1);
    SPY_CHECK_ARG(blocks * SM_THREADS < (1ll << 32) && (int64_t)n_seq * VF_BLOCKS * SM_THREADS < (1ll << 32));
    if (scratch_bytes < verify_scratch(n_row, n_seq)) return SPY_HIP_ENOSPACE;
    SPY_CHECK_ARG(scratch && ((uintptr_t)scratch & 255) == 0);
    verify_args a;
    a.target = sample_args_of(logits, param);
    a.draft = draft_logits ? sample_args_of(draft_logits, draft_param) : a.target;
    if (!draft_logits) a.draft.logits = nullptr;
    a.drafted = drafted; a.row_start = row_start; a.accept = accept; a.n_seq = n_seq; a.n_row = (int)n_row;
    a.tokens = tokens; a.accepted = accepted; a.probs = probs; a.err = spy_hip_err_flag_ptr();
    a.cuts = (sample_cut *)scratch; a.kept = (u64 *)((uint8_t *)scratch + verify_cuts(n_row)); a.sums = a.kept + n_row * SM_KEPT; a.arrived = (int32_t *)(a.sums + (int64_t)n_seq * VF_PARTS); a.owner = a.arrived + n_seq;
    const size_t lds = sample_lds(a.target);
    rc = spy_raise_lds_limit((const void *)verify_cut_kernel, lds);
    if (rc) return rc;
    verify_cut_kernel<<<dim3((unsigned)blocks), dim3(SM_THREADS), lds, (hipStream_t)stream>>>(a);
    rc = SPY_LAUNCH_RC();
    if (rc) return rc;
    verify_draw_kernel<<<dim3((unsigned)n_seq * VF_BLOCKS), dim3(SM_THREADS), 0, (hipStream_t)stream>>>(a);
    return SPY_LAUNCH_RC();
}
