// Drafted tokens against what the target model would have drawn (sample.cuh has the distributions): token d of row i is taken where a_i q_i(d) < p_i(d), p the target's and q the
// draft's distribution and a_i a given random number; the first that is not taken is replaced by one drawn from max(p_i - q_i, 0), and behind the last one that is taken one is drawn from p.
// Tokens that come out are distributed as the target's alone: min(p, q) of d is what the draft proposes and is taken, and max(p - q, 0) is what p has beyond that.
//
// First launch: a workgroup for each row and distribution finds what the settings leave -- the last rank word, the sum of the weights and d's own (sample_row_of<true>).  Second launch: a
// workgroup for each request finds the row where its drafts end and draws there.  p and q are weights over their sums, in 64 bits; p - q as multiples of 2^-60, so that sums of it are
// exact in any order.
#include "paged.cuh"
#include "sample.cuh"

int *spy_hip_err_flag_ptr();

struct verify_args {
    sample_args target, draft;
    const int32_t *drafted, *row_start;
    const float *accept;
    int n_seq, n_row;
    int32_t *tokens, *accepted;
    float *probs;
    sample_cut *cuts;                    // of the target's rows, then of the draft's
    int *err;
};

__global__ __launch_bounds__(SM_THREADS) void verify_cut_kernel(verify_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int side = (int)blockIdx.x >= a.n_row, r = blockIdx.x - side * a.n_row, lane = threadIdx.x & 63;
    int row0 = -1, row1 = -1;                                                     // of the row's request: the first that ends behind it
    for (int base = 0; base < a.n_seq; base += 64) {
        const int s = min(base + lane, a.n_seq - 1), from = a.row_start[s], to = a.row_start[s + 1];
        const unsigned long long past = __ballot(base + lane < a.n_seq && to > r);
        if (!past) continue;
        const int at = __builtin_amdgcn_readfirstlane(__ffsll(past) - 1);
        row0 = __builtin_amdgcn_readlane(from, at);
        row1 = __builtin_amdgcn_readlane(to, at);
        break;
    }
    if (row0 < 0 || r < row0 || row1 > a.n_row || (side && r == row1 - 1)) return;
    const int d = r < row1 - 1 ? a.drafted[r] : -1;
    sample_row_of<true>(side ? a.draft : a.target, smem, r, d, a.cuts + side * (int64_t)a.n_row + r);
}

__global__ __launch_bounds__(SM_THREADS) void verify_draw_kernel(verify_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    sample_shared &s = *(sample_shared *)smem;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), row0 = a.row_start[blockIdx.x], row1 = a.row_start[blockIdx.x + 1];
    if (row0 < 0 || row1 < row0 || row1 > a.n_row) { if (a.err) *a.err = 1; return; }
    if (row0 == row1) return;
    const bool drawn_from = a.draft.logits != nullptr;                            // else a draft is certain of its token
    const auto share = [](u64 w, u64 all) { return all ? (double)w / (double)all : 0.0; };
    int stop = row1 - 1;
    for (int base = row0; base < row1 - 1; base += 64) {
        const int r = min(base + lane, row1 - 2);
        const float u = a.accept[r] > 0.0f ? fminf(a.accept[r], 0.99999994f) : 0.0f;
        const double p = share(a.cuts[r].weight, a.cuts[r].total), q = drawn_from ? share(a.cuts[a.n_row + (int64_t)r].weight, a.cuts[a.n_row + (int64_t)r].total) : 1.0;
        const unsigned long long not_taken = __ballot(!((double)u * q < p));
        if (not_taken) { stop = min(base + __builtin_amdgcn_readfirstlane(__ffsll(not_taken) - 1), row1 - 2); break; }
    }
    const sample_cut c = a.cuts[stop];
    const bool at_end = stop == row1 - 1;
    const int drafted = at_end ? -1 : a.drafted[stop];
    for (int r = row0 + t; r < row1; r += SM_THREADS) {
        if (r == stop) continue;
        a.tokens[r] = r < stop ? a.drafted[r] : -1;
        if (a.probs) a.probs[r] = r < stop ? (float)share(a.cuts[r].weight, a.cuts[r].total) : 0.0f;
    }
    if (t == 0) {
        a.accepted[blockIdx.x] = stop - row0;
        if (!c.total) { a.tokens[stop] = -1; if (a.probs) a.probs[stop] = 0.0f; }
    }
    if (!c.total) return;                                                         // a row without a logit above -inf
    const sample_args &g = a.target;
    sample_row row;
    row.g = (const float *)(g.logits + stop * g.stride);
    row.n = g.n; row.begin = wave * g.part; row.part = g.part; row.held = g.held; row.infinite = c.infinite;
    f4 *const held = (f4 *)(smem + sizeof(sample_shared));
    row.lds = held + wave * (g.held / 4);
    row.load(0);
    struct left {                                                                 // what settings leave of a row
        weigher weigh;
        float last_l;
        int last_i;
        __device__ __forceinline__ left(const sample_args &g, const sample_cut &c, int r) {
            const float temp = g.temperature ? g.temperature[r] : 1.0f;
            weigh = weigher_of(temp > 0.0f ? temp : 1.0f, c.top);                 // (the only token left of a greedy row has the largest logit: any temperature)
            last_l = c.last == ~0ull ? -INFINITY : logit_of(c.last);
            last_i = (int)(uint32_t)min(c.last & 0xFFFFFFFFull, 0x7FFFFFFFull);
        }
        __device__ __forceinline__ bool has(float v, int i) const { return (v > -INFINITY) & ((v > last_l) | ((v == last_l) & (i <= last_i))); }
    };
    const left p(g, c, stop);
    sample_cut cq = {0, 0, 0, 0.0f, 0};
    const bool beyond_q = !at_end && drawn_from;
    if (beyond_q) cq = a.cuts[a.n_row + (int64_t)stop];
    const left q(a.draft, cq, stop);
    const float *const gq = (const float *)(a.draft.logits + stop * a.draft.stride);
    const double one_p = 1.0 / (double)c.total, one_q = cq.total ? 1.0 / (double)cq.total : 0.0;
    bool as_p = at_end;                                                           // from p itself
    const auto weight = [&](float v, int i) -> u64 {
        if (!p.has(v, i)) return 0;
        const u64 w = p.weigh(v);
        if (as_p) return w;
        if (!beyond_q) return i == drafted ? 0 : w;
        float l = gq[i];
        l = cq.infinite ? (l == INFINITY ? 0.0f : -INFINITY) : l;                 // (a NaN is not left by any setting)
        const double more = (double)w * one_p - (q.has(l, i) && cq.total ? (double)q.weigh(l) * one_q : 0.0);
        return more > 0.0 ? (u64)(more * 0x1p60) : 0;
    };
    for (;;) {
        u64 sum = 0;
        row.groups([&](f4 v, int i) {
            bool some = false;
#pragma unroll
            for (int e = 0; e < 4; e++) some |= p.has(v[e], i + e);
            if (!__any(some)) return;
#pragma unroll
            for (int e = 0; e < 4; e++) sum += weight(v[e], i + e);
        });
        sum = of_lane(wave_scan(sum), 63);
        if (lane == 0) s.part[wave] = sum;
        __syncthreads();
        if (as_p || of_lane(row_scan(s.part[lane & 15]), 15)) break;
        as_p = true;                                                              // p and q are the same but for their roundings
        __syncthreads();
    }
    const float u = g.uniform[stop];
    draw_by_parts(g, s, row, held, u, weight, [&](int i, u64, u64) {
        a.tokens[stop] = i;
        if (a.probs) a.probs[stop] = (float)share(p.weigh(row.clean(f4{row.g[i], 0.0f, 0.0f, 0.0f})[0]), c.total);
    });
}

extern "C" size_t spy_hip_sample_verify_scratch_size(const spy_hip_tensor *logits, int32_t n_seq) {
    return logits && n_seq > 0 && logits->ne[1] > 0 && logits->ne[1] < (1 << 22) ? (size_t)logits->ne[1] * 2 * sizeof(sample_cut) : 0;
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
    SPY_CHECK_ARG(blocks * SM_THREADS < (1ll << 32) && (int64_t)n_seq * SM_THREADS < (1ll << 32));
    if (scratch_bytes < (size_t)n_row * 2 * sizeof(sample_cut)) return SPY_HIP_ENOSPACE;
    SPY_CHECK_ARG(scratch && ((uintptr_t)scratch & 255) == 0);
    verify_args a;
    a.target = sample_args_of(logits, param);
    a.draft = draft_logits ? sample_args_of(draft_logits, draft_param) : a.target;
    if (!draft_logits) a.draft.logits = nullptr;
    a.drafted = drafted; a.row_start = row_start; a.accept = accept; a.n_seq = n_seq; a.n_row = (int)n_row;
    a.tokens = tokens; a.accepted = accepted; a.probs = probs; a.cuts = (sample_cut *)scratch; a.err = spy_hip_err_flag_ptr();
    const size_t lds = sample_lds(a.target);
    rc = spy_raise_lds_limit((const void *)verify_cut_kernel, lds);
    if (!rc) rc = spy_raise_lds_limit((const void *)verify_draw_kernel, lds);
    if (rc) return rc;
    verify_cut_kernel<<<dim3((unsigned)blocks), dim3(SM_THREADS), lds, (hipStream_t)stream>>>(a);
    rc = SPY_LAUNCH_RC();
    if (rc) return rc;
    verify_draw_kernel<<<dim3((unsigned)n_seq), dim3(SM_THREADS), lds, (hipStream_t)stream>>>(a);
    return SPY_LAUNCH_RC();
}
