// Attention of sequences that begin alike: what a group of them has in common is attended to by all its rows together, the rest by each sequence.
//
// For a row, whose keys are those in common, C, and its sequence's own, S: out = (sum over C and S of e^(x_j - m) V_j) / (sum over C and S of e^(x_j - m)).  Both sums are taken in pieces, each
// with an m of its own, by the kernels of paged_attn.cuh: C with the group as one sequence whose new tokens are all its sequences' and which sees all of C, S from the first position on
// that is not in common.  A second launch scales the pieces' (o, l) to the largest m and adds them up.
// What is gained: K and V of C are read once for a group, in tiles of up to 128 rows of the matrix instructions, instead of once for each sequence, which has few.
//
// Chunks by four waves, so that a compute unit has two workgroups at a time, of which one's tiles of few rows read memory beside the other's products (one term of a probability: 61, 39 and 85 us for the
// three cases that follow, by eight waves, as in paged_attn.hip, 72, 49 and 102).  64 requests behind four prompts of 8000 tokens, 32 heads to 8, 128 wide: 63 us, 6 of them the second launch; the rest reads at 4.9 TB/s.  32 requests behind one of 20000, 8 bits: 43.5 us, where each
// workgroup has ten steps of 64 keys, 2.5 us each with one wave on a SIMD, a start and 64 KB to write.  965 rows of 8 requests behind 2000 tokens, 32 heads: 85 us; 288 workgroups of 31 such steps on 256 compute
// units, then 15 us of the second launch.  4 requests of one token behind 600: 13 us, two launches' latency.
#include "paged_few_q8.cuh"

template <int D, int WAVES, int MODE> using shared_few = std::conditional_t<MODE & ATTN_Q8, few_q8_shared<D, WAVES>, few_shared<D, WAVES>>;
template <int D, int WAVES, int MODE> static __device__ __forceinline__ void attn_shared_few(const attn_more &a, shared_few<D, WAVES, MODE> &sh, int block, bool common) {
    if constexpr (MODE & ATTN_Q8) attn_few_q8<D, true, WAVES, MODE>(a, sh, block, common);
    else attn_few<D, true, WAVES, MODE>(a, sh, block, common);
}
template <int D, int MODE> __global__ __launch_bounds__(256, D == 256 && !(MODE & ATTN_Q8) ? 1 : 2) void attn_shared_few_kernel(attn_more a) {
    __shared__ shared_few<D, 4, MODE> sh;
    const int block = blockIdx.x;
    const bool common = block < a.common.few_blocks;
    attn_shared_few<D, 4, MODE>(a, sh, common ? block : block - a.common.few_blocks, common);
}
// Whether a tile over keys in common has rows of a sequence that has a.few rows at most.  By every lane of a wave, 64 sequences per round from the group's first on.
static __device__ __forceinline__ bool shared_tile_has_few(const attn_more &a, const span_tile &found) {
    const row_tile rt(a, found.sq, found.count - 1 - found.tile, CHUNK_ROWS, true);        // as attn_chunk has it
    const int lane = threadIdx.x & 63, first = found.sq.row0 + rt.first(), last = found.sq.row0 + rt.last(), few = a.few / a.group;
    for (int base = found.sq.s; base < a.b.n_seq; base += 64) {
        const int s = min(base + lane, a.b.n_seq - 1), from = a.b.row_start[s], to = a.b.row_start[s + 1];
        if (__any(from <= last && to > max(first, from) && to - from <= few)) return true;
        if (__any(from > last)) break;
    }
    return false;
}
// What takes longest first: chunks over the keys in common, and over a sequence's own, then tiles of few rows.  TWO: a probability enters a chunk's product as two fp16 terms.  Without it (F16 outputs,
// sequences of many rows in the batch) it does so where paged_attn.hip has two, in tiles over keys in common that have rows of a sequence of few; the other rows of the tile have more bits than
// they need.  One term for all keys in common, before: 61 us instead of 63 for the 64 requests, 38.9 instead of 43.5 for the 32, and 266 instead of 284 for a chunk of 2048 tokens and eight single ones behind
// 4000, 32 heads to 8; two for all: 111 us instead of 85 for the 965 rows.
template <int D, bool TWO, int MODE> __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_shared_mixed_kernel(attn_more a) {
    __shared__ union { shared_few<D, 4, MODE> few; std::conditional_t<MODE & ATTN_Q8, chunk_shared_q8<D, 1>, chunk_shared<D, 1>> chunk; } sh;
    int block = blockIdx.x;
    if (block < a.common.chunk_blocks + a.chunk_blocks) {
        const bool common = block < a.common.chunk_blocks;
        if (!common) block -= a.common.chunk_blocks;
        span_tile found;
        if (!find_span(a, common, block % ((common ? a.common.chunk_tiles : a.chunk_tiles) * a.G) / a.G, found)) return;
        if (!TWO && common && shared_tile_has_few(a, found)) attn_chunk<D, true, MODE, 1>(a, sh.chunk, block, true, found);
        else attn_chunk<D, TWO, MODE, 1>(a, sh.chunk, block, common, found);
        return;
    }
    block -= a.common.chunk_blocks + a.chunk_blocks;
    const bool common = block < a.common.few_blocks;
    attn_shared_few<D, 4, MODE>(a, sh.few, common ? block : block - a.common.few_blocks, common);
}

template <int D, int MODE> static int attn_shared_launch(const attn_more &a, bool two, hipStream_t st) {
    const unsigned few = a.common.few_blocks + a.few_blocks, chunk = a.common.chunk_blocks + a.chunk_blocks;
    if (!chunk) attn_shared_few_kernel<D, MODE><<<dim3(few), dim3(256), 0, st>>>(a);
    else if (two) attn_shared_mixed_kernel<D, true, MODE><<<dim3(chunk + few), dim3(256), 0, st>>>(a);
    else attn_shared_mixed_kernel<D, false, MODE><<<dim3(chunk + few), dim3(256), 0, st>>>(a);
    return SPY_LAUNCH_RC();
}
template <int MODE> static int attn_shared_launch(const attn_more &a, int64_t hd, bool two, hipStream_t st) {
    return hd == 64 ? attn_shared_launch<64, MODE>(a, two, st) : hd == 128 ? attn_shared_launch<128, MODE>(a, two, st) : attn_shared_launch<256, MODE>(a, two, st);
}
int spy_attn_shared_q8(const attn_more &a, int64_t hd, bool two, hipStream_t st);        // paged_shared_q8.hip
