// Attention of sequences that begin alike: what a group of them has in common is attended to by all its rows together, the rest by each sequence.
//
// For a row, whose keys are those in common, C, and its sequence's own, S: out = (sum over C and S of e^(x_j - m) V_j) / (sum over C and S of e^(x_j - m)).  Both sums are taken in pieces, each
// with an m of its own, by the kernels of paged_attn.cuh: C with the group as one sequence whose new tokens are all its sequences' and which sees all of C, S from the first position on
// that is not in common.  A second launch scales the pieces' (o, l) to the largest m and adds them up.
// What is gained: K and V of C are read once for a group, in tiles of up to 128 rows of the matrix instructions, instead of once for each sequence, which has few.
//
// Chunks by four waves, so that a compute unit has two workgroups at a time, of which one's tiles of few rows read memory beside the other's products (by eight waves, as in paged_attn.hip: 72, 49 and 102 us for the
// three cases that follow).  64 requests behind four prompts of 8000 tokens, 32 heads to 8, 128 wide: 61 us, 6 of them the second launch; the rest reads at 5 TB/s.  32 requests behind one of 20000, 8 bits: 38.5 us, where each
// workgroup has ten steps of 64 keys, 2.1 us each with one wave on a SIMD, a start and 64 KB to write.  965 rows of 8 requests behind 2000 tokens, 32 heads: 85 us; 288 workgroups of 31 such steps on 256 compute
// units, then 15 us of the second launch.  4 requests of one token behind 600: 13 us, two launches' latency.
#include "paged_few_q8.cuh"

template <int D, int WAVES, int MODE> using shared_few = std::conditional_t<MODE & ATTN_Q8, few_q8_shared<D, WAVES>, few_shared<D, WAVES>>;
template <int D, bool F32OUT, int WAVES, int MODE> static __device__ __forceinline__ void attn_shared_few(const attn_more &a, shared_few<D, WAVES, MODE> &sh, int block, bool common) {
    if constexpr (MODE & ATTN_Q8) attn_few_q8<D, F32OUT, WAVES, MODE>(a, sh, block, common);
    else attn_few<D, F32OUT, WAVES, MODE>(a, sh, block, common);
}
template <int D, bool F32OUT, int MODE> __global__ __launch_bounds__(256, D == 256 && !(MODE & ATTN_Q8) ? 1 : 2) void attn_shared_few_kernel(attn_more a) {
    __shared__ shared_few<D, 4, MODE> sh;
    const int block = blockIdx.x;
    const bool common = block < a.common.few_blocks;
    attn_shared_few<D, F32OUT, 4, MODE>(a, sh, common ? block : block - a.common.few_blocks, common);
}
// What takes longest first: chunks over the keys in common, and over a sequence's own, then tiles of few rows
template <int D, bool F32OUT, int MODE> __global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attn_shared_mixed_kernel(attn_more a) {
    __shared__ union { shared_few<D, 4, MODE> few; std::conditional_t<MODE & ATTN_Q8, chunk_shared_q8<D, 1>, chunk_shared<D, 1>> chunk; } sh;
    int block = blockIdx.x;
    if (block < a.common.chunk_blocks + a.chunk_blocks) {
        const bool common = block < a.common.chunk_blocks;
        attn_chunk<D, F32OUT, MODE, 1>(a, sh.chunk, common ? block : block - a.common.chunk_blocks, common);
        return;
    }
    block -= a.common.chunk_blocks + a.chunk_blocks;
    const bool common = block < a.common.few_blocks;
    attn_shared_few<D, F32OUT, 4, MODE>(a, sh.few, common ? block : block - a.common.few_blocks, common);
}

template <int D, bool F32OUT, int MODE> static int attn_shared_launch(const attn_more &a, hipStream_t st) {
    const unsigned few = a.common.few_blocks + a.few_blocks, chunk = a.common.chunk_blocks + a.chunk_blocks;
    if (chunk) attn_shared_mixed_kernel<D, F32OUT, MODE><<<dim3(chunk + few), dim3(256), 0, st>>>(a);
    else attn_shared_few_kernel<D, F32OUT, MODE><<<dim3(few), dim3(256), 0, st>>>(a);
    return SPY_LAUNCH_RC();
}
template <int MODE> static int attn_shared_launch(const attn_more &a, int64_t hd, bool f32, hipStream_t st) {
    if (hd == 64) return f32 ? attn_shared_launch<64, true, MODE>(a, st) : attn_shared_launch<64, false, MODE>(a, st);
    if (hd == 128) return f32 ? attn_shared_launch<128, true, MODE>(a, st) : attn_shared_launch<128, false, MODE>(a, st);
    return f32 ? attn_shared_launch<256, true, MODE>(a, st) : attn_shared_launch<256, false, MODE>(a, st);
}
int spy_attn_shared_q8(const attn_more &a, int64_t hd, bool f32, hipStream_t st);        // paged_shared_q8.hip
