// Attention over pages of 8 bits: paged_attn.cuh with fp16(d * q) for the elements of K and V, so that its results are those of pages that hold these as fp16, bit for bit.
// Few rows: paged_few_q8.cuh, bound by memory.  Chunks: attn_chunk of paged_attn.cuh, bound by instructions, with 14 vector instructions to 8 elements on top of what fp16 pages take: 512 tokens on 7680, 32 heads
// to 8, 128 wide 106 us (fp16 pages: 88), F32 out 128 (112); the cache is half the bytes, which matters for few rows alone.
#include "paged_few_q8.cuh"

// waves on a SIMD that the tiles in LDS, and the registers, leave room for (128 wide: 131 registers; four waves with 128 took 146.7 us instead of 144.7 for the 64 requests)
template <int D, bool F32OUT> __global__ __launch_bounds__(256, 512 / D > 4 ? 4 : 512 / D > 2 ? 3 : 2) void attn_q8_few_kernel(attn_more a) {
    __shared__ few_q8_shared<D, 4> sh;
    attn_few_q8<D, F32OUT, 4, ATTN_Q8>(a, sh, blockIdx.x);
}
template <int D, bool F32OUT> __global__ __launch_bounds__(256 * chunk_groups(D)) void attn_q8_mixed_kernel(attn_more a) {
    __shared__ union { few_q8_shared<D, 4 * chunk_groups(D)> few; chunk_shared_q8<D> chunk; } sh;
    if ((int)blockIdx.x < a.chunk_blocks) attn_chunk<D, F32OUT, ATTN_Q8>(a, sh.chunk, blockIdx.x);
    else attn_few_q8<D, F32OUT, 4 * chunk_groups(D), ATTN_Q8>(a, sh.few, blockIdx.x - a.chunk_blocks);
}

extern "C" size_t spy_hip_paged_attention_q8_scratch_size(const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_paged_batch *batch) {
    attn_plan p;
    return attn_make_plan(q, k_pages, batch, true, p) ? 0 : p.scratch;
}

template <int D, bool F32OUT> static int attn_q8_launch(const attn_more &a, const attn_plan &p, hipStream_t st) {
    if (a.chunk_blocks) attn_q8_mixed_kernel<D, F32OUT><<<dim3((unsigned)(a.chunk_blocks + a.few_blocks)), dim3(256 * chunk_groups(D)), 0, st>>>(a);
    else attn_q8_few_kernel<D, F32OUT><<<dim3((unsigned)a.few_blocks), dim3(256), 0, st>>>(a);
    const int rc = SPY_LAUNCH_RC();
    return rc ? rc : spy_attn_join(a, p, D, F32OUT, st);
}

extern "C" int spy_hip_paged_attention_q8(void *stream, const spy_hip_tensor *q, const spy_hip_tensor *k_pages, const spy_hip_tensor *k_scales, const spy_hip_tensor *v_pages,
                                          const spy_hip_tensor *v_scales, const spy_hip_tensor *out, const spy_hip_paged_batch *batch, float scale, int32_t causal, int32_t window, void *scratch,
                                          size_t scratch_bytes) {
    SPY_CHECK_ARG(q && k_pages && k_scales && v_pages && v_scales && out);
    attn_plan p;
    attn_more a = {};
    int rc = attn_make_plan(q, k_pages, batch, true, p);
    if (!rc) rc = attn_check(q, k_pages, k_scales, v_pages, v_scales, out, batch, scale, causal, window, p.scratch, scratch, scratch_bytes, a);
    if (rc) return rc;
    attn_use_plan(p, scratch, a);
    attn_use_scales(k_scales, v_scales, a);
    hipStream_t st = (hipStream_t)stream;
    const int64_t hd = k_pages->ne[0];
    const bool f32 = out->type == SPY_HIP_F32;
    if (hd == 64) return f32 ? attn_q8_launch<64, true>(a, p, st) : attn_q8_launch<64, false>(a, p, st);
    if (hd == 128) return f32 ? attn_q8_launch<128, true>(a, p, st) : attn_q8_launch<128, false>(a, p, st);
    return f32 ? attn_q8_launch<256, true>(a, p, st) : attn_q8_launch<256, false>(a, p, st);
}
