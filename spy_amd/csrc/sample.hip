// A token drawn from each row of logits (sample.cuh).
#include "sample.cuh"

__global__ __launch_bounds__(SM_THREADS) void sample_kernel(sample_args a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    sample_row_of<false>(a, smem, blockIdx.x, 0, nullptr, nullptr);
}

extern "C" size_t spy_hip_sample_scratch_size(const spy_hip_tensor *logits) {
    (void)logits;
    return 0;
}

extern "C" int spy_hip_sample(void *stream, const spy_hip_tensor *logits, const spy_hip_sample_param *param, int32_t *tokens, float *probs, void *scratch, size_t scratch_bytes) {
    (void)scratch; (void)scratch_bytes;
    SPY_CHECK_ARG(logits && param && tokens && logits->data && param->uniform);
    int rc = sample_check(logits, param);
    if (rc) return rc;
    SPY_CHECK_ARG((((uintptr_t)tokens | (uintptr_t)probs) & 3) == 0);
    sample_args a = sample_args_of(logits, param);
    a.tokens = tokens; a.probs = probs;
    const size_t lds = sample_lds(a);
    rc = spy_raise_lds_limit((const void *)sample_kernel, lds);
    if (rc) return rc;
    sample_kernel<<<dim3((unsigned)logits->ne[1]), dim3(SM_THREADS), lds, (hipStream_t)stream>>>(a);
    return SPY_LAUNCH_RC();
}
