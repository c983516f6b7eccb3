// Attention of sequences that begin alike over pages of 8 bits: the kernels of paged_shared.cuh, in an object of their own.
#include "paged_shared.cuh"

int spy_attn_shared_q8(const attn_more &a, int64_t hd, bool two, hipStream_t st) { return attn_shared_launch<ATTN_SHARED | ATTN_Q8>(a, hd, two, st); }
