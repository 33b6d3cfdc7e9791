// Attention over a paged cache (paged_attn.cuh): one new token per row, i8 caches.
#include "paged_attn.cuh"

using namespace gpt2q;

cudaError_t gpt2q::launch_paged_attn_i8(const PagedAttn& p, int dtype, cudaStream_t st) {
    if (dtype == GPT2Q_F32) return by_dim<int8_t, float, false>(p, st);
    return dtype == GPT2Q_F16 ? by_dim<int8_t, __half, false>(p, st) : by_dim<int8_t, bf16, false>(p, st);
}
