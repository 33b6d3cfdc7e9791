// Attention over a paged cache (paged_attn.cuh): one new token per row, e4m3 caches.
#include "paged_attn.cuh"

using namespace gpt2q;

cudaError_t gpt2q::launch_paged_attn_e4m3(const PagedAttn& p, int dtype, cudaStream_t st) {
    if (dtype == GPT2Q_F32) return by_dim<__nv_fp8_e4m3, float, false>(p, st);
    return dtype == GPT2Q_F16 ? by_dim<__nv_fp8_e4m3, __half, false>(p, st) : by_dim<__nv_fp8_e4m3, bf16, false>(p, st);
}
