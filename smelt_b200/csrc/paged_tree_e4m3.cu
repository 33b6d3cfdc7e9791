// Attention over a paged cache (paged_attn.cuh): a tree of drafted tokens per row, e4m3 caches.
#include "paged_attn.cuh"

using namespace gpt2q;

cudaError_t gpt2q::launch_paged_tree_e4m3(const PagedAttn& p, int dtype, cudaStream_t st) {
    if (dtype == GPT2Q_F32) return by_dim<__nv_fp8_e4m3, float, true>(p, st);
    return dtype == GPT2Q_F16 ? by_dim<__nv_fp8_e4m3, __half, true>(p, st) : by_dim<__nv_fp8_e4m3, bf16, true>(p, st);
}
