// Attention over a paged cache (paged_attn.cuh): a tree of drafted tokens per row, caches of 32 and 16 bits.
#include "paged_attn.cuh"

using namespace gpt2q;

cudaError_t gpt2q::launch_paged_tree(const PagedAttn& p, int cache_dtype, int dtype, cudaStream_t st) {
    if (cache_dtype == GPT2Q_I8) return launch_paged_tree_i8(p, dtype, st);
    if (cache_dtype == GPT2Q_E4M3) return launch_paged_tree_e4m3(p, dtype, st);
    if (cache_dtype == GPT2Q_F32) return by_dim<float, float, true>(p, st);
    if (cache_dtype == GPT2Q_F16)
        return dtype == GPT2Q_F32 ? by_dim<__half, float, true>(p, st) : by_dim<__half, __half, true>(p, st);
    return dtype == GPT2Q_F32 ? by_dim<bf16, float, true>(p, st) : by_dim<bf16, bf16, true>(p, st);
}
