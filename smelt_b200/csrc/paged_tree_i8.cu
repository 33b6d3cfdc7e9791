// Attention over a paged cache (paged_attn.cuh): a tree of drafted tokens per row, i8 caches.
#include "paged_attn.cuh"

using namespace gpt2q;

cudaError_t gpt2q::launch_paged_tree_i8(const PagedAttn& p, int dtype, cudaStream_t st) {
    if (dtype == GPT2Q_F32) return by_dim<int8_t, float, true>(p, st);
    return dtype == GPT2Q_F16 ? by_dim<int8_t, __half, true>(p, st) : by_dim<int8_t, bf16, true>(p, st);
}
