// Attention over a paged cache (paged_attn.cuh): one new token per row, caches of 32 and 16 bits; and the layout of the
// workspace that all of its variants share.
#include "paged_attn.cuh"

using namespace gpt2q;

// Layout of the workspace: per block its last row's whereabouts, two partial results, and one more
// per warp.
uint64_t gpt2q::paged_attn_workspace(int dim, int group) {
    const uint64_t hd = dim <= 64 ? 64 : dim <= 128 ? 128 : 256, hb = group > 8 ? 16 : 8;
    return MAX_CTAS * (16 + 2 * hb * (hd * 4 + 8) + MAX_WARPS * hb * (hd + 4) * 4);
}

cudaError_t gpt2q::launch_paged_attn(PagedAttn p, int cache_dtype, int dtype, void* work, cudaStream_t st) {
    const bool tree = p.first != nullptr;
    const uint64_t hd = p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256, hb = tree || p.group > 8 ? 16 : 8;
    p.page_shift = -1;
    for (int s = 0; s < 31; ++s)
        if (p.page == 1 << s) p.page_shift = s;
    if (tree && paged_tree_tc_serves(p, cache_dtype, dtype)) {
        bool taken = false;
        const cudaError_t e = launch_paged_tree_tc(p, cache_dtype, dtype, work, st, &taken);
        if (taken || e != cudaSuccess) return e;
    }
    char* at = static_cast<char*>(work);
    p.meta = reinterpret_cast<int4*>(at);
    at += MAX_CTAS * 16;
    p.block_part = reinterpret_cast<float*>(at);
    at += MAX_CTAS * 2 * hb * hd * 4;
    p.warp_part = reinterpret_cast<float*>(at);
    at += MAX_CTAS * MAX_WARPS * hb * (hd + 4) * 4;
    p.block_ml = reinterpret_cast<float2*>(at);
    if (tree) return launch_paged_tree(p, cache_dtype, dtype, st);
    if (cache_dtype == GPT2Q_I8) return launch_paged_attn_i8(p, dtype, st);
    if (cache_dtype == GPT2Q_E4M3) return launch_paged_attn_e4m3(p, dtype, st);
    if (cache_dtype == GPT2Q_F32) return by_dim<float, float, false>(p, st);
    if (cache_dtype == GPT2Q_F16)
        return dtype == GPT2Q_F32 ? by_dim<__half, float, false>(p, st) : by_dim<__half, __half, false>(p, st);
    return dtype == GPT2Q_F32 ? by_dim<bf16, float, false>(p, st) : by_dim<bf16, bf16, false>(p, st);
}
