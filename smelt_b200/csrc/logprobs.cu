// Log probabilities of given tokens, entropy and top alternatives (gpt2q_logprobs), and their
// gradient (gpt2q_logprobs_grad): gpt2q.h states the definitions.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "device_op.cuh"
#include "gpt2q.h"

namespace gpt2q {
void set_global_error(const std::string& msg);  // runtime.cu
}

using namespace gpt2q;

namespace {

struct LpParams {
    const void* x;
    long long ld;
    int rows, vocab, top;
    float inv_t;
    const void* targets;
    int i64;
    float *lp, *entropy, *stats;
    int* ids;
    float* top_lp;
};

__device__ __forceinline__ long long target_of(const void* t, int i64, int r) {
    return i64 ? static_cast<const long long*>(t)[r] : (long long)static_cast<const int*>(t)[r];
}

// Rank of a logit among alternatives: larger value first, equal values by rising index. -0 counts
// as +0 and NaN as -inf.
__device__ __forceinline__ unsigned long long rank_key(float x, int index) {
    x = isnan(x) ? -INFINITY : x + 0.f;
    unsigned b = __float_as_uint(x);
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((unsigned long long)b << 32) | (unsigned)~index;
}

template <class T>
__device__ T block_reduce(T v, T* red, T (*op)(T, T)) {
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < (int)blockDim.x / 32; ++w) v = op(v, red[w]);
    return v;
}
__device__ float op_add(float a, float b) { return a + b; }
__device__ float op_max(float a, float b) { return fmaxf(a, b); }
__device__ unsigned long long op_maxu(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// One block per row.
template <class T>
__global__ void __launch_bounds__(256) k_logprobs_simple(const LpParams p) {
    __shared__ float redf[8];
    __shared__ unsigned long long redu[8];
    tc::pdl_trigger();
    tc::pdl_wait();
    const int r = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + r * p.ld;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += 256) m = fmaxf(m, to_f(x[i]));
    m = block_reduce(m, redf, op_max);
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < p.vocab; i += 256) {
        const float z = (to_f(x[i]) - m) * p.inv_t;
        const float e = expf(z);
        s += e;
        t += e * (z < -1000.f ? -1000.f : z);
    }
    s = block_reduce(s, redf, op_add);
    t = block_reduce(t, redf, op_add);
    const bool empty = m == -INFINITY && s != s && block_reduce([&] {
        float nan = 0.f;
        for (int i = threadIdx.x; i < p.vocab; i += 256) nan += isnan(to_f(x[i])) ? 1.f : 0.f;
        return nan;
    }(), redf, op_add) == 0.f;
    const float ls = empty ? -INFINITY : logf(s);
    const float h = empty ? 0.f : ls - t / s;
    auto lp_of = [&](float v) { return empty ? -INFINITY : (v - m) * p.inv_t - ls; };
    if (threadIdx.x == 0) {
        if (p.lp) {
            const long long tg = target_of(p.targets, p.i64, r);
            p.lp[r] = tg < 0 ? 0.f : tg >= p.vocab ? NAN : lp_of(to_f(x[tg]));
        }
        if (p.entropy) p.entropy[r] = h;
        if (p.stats) p.stats[3LL * r] = m, p.stats[3LL * r + 1] = ls, p.stats[3LL * r + 2] = h;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < p.vocab; i += 256) {
            const unsigned long long key = rank_key(to_f(x[i]), i);
            if (key < last && key > best) best = key;
        }
        last = block_reduce(best, redu, op_maxu);
        if (threadIdx.x == 0) {
            const int i = (int)~(unsigned)last;
            if (p.ids) p.ids[(long long)r * p.top + k] = i;
            if (p.top_lp) p.top_lp[(long long)r * p.top + k] = lp_of(to_f(x[i]));
        }
    }
}

struct GradParams {
    const void* x;
    void* dx;
    long long ld, ldo;
    int rows, vocab;
    float inv_t;
    const void* targets;
    int i64;
    const float *stats, *d_lp, *d_ent;
};

template <class T>
__global__ void __launch_bounds__(256) k_logprobs_grad_simple(const GradParams p) {
    tc::pdl_trigger();
    tc::pdl_wait();
    const int r = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + r * p.ld;
    T* dx = static_cast<T*>(p.dx) + r * p.ldo;
    const float m = p.stats[3LL * r], ls = p.stats[3LL * r + 1], h = p.stats[3LL * r + 2];
    float g = p.d_lp ? p.d_lp[r] : 0.f;
    const float ge = p.d_ent ? p.d_ent[r] : 0.f;
    long long tg = -1;
    if (p.d_lp) {
        tg = target_of(p.targets, p.i64, r);
        if (tg < 0) g = 0.f;
        if (tg >= p.vocab) g = NAN;
    }
    const bool empty = m == -INFINITY && ls == -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += 256) {
        const float lp = (to_f(x[i]) - m) * p.inv_t - ls;
        const float pr = expf(lp);
        const float lc = lp < -1000.f ? -1000.f : lp;
        const float d = (i == tg ? g : 0.f) - pr * (g + ge * (lc + h));
        dx[i] = from_f<T>(empty ? 0.f : d * p.inv_t);
    }
}

int refuse(const char* who, const char* msg) {
    set_global_error(std::string(who) + ": " + msg);
    return GPT2Q_EARG;
}

int check(const char* who, const void* x, int dtype, int64_t ld, int n_rows, int vocab, float temperature) {
    if (n_rows < 0) return refuse(who, "n_rows < 0");
    if (vocab < 1 || ld < vocab) return refuse(who, "vocab must be >= 1 and ld >= vocab");
    if (dtype < GPT2Q_F32 || dtype > GPT2Q_BF16) return refuse(who, "unknown dtype");
    if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(1.f / temperature))
        return refuse(who, "temperature must be positive and finite");
    if (n_rows > 0 && !x) return refuse(who, "null logits");
    if (reinterpret_cast<uintptr_t>(x) % (dtype == GPT2Q_F32 ? 4 : 2)) return refuse(who, "unaligned logits");
    return GPT2Q_OK;
}

}  // namespace

extern "C" int gpt2q_logprobs(const void* d_logits, int dtype, int64_t ld, int n_rows, int vocab, float temperature,
                              const void* d_targets, int targets_i64, int top, float* d_lp, float* d_entropy,
                              float* d_stats, int32_t* d_top_ids, float* d_top_lp, void* stream) {
    const char* who = "gpt2q_logprobs";
    const int rc = check(who, d_logits, dtype, ld, n_rows, vocab, temperature);
    if (rc) return rc;
    if (top < 0 || top > GPT2Q_TOP_MAX || top > vocab) return refuse(who, "top out of range [0, min(vocab, GPT2Q_TOP_MAX)]");
    if (n_rows > 0 && d_lp && !d_targets) return refuse(who, "null targets");
    if (n_rows == 0) return GPT2Q_OK;
    LpParams p{d_logits, ld, n_rows, vocab, top, 1.f / temperature, d_targets, targets_i64 != 0,
               d_lp, d_entropy, d_stats, d_top_ids, d_top_lp};
    if (!d_top_ids && !d_top_lp) p.top = 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == GPT2Q_F32)
        e = launch_dependent(k_logprobs_simple<float>, dim3(n_rows), dim3(256), 0, st, p);
    else if (dtype == GPT2Q_F16)
        e = launch_dependent(k_logprobs_simple<__half>, dim3(n_rows), dim3(256), 0, st, p);
    else
        e = launch_dependent(k_logprobs_simple<bf16>, dim3(n_rows), dim3(256), 0, st, p);
    if (e != cudaSuccess) {
        set_global_error(std::string(who) + ": " + cudaGetErrorString(e));
        return GPT2Q_ECUDA;
    }
    return GPT2Q_OK;
}

extern "C" int gpt2q_logprobs_grad(const void* d_logits, int dtype, int64_t ld, int n_rows, int vocab, float temperature,
                                   const void* d_targets, int targets_i64, const float* d_stats, const float* d_lp,
                                   const float* d_ent, void* d_dlogits, int64_t ld_out, void* stream) {
    const char* who = "gpt2q_logprobs_grad";
    const int rc = check(who, d_logits, dtype, ld, n_rows, vocab, temperature);
    if (rc) return rc;
    if (ld_out < vocab) return refuse(who, "ld_out < vocab");
    if (n_rows == 0) return GPT2Q_OK;
    if (!d_stats || !d_dlogits) return refuse(who, "null stats or dlogits");
    if (d_lp && !d_targets) return refuse(who, "null targets");
    if (reinterpret_cast<uintptr_t>(d_dlogits) % (dtype == GPT2Q_F32 ? 4 : 2)) return refuse(who, "unaligned dlogits");
    if (d_dlogits == d_logits && ld_out != ld) return refuse(who, "in place ld_out must equal ld");
    const GradParams p{d_logits, d_dlogits, ld, ld_out, n_rows, vocab, 1.f / temperature, d_targets, targets_i64 != 0,
                       d_stats, d_lp, d_ent};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == GPT2Q_F32)
        e = launch_dependent(k_logprobs_grad_simple<float>, dim3(n_rows), dim3(256), 0, st, p);
    else if (dtype == GPT2Q_F16)
        e = launch_dependent(k_logprobs_grad_simple<__half>, dim3(n_rows), dim3(256), 0, st, p);
    else
        e = launch_dependent(k_logprobs_grad_simple<bf16>, dim3(n_rows), dim3(256), 0, st, p);
    if (e != cudaSuccess) {
        set_global_error(std::string(who) + ": " + cudaGetErrorString(e));
        return GPT2Q_ECUDA;
    }
    return GPT2Q_OK;
}
