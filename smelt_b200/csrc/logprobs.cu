// Log probabilities of given tokens, entropy and top alternatives (gpt2q_logprobs), and their
// gradient (gpt2q_logprobs_grad): gpt2q.h states the definitions.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include <cooperative_groups.h>

#include "device_op.cuh"
#include "gpt2q.h"

namespace gpt2q {
void set_global_error(const std::string& msg);  // runtime.cu
}

using namespace gpt2q;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int THREADS = 256;
constexpr int CANDIDATES = 2048;

__device__ __forceinline__ float ex2(float x) {  // 2^x to 2 ulp; results under 2^-126 are 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}

// One 16-byte vector of a row. Rows start anywhere, so vectors are counted from the row's first
// 16-byte boundary at or before it: vector v holds the elements v * VE - shift + [0, VE) of the row,
// and only its first and last vector are partly outside; those are loaded element by element.
template <class T>
struct Row {
    static constexpr int VE = 16 / sizeof(T);
    const T* x;  // the row's first element
    int shift, vocab, vectors;
    __device__ Row(const T* row, int vocab_) : x(row), vocab(vocab_) {
        shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        vectors = (vocab + shift + VE - 1) / VE;
    }
    __device__ __forceinline__ int first(int v) const { return v * VE - shift; }
    __device__ __forceinline__ uint4 load(int v) const {
        const int e = first(v);
        if (e >= 0 && e + VE <= vocab) return __ldcg(reinterpret_cast<const uint4*>(x + e));
        return edge(e);
    }
    __device__ __noinline__ uint4 edge(int e) const {  // elements outside the row read as -inf
        union {
            uint4 u;
            T t[VE];
        } r;
#pragma unroll
        for (int i = 0; i < VE; ++i) r.t[i] = e + i >= 0 && e + i < vocab ? x[e + i] : from_f<T>(-INFINITY);
        return r.u;
    }
};

// a vector of -inf
template <class T>
__device__ __forceinline__ uint4 nothing() {
    constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u;
    return make_uint4(w, w, w, w);
}

template <class T>
__device__ __forceinline__ void unpack(const uint4& u, float2* f) {  // VE / 2 pairs
    if constexpr (sizeof(T) == 4) {
        f[0] = make_float2(__uint_as_float(u.x), __uint_as_float(u.y));
        f[1] = make_float2(__uint_as_float(u.z), __uint_as_float(u.w));
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, bf16>::value)
                f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            else
                f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        }
    }
}

struct LpParams {
    const void* x;
    long long ld;
    int rows, vocab, top, parts;
    float inv_t;
    const void* targets;
    int i64;
    float *lp, *entropy, *stats;
    int* ids;
    float* top_lp;
};

__device__ __forceinline__ long long target_of(const void* t, int i64, int r) {
    return i64 ? __ldcg(static_cast<const long long*>(t) + r) : (long long)__ldcg(static_cast<const int*>(t) + r);
}

// Rank of a logit among alternatives: larger value first, equal values by rising index. -0 counts
// as +0 and NaN as -inf. Every element's key is above 0.
__device__ __forceinline__ unsigned long long rank_key(float x, int index) {
    x = isnan(x) ? -INFINITY : x + 0.f;
    unsigned b = __float_as_uint(x);
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return ((unsigned long long)b << 32) | (unsigned)~index;
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? b ^ 0x80000000u : ~b);
}
__device__ __forceinline__ unsigned long long maxu(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// The sums of a part of a row: m the largest logit, s = sum 2^z and t = sum 2^z z over
// z = (x - m) c, c = log2(e) / temperature. A part of nothing but -inf has m = -inf, s = t = 0.
struct Sums {
    float m, s, t;
};
__device__ __forceinline__ Sums merge(const Sums& a, const Sums& b, float c) {
    const float m = fmaxf(a.m, b.m);
    const float r = m == -INFINITY ? 0.f : m;
    // a part without mass has z = -inf; the clamp keeps 0 * z at 0
    const float za = fmaxf((a.m - r) * c, -2000.f), zb = fmaxf((b.m - r) * c, -2000.f);
    const float wa = ex2(za), wb = ex2(zb);
    return Sums{m, a.s * wa + b.s * wb, wa * (a.t + za * a.s) + wb * (b.t + zb * b.s)};
}

struct LpShared {
    Sums warp[THREADS / 32];
    Sums part;                                   // this block's, read by the cluster's first block
    unsigned long long group[THREADS / 2];       // best of every group of threads
    unsigned long long top[GPT2Q_TOP_MAX];       // this block's alternatives, in order
    unsigned long long threshold;
    unsigned long long best[THREADS / 32];
    int n_scan, n_cand;
    short scan[THREADS];
    unsigned long long cand[CANDIDATES];
};

// One pass over the logits. A cluster of `parts` blocks shares a row (one where there are rows
// enough), each block a consecutive range of vectors. A thread takes a batch of 32 elements at a
// time: the batch's largest logit first, so that the running sums are rescaled at most once per
// batch, then the exponentials.
//
// Alternatives need no second pass: the k-th best of the groups' best logits (a group is 2 to 8
// threads) is reached by k elements at least, so only elements from there on matter, and only
// threads whose own best reaches it can hold any. Those threads' elements, a small part of the
// row, are read once more from L2, and what passes (a few dozen) is ranked by counting. Rows that
// put more than CANDIDATES elements above the threshold take one round of search per alternative.
template <class T, bool TOP>
__global__ void __launch_bounds__(THREADS, 4) k_logprobs(const __grid_constant__ LpParams p) {
    constexpr int VE = Row<T>::VE, U = 32 / VE;  // vectors of a batch
    __shared__ LpShared sh;
    namespace cg = cooperative_groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    tc::pdl_trigger();
    tc::pdl_wait();
    const T* x = static_cast<const T*>(p.x) + (long long)r * p.ld;
    const Row<T> row(x, p.vocab);
    const int share = (row.vectors + p.parts - 1) / p.parts;
    const int v0 = share * part, v1 = min(v0 + share, row.vectors);
    const float c = p.inv_t * LOG2E;
    const bool leader = part == 0 && tid == 0;
    long long target = -1;
    float xt = 0.f;
    if (leader && p.lp) {
        target = target_of(p.targets, p.i64, r);
        if (target >= 0 && target < p.vocab) xt = to_f(x[target]);
    }

    float m = -INFINITY;
    float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
    int at = v0 + tid;  // the vector that holds this thread's best logit first
    for (int v = v0 + tid; v < v1; v += U * THREADS) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int vu = v + u * THREADS;
            raw[u] = vu < v1 ? row.load(vu) : nothing<T>();
        }
        float bm = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float2 f[VE / 2];
            unpack<T>(raw[u], f);
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) bm = fmaxf(bm, fmaxf(f[i].x, f[i].y));
        }
        if (bm > m) {
            const float z = fmaxf((m - bm) * c, -2000.f), w = ex2(z);
            t = make_float2(w * fmaf(z, s.x, t.x), w * fmaf(z, s.y, t.y));
            s = make_float2(w * s.x, w * s.y);
            m = bm;
            if constexpr (TOP) {
#pragma unroll
                for (int u = U - 1; u >= 0; --u) {
                    float2 f[VE / 2];
                    unpack<T>(raw[u], f);
                    float um = -INFINITY;
#pragma unroll
                    for (int i = 0; i < VE / 2; ++i) um = fmaxf(um, fmaxf(f[i].x, f[i].y));
                    if (um == bm) at = v + u * THREADS;
                }
            }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const float2 nm = make_float2(-ref, -ref), cc = make_float2(c, c);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float2 f[VE / 2];
            unpack<T>(raw[u], f);
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) {
                const float2 z = mul2(add2(f[i], nm), cc);
                const float2 e = make_float2(ex2(z.x), ex2(z.y));
                s = add2(s, e);
                t = fma2(e, make_float2(fmaxf(z.x, -2000.f), fmaxf(z.y, -2000.f)), t);
            }
        }
    }
    const float mine = m;
    Sums a{m, s.x + s.y, t.x + t.y};
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                     __shfl_xor_sync(0xffffffffu, a.t, o)};
        a = (lane & o) ? merge(b, a, c) : merge(a, b, c);  // the same order in both lanes
    }
    if (lane == 0) sh.warp[warp] = a;
    if (tid == 0) sh.n_scan = 0, sh.n_cand = 0, sh.threshold = 0;

    if constexpr (TOP) {
        const int K = p.top;
        const bool any = v0 + tid < v1;
        // at most the thread's best element's key: its value, and the last index of its vector
        unsigned long long key = any ? rank_key(mine, row.first(at) + VE - 1) : 0;
        const int g = K <= 20 ? 8 : K <= 40 ? 4 : 2;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1)
            if (o < g) key = maxu(key, __shfl_xor_sync(0xffffffffu, key, o));
        if (lane % g == 0) sh.group[tid / g] = key;
        __syncthreads();
        const int G = THREADS / g;
        if (tid < G) {
            const unsigned long long k0 = sh.group[tid];
            int above = 0;
            for (int i = 0; i < G; ++i) above += sh.group[i] > k0 || (sh.group[i] == k0 && i < tid);
            if (above == K - 1) sh.threshold = k0;  // 0 where fewer than K groups hold anything
        }
        __syncthreads();
        const unsigned long long thr = sh.threshold;
        // the thread's best possible key: its value at the first index of its vector
        if (any && rank_key(mine, max(0, row.first(at))) >= thr) sh.scan[atomicAdd(&sh.n_scan, 1)] = (short)tid;
        __syncthreads();
        const int per = (v1 - v0 + THREADS - 1) / THREADS;
        for (int i = tid; i < sh.n_scan * per; i += THREADS) {
            const int v = v0 + sh.scan[i / per] + (i % per) * THREADS;
            if (v < v1) {
                float2 f[VE / 2];
                unpack<T>(row.load(v), f);
                const int e = row.first(v);
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    const float y = j & 1 ? f[j / 2].y : f[j / 2].x;
                    const unsigned long long k = rank_key(y, e + j);
                    if (k >= thr && e + j >= 0 && e + j < p.vocab) {
                        const int n = atomicAdd(&sh.n_cand, 1);
                        if (n < CANDIDATES) sh.cand[n] = k;
                    }
                }
            }
        }
        if (tid < GPT2Q_TOP_MAX) sh.top[tid] = 0;
        __syncthreads();
        const int n = sh.n_cand;
        if (n <= CANDIDATES) {
            for (int i = tid; i < n; i += THREADS) {
                const unsigned long long k = sh.cand[i];
                int above = 0;
                for (int j = 0; j < n; ++j) above += sh.cand[j] > k;
                if (above < K) sh.top[above] = k;
            }
        } else {
            unsigned long long last = ~0ull;
            for (int q = 0; q < K && last; ++q) {
                unsigned long long best = 0;
                const int e1 = min(p.vocab, row.first(v1));
                for (int e = max(0, row.first(v0)) + tid; e < e1; e += THREADS) {
                    const unsigned long long k = rank_key(to_f(x[e]), e);
                    if (k < last) best = maxu(best, k);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) best = maxu(best, __shfl_xor_sync(0xffffffffu, best, o));
                if (lane == 0) sh.best[warp] = best;
                __syncthreads();
                last = sh.best[0];
                for (int w = 1; w < THREADS / 32; ++w) last = maxu(last, sh.best[w]);
                if (tid == 0) sh.top[q] = last;
                __syncthreads();
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        a = sh.warp[0];
        for (int w = 1; w < THREADS / 32; ++w) a = merge(a, sh.warp[w], c);
        sh.part = a;
    }
    if (p.parts > 1) {
        cg::this_cluster().sync();
        if (part == 0) {
            if (tid == 0) {
                for (int q = 1; q < p.parts; ++q) a = merge(a, cg::this_cluster().map_shared_rank(&sh, q)->part, c);
                sh.part = a;
            }
            if constexpr (TOP) {
                for (int i = tid; i < p.parts * p.top; i += THREADS)
                    sh.cand[i] = cg::this_cluster().map_shared_rank(&sh, i / p.top)->top[i % p.top];
                __syncthreads();
                const int n = p.parts * p.top;
                for (int i = tid; i < n; i += THREADS) {
                    const unsigned long long k = sh.cand[i];  // 0: the block has fewer elements than that
                    int above = 0;
                    for (int j = 0; j < n; ++j) above += sh.cand[j] > k;
                    if (k && above < p.top) sh.top[above] = k;
                }
            }
        }
        cg::this_cluster().sync();  // no block leaves while its shared memory may be read
    }
    if (part != 0) return;
    __syncthreads();
    a = sh.part;
    const bool empty = a.m == -INFINITY && a.s == 0.f;
    const float ls = empty ? -INFINITY : logf(a.s);
    auto lp_of = [&](float v) { return empty ? -INFINITY : (v - a.m) * p.inv_t - ls; };
    if (tid == 0) {
        const float h = empty ? 0.f : ls - a.t / a.s * LN2;
        if (p.lp) p.lp[r] = target < 0 ? 0.f : target >= p.vocab ? NAN : lp_of(xt);
        if (p.entropy) p.entropy[r] = h;
        if (p.stats) p.stats[3LL * r] = a.m, p.stats[3LL * r + 1] = ls, p.stats[3LL * r + 2] = h;
    }
    if constexpr (TOP) {
        for (int k = tid; k < p.top; k += THREADS) {
            const unsigned long long key = sh.top[k];
            if (p.ids) p.ids[(long long)r * p.top + k] = (int)~(unsigned)key;
            if (p.top_lp) p.top_lp[(long long)r * p.top + k] = lp_of(key_value(key));
        }
    }
}

template <class T>
cudaError_t launch_logprobs(LpParams p, cudaStream_t st) {
    // blocks per row: enough for eight per SM in all, as long as every thread has a batch
    const int batches = (p.vocab + 32 * THREADS - 1) / (32 * THREADS);
    p.parts = 1;
    while (p.parts < 8 && p.parts < batches && (long long)p.rows * p.parts < 148 * 8) p.parts *= 2;
    if ((long long)p.rows * p.parts > INT32_MAX) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.rows * p.parts);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.parts;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    return p.top ? cudaLaunchKernelEx(&cfg, k_logprobs<T, true>, p) : cudaLaunchKernelEx(&cfg, k_logprobs<T, false>, p);
}

struct GradParams {
    const void* x;
    void* dx;
    long long ld, ldo;
    int rows, vocab, chunks;
    float inv_t;
    const void* targets;
    int i64;
    const float *stats, *d_lp, *d_ent;
};

// 16 bytes from byte `by` (a multiple of the element's size, under 16) of the 32 bytes (a, b).
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int by) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (by & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (by & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const int bits = (by & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// One element in, one out: d_j = -p_j (A + B log2 p_j), the target's plus g / temperature. A block
// takes four vectors per thread of one row. Vectors are the output's; where the input row lies
// differently against the 16-byte boundaries, its 16 bytes are cut from two aligned vectors, the
// second of which the neighbouring lane holds.
template <class T>
__global__ void __launch_bounds__(THREADS) k_logprobs_grad(const __grid_constant__ GradParams p) {
    constexpr int VE = Row<T>::VE, U = 4;
    tc::pdl_trigger();
    tc::pdl_wait();
    const int r = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
    const Row<T> in(static_cast<const T*>(p.x) + (long long)r * p.ld, p.vocab);
    T* dx = static_cast<T*>(p.dx) + (long long)r * p.ldo;
    const Row<T> out(dx, p.vocab);
    const int v = chunk * U * THREADS + threadIdx.x;
    // element e of the output's vector is e + off of the input's, counted from its boundary
    const int off = in.shift - out.shift;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int vu = v + u * THREADS, e = out.first(vu);
        if (off == 0) {
            raw[u] = vu < out.vectors ? in.load(vu) : nothing<T>();
        } else {
            const int q = vu * VE + off, v0 = q >= 0 ? q / VE : -1;  // off > -VE
            const int e0 = in.first(v0);
            const uint4* src = reinterpret_cast<const uint4*>(in.x - in.shift) + v0;
            uint4 a = nothing<T>(), b;
            if (e0 >= 0 && e0 + VE <= p.vocab) a = __ldcg(src);
            b.x = __shfl_down_sync(0xffffffffu, a.x, 1);
            b.y = __shfl_down_sync(0xffffffffu, a.y, 1);
            b.z = __shfl_down_sync(0xffffffffu, a.z, 1);
            b.w = __shfl_down_sync(0xffffffffu, a.w, 1);
            if (e0 >= 0 && e0 + 2 * VE <= p.vocab) {
                if ((threadIdx.x & 31) == 31) b = __ldcg(src + 1);
                raw[u] = shifted(a, b, (q - v0 * VE) * (int)sizeof(T));
            } else {
                raw[u] = vu < out.vectors ? in.edge(e) : nothing<T>();
            }
        }
    }
    const float m = __ldcg(p.stats + 3LL * r), ls = __ldcg(p.stats + 3LL * r + 1), h = __ldcg(p.stats + 3LL * r + 2);
    float g = p.d_lp ? __ldcg(p.d_lp + r) : 0.f;
    const float ge = p.d_ent ? __ldcg(p.d_ent + r) : 0.f;
    long long target = -1;
    if (p.d_lp) {
        target = target_of(p.targets, p.i64, r);
        if (target < 0) g = 0.f;
        if (target >= p.vocab) g = NAN;
    }
    const bool empty = m == -INFINITY && ls == -INFINITY;
    const float A = -p.inv_t * (g + ge * h), B = -p.inv_t * ge * LN2, hit = p.inv_t * g;
    const float c = p.inv_t * LOG2E, l2 = -ls * LOG2E;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int vu = v + u * THREADS, e = out.first(vu);
        if (vu >= out.vectors) break;
        float2 f[VE / 2];
        unpack<T>(raw[u], f);
        union {
            uint4 u4;
            T t[VE];
        } o;
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            const float2 z = fma2(add2(f[i], make_float2(-m, -m)), make_float2(c, c), make_float2(l2, l2));
            const float2 q = make_float2(ex2(z.x), ex2(z.y));
            // log2 p of a masked element is -inf; the clamp keeps its 0 * log2 p at 0
            const float2 k = fma2(make_float2(fmaxf(z.x, -2000.f), fmaxf(z.y, -2000.f)), make_float2(B, B), make_float2(A, A));
            float2 d = mul2(q, k);
            if (target == e + 2 * i) d.x += hit;
            if (target == e + 2 * i + 1) d.y += hit;
            if (empty) d = make_float2(0.f, 0.f);
            o.t[2 * i] = from_f<T>(d.x);
            o.t[2 * i + 1] = from_f<T>(d.y);
        }
        if (e >= 0 && e + VE <= p.vocab) {
            *reinterpret_cast<uint4*>(dx + e) = o.u4;
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i)
                if (e + i >= 0 && e + i < p.vocab) dx[e + i] = o.t[i];
        }
    }
}

template <class T>
cudaError_t launch_grad(GradParams p, cudaStream_t st) {
    constexpr int per = 4 * THREADS * Row<T>::VE;
    p.chunks = (p.vocab + Row<T>::VE - 1 + per - 1) / per;
    if ((long long)p.rows * p.chunks > INT32_MAX) return cudaErrorInvalidConfiguration;
    return launch_dependent(k_logprobs_grad<T>, dim3((unsigned)p.rows * p.chunks), dim3(THREADS), 0, st, p);
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
    LpParams p{d_logits, ld, n_rows, vocab, top, 1, 1.f / temperature, d_targets, targets_i64 != 0,
               d_lp, d_entropy, d_stats, d_top_ids, d_top_lp};
    if (!d_top_ids && !d_top_lp) p.top = 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == GPT2Q_F32)
        e = launch_logprobs<float>(p, st);
    else if (dtype == GPT2Q_F16)
        e = launch_logprobs<__half>(p, st);
    else
        e = launch_logprobs<bf16>(p, st);
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
    const GradParams p{d_logits, d_dlogits, ld, ld_out, n_rows, vocab, 1, 1.f / temperature, d_targets, targets_i64 != 0,
                       d_stats, d_lp, d_ent};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (dtype == GPT2Q_F32)
        e = launch_grad<float>(p, st);
    else if (dtype == GPT2Q_F16)
        e = launch_grad<__half>(p, st);
    else
        e = launch_grad<bf16>(p, st);
    if (e != cudaSuccess) {
        set_global_error(std::string(who) + ": " + cudaGetErrorString(e));
        return GPT2Q_ECUDA;
    }
    return GPT2Q_OK;
}
