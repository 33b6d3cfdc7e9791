// Log probabilities of given tokens, entropy and top alternatives (gpt2q_logprobs), and their
// gradient (gpt2q_logprobs_grad): gpt2q.h states the definitions.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include <cooperative_groups.h>

#include "device_op.cuh"
#include "gpt2q.h"
#include "logprobs.h"

namespace gpt2q {
void set_global_error(const std::string& msg);  // runtime.cu
}

using namespace gpt2q;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int THREADS = 256;  // of the gradient
constexpr int CANDIDATES = 2048;

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

// VE / 2 pairs rounded to a vector
template <class T>
__device__ __forceinline__ uint4 packed(const float2* f) {
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, bf16>::value) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[i].x, f[i].y);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// the largest of a vector's elements that are numbers (-inf or NaN where none is)
template <class T>
__device__ __forceinline__ float largest(const uint4& u) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    } else {
        using T2 = std::conditional_t<std::is_same<T, bf16>::value, __nv_bfloat162, __half2>;
        const T2* h = reinterpret_cast<const T2*>(&u);
        const T2 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(to_f(a.x), to_f(a.y));
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
// The sums of all lanes' parts, in every lane: brought to the largest m, then added as a tree.
__device__ __forceinline__ Sums join(const Sums& a, float c) {
    Sums r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r.m) : "f"(a.m));
    // a part without mass has z = -inf; the clamp keeps 0 * z at 0
    const float z = fmaxf((a.m - (r.m == -INFINITY ? 0.f : r.m)) * c, -2000.f), w = ex2(z);
    r.s = a.s * w;
    r.t = w * fmaf(z, a.s, a.t);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
        r.t += __shfl_xor_sync(0xffffffffu, r.t, o);
    }
    return r;
}

template <int THREADS>
struct LpShared {
    Sums warp[THREADS / 32];
    Sums part[8];                          // of every block of the cluster (first block)
    unsigned long long key[THREADS];       // best of every thread
    unsigned long long group[128];         // best of every group of threads
    unsigned long long every[128];         // those of the whole cluster
    unsigned long long threshold;
    unsigned long long best[THREADS / 32];
    unsigned long long top[GPT2Q_TOP_MAX];  // the alternatives, in order (first block)
    int n_cand;
    unsigned long long cand[CANDIDATES];   // (first block)
};
struct LpSharedSums {  // without alternatives
    Sums warp[8];
    Sums part[8];
};

// One pass over the logits. A cluster of `parts` blocks shares a row (one where there are rows
// enough); their warps take 32 vectors each in turn, so that every block sees all parts of the row. A
// thread takes a batch of 32 elements at a time: the batch's largest logit first, so that the running
// sums are rescaled at most once per batch, then the exponentials.
//
// Alternatives need no second pass. Each thread keeps its best logit, the vector that holds it and
// the best of its other vectors. The k-th best of the bests of 64 or 128 groups of threads is
// reached by at least k elements, so only elements from there on matter: those lie in the best
// vectors of the threads that reach it (a few more than k), and in other vectors only of threads
// whose second best reaches it (a few). These are read once more, and what passes is ranked by
// counting. Rereading every vector of the first kind of thread, which needs no second best, cost 42
// thousand cycles a row in a call of 4096 rows, as the row had left L2 by then. Rows that put more
// than CANDIDATES elements above the threshold take one round of search per alternative.
// Measured: 4093 rows of 50257 fp32 125 us (6.6 TB/s, the memory's rate), 256 rows of 128000 bf16 with 20
// alternatives 21.3 us (15 without), one row of 50257 with 5 alternatives 5.8 us.
template <class T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_logprobs(const __grid_constant__ LpParams p) {
    constexpr int VE = Row<T>::VE, U = 32 / VE;  // vectors of a batch
    __shared__ std::conditional_t<TOP, LpShared<THREADS>, LpSharedSums> sh;
    namespace cg = cooperative_groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    // without alternatives nothing else tells a block that the first one of its cluster has started
    // when it writes into that one's shared memory
    if (!TOP && p.parts > 1) tc::cluster_arrive_relaxed();
    tc::pdl_trigger();
    tc::pdl_wait();
    const T* x = static_cast<const T*>(p.x) + (long long)r * p.ld;
    const Row<T> row(x, p.vocab);
    // blocks of 128 threads have a row each, and addresses with a constant stride (1 us of 130 in 4093 rows)
    const int stride = THREADS == 128 ? THREADS : p.parts * THREADS, v1 = row.vectors;
    const int v0 = (warp * p.parts + part) * 32 + lane;  // this thread's vectors: v0, v0 + stride, ...
    const float c = p.inv_t * LOG2E;
    long long target = -1;
    float xt = 0.f;
    if (part == 0 && tid == 0 && p.lp) {
        target = target_of(p.targets, p.i64, r);
        if (target >= 0 && target < p.vocab) xt = to_f(x[target]);
    }

    float m = -INFINITY, second = -INFINITY;
    float2 s = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
    int at = v0;  // the first vector that holds this thread's best logit
    // a batch whose vectors all lie inside the row takes no checks of its own
    const int in0 = row.shift ? 1 : 0, in1 = min(v1, (p.vocab + row.shift) / VE);
    const uint4* vec = reinterpret_cast<const uint4*>(x - row.shift);
    auto sums = [&](const uint4& raw, float2 nm, float2 cc) {
        float2 f[VE / 2];
        unpack<T>(raw, f);
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
            const float2 z = mul2(add2(f[i], nm), cc);
            const float2 e = make_float2(ex2(z.x), ex2(z.y));
            s = add2(s, e);
            t = fma2(e, make_float2(fmaxf(z.x, -2000.f), fmaxf(z.y, -2000.f)), t);
        }
    };
    for (int v = v0; v < v1; v += U * stride) {
        uint4 raw[U];
        const bool inside = v >= in0 && v + (U - 1) * stride < in1;
        if (inside) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = __ldcg(vec + v + u * stride);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = v + u * stride < v1 ? row.load(v + u * stride) : nothing<T>();
        }
        float bm = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float um = largest<T>(raw[u]);
            if constexpr (TOP) {
                // the first vector counts as the best until a larger one comes
                if (u > 0 || v != v0) second = fmaxf(second, fminf(bm, um));
                if (um > bm) at = v + u * stride;
            }
            bm = fmaxf(bm, um);
        }
        if (bm > m) {
            const float z = fmaxf((m - bm) * c, -2000.f), w = ex2(z);
            t = make_float2(w * fmaf(z, s.x, t.x), w * fmaf(z, s.y, t.y));
            s = make_float2(w * s.x, w * s.y);
            m = bm;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const float2 nm = make_float2(-ref, -ref), cc = make_float2(c, c);
        if (inside) {
#pragma unroll
            for (int u = 0; u < U; ++u) sums(raw[u], nm, cc);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (v + u * stride < v1) sums(raw[u], nm, cc);
        }
    }
    if constexpr (TOP) {
        // at most the key of the thread's best element: its value, and its vector's last index. Neighbouring
        // threads are of different groups, and neighbouring warps' vectors of different blocks, so that likely
        // tokens that lie together count as many: with a range of 6000 allowed ids, 20 alternatives of one row
        // took 308 us from consecutive threads and ranges (no threshold left of 13000 candidates), 6.0 so
        unsigned long long key = v0 < v1 ? rank_key(m, row.first(at) + VE - 1) : (unsigned)blockIdx.x * THREADS + tid;
        const int groups = (p.top <= 20 ? 64 : 128) / p.parts;
        for (int o = 16; o >= groups; o >>= 1) key = maxu(key, __shfl_xor_sync(0xffffffffu, key, o));
        sh.key[tid] = key;
        __syncthreads();
        if (tid < groups) {
            // groups below 32 have their warps' keys in the first lanes of each
            for (int i = tid + max(groups, 32); i < THREADS; i += max(groups, 32)) key = maxu(key, sh.key[i]);
            sh.group[tid] = key;
        }
        if (tid == 0) sh.n_cand = 0, sh.threshold = 0;
    }
    const Sums none{-INFINITY, 0.f, 0.f};
    Sums a = join(Sums{m, s.x + s.y, t.x + t.y}, c);
    if (lane == 0) sh.warp[warp] = a;
    auto* first = p.parts > 1 ? cg::this_cluster().map_shared_rank(&sh, 0) : &sh;

    if constexpr (TOP) {
        const int groups = (p.top <= 20 ? 64 : 128) / p.parts;
        const int total = groups * p.parts;
        const unsigned long long* keys = sh.group;
        if (p.parts > 1) {
            cg::this_cluster().sync();
            if (tid < total) sh.every[tid] = cg::this_cluster().map_shared_rank(&sh, tid / groups)->group[tid % groups];
            keys = sh.every;
        }
        __syncthreads();
        // the `top`-th of the groups' keys, which are all different (the keys of groups without a
        // vector, below 2^32, pass for no threshold); four or fewer threads count for a key
        {
            const int share_n = THREADS / total, k = tid / share_n, i0 = tid % share_n;
            const unsigned long long k0 = keys[k];
            int above = 0;
#pragma unroll 8
            for (int i = i0; i < total; i += share_n) above += keys[i] > k0;
            for (int o = 1; o < share_n; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
            if (above == p.top - 1 && i0 == 0) sh.threshold = k0 >> 32 ? k0 : 0;
        }
        __syncthreads();
        const unsigned long long thr = sh.threshold;
        const float least = thr ? key_value(thr) : -INFINITY;
        auto take = [&](const uint4& raw, int v) {
            float2 f[VE / 2];
            unpack<T>(raw, f);
            const int e = row.first(v);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float y = j & 1 ? f[j / 2].y : f[j / 2].x;
                if (y < least || e + j < 0 || e + j >= p.vocab) continue;
                const unsigned long long k = rank_key(y, e + j);
                if (k >= thr) {
                    const int n = atomicAdd(&first->n_cand, 1);
                    if (n < CANDIDATES) first->cand[n] = k;
                }
            }
        };
        // the best keys possible: of the best element, and of the other vectors' best
        const int other = at == v0 ? at + stride : v0;
        const bool every = other < v1 && second >= least && rank_key(second, max(0, row.first(other))) >= thr;
        if (!every && v0 < v1 && m >= least && rank_key(m, max(0, row.first(at))) >= thr) take(row.load(at), at);
        for (unsigned todo = __ballot_sync(0xffffffffu, every); todo; todo &= todo - 1) {
            // the warp rereads all vectors of one of its threads, four loads at a time
            const int v2 = v0 - lane + __ffs(todo) - 1;
            for (int v = v2 + lane * stride; v < v1; v += 4 * 32 * stride) {
                uint4 raw[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) raw[q] = v + q * 32 * stride < v1 ? row.load(v + q * 32 * stride) : nothing<T>();
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (v + q * 32 * stride < v1) take(raw[q], v + q * 32 * stride);
            }
        }
    } else {
        __syncthreads();
        if (p.parts > 1) tc::cluster_wait();
    }
    if (warp == 0) {
        a = join(lane < THREADS / 32 ? sh.warp[lane] : none, c);
        if (lane == 0) first->part[part] = a;
    }
    if (p.parts > 1)
        cg::this_cluster().sync();  // after it only the first block's shared memory is used
    else
        __syncthreads();
    if (part != 0) return;
    if (warp == 0) {
        a = join(lane < p.parts ? sh.part[lane] : none, c);
        if (lane == 0) sh.warp[0] = a;
    }
    if constexpr (TOP) {
        const int n = sh.n_cand;
        if (n <= CANDIDATES) {
            for (int i = tid; i < n; i += THREADS) {
                const unsigned long long k = sh.cand[i];
                int above = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) above += sh.cand[j] > k;
                if (above < p.top) sh.top[above] = k;
            }
        } else {
            unsigned long long last = ~0ull;
            for (int q = 0; q < p.top; ++q) {
                unsigned long long best = 0;
                for (int e = tid; e < p.vocab; e += THREADS) {
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
    a = sh.warp[0];
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

template <class T, int THREADS>
cudaError_t launch_rows_by(LpParams p, cudaStream_t st) {
    if ((long long)p.rows * p.parts > INT32_MAX) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.rows * p.parts);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = p.parts;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.parts > 1 ? 2 : 1;
    return p.top ? cudaLaunchKernelEx(&cfg, k_logprobs<T, true, THREADS>, p)
                 : cudaLaunchKernelEx(&cfg, k_logprobs<T, false, THREADS>, p);
}

template <class T>
cudaError_t launch_rows(LpParams p, cudaStream_t st) {
    // Blocks per row: as many as still run at the same time (four of 256 threads per SM), while a
    // thread has a batch. 256 rows of 128000 bf16, 20 alternatives: 29.6, 21.4, 25.3 and 35.0 us with
    // 1, 2, 4 and 8 blocks per row; one row: 15.8, 11.1, 7.7, 6.6 us.
    const int batches = (p.vocab + 32 * 256 - 1) / (32 * 256);
    p.parts = 1;
    while (p.parts < 8 && p.parts < batches && (long long)p.rows * p.parts * 2 <= 148 * 4) p.parts *= 2;
    // With more rows than run at once, eight blocks of 128 threads per SM overlap one row's end with
    // other rows' loads better than four of 256 (2000 rows of 50257 bf16: 44 and 46 us, with 20
    // alternatives 62 and 66), but for many alternatives, whose ranking is shared by the threads (64 of
    // 4096 fp32 rows: 228 and 190 us).
    if (p.rows > 148 * 4 && p.top <= 20) return launch_rows_by<T, 128>(p, st);
    return launch_rows_by<T, 256>(p, st);
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

// 16 bytes from byte `by` (a multiple of the element's size, under 16) of the 32 bytes (a, b). `by`
// is the same in all lanes of a row, so the branch is uniform.
__device__ __forceinline__ uint4 shifted(const uint4& a, const uint4& b, int by) {
    const int bits = (by & 3) * 8;
    switch (by >> 2) {
        case 0:
            return make_uint4(__funnelshift_r(a.x, a.y, bits), __funnelshift_r(a.y, a.z, bits),
                              __funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits));
        case 1:
            return make_uint4(__funnelshift_r(a.y, a.z, bits), __funnelshift_r(a.z, a.w, bits),
                              __funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits));
        case 2:
            return make_uint4(__funnelshift_r(a.z, a.w, bits), __funnelshift_r(a.w, b.x, bits),
                              __funnelshift_r(b.x, b.y, bits), __funnelshift_r(b.y, b.z, bits));
        default:
            return make_uint4(__funnelshift_r(a.w, b.x, bits), __funnelshift_r(b.x, b.y, bits),
                              __funnelshift_r(b.y, b.z, bits), __funnelshift_r(b.z, b.w, bits));
    }
}

// One element in, one out: d_j = -p_j (A + B log2 p_j), the target's plus g / temperature; without an
// entropy gradient (ENT false) B is 0. A block takes four vectors per thread of one row at a time. Vectors are
// the output's; where the input row lies differently against the 16-byte boundaries, its 16 bytes are
// cut from two aligned vectors, the second of which the neighbouring lane holds. Only warps at a
// row's ends check where they are.
// Measured: 4096 rows of 50257 bf16, input rows padded by 7, 142 us (5.8 TB/s; 130 us where both rows lie alike),
// 64 rows of fp32 6.6 us.
template <class T, bool ENT>
__global__ void __launch_bounds__(THREADS) k_logprobs_grad(const __grid_constant__ GradParams p) {
    constexpr int VE = Row<T>::VE, U = 4;
    tc::pdl_trigger();
    tc::pdl_wait();
    const int r = blockIdx.x / p.chunks, chunk = blockIdx.x - r * p.chunks;
    const Row<T> in(static_cast<const T*>(p.x) + (long long)r * p.ld, p.vocab);
    T* dx = static_cast<T*>(p.dx) + (long long)r * p.ldo;
    const Row<T> out(dx, p.vocab);
    const int lane = threadIdx.x & 31;
    // the output's vector v begins `off` elements into the input's vector v + down
    const int off = (in.shift - out.shift + VE) % VE, down = in.shift < out.shift ? -1 : 0;
    const uint4* src0 = reinterpret_cast<const uint4*>(in.x - in.shift) + down + lane;
    float m = __ldcg(p.stats + 3LL * r), ls = __ldcg(p.stats + 3LL * r + 1), h = __ldcg(p.stats + 3LL * r + 2);
    float g = p.d_lp ? __ldcg(p.d_lp + r) : 0.f;
    const float ge = ENT ? __ldcg(p.d_ent + r) : 0.f;
    int target = -1;
    if (p.d_lp) {
        const long long t = target_of(p.targets, p.i64, r);
        target = t >= 0 && t < p.vocab ? (int)t : -1;
        if (t < 0) g = 0.f;
        if (t >= p.vocab) g = NAN;
    }
    float A = -p.inv_t * (g + ge * h), B = -p.inv_t * ge * LN2, hit = p.inv_t * g;
    if (m == -INFINITY && ls == -INFINITY) m = 0.f, ls = INFINITY, A = B = hit = 0.f;  // a row of nothing but -inf: all zeros
    const float c = p.inv_t * LOG2E, l2 = -ls * LOG2E;
    // a warp's U * 32 vectors lie side by side
    for (int wv = chunk * U * THREADS + (threadIdx.x & ~31) * U; wv < out.vectors; wv += p.chunks * U * THREADS) {
        const uint4* src = src0 + wv;
        uint4 raw[U];
        bool inner[U];  // all of the warp's vectors, and those they are cut from, are inside the row
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int w0 = wv + u * 32;
            inner[u] = w0 >= 2 && (w0 + 34) * VE <= p.vocab;
            if (inner[u])
                raw[u] = __ldcg(src + u * 32);
            else if (w0 < out.vectors)
                raw[u] = in.edge(out.first(w0 + lane));
        }
        if (off && inner[0]) {
            // lane i's second vector is lane i + 1's, lane 31's that of lane 0 one step on; the last
            // inner step's is loaded for it
            int last = 0;
#pragma unroll
            for (int u = 1; u < U; ++u) last += inner[u];
            uint4 more = raw[0];
            if (lane == 0) more = __ldcg(src + last * 32 + 32);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!inner[u]) continue;
                uint4 b = u + 1 < U && u < last ? raw[u + 1 < U ? u + 1 : u] : more;
                if (lane != 0) b = raw[u];
                b.x = __shfl_sync(0xffffffffu, b.x, (lane + 1) & 31);
                b.y = __shfl_sync(0xffffffffu, b.y, (lane + 1) & 31);
                b.z = __shfl_sync(0xffffffffu, b.z, (lane + 1) & 31);
                b.w = __shfl_sync(0xffffffffu, b.w, (lane + 1) & 31);
                raw[u] = shifted(raw[u], b, off * (int)sizeof(T));
            }
        } else if (off) {
            // the row's beginning: its inner steps one by one
#pragma unroll
            for (int u = 1; u < U; ++u) {
                if (!inner[u]) continue;
                raw[u] = in.edge(out.first(wv + u * 32 + lane));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = wv + u * 32 + lane, e = out.first(v);
            if (!inner[u] && v >= out.vectors) continue;
            float2 f[VE / 2];
            unpack<T>(raw[u], f);
#pragma unroll
            for (int i = 0; i < VE / 2; ++i) {
                const float2 z = fma2(add2(f[i], make_float2(-m, -m)), make_float2(c, c), make_float2(l2, l2));
                const float2 q = make_float2(ex2(z.x), ex2(z.y));
                if constexpr (ENT) {
                    // log2 p of a masked element is -inf; the clamp keeps its 0 * log2 p at 0
                    const float2 k = make_float2(fmaxf(z.x, -2000.f), fmaxf(z.y, -2000.f));
                    f[i] = mul2(q, fma2(k, make_float2(B, B), make_float2(A, A)));
                } else {
                    f[i] = mul2(q, make_float2(A, A));
                }
            }
            if ((unsigned)(target - e) < (unsigned)VE && target >= 0) {
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    if (target == e + i) (i & 1 ? f[i / 2].y : f[i / 2].x) += hit;
            }
            union {
                uint4 u4;
                T t[VE];
            } o;
            o.u4 = packed<T>(f);
            if (inner[u] || (e >= 0 && e + VE <= p.vocab)) {
                *reinterpret_cast<uint4*>(dx + e) = o.u4;
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    if (e + i >= 0 && e + i < p.vocab) dx[e + i] = o.t[i];
            }
        }
    }
}

template <class T>
cudaError_t launch_grad(GradParams p, cudaStream_t st) {
    constexpr int per = 4 * THREADS * Row<T>::VE;
    // blocks per row: one batch of four vectors per thread each while the call has fewer blocks than
    // run at once (five per SM), else as few as fill the GPU four times over, so that a thread's reading of the row's
    // statistics and alignment serves many batches
    const int most = (p.vocab + Row<T>::VE - 1 + per - 1) / per;
    p.chunks = (int)std::clamp<long long>(148LL * 5 * 4 / p.rows, 1, most);
    if ((long long)p.rows * p.chunks > INT32_MAX) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)p.rows * p.chunks);
    return p.d_ent ? launch_dependent(k_logprobs_grad<T, true>, grid, dim3(THREADS), 0, st, p)
                   : launch_dependent(k_logprobs_grad<T, false>, grid, dim3(THREADS), 0, st, p);
}

int refuse(const char* who, const char* msg) {
    set_global_error(std::string(who) + ": " + msg);
    return GPT2Q_EARG;
}

int check(const char* who, const void* x, int dtype, int64_t ld, int n_rows, int vocab, float temperature) {
    if (n_rows < 0) return refuse(who, "n_rows < 0");
    if (vocab < 1 || ld < vocab) return refuse(who, "vocab must be >= 1 and ld >= vocab");
    if (vocab > 1 << 30) return refuse(who, "vocab must be at most 2^30");  // the kernels count a row's elements in 32 bits
    if (dtype < GPT2Q_F32 || dtype > GPT2Q_BF16) return refuse(who, "unknown dtype");
    // below about 1e-36 the kernels' factors leave fp32, and 0 times one of them would be NaN
    if (!(temperature >= 1e-30f) || !std::isfinite(temperature)) return refuse(who, "temperature must be finite and at least 1e-30");
    if (n_rows > 0 && !x) return refuse(who, "null logits");
    if (reinterpret_cast<uintptr_t>(x) % (dtype == GPT2Q_F32 ? 4 : 2)) return refuse(who, "unaligned logits");
    return GPT2Q_OK;
}

}  // namespace

cudaError_t gpt2q::launch_logprobs(const float* logits, int ld, int rows, int vocab, const int32_t* targets, int top,
                                   float* lp, float* entropy, float* stats, int32_t* top_ids, float* top_lp, cudaStream_t st) {
    return launch_rows<float>(LpParams{logits, ld, rows, vocab, top, 1, 1.f, targets, 0, lp, entropy, stats, top_ids, top_lp}, st);
}

cudaError_t gpt2q::launch_logprobs_grad(float* logits, int ld, int rows, int vocab, const int32_t* targets, const float* stats,
                                        const float* d_lp, const float* d_ent, cudaStream_t st) {
    return launch_grad<float>(GradParams{logits, logits, ld, ld, rows, vocab, 1, 1.f, targets, 0, stats, d_lp, d_ent}, st);
}

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
        e = launch_rows<float>(p, st);
    else if (dtype == GPT2Q_F16)
        e = launch_rows<__half>(p, st);
    else
        e = launch_rows<bf16>(p, st);
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
    if (d_dlogits != d_logits && ld_out == ld) {
        // rows of the one that lie over rows of the other; those of both side by side in one buffer do not
        const int size = dtype == GPT2Q_F32 ? 4 : 2;
        const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(d_dlogits) - reinterpret_cast<uintptr_t>(d_logits)) / size;
        const int64_t apart = off < 0 ? -off : off, in_row = apart % ld;
        if (apart < (n_rows - 1) * ld + vocab && (in_row < vocab || (in_row > ld - vocab && apart / ld < n_rows - 1)))
            return refuse(who, "dlogits overlap the logits");
    }
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
