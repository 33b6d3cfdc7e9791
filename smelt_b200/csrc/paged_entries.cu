// Kernels that move the entries of a paged cache: append with position rotation (and quantisation), read, commit.
#include <cuda_fp8.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "device_op.cuh"
#include "gpt2q.h"
#include "paged.h"

using namespace gpt2q;

namespace {

// Where position `pos` of a table row lies; page -1: nowhere, and `slot` is the status bit.
struct Place {
    int page, slot;
};
template <class P>
__device__ __forceinline__ Place place(const P& p, int row, int pos) {
    if (row < 0 || row >= p.n_rows) return {-1, GPT2Q_STATUS_ROW};
    if (pos < 0) return {-1, GPT2Q_STATUS_POSITION};
    const int pg = pos / p.page;
    if (pg >= p.width) return {-1, GPT2Q_STATUS_POSITION};
    const int id = __ldcg(p.table + (long long)row * p.ld + pg);
    if (id < 0 || id >= p.n_pages) return {-1, GPT2Q_STATUS_PAGE};
    return {id, pos - pg * p.page};
}

// ------------------------------------------------------------------ 8-bit codes
template <class TC>
constexpr float code_top() { return std::is_same<TC, int8_t>::value ? 127.f : 448.f; }

// |x| as a number whose order is that of magnitudes, with NaN above infinity
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of an entry of largest magnitude `top`, and its codes: x * (T / top) rounded once more, to nearest even. The
// quotients and the product are fp32 operations of their own (no fused product), so that the codes of given values
// are the same wherever they are computed.
template <class TC>
struct Scale {
    float scale, inverse;
    __device__ __forceinline__ explicit Scale(uint32_t top) {
        constexpr uint32_t LEAST = 27u << 23;  // 2^-100: T / top stays finite, the scale a normal number
        const float t = __uint_as_float(top);
        const bool some = top >= LEAST && top < 0x7f800000u;
        // (at most the number whose product with T is finite)
        scale = some ? fminf(__fdiv_rn(t, code_top<TC>()), __fdiv_rd(3.402823466e38f, code_top<TC>()))
                     : top < LEAST ? 0.f : __uint_as_float(0x7fffffffu);
        inverse = some ? __fdiv_rn(code_top<TC>(), t) : 0.f;
    }
    // four codes; 0 where there is no finite scale
    __device__ __forceinline__ uint32_t codes(const float* x) const {
        if (inverse == 0.f) return 0;
        if constexpr (std::is_same<TC, int8_t>::value) {
            uint32_t r[4];
            // 1.5 * 2^23 + y has the rounded y in its lowest bits
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inverse), 12582912.f));
            return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
        } else {
            uint32_t r;
            asm("{\n\t.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\tmov.b32 %0, {a, b};\n\t}"
                : "=r"(r)
                : "f"(__fmul_rn(x[0], inverse)), "f"(__fmul_rn(x[1], inverse)), "f"(__fmul_rn(x[2], inverse)), "f"(__fmul_rn(x[3], inverse)));
            return r;
        }
    }
};
// two codes as values before the scale
template <class TC>
__device__ __forceinline__ float2 decode2(uint32_t v) {  // the lower 16 bits
    if constexpr (std::is_same<TC, int8_t>::value) {
        return make_float2((float)(int8_t)(v & 0xff), (float)(int8_t)(v >> 8 & 0xff));
    } else {
        uint32_t h;
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(h) : "r"(v));
        return __half22float2(*reinterpret_cast<const __half2*>(&h));
    }
}

// ------------------------------------------------------------------ append
// A unit is two chunks of V consecutive elements of a head, chosen so that neighbouring threads' chunks
// are neighbours: the (a, b) of V rotated pairs, or chunks that are rotated within themselves
// (interleaved pairs) or only copied; a head has dim / (2 V) of them. A thread takes one unit index of one
// token and walks over the token's heads (queries, keys, values), `groups` threads sharing a unit
// index, so that the sines and cosines of its V pairs are computed once per thread. The angle is
// the fractional part of position * turns, formed in fp64 (fp32 would lose 2^-24 * position turns:
// 0.4 rad at a position of a million), then sincospif in fp32. Bound by the memory in a prompt;
// loading four heads at a time was slower (117 against 88 us at 16 thousand tokens of 48 heads), as it
// halved the threads an SM holds.
//
// Into an 8-bit cache the threads of a unit row, neighbouring lanes, hold an entry between them: its largest magnitude
// goes round by shuffles, and each writes 16 codes. 24 prompts of 60 to 2600 tokens, 48 heads of 128, bf16 to e4m3: 94 us (59 at the
// memory rate).
constexpr int BLOCKS = 4;  // of 256 threads per SM (64 registers a thread): 80 us at 16 thousand tokens; 88, 86, 90 with 3, 5, 6

template <class TI, class TC, int V>
__global__ void __launch_bounds__(256, BLOCKS) k_paged_append(const __grid_constant__ AppendParams p) {
    tc::pdl_trigger();
    tc::pdl_wait();
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int u = (int)(id & ((1 << p.unit_shift) - 1));
    const long long rest = id >> p.unit_shift;
    const int g = (int)(rest % p.groups);
    const long long ti = rest / p.groups;
    constexpr bool Q8 = sizeof(TC) == 1;
    const bool idle = u * 2 * V >= p.dim;
    if (ti >= p.n_tokens || (!Q8 && idle)) return;
    const int pos = p.pos ? __ldcg(p.pos + ti) : p.pos0 + (int)ti;
    const Place to = pos < 0 ? Place{-1, 0} : place(p, p.pos ? (p.seq ? __ldcg(p.seq + ti) : (int)ti) : 0, p.slot ? __ldcg(p.slot + ti) : pos);
    if (pos >= 0 && to.page < 0 && p.status && u == 0 && g == 0) atomicOr(p.status, to.slot);
    // the token's entry in a pool, before the head
    const long long at = to.page < 0 ? -1 : (long long)to.page * p.c_ps + (long long)to.slot * p.c_ts;
    // the unit's chunks in queries and keys (values: those of plain copies), and whether each is rotated
    const int va = V == 1 ? 2 * u : u * V, vb = V == 1 ? va + 1 : va + p.dim / 2;
    int ca = va, cb = vb;
    if (!p.interleaved && p.rot) {
        const int w = u - p.rot / (2 * V);  // units after the rotated pairs
        ca = w < 0 ? u * V : p.rot + w * V;
        cb = w < 0 ? ca + p.rot / 2 : ca + (p.dim - p.rot) / 2;
    }
    const bool turn_a = pos >= 0 && ca < p.rot, turn_b = pos >= 0 && cb < p.rot;
    float cs[V], sn[V];
    if (turn_a) {  // turn_b only where turn_a
#pragma unroll
        for (int e = 0; e < V; ++e) {
            // pair of element e: of (a[e], b[e]), or with interleaved pairs of a's V / 2 pairs, then b's
            const bool own = !p.interleaved || V == 1 || e < V / 2;
            const int pair = !p.interleaved || V == 1 ? u * V + e : own ? ca / 2 + e : cb / 2 + e - V / 2;
            double t = own || turn_b ? (double)pos * p.turns[pair] : 0.0;
            t -= rint(t);
            sincospif((float)(2.0 * t), &sn[e], &cs[e]);
        }
    }
    const int heads = p.n_q + 2 * p.n_kv;
    [[maybe_unused]] const unsigned mates = Q8 ? ((2u << ((1 << p.unit_shift) - 1)) - 1) << (threadIdx.x & 31 & ~((1 << p.unit_shift) - 1)) : 0;
    for (int h = g; h < heads; h += p.groups) {
        const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
        if (is_q ? idle : at < 0) continue;
        const int hk = is_q ? h : is_v ? h - p.n_q - p.n_kv : h - p.n_q;
        const TI* src = is_q ? static_cast<const TI*>(p.q) + ti * p.q_ts + hk * p.q_hs
                             : is_v ? static_cast<const TI*>(p.v) + ti * p.v_ts + hk * p.v_hs
                                    : static_cast<const TI*>(p.k) + ti * p.k_ts + hk * p.k_hs;
        const int oa = is_v ? va : ca, ob = is_v ? vb : cb;
        float a[V] = {}, b[V] = {};
        if (!idle) {
            load_vec<TI, V>(src + oa, a);
            load_vec<TI, V>(src + ob, b);
        }
        if (!is_v && turn_a) {
            if (!p.interleaved || V == 1) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float x = a[e], y = b[e];
                    a[e] = x * cs[e] - y * sn[e];
                    b[e] = y * cs[e] + x * sn[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e + 1 < V; e += 2) {
                    float x = a[e], y = a[e + 1];
                    a[e] = x * cs[e / 2] - y * sn[e / 2];
                    a[e + 1] = y * cs[e / 2] + x * sn[e / 2];
                    if (turn_b) {
                        x = b[e], y = b[e + 1];
                        b[e] = x * cs[V / 2 + e / 2] - y * sn[V / 2 + e / 2];
                        b[e + 1] = y * cs[V / 2 + e / 2] + x * sn[V / 2 + e / 2];
                    }
                }
            }
        }
        if (is_q) {
            TI* dst = static_cast<TI*>(p.qo) + ti * p.qo_ts + hk * p.qo_hs;
            store_vec<TI, V>(dst + oa, a);
            store_vec<TI, V>(dst + ob, b);
        } else if constexpr (Q8) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < V; ++e) top = max(top, max(magnitude(a[e]), magnitude(b[e])));
            for (int o = 1; o < 1 << p.unit_shift; o <<= 1) top = max(top, __shfl_xor_sync(mates, top, o));
            const Scale<TC> s(top);
            TC* dst = static_cast<TC*>(is_v ? p.vc : p.kc) + at + hk * p.c_hs;
            if (!idle) {
                *reinterpret_cast<uint2*>(dst + oa) = make_uint2(s.codes(a), s.codes(a + 4));
                *reinterpret_cast<uint2*>(dst + ob) = make_uint2(s.codes(b), s.codes(b + 4));
            }
            if (u == 0) (is_v ? p.v_scale : p.k_scale)[(long long)to.page * p.s_ps + hk * p.s_hs + (long long)to.slot * p.s_ts] = s.scale;
        } else {
            TC* dst = static_cast<TC*>(is_v ? p.vc : p.kc) + at + hk * p.c_hs;
            store_vec<TC, V>(dst + oa, a);
            store_vec<TC, V>(dst + ob, b);
        }
    }
}


// The same into an 8-bit cache for tensors that are not 16-byte aligned, or a rotation of no whole chunks: a warp takes one
// entry (or query) element by element, lane l elements l, l + 32, ...; the partner of a rotated element is loaded again.
template <class TI, class TC>
__global__ void __launch_bounds__(256) k_paged_append_any(const __grid_constant__ AppendParams p) {
    tc::pdl_trigger();
    tc::pdl_wait();
    const int heads = p.n_q + 2 * p.n_kv, lane = threadIdx.x & 31;
    const long long id = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5;
    const long long ti = id / heads;
    const int h = (int)(id - ti * heads);
    if (ti >= p.n_tokens) return;
    const int pos = p.pos ? __ldcg(p.pos + ti) : p.pos0 + (int)ti;
    const Place to = pos < 0 ? Place{-1, 0} : place(p, p.pos ? (p.seq ? __ldcg(p.seq + ti) : (int)ti) : 0, p.slot ? __ldcg(p.slot + ti) : pos);
    if (pos >= 0 && to.page < 0 && p.status && h == 0 && lane == 0) atomicOr(p.status, to.slot);
    const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
    if (!is_q && to.page < 0) return;
    const int hk = is_q ? h : is_v ? h - p.n_q - p.n_kv : h - p.n_q;
    const TI* src = is_q ? static_cast<const TI*>(p.q) + ti * p.q_ts + hk * p.q_hs
                         : is_v ? static_cast<const TI*>(p.v) + ti * p.v_ts + hk * p.v_hs
                                : static_cast<const TI*>(p.k) + ti * p.k_ts + hk * p.k_hs;
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int e = i * 32 + lane;
        x[i] = e < p.dim ? to_f(src[e]) : 0.f;
        if (!is_v && pos >= 0 && e < p.rot) {
            const int half = p.rot / 2;
            const bool second = p.interleaved ? e & 1 : e >= half;
            const int pair = p.interleaved ? e / 2 : second ? e - half : e;
            const float other = to_f(src[p.interleaved ? e ^ 1 : second ? e - half : e + half]);
            double t = (double)pos * p.turns[pair];
            t -= rint(t);
            float sn, cs;
            sincospif((float)(2.0 * t), &sn, &cs);
            x[i] = second ? x[i] * cs + other * sn : x[i] * cs - other * sn;
        }
        top = max(top, magnitude(x[i]));
    }
    if (is_q) {
        __syncwarp();  // q_out may be q: every lane has its partner
        TI* dst = static_cast<TI*>(p.qo) + ti * p.qo_ts + hk * p.qo_hs;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i * 32 + lane < p.dim) dst[i * 32 + lane] = from_f<TI>(x[i]);
        return;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    const Scale<TC> s(top);
    uint8_t* dst = static_cast<uint8_t*>(is_v ? p.vc : p.kc) + (long long)to.page * p.c_ps + (long long)to.slot * p.c_ts + hk * p.c_hs;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
        const uint32_t c = s.codes(x + i);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((i + j) * 32 + lane < p.dim) dst[(i + j) * 32 + lane] = (uint8_t)(c >> 8 * j);
    }
    if (lane == 0) (is_v ? p.v_scale : p.k_scale)[(long long)to.page * p.s_ps + hk * p.s_hs + (long long)to.slot * p.s_ts] = s.scale;
}

template <class TI, class TC>
cudaError_t append(AppendParams p, bool vec, cudaStream_t st) {
    const long long heads = (long long)p.n_q + 2LL * p.n_kv;
    long long blocks;
    if (sizeof(TC) == 1 && !vec) {
        blocks = ((long long)p.n_tokens * heads + 7) / 8;
        if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
        return launch_dependent(k_paged_append_any<TI, TC>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    }
    const int units = p.dim / (vec ? 16 : 2);
    while ((1 << p.unit_shift) < units) ++p.unit_shift;
    // heads a thread walks over: one while the call has fewer threads than the GPU holds, so that a
    // decode step is one round of loads; up to 8 in a large call, where the angles' arithmetic
    // would otherwise be repeated for every head
    const long long threads = ((long long)p.n_tokens << p.unit_shift) * heads;
    const long long walk = std::clamp<long long>(threads / (148 * 2048), 1, 8);
    p.groups = (int)((heads + walk - 1) / walk);
    blocks = ((((long long)p.n_tokens * p.groups) << p.unit_shift) + 255) / 256;
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    if constexpr (sizeof(TC) > 1)
        if (!vec) return launch_dependent(k_paged_append<TI, TC, 1>, dim3((unsigned)blocks), dim3(256), 0, st, p);
    return launch_dependent(k_paged_append<TI, TC, 8>, dim3((unsigned)blocks), dim3(256), 0, st, p);
}

// ------------------------------------------------------------------ read
// A warp per token, whose place is looked up once: its lanes take the token's heads' elements, 16 bytes of output each and
// neighbours side by side, READ of them at a time with all loads on their way before the first is used. (Threads that each
// looked up their own token took 188 us for 100 thousand tokens with 16 codes each, 232 with 8.) Bound by the memory.
constexpr int READ = 8;

template <class TC, class TO, bool VEC>
__global__ void __launch_bounds__(256) k_paged_read(const __grid_constant__ EntryParams p, int chunks) {
    constexpr int N = 16 / sizeof(TO), B = N * sizeof(TC);  // elements, and their bytes in the cache: 4, 8 or 16
    using Raw = std::conditional_t<B == 16, uint4, std::conditional_t<B == 8, uint2, unsigned>>;
    tc::pdl_trigger();
    tc::pdl_wait();
    const int ti = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (ti >= p.n_tokens) return;
    const int pos = __ldcg(p.pos + ti);
    const Place at = pos < 0 ? Place{-1, 0} : place(p, p.seq ? __ldcg(p.seq + ti) : ti, pos);
    const bool there = at.page >= 0;
    if (pos >= 0 && !there && p.status && lane == 0) atomicOr(p.status, at.slot);
    const float none = pos < 0 ? 0.f : __uint_as_float(0x7fffffffu);  // padding, or out of range
    const long long off = (long long)at.page * p.c_ps + (long long)at.slot * p.c_ts, s_off = (long long)at.page * p.s_ps + (long long)at.slot * p.s_ts;
    const unsigned units = 2u * p.n_kv * chunks;
    for (unsigned u0 = lane; u0 < units; u0 += 32 * READ) {
        Raw raw[READ];
        float scale[READ];
#pragma unroll
        for (int i = 0; i < READ; ++i) {
            const unsigned u = u0 + i * 32;
            if (u >= units || !there) continue;
            const int hh = u / (unsigned)chunks, c = u - hh * chunks, h = hh < p.n_kv ? hh : hh - p.n_kv;
            raw[i] = __ldcg(reinterpret_cast<const Raw*>(static_cast<const TC*>(hh < p.n_kv ? p.kc : p.vc) + off + h * p.c_hs + c * N));
            if constexpr (sizeof(TC) == 1) scale[i] = __ldcg((hh < p.n_kv ? p.k_scale : p.v_scale) + s_off + h * p.s_hs);
        }
#pragma unroll
        for (int i = 0; i < READ; ++i) {
            const unsigned u = u0 + i * 32;
            if (u >= units) continue;
            const int hh = u / (unsigned)chunks, c = u - hh * chunks, h = hh < p.n_kv ? hh : hh - p.n_kv;
            TO* dst = (hh < p.n_kv ? static_cast<TO*>(p.k) + ti * p.k_ts + h * p.k_hs : static_cast<TO*>(p.v) + ti * p.v_ts + h * p.v_hs) + c * N;
            union {
                uint4 u4;
                TO t[N];
            } r;
            if (there) {
                if constexpr (sizeof(TC) == 1) {
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[i]);
#pragma unroll
                    for (int e = 0; e < N; e += 2) {
                        const float2 v = decode2<TC>(w[e / 4] >> (e & 2) * 8);
                        r.t[e] = from_f<TO>(v.x * scale[i]), r.t[e + 1] = from_f<TO>(v.y * scale[i]);
                    }
                } else {
                    const TC* v = reinterpret_cast<const TC*>(&raw[i]);
#pragma unroll
                    for (int e = 0; e < N; ++e) r.t[e] = from_f<TO>(to_f(v[e]));
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) r.t[e] = from_f<TO>(none);
            }
            if constexpr (VEC) {
                *reinterpret_cast<uint4*>(dst) = r.u4;
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) dst[e] = r.t[e];
            }
        }
    }
}

template <class TC, class TO>
cudaError_t read(const EntryParams& p, bool vec, cudaStream_t st) {
    const int chunks = p.dim * (int)sizeof(TO) / 16;
    if (2LL * p.n_kv * chunks > INT32_MAX) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)(((long long)p.n_tokens + 7) / 8));
    return vec ? launch_dependent(k_paged_read<TC, TO, true>, grid, dim3(256), 0, st, p, chunks)
               : launch_dependent(k_paged_read<TC, TO, false>, grid, dim3(256), 0, st, p, chunks);
}

// ------------------------------------------------------------------ commit
// A block looks up 256 tokens of a row's list at once, a thread each, and finds where the list ends. Then every thread owns
// 16 bytes of one (pool, head) - or its scale - and carries them through the list in order, eight entries at a time: loads, then
// stores. Tokens rise, so an entry is never behind the place that it goes to, and a place that is written lies before every
// entry that is still to be read. Bound by latency: the list, the table, then a round of loads for eight tokens (looked up eight at a time
// in turn, 256 rows of up to 14 tokens took 12.9 us a call).
constexpr int MOVES = 8, LIST = 256;

template <bool Q8>
__global__ void __launch_bounds__(LIST) k_paged_commit(const __grid_constant__ EntryParams p, int chunks, int size) {
    __shared__ int2 s_from[LIST], s_to[LIST];  // page, slot
    __shared__ int s_a[LIST + 1], s_end;
    tc::pdl_trigger();
    tc::pdl_wait();
    const int row = blockIdx.x, tid = threadIdx.x, id = blockIdx.y * LIST + tid;
    const int pools = 2 * p.n_kv * chunks;  // threads of codes; then, of an 8-bit cache, those of scales
    const bool scales = Q8 && id >= pools, here = id < pools + (Q8 ? 2 * p.n_kv : 0);
    const int hh = scales ? id - pools : id / chunks, c = scales ? 0 : id - hh * chunks;
    const bool is_v = hh >= p.n_kv;
    const int h = is_v ? hh - p.n_kv : hh;
    char* base = scales ? reinterpret_cast<char*>((is_v ? p.v_scale : p.k_scale) + h * p.s_hs)
                        : static_cast<char*>(is_v ? p.vc : p.kc) + h * p.c_hs * size + c * 16;
    const long long ps = scales ? p.s_ps * 4 : p.c_ps * size, ts = scales ? p.s_ts * 4 : p.c_ts * size;
    const int len = max(__ldcg(p.lens + row), 0);
    const int* accept = p.accept + row * p.accept_ld;
    int kept = 0;
    for (bool more = true; more && kept < p.n_accept;) {
        const int i = kept + tid, a = i < p.n_accept ? __ldcg(accept + i) : -1;
        if (tid == 0) {
            s_end = LIST;
            s_a[0] = kept ? s_a[LIST] : -1;  // the token before
        }
        __syncthreads();
        s_a[tid + 1] = a;
        Place x{-1, GPT2Q_STATUS_POSITION}, y = x;
        if (a >= 0 && a <= INT32_MAX - len) x = place(p, row, len + a);
        if (a >= 0 && i <= INT32_MAX - len) y = place(p, row, len + i);
        s_from[tid] = make_int2(x.page, x.slot);
        s_to[tid] = make_int2(y.page, y.slot);
        __syncthreads();
        const bool rises = a > s_a[tid];
        if (a < 0 || !rises || x.page < 0 || y.page < 0) atomicMin(&s_end, tid);
        __syncthreads();
        const int n = s_end;
        more = n == LIST;
        if (tid == n && a >= 0 && blockIdx.y == 0 && p.status)
            atomicOr(p.status, !rises ? GPT2Q_STATUS_POSITION : x.page < 0 ? x.slot : y.slot);
        for (int j = 0; j < n && here; j += MOVES) {
            uint4 v[MOVES];
#pragma unroll
            for (int k = 0; k < MOVES; ++k) {
                if (j + k >= n || s_a[j + k + 1] == kept + j + k) continue;
                const int2 at = s_from[j + k];
                const char* from = base + at.x * ps + at.y * ts;
                if (Q8 && scales)
                    v[k].x = __ldcg(reinterpret_cast<const unsigned*>(from));
                else
                    v[k] = __ldcg(reinterpret_cast<const uint4*>(from));
            }
#pragma unroll
            for (int k = 0; k < MOVES; ++k) {
                if (j + k >= n || s_a[j + k + 1] == kept + j + k) continue;
                const int2 at = s_to[j + k];
                char* to = base + at.x * ps + at.y * ts;
                if (Q8 && scales)
                    *reinterpret_cast<unsigned*>(to) = v[k].x;
                else
                    *reinterpret_cast<uint4*>(to) = v[k];
            }
        }
        kept += n;
        __syncthreads();  // before the list's next part
    }
    if (id == 0) p.new_lens[row] = len + kept;
}

}  // namespace

cudaError_t gpt2q::launch_append(AppendParams p, int cache, int dtype, bool vec, cudaStream_t st) {
    if (cache == GPT2Q_F32) return append<float, float>(p, vec, st);
    if (cache == GPT2Q_F16) return dtype == GPT2Q_F32 ? append<float, __half>(p, vec, st) : append<__half, __half>(p, vec, st);
    if (cache == GPT2Q_BF16) return dtype == GPT2Q_F32 ? append<float, bf16>(p, vec, st) : append<bf16, bf16>(p, vec, st);
    if (cache == GPT2Q_I8)
        return dtype == GPT2Q_F32 ? append<float, int8_t>(p, vec, st)
                                  : dtype == GPT2Q_F16 ? append<__half, int8_t>(p, vec, st) : append<bf16, int8_t>(p, vec, st);
    return dtype == GPT2Q_F32 ? append<float, __nv_fp8_e4m3>(p, vec, st)
                              : dtype == GPT2Q_F16 ? append<__half, __nv_fp8_e4m3>(p, vec, st) : append<bf16, __nv_fp8_e4m3>(p, vec, st);
}

cudaError_t gpt2q::launch_read(const EntryParams& p, int cache, int dtype, bool vec, cudaStream_t st) {
    if (cache == GPT2Q_F32) return read<float, float>(p, vec, st);
    if (cache == GPT2Q_F16) return dtype == GPT2Q_F32 ? read<__half, float>(p, vec, st) : read<__half, __half>(p, vec, st);
    if (cache == GPT2Q_BF16) return dtype == GPT2Q_F32 ? read<bf16, float>(p, vec, st) : read<bf16, bf16>(p, vec, st);
    if (cache == GPT2Q_I8)
        return dtype == GPT2Q_F32 ? read<int8_t, float>(p, vec, st)
                                  : dtype == GPT2Q_F16 ? read<int8_t, __half>(p, vec, st) : read<int8_t, bf16>(p, vec, st);
    return dtype == GPT2Q_F32 ? read<__nv_fp8_e4m3, float>(p, vec, st)
                              : dtype == GPT2Q_F16 ? read<__nv_fp8_e4m3, __half>(p, vec, st) : read<__nv_fp8_e4m3, bf16>(p, vec, st);
}

cudaError_t gpt2q::launch_commit(const EntryParams& p, int cache, cudaStream_t st) {
    const int size = size_of(cache), chunks = p.dim * size / 16;
    const long long threads = 2LL * p.n_kv * (chunks + (size == 1 ? 1 : 0));
    if (threads > 65535LL * 256) return cudaErrorInvalidConfiguration;
    const dim3 grid(p.n_rows, (unsigned)((threads + 255) / 256));
    return size == 1 ? launch_dependent(k_paged_commit<true>, grid, dim3(256), 0, st, p, chunks, size)
                     : launch_dependent(k_paged_commit<false>, grid, dim3(256), 0, st, p, chunks, size);
}
