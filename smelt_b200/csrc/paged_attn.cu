// Attention of one new token per row over a paged key/value cache (gpt2q_paged_attention).
//
//   out[r][h] = sum_j softmax_j(scale q[r][h] . K[j]) V[j]
//
// Every cached byte is used once, for the few query heads that share its kv head, so the bound is
// the memory: 4 FLOP per element and query head against 2 or 4 bytes. The work is one flat list of
// tiles of TK keys, ordered by row, kv head and position. The grid is one block per SM; block and
// warp take consecutive ranges of equal length, whatever the rows' lengths are, so that one long
// row and many short ones both keep every SM's loads busy to the end. A range's first and last
// (row, head) are usually incomplete: their running maximum, sum and weighted values meet first
// inside the block, through shared memory, and then over the blocks in a second small kernel.
// Nothing is accumulated with atomics, so results are the same on every run.
//
// A warp streams its tiles through a ring of three shared-memory stages of its own (cp.async, 16
// bytes per lane; the page of every key is looked up one tile ahead), so warps never wait for each
// other while they stream.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "device_op.cuh"
#include "gpt2q.h"
#include "paged.h"

using namespace gpt2q;

namespace {

constexpr int STAGES = 3;
constexpr int MAX_WARPS = 8;
constexpr int MAX_CTAS = 148;  // one per SM of a B200
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// TC: cache type, TI: type of q and out, HD: head dim rounded up, HB: query heads a tile is used for.
template <class TC_, class TI_, int HD_, int HB_>
struct Cfg {
    using TC = TC_;
    using TI = TI_;
    static constexpr int HD = HD_, HB = HB_;
    static constexpr bool F32 = std::is_same<TC, float>::value;
    static constexpr bool HALF = std::is_same<TC, __half>::value;
    static constexpr int ROWB = HD * (int)sizeof(TC);
    static constexpr int CHP = ROWB / 16;  // 16-byte chunks of a row
    // keys of a tile: 8 KB of keys and values (16 KB at 256 dims)
    static constexpr int TK = F32 ? (HD == 64 ? 16 : 8) : (HD == 64 ? 32 : 16);
    static constexpr int LPK = 32 / TK;  // lanes per key (fp32 cache)
    static constexpr int GR = TK < 16 ? TK : 16, NG = TK / GR;  // keys of one page lookup where pages allow it
    static constexpr int ITS = TK * CHP / 32, RPI = 32 / CHP > 0 ? 32 / CHP : 1;  // copies of a tile, rows of one copy
    static constexpr int STAGE = 2 * TK * ROWB;
    static constexpr int HS = HD + 4;  // floats of a partial result's row
    // 16-bit pieces of the query and of the weights. Queries of the cache's type are exact in one;
    // fp32 ones take two fp16 (22 bits) or three bf16 (24 bits). Weights take as many, and two where
    // the output has 16 bits: one piece would add an error as large as the output's own rounding.
    static constexpr int SQ = F32 || !std::is_same<TI, float>::value ? 1 : HALF ? 2 : 3;
    static constexpr int sp() { return SQ == 1 ? 2 : SQ; }
    static constexpr int MT = TK / 16, NT = HB / 8, KD = HD / 16;
    // fp16 weights are held times 2^10, so that small ones stay normal numbers
    static constexpr float shift() { return HALF ? 10.f : 0.f; }
    static constexpr float UNSHIFT = HALF ? 1.f / 1024.f : 1.f;
};

struct Walk {
    int row, vh, j, nt, start, end;
    bool over;
};

struct Piece {
    long long first;  // index of its segment's first tile
    int nt, row, vh;  // nt = 0: none
    const float* data;
};

template <class C>
__device__ __forceinline__ void enter(const PagedAttn& p, Walk& w, int row) {
    w.row = row;
    const int len = row < p.n_rows ? __ldcg(p.lens + row) : 0;
    w.over = len > p.cap;
    w.end = w.over ? p.cap : len;
    w.start = p.window > 0 && w.end > p.window ? w.end - p.window : 0;
    // tiles begin at multiples of TK, so that a group of GR keys lies in one page
    w.nt = w.end > 0 ? (w.end + C::TK - 1) / C::TK - w.start / C::TK : 0;
}

template <class C>
__device__ __forceinline__ void advance(const PagedAttn& p, Walk& w) {
    if (++w.j < w.nt) return;
    w.j = 0;
    if (++w.vh < p.n_vh) return;
    w.vh = 0;
    do {
        enter<C>(p, w, w.row + 1);
    } while (w.nt == 0 && w.row < p.n_rows);
}

template <class TC>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<TC, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// (a, b) rounded to a pair of the type; a and b become what the pair leaves over
template <class T>
__device__ __forceinline__ uint32_t take_pair(float& a, float& b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        a -= f.x;
        b -= f.y;
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        const float2 f = __bfloat1622float2(h);
        a -= f.x;
        b -= f.y;
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ex2(float x) {  // 2^x to 2 ulp; results under 2^-126 are 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four elements of one head's result to the output and, when wanted, its fp16 hi/lo copies.
template <class TI>
__device__ __forceinline__ void write4(const PagedAttn& p, int row, int head, int d, const float* r) {
    if (p.out) store_vec<TI, 4>(static_cast<TI*>(p.out) + row * p.o_ts + head * p.o_hs + d, r);
    if (p.hl.hi) {
        const long long at = (long long)row * p.hl.ld + head * p.dim + d;
        float lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = r[i] - __half2float(__float2half_rn(r[i]));
        store_vec<__half, 4>(p.hl.hi + at, r);
        store_vec<__half, 4>(p.hl.lo + at, lo);
    }
}
template <class TI>
__device__ __forceinline__ void write1(const PagedAttn& p, int row, int head, int d, float r) {
    if (p.out) static_cast<TI*>(p.out)[row * p.o_ts + head * p.o_hs + d] = from_f<TI>(r);
    if (p.hl.hi) {
        const long long at = (long long)row * p.hl.ld + head * p.dim + d;
        const __half h = __float2half_rn(r);
        p.hl.hi[at] = h;
        p.hl.lo[at] = __float2half_rn(r - __half2float(h));
    }
}
// l of a row whose keys all have weight 0 is 0: its result is 0 and its logarithm -inf
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * LN2; }

template <class C>
__global__ void __launch_bounds__(MAX_WARPS * 32, 1) k_paged_attn(const __grid_constant__ PagedAttn p) {
    using TC = typename C::TC;
    using TI = typename C::TI;
    constexpr int HB = C::HB, HD = C::HD, TK = C::TK, NT = C::NT > 0 ? C::NT : 1, MT = C::MT > 0 ? C::MT : 1;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long cum[MAX_WARPS * 32 + 1];
    __shared__ long long wsum[MAX_WARPS];
    __shared__ Piece pieces[2 * MAX_WARPS];
    __shared__ float pm[2 * MAX_WARPS][HB], pl[2 * MAX_WARPS][HB];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nthr = blockDim.x, nw = nthr >> 5;
    const int hv = p.heads_per_block;                    // heads a block's partial results hold
    const int qrow = HD * (int)sizeof(TI);               // bytes of a staged query
    unsigned char* ring = smem + (size_t)warp * p.warp_bytes;
    unsigned char* qring = ring + STAGES * C::STAGE;
    float* pbuf = reinterpret_cast<float*>(qring + STAGES * hv * qrow);  // fp32 cache: the tile's weights
    const uint32_t ring32 = tc::smem_u32(ring), q32 = tc::smem_u32(qring);
    const int nch = p.dim * (int)sizeof(TC) / 16, nqch = p.dim * (int)sizeof(TI) / 16;

    if (lane < 2) pieces[2 * warp + lane].nt = 0;
    // dims past the head's own are zero in the ring and are never written again
    if (nch < C::CHP)
        for (int r = lane; r < STAGES * 2 * TK; r += 32)
            for (int c = 0; c < C::CHP; ++c) {
                const int rr = r % TK;
                const int swz = C::F32 ? (rr * C::LPK) & 7 : rr & 7;
                if (c >= nch) *reinterpret_cast<uint4*>(ring + r * C::ROWB + ((c ^ swz) * 16)) = make_uint4(0, 0, 0, 0);
            }
    if (nch < C::CHP)
        for (int i = lane; i < STAGES * hv * (qrow / 16); i += 32)
            if (i % (qrow / 16) >= nqch) *reinterpret_cast<uint4*>(qring + i * 16) = make_uint4(0, 0, 0, 0);
    tc::pdl_trigger();
    tc::pdl_wait();

    // ---- this block's and this warp's range of tiles ----
    const int nc = (p.n_rows + nthr - 1) / nthr;  // rows a thread counts
    Walk w;
    long long mine = 0;
    for (int r = tid * nc; r < min((tid + 1) * nc, p.n_rows); ++r) {
        enter<C>(p, w, r);
        mine += w.nt;
    }
    mine *= p.n_vh;
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    long long before = 0, total = 0;
    for (int i = 0; i < nw; ++i) {
        if (i < warp) before += wsum[i];
        total += wsum[i];
    }
    cum[tid] = before + inc - mine;
    __syncthreads();
    const long long per = ((total + gridDim.x - 1) / gridDim.x + nw - 1) / nw * nw;
    const long long ca = per * blockIdx.x, cb = min(ca + per, total);
    const long long a = ca + per / nw * warp, b = min(a + per / nw, cb);
    const int n = (int)max(0LL, b - a);

    if (n > 0) {
        // the row, head and tile that index a lies in
        int lo = 0, hi = nthr - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cum[mid] <= a)
                lo = mid;
            else
                hi = mid - 1;
        }
        long long rem = a - cum[lo];
        int row = lo * nc;
        enter<C>(p, w, row);
        while (rem >= (long long)w.nt * p.n_vh) {
            rem -= (long long)w.nt * p.n_vh;
            enter<C>(p, w, ++row);
        }
        w.vh = (int)(rem / w.nt);
        w.j = (int)(rem - (long long)w.vh * w.nt);
        // L is the next tile to load, N the one after it, whose pages are on their way
        Walk L = w, N;
        const int kr = lane & (TK - 1);
        const bool grouped = p.grouped != 0;
        int page[C::NG], npage[C::NG];
        // page ids of a tile: of every group of GR keys (the same load in all lanes) where a page is
        // a multiple of GR, else of the lane's own key, in element 0
        auto look = [&](const Walk& t, int* out) {
            const int k0 = (t.start / TK + t.j) * TK;
            const int* ids = p.table + (long long)t.row * p.ld;
            if (grouped) {
#pragma unroll
                for (int g = 0; g < C::NG; ++g) {
                    const int key = k0 + g * C::GR;
                    out[g] = key < t.end && key + C::GR > t.start
                                 ? __ldcg(ids + (p.page_shift >= 0 ? key >> p.page_shift : key / p.page))
                                 : 0;
                }
            } else {
                const int key = k0 + kr;
                out[0] = key < t.end && key >= t.start ? __ldcg(ids + (p.page_shift >= 0 ? key >> p.page_shift : key / p.page)) : 0;
            }
        };
        look(L, page);
        int loaded = 0, qload = -1;  // tiles and queries put into the rings
        uint32_t badmask = 0;        // stages with a page id out of range
        if (n > 1) {
            N = L;
            advance<C>(p, N);
            look(N, npage);
        }
        const int lr = lane / C::CHP, lc = lane % C::CHP;  // the lane's row and chunk of a copy
        auto issue = [&](int stage) {
            const int kvh = L.vh / p.blocks_per_kv;
            if (loaded == 0 || L.j == 0) {
                qload = qload + 1 == STAGES ? 0 : qload + 1;
                const int h0 = (L.vh - kvh * p.blocks_per_kv) * HB;
                const char* q = static_cast<const char*>(p.q) +
                                ((long long)L.row * p.q_ts + (long long)(kvh * p.group + h0) * p.q_hs) * (int)sizeof(TI);
                for (int i = lane; i < hv * (qrow / 16); i += 32) {
                    const int h = i / (qrow / 16), c = i - h * (qrow / 16);
                    const bool there = h0 + h < p.group;
                    if (c < nqch)
                        cp16(q32 + qload * hv * qrow + i * 16, q + (there ? h * p.q_hs * (int)sizeof(TI) + c * 16 : 0), there);
                }
            }
            const int k0 = (L.start / TK + L.j) * TK;
            const uint32_t dst = ring32 + stage * C::STAGE;
            const unsigned long long hoff = (unsigned long long)kvh * p.hs16 * 16;
            const long long vk = static_cast<const char*>(p.v) - static_cast<const char*>(p.k);
            bool bad = false;
            if (grouped) {
                const int lo = L.start - k0, hi = L.end - k0;  // rows lo <= r < hi are wanted
                const unsigned long long step = (unsigned long long)p.ts16 * 16 * C::RPI;
                const char* src = nullptr;
#pragma unroll
                for (int it = 0; it < C::ITS; ++it) {
                    const int r0 = C::CHP > 32 ? it * 32 / C::CHP : it * C::RPI;
                    const int r = r0 + (C::CHP > 32 ? 0 : lr), c = C::CHP > 32 ? (it * 32 + lane) % C::CHP : lc;
                    if (r0 % C::GR == 0 && (C::CHP <= 32 || it * 32 % C::CHP == 0)) {
                        const int id = page[r0 / C::GR];
                        const bool ok = (unsigned)id < (unsigned)p.n_pages;
                        bad |= !ok;
                        const int key = k0 + r0;
                        const int slot = p.page_shift >= 0 ? key & (p.page - 1) : key % p.page;
                        src = static_cast<const char*>(p.k) + hoff +
                              ((unsigned long long)(unsigned)(ok ? id : 0) * p.ps16 +
                               (unsigned long long)(unsigned)(slot + (C::CHP > 32 ? 0 : lr)) * p.ts16) * 16 +
                              (C::CHP > 32 ? 0 : lc * 16);
                    }
                    const int swz = C::F32 ? (r * C::LPK) & 7 : r & 7;
                    const uint32_t d = dst + r * C::ROWB + ((c ^ swz) * 16);
                    const bool there = r >= lo && r < hi;
                    if (c < nch) {
                        const char* at = src + (C::CHP > 32 ? c * 16 : 0);
                        cp16(d, at, there);
                        cp16(d + TK * C::ROWB, at + vk, there);
                    }
                    if (C::CHP <= 32 || (it + 1) * 32 % C::CHP == 0) src += step;
                }
            } else {
                const int key = k0 + kr;
                long long at = -1;
                if (key < L.end && key >= L.start) {
                    const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.page;
                    if ((unsigned)page[0] < (unsigned)p.n_pages)
                        at = (long long)(hoff + ((unsigned long long)(unsigned)page[0] * p.ps16 +
                                                 (unsigned long long)(unsigned)(key - pg * p.page) * p.ts16) * 16);
                    else
                        bad = true;
                }
#pragma unroll
                for (int it = 0; it < C::ITS; ++it) {
                    const int idx = it * 32 + lane, r = idx / C::CHP, c = idx % C::CHP;
                    const long long o = __shfl_sync(0xffffffffu, at, r);
                    if (c < nch) {
                        const int swz = C::F32 ? (r * C::LPK) & 7 : r & 7;
                        const uint32_t d = dst + r * C::ROWB + ((c ^ swz) * 16);
                        const char* src = static_cast<const char*>(p.k) + (o >= 0 ? o + c * 16 : 0);
                        cp16(d, src, o >= 0);
                        cp16(d + TK * C::ROWB, src + vk, o >= 0);
                    }
                }
            }
            badmask = (badmask & ~(1u << stage)) | ((__any_sync(0xffffffffu, bad) ? 1u : 0u) << stage);
            ++loaded;
            L = N;
#pragma unroll
            for (int g = 0; g < C::NG; ++g) page[g] = npage[g];
            if (loaded + 1 < n) {
                advance<C>(p, N);
                look(N, npage);
            }
        };

        // running state of the current (row, head block)
        float m[C::F32 ? HB : 2 * NT], l[C::F32 ? HB : 2 * NT], fac[2 * NT];
        float O[C::F32 ? HB : C::KD][C::F32 ? (HD + 127) / 128 : NT][4];
        uint32_t qf[C::F32 ? 1 : C::SQ][NT][C::F32 ? 1 : C::KD][2];
        const float sl2 = p.scale * LOG2E;
        int quse = -1;
        int bad = 0;  // status bits of the current row
        bool fresh = true;

#pragma unroll
        for (int s = 0; s < STAGES - 1; ++s) {
            if (loaded < n) issue(s);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        int stage = 0;
        for (int i = 0; i < n; ++i) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();
            if (loaded < n) issue(stage == 0 ? STAGES - 1 : stage - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");

            if (fresh) {
                fresh = false;
                bad = w.over ? GPT2Q_STATUS_POSITION : 0;
                quse = quse + 1 == STAGES ? 0 : quse + 1;
                const unsigned char* q = qring + quse * hv * qrow;
#pragma unroll
                for (int k = 0; k < (C::F32 ? HB : 2 * NT); ++k) m[k] = -INFINITY, l[k] = 0.f;
#pragma unroll
                for (int x = 0; x < (C::F32 ? HB : C::KD); ++x)
#pragma unroll
                    for (int y = 0; y < (C::F32 ? (HD + 127) / 128 : NT); ++y)
#pragma unroll
                        for (int z = 0; z < 4; ++z) O[x][y][z] = 0.f;
                if constexpr (!C::F32) {
                    // B fragments of the queries: head lane / 4, dims 2 (lane % 4) + {0, 1, 8, 9}
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int h = nt * 8 + (lane >> 2);
                        const TI* qh = reinterpret_cast<const TI*>(q + h * qrow) + (lane & 3) * 2;
                        float down = 1.f, up = 1.f;
                        if constexpr (C::SQ > 1 && C::HALF) {
                            // fp16 pieces of an fp32 query: scaled by a power of two so that the
                            // head's largest element lies in [1, 2), undone on the scores
                            float top = 0.f;
#pragma unroll
                            for (int k = 0; k < HD / 8; ++k)
                                if (h < hv) top = fmaxf(top, fmaxf(fabsf(to_f(qh[k * 8])), fabsf(to_f(qh[k * 8 + 1]))));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                            int e = (int)(__float_as_uint(top) >> 23);  // biased exponent
                            e = e == 0 || e == 255 ? 127 : min(max(e, 2), 252);
                            down = __uint_as_float((uint32_t)(254 - e) << 23);
                            up = __uint_as_float((uint32_t)e << 23);
                        }
#pragma unroll
                        for (int k = 0; k < C::KD; ++k)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                if constexpr (C::SQ == 1) {
                                    qf[0][nt][k][x] = h < hv ? *reinterpret_cast<const uint32_t*>(qh + k * 16 + x * 8) : 0u;
                                } else {
                                    float u = 0.f, v = 0.f;
                                    if (h < hv) u = to_f(qh[k * 16 + x * 8]) * down, v = to_f(qh[k * 16 + x * 8 + 1]) * down;
#pragma unroll
                                    for (int s = 0; s < C::SQ; ++s) qf[s][nt][k][x] = take_pair<TC>(u, v);
                                }
                            }
                        // a score's columns are heads 2 (lane % 4) + {0, 1}
                        fac[2 * nt] = sl2 * __shfl_sync(0xffffffffu, up, (lane & 3) * 8);
                        fac[2 * nt + 1] = sl2 * __shfl_sync(0xffffffffu, up, (lane & 3) * 8 + 4);
                    }
                }
            }
            if ((badmask >> stage) & 1u) bad |= GPT2Q_STATUS_PAGE;
            const int k0 = (w.start / TK + w.j) * TK, klo = w.start - k0, khi = w.end - k0;
            const bool cut = klo > 0 || khi < TK;  // some of the tile's keys are not the row's
            const uint32_t kt = ring32 + stage * C::STAGE, vt = kt + TK * C::ROWB;

            if constexpr (!C::F32) {
                // S^T = K q^T: keys are the rows of the product, heads its columns
                float s[MT][NT][2][4];
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int z = 0; z < 4; ++z) s[x][y][0][z] = s[x][y][1][z] = 0.f;
#pragma unroll
                for (int k = 0; k < C::KD; ++k) {
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        const int r = x * 16 + (lane & 15), c = 2 * k + (lane >> 4);
                        uint32_t af[4];
                        ldsm4(af, kt + r * C::ROWB + ((c ^ (r & 7)) * 16));
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int t = 0; t < C::SQ; ++t) mma16816<TC>(s[x][y][k & 1], af, qf[t][y][k][0], qf[t][y][k][1]);
                    }
                }
                bool moved = false;
                float al[2 * NT];
#pragma unroll
                for (int y = 0; y < NT; ++y)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int x = 0; x < MT; ++x)
#pragma unroll
                            for (int z = c; z < 4; z += 2) {
                                float v = (s[x][y][0][z] + s[x][y][1][z]) * fac[2 * y + c];
                                const int r = x * 16 + (lane >> 2) + (z >> 1) * 8;
                                if (cut && (r < klo || r >= khi)) v = -INFINITY;
                                s[x][y][0][z] = v;
                                mx = fmaxf(mx, v);
                            }
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const int k = 2 * y + c;
                        const float mn = fmaxf(m[k], mx);
                        const float ms = mn == -INFINITY ? 0.f : mn;
                        al[k] = ex2(m[k] - ms);
                        moved |= m[k] != mn;
                        m[k] = mn;
                        float sum = 0.f;
#pragma unroll
                        for (int x = 0; x < MT; ++x)
#pragma unroll
                            for (int z = c; z < 4; z += 2) {
                                const float e = ex2(s[x][y][0][z] - ms + C::shift());
                                s[x][y][0][z] = e;
                                sum += e;
                            }
                        l[k] = l[k] * al[k] + sum;
                    }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int d = 0; d < C::KD; ++d)
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int z = 0; z < 4; ++z) O[d][y][z] *= al[2 * y + (z & 1)];
                }
                // O^T += V^T P^T: the weights, transposed 8 x 8 in registers, are the B operand
                uint32_t pf[C::sp()][MT][NT][2];
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int t = 0; t < C::sp(); ++t) {
                            pf[t][x][y][0] = movm(take_pair<TC>(s[x][y][0][0], s[x][y][0][1]));
                            pf[t][x][y][1] = movm(take_pair<TC>(s[x][y][0][2], s[x][y][0][3]));
                        }
#pragma unroll
                for (int d = 0; d < C::KD; ++d) {
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        const int r = x * 16 + (lane & 7) + ((lane >> 4) & 1) * 8, c = 2 * d + ((lane >> 3) & 1);
                        uint32_t af[4];
                        ldsm4t(af, vt + r * C::ROWB + ((c ^ (r & 7)) * 16));
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int t = 0; t < C::sp(); ++t) mma16816<TC>(O[d][y], af, pf[t][x][y][0], pf[t][x][y][1]);
                    }
                }
            } else {
                // CUDA cores: LPK lanes share a key and take its chunks in turn
                const unsigned char* q = qring + quse * hv * qrow;
                const unsigned char* kp = ring + stage * C::STAGE;
                const unsigned char* vp = kp + TK * C::ROWB;
                const int key = lane / C::LPK, part = lane % C::LPK;
                float s[HB];
#pragma unroll
                for (int h = 0; h < HB; ++h) s[h] = 0.f;
#pragma unroll 4
                for (int c = part; c < nch; c += C::LPK) {
                    const float4 kv = *reinterpret_cast<const float4*>(kp + key * C::ROWB + ((c ^ ((key * C::LPK) & 7)) * 16));
#pragma unroll
                    for (int h = 0; h < HB; ++h)
                        if (h < hv) {
                            const float4 qv = *reinterpret_cast<const float4*>(q + h * qrow + c * 16);
                            s[h] = fmaf(kv.x, qv.x, s[h]);
                            s[h] = fmaf(kv.y, qv.y, s[h]);
                            s[h] = fmaf(kv.z, qv.z, s[h]);
                            s[h] = fmaf(kv.w, qv.w, s[h]);
                        }
                }
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    float v = s[h];
#pragma unroll
                    for (int o = 1; o < C::LPK; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    v = key >= klo && key < khi ? v * sl2 : -INFINITY;
                    float mx = v;
#pragma unroll
                    for (int o = C::LPK; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float mn = fmaxf(m[h], mx);
                    const float ms = mn == -INFINITY ? 0.f : mn;
                    const float al = ex2(m[h] - ms);
                    const float e = ex2(v - ms);
                    m[h] = mn;
                    l[h] = l[h] * al + (part == 0 ? e : 0.f);
#pragma unroll
                    for (int y = 0; y < (HD + 127) / 128; ++y)
#pragma unroll
                        for (int z = 0; z < 4; ++z) O[h][y][z] *= al;
                    if (part == 0) pbuf[key * HB + h] = e;
                }
                __syncwarp();
                constexpr int KH = HD == 64 ? 2 : 1;  // keys the warp takes at once
                const int c0 = HD == 64 ? lane & 15 : lane, k0 = HD == 64 ? lane >> 4 : 0;
#pragma unroll
                for (int k = 0; k < TK; k += KH) {
                    const int r = k + k0;
                    float e[HB];
                    if constexpr (HB % 4 == 0) {
#pragma unroll
                        for (int h = 0; h < HB; h += 4) *reinterpret_cast<float4*>(e + h) = *reinterpret_cast<const float4*>(pbuf + r * HB + h);
                    } else {
#pragma unroll
                        for (int h = 0; h < HB; ++h) e[h] = pbuf[r * HB + h];
                    }
#pragma unroll
                    for (int y = 0; y < (HD + 127) / 128; ++y) {
                        const float4 v = *reinterpret_cast<const float4*>(vp + r * C::ROWB + (((c0 + 32 * y) ^ ((r * C::LPK) & 7)) * 16));
#pragma unroll
                        for (int h = 0; h < HB; ++h) {
                            O[h][y][0] = fmaf(e[h], v.x, O[h][y][0]);
                            O[h][y][1] = fmaf(e[h], v.y, O[h][y][1]);
                            O[h][y][2] = fmaf(e[h], v.z, O[h][y][2]);
                            O[h][y][3] = fmaf(e[h], v.w, O[h][y][3]);
                        }
                    }
                }
            }

            const bool last = i == n - 1;
            if (last || w.j + 1 == w.nt) {
                // the segment ends, here or in this warp's range
                fresh = true;
                const long long first = a + i - w.j;  // its first tile
                const bool whole = first >= a && w.j + 1 == w.nt;
                const int kvh = w.vh / p.blocks_per_kv, h0 = (w.vh - kvh * p.blocks_per_kv) * HB;
                const int head0 = kvh * p.group + h0, nh = min(HB, p.group - h0);
                if (bad && p.status && lane == 0) atomicOr(p.status, bad);
#pragma unroll
                for (int k = 0; k < (C::F32 ? HB : 2 * NT); ++k) {
#pragma unroll
                    for (int o = C::F32 ? 1 : 4; o < 32; o <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], o);
                    l[k] *= C::UNSHIFT;
                    if (bad) l[k] = NAN;
                }
                if constexpr (C::F32 && HD == 64) {
#pragma unroll
                    for (int h = 0; h < HB; ++h)
#pragma unroll
                        for (int z = 0; z < 4; ++z) O[h][0][z] += __shfl_xor_sync(0xffffffffu, O[h][0][z], 16);
                }
                const int ps = 2 * warp + (first < a ? 0 : 1);
                float* dst = nullptr;
                if (!whole) {
                    // in the middle of a range to memory, at its end into the drained ring
                    dst = last ? reinterpret_cast<float*>(ring)
                               : p.warp_part + ((long long)blockIdx.x * MAX_WARPS + warp) * HB * C::HS;
                    if (lane == 0) pieces[ps] = Piece{first, w.nt, w.row, w.vh, dst};
                    __syncwarp();
                }
                if constexpr (!C::F32) {
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int h = y * 8 + (lane & 3) * 2 + c, k = 2 * y + c;
                            if (h < nh) {
                                const float f = whole ? inverse(l[k]) * C::UNSHIFT : C::UNSHIFT;
#pragma unroll
                                for (int d = 0; d < C::KD; ++d)
#pragma unroll
                                    for (int z = 0; z < 2; ++z) {
                                        const int at = d * 16 + z * 8 + (lane >> 2);
                                        const float v = O[d][y][2 * z + c] * f;
                                        if (at < p.dim) {
                                            if (whole)
                                                write1<TI>(p, w.row, head0 + h, at, v);
                                            else
                                                dst[h * C::HS + at] = v;
                                        }
                                    }
                                if (lane < 4) {
                                    if (!whole)
                                        pm[ps][h] = m[k], pl[ps][h] = l[k];
                                    else if (p.lse)
                                        p.lse[(long long)w.row * p.n_heads + head0 + h] = log_sum(m[k], l[k]);
                                }
                            }
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < HB; ++h)
                        if (h < nh) {
                            const float f = whole ? inverse(l[h]) : 1.f;
#pragma unroll
                            for (int y = 0; y < (HD + 127) / 128; ++y) {
                                const int at = (HD == 64 ? lane & 15 : lane + 32 * y) * 4;
                                float v[4];
#pragma unroll
                                for (int z = 0; z < 4; ++z) v[z] = O[h][y][z] * f;
                                if (at < p.dim && !(HD == 64 && lane > 15)) {
                                    if (whole)
                                        write4<TI>(p, w.row, head0 + h, at, v);
                                    else
                                        *reinterpret_cast<float4*>(dst + h * C::HS + at) = make_float4(v[0], v[1], v[2], v[3]);
                                }
                            }
                            if (lane == 0) {
                                if (!whole)
                                    pm[ps][h] = m[h], pl[ps][h] = l[h];
                                else if (p.lse)
                                    p.lse[(long long)w.row * p.n_heads + head0 + h] = log_sum(m[h], l[h]);
                            }
                        }
                }
            }
            if (!last) advance<C>(p, w);
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
    }
    __syncthreads();

    // ---- the block's pieces, joined where they belong to one (row, head block) ----
    int chain = 0, tail_row = -1, tail_vh = 0;
    long long tail_last = 0;
    for (int i = 0; i < 2 * nw;) {
        if (pieces[i].nt == 0) {
            ++i;
            continue;
        }
        const Piece P = pieces[i];
        int e = i + 1;
        for (int j = i + 1; j < 2 * nw; ++j)
            if (pieces[j].nt) {
                if (pieces[j].first != P.first) break;
                e = j + 1;
            }
        const bool whole = P.first >= ca && P.first + P.nt <= cb;
        if (P.first >= ca && !whole) tail_row = P.row, tail_vh = P.vh, tail_last = (P.first + P.nt - 1) / per;
        const int kvh = P.vh / p.blocks_per_kv, h0 = (P.vh - kvh * p.blocks_per_kv) * HB;
        const int nh = min(HB, p.group - h0);
        for (int h = 0; h < nh; ++h) {
            if ((chain * hv + h) % nw != warp) continue;
            float M = -INFINITY, Ls = 0.f;
            for (int j = i; j < e; ++j)
                if (pieces[j].nt) M = fmaxf(M, pm[j][h]);
            const float ms = M == -INFINITY ? 0.f : M;
            for (int j = i; j < e; ++j)
                if (pieces[j].nt) Ls += pl[j][h] * ex2(pm[j][h] - ms);
            const float f = whole ? inverse(Ls) : 1.f;
            const long long ci = ((long long)blockIdx.x * 2 + (P.first < ca ? 0 : 1)) * HB + h;
            for (int d = lane * 4; d < p.dim; d += 128) {
                float r[4] = {0.f, 0.f, 0.f, 0.f};
                for (int j = i; j < e; ++j)
                    if (pieces[j].nt) {
                        const float4 v = *reinterpret_cast<const float4*>(pieces[j].data + h * C::HS + d);
                        const float wt = ex2(pm[j][h] - ms);
                        r[0] = fmaf(v.x, wt, r[0]);
                        r[1] = fmaf(v.y, wt, r[1]);
                        r[2] = fmaf(v.z, wt, r[2]);
                        r[3] = fmaf(v.w, wt, r[3]);
                    }
#pragma unroll
                for (int z = 0; z < 4; ++z) r[z] *= f;
                if (whole)
                    write4<TI>(p, P.row, kvh * p.group + h0 + h, d, r);
                else
                    *reinterpret_cast<float4*>(p.block_part + ci * HD + d) = make_float4(r[0], r[1], r[2], r[3]);
            }
            if (lane == 0) {
                if (!whole)
                    p.block_ml[ci] = make_float2(M, Ls);
                else if (p.lse)
                    p.lse[(long long)P.row * p.n_heads + kvh * p.group + h0 + h] = log_sum(M, Ls);
            }
        }
        ++chain;
        i = e;
    }
    if (tid == 0) p.meta[blockIdx.x] = make_int4(tail_row, tail_vh, (int)tail_last, 0);

    // ---- rows without a cached token ----
    for (int r = blockIdx.x; r < p.n_rows; r += gridDim.x) {
        if (__ldcg(p.lens + r) > 0) continue;
        const float zero[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i = tid * 4; i < p.n_heads * p.dim; i += nthr * 4) write4<TI>(p, r, i / p.dim, i % p.dim, zero);
        if (p.lse)
            for (int h = tid; h < p.n_heads; h += nthr) p.lse[(long long)r * p.n_heads + h] = -INFINITY;
    }
}

// Joins the pieces of a (row, head block) that lies in several blocks' ranges: block c of the first
// kernel has its beginning (slot 1), the blocks after it up to `last` the rest (slot 0). One block
// per (c, head).
template <class TI, int HD, int HB>
__global__ void __launch_bounds__(128) k_paged_attn_join(const __grid_constant__ PagedAttn p) {
    __shared__ float4 part[128];
    tc::pdl_trigger();
    tc::pdl_wait();
    const int c = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int4 meta = __ldcg(p.meta + c);
    if (meta.x < 0) return;
    const int kvh = meta.y / p.blocks_per_kv, h0 = (meta.y - kvh * p.blocks_per_kv) * HB;
    if (h0 + h >= p.group) return;
    const int n = meta.z - c + 1;
    auto at = [&](int i) { return ((long long)(c + i) * 2 + (i == 0 ? 1 : 0)) * HB + h; };
    float M = -INFINITY, L = 0.f;
    for (int i = lane; i < n; i += 32) M = fmaxf(M, __ldcg(p.block_ml + at(i)).x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ms = M == -INFINITY ? 0.f : M;
    for (int i = lane; i < n; i += 32) {
        const float2 ml = __ldcg(p.block_ml + at(i));
        L += ml.y * ex2(ml.x - ms);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    constexpr int DG = HD / 4, PG = 128 / DG;  // threads over dims, and over pieces
    const int d = tid % DG * 4, g = tid / DG;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < p.dim)
#pragma unroll 4
        for (int i = g; i < n; i += PG) {
            const float wt = ex2(__ldcg(p.block_ml + at(i)).x - ms);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.block_part + at(i) * HD + d));
            r.x = fmaf(v.x, wt, r.x);
            r.y = fmaf(v.y, wt, r.y);
            r.z = fmaf(v.z, wt, r.z);
            r.w = fmaf(v.w, wt, r.w);
        }
    part[tid] = r;
    __syncthreads();
    const int head = kvh * p.group + h0 + h;
    if (g == 0 && d < p.dim) {
#pragma unroll
        for (int k = 1; k < PG; ++k) {
            const float4 v = part[tid + k * DG];
            r.x += v.x, r.y += v.y, r.z += v.z, r.w += v.w;
        }
        const float f = inverse(L);
        const float o[4] = {r.x * f, r.y * f, r.z * f, r.w * f};
        write4<TI>(p, meta.x, head, d, o);
    }
    if (tid == 0 && p.lse) p.lse[(long long)meta.x * p.n_heads + head] = log_sum(M, L);
}

constexpr size_t SMEM_LIMIT = 227 * 1024 - 8 * 1024;  // dynamic; the rest for the static arrays

template <class C>
cudaError_t launch(PagedAttn p, cudaStream_t st) {
    p.blocks_per_kv = (p.group + C::HB - 1) / C::HB;
    p.n_vh = p.n_kv * p.blocks_per_kv;
    p.heads_per_block = std::min(p.group, C::HB);
    size_t wb = STAGES * C::STAGE + (size_t)STAGES * p.heads_per_block * C::HD * sizeof(typename C::TI);
    if (C::F32) wb += (size_t)C::TK * C::HB * 4;
    p.grouped = p.page % C::GR == 0;
    p.warp_bytes = (int)((wb + 127) / 128 * 128);
    const int nw = (int)std::min<size_t>(MAX_WARPS, SMEM_LIMIT / p.warp_bytes);
    // no more blocks than the longest rows the table can hold would fill
    const long long longest = p.window > 0 ? std::min(p.window, p.cap) : p.cap;
    const long long tiles = ((longest + C::TK - 1) / C::TK + (p.window > 0 ? 1 : 0)) * p.n_vh;
    const long long want = tiles > MAX_CTAS * 8LL ? MAX_CTAS : (tiles * p.n_rows + nw - 1) / nw;
    const int grid = (int)std::clamp<long long>(want, 1, MAX_CTAS);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    const size_t smem = (size_t)nw * p.warp_bytes;
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        e = cudaFuncSetAttribute(k_paged_attn<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    e = launch_dependent(k_paged_attn<C>, dim3(grid), dim3(nw * 32), smem, st, p);
    if (e != cudaSuccess || grid == 1) return e;
    return launch_dependent(k_paged_attn_join<typename C::TI, C::HD, C::HB>, dim3(grid, p.heads_per_block), dim3(128), 0, st, p);
}

template <class TC, class TI, int HD>
cudaError_t by_heads(const PagedAttn& p, cudaStream_t st) {
    if constexpr (std::is_same<TC, float>::value) {
        if (p.group == 1) return launch<Cfg<TC, TI, HD, 1>>(p, st);
        if (p.group == 2) return launch<Cfg<TC, TI, HD, 2>>(p, st);
        if (p.group <= 4) return launch<Cfg<TC, TI, HD, 4>>(p, st);
        return launch<Cfg<TC, TI, HD, 8>>(p, st);
    } else {
        if constexpr (std::is_same<TC, TI>::value && HD <= 128)
            if (p.group > 8) return launch<Cfg<TC, TI, HD, 16>>(p, st);
        return launch<Cfg<TC, TI, HD, 8>>(p, st);
    }
}

template <class TC, class TI>
cudaError_t by_dim(const PagedAttn& p, cudaStream_t st) {
    if (p.dim <= 64) return by_heads<TC, TI, 64>(p, st);
    if (p.dim <= 128) return by_heads<TC, TI, 128>(p, st);
    return by_heads<TC, TI, 256>(p, st);
}

}  // namespace

// Layout of the workspace: per block its last row's whereabouts, two partial results, and one more
// per warp.
uint64_t gpt2q::paged_attn_workspace(int dim, int group) {
    const uint64_t hd = dim <= 64 ? 64 : dim <= 128 ? 128 : 256, hb = group > 8 ? 16 : 8;
    return MAX_CTAS * (16 + 2 * hb * (hd * 4 + 8) + MAX_WARPS * hb * (hd + 4) * 4);
}

cudaError_t gpt2q::launch_paged_attn(PagedAttn p, int cache_dtype, int dtype, void* work, cudaStream_t st) {
    const uint64_t hd = p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256, hb = p.group > 8 ? 16 : 8;
    char* at = static_cast<char*>(work);
    p.meta = reinterpret_cast<int4*>(at);
    at += MAX_CTAS * 16;
    p.block_part = reinterpret_cast<float*>(at);
    at += MAX_CTAS * 2 * hb * hd * 4;
    p.warp_part = reinterpret_cast<float*>(at);
    at += MAX_CTAS * MAX_WARPS * hb * (hd + 4) * 4;
    p.block_ml = reinterpret_cast<float2*>(at);
    p.page_shift = -1;
    for (int s = 0; s < 31; ++s)
        if (p.page == 1 << s) p.page_shift = s;
    if (cache_dtype == GPT2Q_F32) return by_dim<float, float>(p, st);
    if (cache_dtype == GPT2Q_F16)
        return dtype == GPT2Q_F32 ? by_dim<__half, float>(p, st) : by_dim<__half, __half>(p, st);
    return dtype == GPT2Q_F32 ? by_dim<bf16, float>(p, st) : by_dim<bf16, bf16>(p, st);
}
