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
// A warp streams its tiles through a ring of two shared-memory stages of its own, so warps never
// wait for each other while they stream. Where a page is a multiple of 16 keys (8 for the short
// tiles of an fp32 cache), one lane starts the tile's copies as TMA boxes of up to 16 keys, swizzled
// in pieces of 128 bytes (all pieces of a key in one box where they are whole); pages are looked up
// a tile ahead. Other page sizes are gathered key by key with cp.async. Measured: 64 query heads on
// 8 kv heads of 128 in bf16 over 131071 keys 94.0 us (5.7 TB/s; four times the keys 349 us, 6.1
// TB/s), 63 rows of 17 to 9000 keys 83.1 us (4.5 TB/s), one row of 1001 keys of 12 heads of 64 12.3
// us, of which the joins and the first tile are most.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <string>
#include <type_traits>

#include "device_op.cuh"
#include "gpt2q.h"
#include "paged.h"

using namespace gpt2q;

namespace {

constexpr int STAGES = 2;
constexpr int MAX_WARPS = 12;
constexpr int LENS = 512;     // rows whose lengths a block keeps in shared memory
constexpr int MAX_CTAS = 148;  // one per SM of a B200
constexpr int WAIT_TRIES = 1 << 19;  // of about 1.5 us: 0.8 s
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
    static constexpr int TK = F32 ? (HD == 256 ? 8 : 4096 / ROWB) : (HD == 256 ? 16 : 4096 / ROWB);
    static __device__ constexpr int lpk() { return 32 / TK; }  // lanes per key (fp32 cache)
    static constexpr int GR = TK < 16 ? TK : 16, NG = TK / GR;  // keys of one page lookup where pages allow it
    static constexpr int BOX = 128 / (int)sizeof(TC);  // dims of a TMA box
    // a tile's rows are cut into pieces of 128 bytes, piece by piece one after the other; the 16-byte
    // chunks of a piece are permuted by the row (the 128-byte swizzle), so that eight rows of one
    // chunk lie in different banks
    static __device__ __forceinline__ int at(int r, int c) {
        return (c >> 3) * (TK * 128) + r * 128 + (((c ^ r) & 7) << 4);
    }
    static constexpr int STAGE = 2 * TK * ROWB;
    static constexpr int HS = HD + 4;  // floats of a partial result's row
    // 16-bit pieces of the query and of the weights. Queries of the cache's type are exact in one;
    // fp32 ones take three (24 bits: two fp16 pieces left scores of 10 off by 1e-6, and the output with
    // them). Weights take two pieces of fp16 (22 bits; the rest is a quarter of ex2's own error), of bf16 three
    // for fp32 outputs and two where the output has 16 bits: one would add an error as large as the output's own
    // rounding, two leave 2^-16 of sum w |v|, which only results that cancel below 2^-8 of that show. A third
    // took 3 to 4 % (63 ragged rows 84.5 to 87.8 us a call, one of 131071 keys 97.1 to 100.0), with the same error
    // against 64 bits.
    static constexpr int SQ = F32 || !std::is_same<TI, float>::value ? 1 : 3;
    static constexpr int sp() { return SQ == 1 || HALF ? 2 : 3; }
    static constexpr int MT = TK / 16, NT = HB / 8, KD = HD / 16;
    // independent sums of a score tile: of even and odd steps where there is no other work to overlap
    // with, and for fp32 queries the lower pieces' apart, as the tensor cores round a running sum down
    static __device__ constexpr int acc() { return SQ > 1 ? 3 : MT * NT == 1 ? 2 : 1; }
    // fp16 weights are held times 2^10, so that small ones stay normal numbers
    static constexpr float shift() { return HALF ? 10.f : 0.f; }
    // rows whose queries are staged per warp: of the two tiles on their way and, where they are not held in
    // registers, of the one worked on
    static constexpr int QS = F32 ? 3 : 2;
    // warps of a block, by the registers that queries and results take
    static constexpr int WARPS = !F32 && SQ * NT * KD * 2 + NT * KD * 4 > 100 ? 8 : MAX_WARPS;
    static constexpr float UNSHIFT = HALF ? 1.f / 1024.f : 1.f;
};

struct Walk {
    int row, kvh, hb, j, nt, start, end;  // hb: block of the kv head's query heads
    bool over;
};

struct Piece {
    long long first;  // index of its segment's first tile
    int nt, row, vh;  // nt = 0: none
    const float* data;
};

// Row `row` of the walk; `lens` holds the first LENS rows' lengths.
template <class C>
__device__ __forceinline__ void enter(const PagedAttn& p, const int* lens, Walk& w, int row) {
    w.row = row;
    const int len = row >= p.n_rows ? 0 : row < LENS ? lens[row] : __ldcg(p.lens + row);
    w.over = len > p.cap;
    w.end = w.over ? p.cap : len;
    w.start = p.window > 0 && w.end > p.window ? w.end - p.window : 0;
    // tiles begin at multiples of TK, so that a group of GR keys lies in one page
    w.nt = w.end > 0 ? (int)((unsigned)(w.end + C::TK - 1) / C::TK - (unsigned)w.start / C::TK) : 0;
}

template <class C>
__device__ __forceinline__ void advance(const PagedAttn& p, const int* lens, Walk& w) {
    if (++w.j < w.nt) return;
    w.j = 0;
    if (++w.hb < p.blocks_per_kv) return;
    w.hb = 0;
    if (++w.kvh < p.n_kv) return;
    w.kvh = 0;
    do {
        enter<C>(p, lens, w, w.row + 1);
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
// the product alone
template <class TC>
__device__ __forceinline__ void mma16816_0(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<TC, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
// coordinates: dim, slot, piece of 128 bytes (0), head, page
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int h, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(0), "r"(h), "r"(page), "r"(bar)
        : "memory");
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
// l of a row whose keys all have weight 0 is 0: its result is 0 and its logarithm -inf
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * LN2; }

// ceil(a / b) and a / b of values that nearly always fit 32 bits (a 64-bit division is a hundred instructions)
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((unsigned long long)a | (unsigned long long)b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

template <class C, bool TMA>
__global__ void __launch_bounds__(C::WARPS * 32, 1)
    k_paged_attn(const __grid_constant__ PagedAttn p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using TC = typename C::TC;
    using TI = typename C::TI;
    constexpr int HB = C::HB, HD = C::HD, TK = C::TK, NT = C::NT > 0 ? C::NT : 1, MT = C::MT > 0 ? C::MT : 1;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ long long cum[MAX_WARPS * 32 + 1];
    __shared__ long long wsum[MAX_WARPS];
    __shared__ int slen[LENS];
    __shared__ Piece pieces[2 * MAX_WARPS];
    __shared__ __align__(8) uint64_t full[MAX_WARPS][2 * STAGES];  // per stage: keys, values
    __shared__ float pm[2 * MAX_WARPS][HB], pl[2 * MAX_WARPS][HB];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nthr = blockDim.x, nw = nthr >> 5;
    const int hv = p.heads_per_block;                    // heads a block's partial results hold
    const int qrow = HD * (int)sizeof(TI);               // bytes of a staged query
    unsigned char* ring = smem + (size_t)warp * p.warp_bytes;
    unsigned char* qring = ring + STAGES * C::STAGE;
    float* pbuf = reinterpret_cast<float*>(qring + C::QS * hv * qrow);  // fp32 cache: the tile's weights
    const uint32_t ring32 = tc::smem_u32(ring), q32 = tc::smem_u32(qring);
    const int nch = p.dim * (int)sizeof(TC) / 16, nqch = p.dim * (int)sizeof(TI) / 16;

    if (lane < 2) pieces[2 * warp + lane].nt = 0;
    if constexpr (TMA) {
        if (lane == 0) {
            for (int i = 0; i < 2 * STAGES; ++i) tc::mbar_init(&full[warp][i], 1);
            tc::fence_mbar_init();
            if (warp == 0) {
                tc::prefetch_tmap(&kmap);
                tc::prefetch_tmap(&vmap);
            }
        }
    }
    // dims past the head's own are zero in the ring and are never written again; TMA fills its last piece
    // of 128 bytes with zeros itself
    const int c_own = TMA ? p.boxes * 8 : nch;
    if (c_own < C::CHP)
        for (int r = lane; r < STAGES * 2 * TK; r += 32)
            for (int c = c_own; c < C::CHP; ++c)
                *reinterpret_cast<uint4*>(ring + r / TK * TK * C::ROWB + C::at(r % TK, c)) = make_uint4(0, 0, 0, 0);
    if (nch < C::CHP)
        for (int i = lane; i < C::QS * hv * (qrow / 16); i += 32)
            if (i % (qrow / 16) >= nqch) *reinterpret_cast<uint4*>(qring + i * 16) = make_uint4(0, 0, 0, 0);
    tc::pdl_trigger();
    tc::pdl_wait();

    // ---- this block's and this warp's range of tiles ----
    const int nc = (p.n_rows + nthr - 1) / nthr;  // rows a thread counts
    Walk w;
    long long mine = 0;
    for (int r = tid; r < min(LENS, p.n_rows); r += nthr) slen[r] = __ldcg(p.lens + r);
    if (nc > 1) __syncthreads();
    for (int r = tid * nc; r < min((tid + 1) * nc, p.n_rows); ++r) {
        enter<C>(p, slen, w, r);  // with nc == 1 the thread's own
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
    const long long wper = quotient(quotient(total + gridDim.x - 1, gridDim.x) + nw - 1, nw), per = wper * nw;
    const long long ca = per * blockIdx.x, cb = min(ca + per, total);
    const long long a = ca + wper * warp, b = min(a + wper, cb);
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
        enter<C>(p, slen, w, row);
        while (rem >= (long long)w.nt * p.n_vh) {
            rem -= (long long)w.nt * p.n_vh;
            enter<C>(p, slen, w, ++row);
        }
        const int vh = (int)quotient(rem, w.nt);
        w.j = (int)(rem - (long long)vh * w.nt);
        w.kvh = vh / p.blocks_per_kv;
        w.hb = vh - w.kvh * p.blocks_per_kv;
        // L is the next tile to load, from key L_key on; its pages are looked up when the tile before
        // it is loaded
        Walk L = w;
        int L_key = ((unsigned)L.start / TK + L.j) * TK;
        const int* L_ids = p.table + (long long)L.row * p.ld;
        int page[C::NG];
        // page ids of a tile: of every group of GR keys (the same load in all lanes) where a page is
        // a multiple of GR, else of the lane's own key, in element 0. -1 for keys the row does not have
        auto look = [&](auto steady) {
#pragma unroll
            for (int g = 0; g < (TMA ? C::NG : 1); ++g) {
                const int key = TMA ? L_key + g * C::GR : L_key + (lane & (TK - 1));
                page[g] = -1;
                if (decltype(steady)::value || (key < L.end && key + (TMA ? C::GR : 1) > L.start))
                    page[g] = __ldcg(L_ids + (p.page_shift >= 0 ? key >> p.page_shift : key / p.page));
            }
        };
        look(std::false_type{});
        int qload = 0;         // where the last queries went
        uint32_t badmask = 0;  // stages with a page id out of range
        bool stuck = false;    // a wait of this lane ran out
        // Starts the copies of tile i's keys (and its row's queries) or values; values come second.
        // steady: the tile and the one after it lie inside the row that the loads are in.
        auto issue = [&](int i, auto values, auto steady) {
            constexpr bool V = decltype(values)::value, ST = decltype(steady)::value;
            const int stage = i % STAGES;
            if (!V && !ST && (i == 0 || L.j == 0)) {
                qload = qload + 1 == C::QS ? 0 : qload + 1;
                const int h0 = L.hb * HB;
                const char* q = static_cast<const char*>(p.q) +
                                ((long long)L.row * p.q_ts + (long long)(L.kvh * p.group + h0) * p.q_hs) * (int)sizeof(TI);
                for (int x = lane; x < hv * (qrow / 16); x += 32) {
                    const int h = x / (qrow / 16), c = x - h * (qrow / 16);
                    const bool there = h0 + h < p.group;
                    if (c < nqch)
                        cp16(q32 + qload * hv * qrow + x * 16, q + (there ? h * p.q_hs * (int)sizeof(TI) + c * 16 : 0), there);
                }
            }
            const uint32_t dst = ring32 + stage * C::STAGE + (V ? TK * C::ROWB : 0);
            bool bad = false;
            if constexpr (TMA) {
                // groups of keys that the row has, and whose page is in the pool
                int bytes = 0;
#pragma unroll
                for (int g = 0; g < C::NG; ++g) {
                    const bool in = (unsigned)page[g] < (unsigned)p.n_pages;
                    if (!V) bad |= !in && (ST || (L_key + g * C::GR < L.end && L_key + (g + 1) * C::GR > L.start));
                    bytes += in ? p.group_bytes : 0;
                }
                if (lane == 0 && !stuck) {
                    tc::mbar_arrive_expect_tx(&full[warp][2 * stage + V], bytes);
                    const uint32_t bar = tc::smem_u32(&full[warp][2 * stage + V]);
#pragma unroll
                    for (int g = 0; g < C::NG; ++g) {
                        if ((unsigned)page[g] >= (unsigned)p.n_pages) continue;
                        const int key = L_key + g * C::GR;
                        const int slot = p.page_shift >= 0 ? key & (p.page - 1) : key % p.page;
                        const CUtensorMap* map = V ? &vmap : &kmap;
                        tma_load(dst + g * (C::GR * 128), map, 0, slot, L.kvh, page[g], bar);
                        for (int x = 1; x < p.box_loads; ++x)
                            tma_load(dst + g * (C::GR * 128) + x * (TK * 128), map, x * C::BOX, slot, L.kvh, page[g], bar);
                    }
                }
            } else {
                const unsigned long long hoff = (unsigned long long)L.kvh * p.hs16 * 16;
                const char* pool = static_cast<const char*>(V ? p.v : p.k);
                const int key = L_key + (lane & (TK - 1));
                long long at = -1;
                if (ST || (key < L.end && key >= L.start)) {
                    const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.page;
                    if ((unsigned)page[0] < (unsigned)p.n_pages)
                        at = (long long)(hoff + ((unsigned long long)(unsigned)page[0] * p.ps16 +
                                                 (unsigned long long)(unsigned)(key - pg * p.page) * p.ts16) * 16);
                    else
                        bad = true;
                }
#pragma unroll
                for (int it = 0; it < TK * C::CHP / 32; ++it) {
                    const int idx = it * 32 + lane, r = idx / C::CHP, c = idx % C::CHP;
                    const long long o = __shfl_sync(0xffffffffu, at, r);
                    if (c < nch) {
                        const uint32_t d = dst + C::at(r, c);
                        cp16(d, pool + (o >= 0 ? o + c * 16 : 0), o >= 0);
                    }
                }
                bad = __any_sync(0xffffffffu, bad);
            }
            if (!V) badmask = (badmask & ~(1u << stage)) | ((bad ? 1u : 0u) << stage);
            if (V && (ST || i + 1 < n)) {
                L_key += TK;
                if (++L.j == L.nt && !ST) {
                    --L.j;
                    advance<C>(p, slen, L);
                    L_key = (unsigned)L.start / TK * TK;
                    L_ids = p.table + (long long)L.row * p.ld;
                }
                look(steady);
            }
        };

        // running state of the current (row, head block)
        float m[C::F32 ? HB : 2 * NT], l[C::F32 ? HB : 2 * NT], fac[2 * NT];
        float O[C::F32 ? HB : C::KD][C::F32 ? (HD + 127) / 128 : NT][4];
        uint32_t qf[C::F32 ? 1 : C::SQ][NT][C::F32 ? 1 : C::KD][2];
        // the scores' factor; the sign goes to the queries, and 0 becomes a factor too small to matter,
        // so that a masked score of -inf stays one
        const float sl2 = fmaxf(fabsf(p.scale) * LOG2E, 1e-37f);
        int quse = 0;
        int bad = 0;  // status bits of the current row
        bool fresh = true;

        // where this lane's ldmatrix rows lie in a tile: chunk 0 of 16 keys' K, transposed V. Chunk k of a piece
        // is k * 32 away by exclusive or, as stages and pieces are multiples of 1024 bytes
        const uint32_t kat = C::at(lane & 15, lane >> 4);
        const uint32_t vat = TK * C::ROWB + C::at((lane & 7) + ((lane >> 4) & 1) * 8, (lane >> 3) & 1);
        // Waits for the copies of a tile's keys (which = 2 * stage) or values (2 * stage + 1). Each lane gives up
        // by itself and then waits for nothing more; what all lanes do together does not depend on it. Lane 0,
        // which starts the copies, starts none after it gave up. Results of a warp with such a lane are NaN.
        auto wait = [&](int which, int i) {
            if constexpr (TMA) {
                for (int tries = 0; !stuck && !tc::mbar_try_wait(&full[warp][which], (i / STAGES) & 1); ++tries) stuck = tries >= WAIT_TRIES;
            } else {
                asm volatile("cp.async.wait_group 3;" ::: "memory");
            }
            __syncwarp();
        };
        // Two tiles are on their way while one is worked on: the next keys come into a tile's keys as
        // soon as its scores are done, the next values into its values at its end.
        auto step = [&](int i, auto steady) {
            constexpr bool ST = decltype(steady)::value;
            const int stage = (i + STAGES) % STAGES;
            int klo = 0, khi = TK;  // the tile's keys that are the row's
            [[maybe_unused]] const uint32_t kt = ring32 + stage * C::STAGE;
            [[maybe_unused]] float s[C::F32 ? HB : 1], S[C::F32 ? 1 : MT][NT][C::acc()][4];  // scores: of a key, or of a tile
            if (ST || i >= 0) {
            if (!ST && fresh) {
                // every load of queries is in the group of its tile's keys
                asm volatile("cp.async.wait_group 3;" ::: "memory");
                __syncwarp();
                fresh = false;
                bad = w.over ? GPT2Q_STATUS_POSITION : 0;
                quse = quse + 1 == C::QS ? 0 : quse + 1;
                [[maybe_unused]] const unsigned char* q = qring + quse * hv * qrow;
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
                        [[maybe_unused]] float down = 1.f, up = 1.f;  // of the queries, and back
                        if constexpr (C::SQ > 1 && C::HALF) {
                            // fp16 pieces of an fp32 query: scaled by a power of two so that the
                            // head's largest element lies in [2^10, 2^11), undone on the scores
                            float top = 0.f;
#pragma unroll
                            for (int k = 0; k < HD / 8; ++k)
                                if (h < hv) top = fmaxf(top, fmaxf(fabsf(to_f(qh[k * 8])), fabsf(to_f(qh[k * 8 + 1]))));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                            int e = (int)(__float_as_uint(top) >> 23);  // biased exponent
                            e = e == 0 || e == 255 ? 127 : min(max(e, 12), 252);
                            down = __uint_as_float((uint32_t)(264 - e) << 23);
                            up = __uint_as_float((uint32_t)(e - 10) << 23);
                        }
#pragma unroll
                        for (int k = 0; k < C::KD; ++k)
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                if constexpr (C::SQ == 1) {
                                    qf[0][nt][k][x] = h < hv ? *reinterpret_cast<const uint32_t*>(qh + k * 16 + x * 8) : 0u;
                                    if (p.scale < 0.f) qf[0][nt][k][x] ^= 0x80008000u;
                                } else {
                                    float u = 0.f, v = 0.f;
                                    const float sd = p.scale < 0.f ? -down : down;
                                    if (h < hv) u = to_f(qh[k * 16 + x * 8]) * sd, v = to_f(qh[k * 16 + x * 8 + 1]) * sd;
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
            static_assert(GPT2Q_STATUS_PAGE == 1, "the mask's bit is the status");
            bad |= (badmask >> stage) & 1u;
            if (!ST && (w.j == 0 || w.j + 1 == w.nt)) {
                const int k0 = ((unsigned)w.start / TK + w.j) * TK;
                klo = w.start - k0;
                khi = w.end - k0;
            }
            wait(2 * stage, i);

            if constexpr (!C::F32) {
                // S^T = K q^T: keys are the rows of the product, heads its columns
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int z = 0; z < 4; ++z) S[x][y][0][z] = S[x][y][C::acc() / 2][z] = S[x][y][C::acc() - 1][z] = 0.f;
#pragma unroll
                for (int k = 0; k < C::KD; ++k) {
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        uint32_t af[4];
                        ldsm4(af, ((kt + kat) ^ ((k & 3) * 32)) + (k >> 2) * (TK * 128) + x * 2048);
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int t = 0; t < C::SQ; ++t) mma16816<TC>(S[x][y][t ? 2 : C::acc() > 1 ? k & 1 : 0], af, qf[t][y][k][0], qf[t][y][k][1]);
                    }
                }
            } else {
                // CUDA cores: LPK lanes share a key and take its chunks in turn
                const unsigned char* q = qring + quse * hv * qrow;
                const unsigned char* kp = ring + stage * C::STAGE;
                // eight neighbouring lanes read eight keys
                const int key = (lane & 7) + (lane >> 3) / C::lpk() * 8, part = (lane >> 3) % C::lpk();
#pragma unroll
                for (int h = 0; h < HB; ++h) s[h] = 0.f;
#pragma unroll 4
                for (int c = part; c < nch; c += C::lpk()) {
                    const float4 kv = *reinterpret_cast<const float4*>(kp + C::at(key, c));
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
            }
            }  // i >= 0
            __syncwarp();
            if (ST || i + STAGES < n) issue(i + STAGES, std::false_type{}, steady);
            asm volatile("cp.async.commit_group;" ::: "memory");
            const bool cut = klo > 0 || khi < TK;
            // the tile's values are there
            auto arrived = [&] {
                if (TMA && cut) {
                    // values that are not the row's may be anything; with weight 0 they have to be finite
                    for (int x = lane; x < TK * p.boxes * 8; x += 32) {
                        const int r = x / (p.boxes * 8), c = x % (p.boxes * 8);
                        if (r < klo || r >= khi)
                            *reinterpret_cast<uint4*>(ring + stage * C::STAGE + TK * C::ROWB + C::at(r, c)) = make_uint4(0, 0, 0, 0);
                    }
                    tc::fence_proxy_async_smem();  // before the stage's next TMA write
                    __syncwarp();
                }
            };
            if (ST || i >= 0) {
            if constexpr (!C::F32) {
                if (cut) {
#pragma unroll
                    for (int x = 0; x < MT; ++x)
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const int r = x * 16 + (lane >> 2) + (z >> 1) * 8;
                            if (r < klo || r >= khi) {
#pragma unroll
                                for (int y = 0; y < NT; ++y) S[x][y][0][z] = S[x][y][C::acc() / 2][z] = S[x][y][C::acc() - 1][z] = -INFINITY;
                            }
                        }
                }
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
                                if (C::acc() == 3) S[x][y][1][z] += S[x][y][2][z];
                                if (C::acc() > 1) S[x][y][0][z] += S[x][y][1][z];
                                mx = fmaxf(mx, S[x][y][0][z]);
                            }
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const int k = 2 * y + c;
                        // m is the largest score before the factor, so that its own weight is exactly 1
                        const float mn = fmaxf(m[k], mx);
                        const float ms = mn == -INFINITY ? 0.f : mn;
                        al[k] = ex2((m[k] - ms) * fac[k]);
                        m[k] = mn;
                        float sum = 0.f;
#pragma unroll
                        for (int x = 0; x < MT; ++x)
#pragma unroll
                            for (int z = c; z < 4; z += 2) {
                                const float e = ex2(fmaf(S[x][y][0][z] - ms, fac[k], C::shift()));
                                S[x][y][0][z] = e;
                                sum += e;
                            }
                        l[k] = l[k] * al[k] + sum;
                    }
                // O^T += V^T P^T: the weights, transposed 8 x 8 in registers, are the B operand. A tile's product
                // is summed by itself and then added to O with rounding to nearest: the tensor cores round a
                // running sum down, which over 600 tiles of 16 keys of values of one sign left fp32 results 2e-5
                // to 6e-5 too small (now 1e-6). It costs 0.4 % of the time on the long row, 0.9 % on ragged ones
                uint32_t pf[C::sp()][MT][NT][2];
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int t = 0; t < C::sp(); ++t) {
                            pf[t][x][y][0] = movm(take_pair<TC>(S[x][y][0][0], S[x][y][0][1]));
                            pf[t][x][y][1] = movm(take_pair<TC>(S[x][y][0][2], S[x][y][0][3]));
                        }
                wait(2 * stage + 1, i);
                arrived();
#pragma unroll
                for (int d = 0; d < C::KD; ++d) {
                    float sum[NT][4];
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        uint32_t af[4];
                        ldsm4t(af, ((kt + vat) ^ ((d & 3) * 32)) + (d >> 2) * (TK * 128) + x * 2048);
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int t = 0; t < C::sp(); ++t)
                                if (x == 0 && t == 0)
                                    mma16816_0<TC>(sum[y], af, pf[t][x][y][0], pf[t][x][y][1]);
                                else
                                    mma16816<TC>(sum[y], af, pf[t][x][y][0], pf[t][x][y][1]);
                    }
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int z = 0; z < 4; z += 2) {
                            const float2 r = fma2(make_float2(O[d][y][z], O[d][y][z + 1]), make_float2(al[2 * y], al[2 * y + 1]),
                                                  make_float2(sum[y][z], sum[y][z + 1]));
                            O[d][y][z] = r.x, O[d][y][z + 1] = r.y;
                        }
                }
            } else {
                const unsigned char* vp = ring + stage * C::STAGE + TK * C::ROWB;
                const int key = (lane & 7) + (lane >> 3) / C::lpk() * 8, part = (lane >> 3) % C::lpk();
#pragma unroll
                for (int h = 0; h < HB; ++h) {
                    float v = s[h];
#pragma unroll
                    for (int o = 8; o < 8 * C::lpk(); o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    v = key >= klo && key < khi ? v * (p.scale * LOG2E) : -INFINITY;
                    float mx = v;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1)  // the lanes of the other keys
                        if (o < 8 || o >= 8 * C::lpk()) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
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
                wait(2 * stage + 1, i);
                arrived();
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
                        const float4 v = *reinterpret_cast<const float4*>(vp + C::at(r, c0 + 32 * y));
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
            }  // i >= 0
            __syncwarp();
            if (ST || i + STAGES < n) issue(i + STAGES, std::true_type{}, steady);
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = -STAGES; i < n; ++i) {
            // tiles inside a row, whose loads stay inside it too, need none of the checks at its ends
            if (i > 0 && !fresh && w.j > 0) {
                for (int run = min(w.nt - STAGES - 2 - w.j, n - STAGES - 1 - i); run > 0; --run, ++i, ++w.j)
                    step(i, std::true_type{});
            }
            step(i, std::false_type{});
            const bool last = i == n - 1;
            if (i >= 0 && (last || w.j + 1 == w.nt)) {
                // the segment ends, here or in this warp's range
                fresh = true;
                const long long first = a + i - w.j;  // its first tile
                const bool whole = first >= a && w.j + 1 == w.nt;
                const int h0 = w.hb * HB, head0 = w.kvh * p.group + h0, nh = min(HB, p.group - h0);
                if (TMA && __any_sync(0xffffffffu, stuck)) bad |= GPT2Q_STATUS_TIMEOUT;
                if (bad && p.status && lane == 0) atomicOr(p.status, bad);
#pragma unroll
                for (int k = 0; k < (C::F32 ? HB : 2 * NT); ++k) {
#pragma unroll
                    for (int o = C::F32 ? 1 : 4; o < 32; o <<= 1) l[k] += __shfl_xor_sync(0xffffffffu, l[k], o);
                    l[k] *= C::UNSHIFT;
                    if (!C::F32) m[k] *= fac[k % (2 * NT)];
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
                    if (lane == 0) pieces[ps] = Piece{first, w.nt, w.row, w.kvh * p.blocks_per_kv + w.hb, dst};
                    __syncwarp();
                }
                if constexpr (!C::F32) {
                    // a lane has dims lane / 4 + {0, 8, 16, ...} of heads 2 (lane % 4) + {0, 1}; the addresses
                    // are one base per head and constants, as this code runs too rarely to stay in the
                    // instruction cache (a flush took 5 us with an address computed per element)
                    const int d0 = lane >> 2;
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int h = y * 8 + (lane & 3) * 2 + c, k = 2 * y + c;
                            if (h >= nh) continue;
                            if (!whole) {
                                float* at = dst + h * C::HS + d0;  // dims past the head's own are 0, and not read
#pragma unroll
                                for (int d = 0; d < 2 * C::KD; ++d) at[d * 8] = O[d / 2][y][2 * (d & 1) + c] * C::UNSHIFT;
                                if (lane < 4) pm[ps][h] = m[k], pl[ps][h] = l[k];
                                continue;
                            }
                            const float f = inverse(l[k]) * C::UNSHIFT;
                            if (p.out) {
                                TI* at = static_cast<TI*>(p.out) + w.row * p.o_ts + (head0 + h) * p.o_hs + d0;
#pragma unroll
                                for (int d = 0; d < 2 * C::KD; ++d)
                                    if (d * 8 < p.dim) at[d * 8] = from_f<TI>(O[d / 2][y][2 * (d & 1) + c] * f);
                            }
                            if (std::is_same<TI, float>::value && p.hl.hi) {
                                const long long o = (long long)w.row * p.hl.ld + (head0 + h) * p.dim + d0;
#pragma unroll
                                for (int d = 0; d < 2 * C::KD; ++d)
                                    if (d * 8 < p.dim) {
                                        const float v = O[d / 2][y][2 * (d & 1) + c] * f;
                                        const __half hi = __float2half_rn(v);
                                        p.hl.hi[o + d * 8] = hi;
                                        p.hl.lo[o + d * 8] = __float2half_rn(v - __half2float(hi));
                                    }
                            }
                            if (p.lse && lane < 4) p.lse[(long long)w.row * p.n_heads + head0 + h] = log_sum(m[k], l[k]);
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
            if (i >= 0 && !last) advance<C>(p, slen, w);
        }
        if (TMA && stuck && lane == 0)
            // copies that may still be on their way get about as long again before the block ends
            for (int k = 0; k < 2 * STAGES; ++k) {
                const uint32_t phase = tc::mbar_test_wait(&full[warp][k], 0);  // the one not completed
                for (int tries = 0; tries < WAIT_TRIES / (2 * STAGES) && !tc::mbar_try_wait(&full[warp][k], phase); ++tries) {}
            }
    }
    __syncthreads();

    // ---- the block's pieces, joined where they belong to one (row, head block) ----
    // lane i has piece i; pieces of one (row, head block) are neighbours and form a chain
    const bool there = lane < 2 * nw && pieces[lane].nt > 0;
    const long long of = there ? pieces[lane].first : -1 - lane;
    const unsigned mates = __match_any_sync(0xffffffffu, of);
    const unsigned heads = __ballot_sync(0xffffffffu, there && __ffs(mates) - 1 == lane);
    const int chains = __popc(heads);
    const int rank = heads >> lane & 1 ? __popc(heads & ((1u << lane) - 1)) : -1;  // which chain this lane heads
    int tail_row = -1, tail_vh = 0;
    long long tail_last = 0;
    if (warp == 0 && chains) {
        const Piece P = pieces[31 - __clz(heads)];  // only the last chain may go on behind the block
        if (P.first >= ca && P.first + P.nt > cb)
            tail_row = P.row, tail_vh = P.vh, tail_last = quotient(P.first + P.nt - 1, per);
    }
    for (int u = warp; u < chains * hv; u += nw) {
        const int ch = u / hv, h = u - ch * hv;
        const int i0 = __ffs(__ballot_sync(0xffffffffu, rank == ch)) - 1;  // the chain's first piece
        const Piece P = pieces[i0];
        unsigned members = __shfl_sync(0xffffffffu, mates, i0);
        const int kvh = P.vh / p.blocks_per_kv, h0 = (P.vh - kvh * p.blocks_per_kv) * HB;
        if (h0 + h >= p.group) continue;
        const bool in = members >> lane & 1;
        const float mm = in ? pm[lane][h] : -INFINITY, ll = in ? pl[lane][h] : 0.f;
        float M = mm;
#pragma unroll
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float wt = ex2(mm - (M == -INFINITY ? 0.f : M));
        float Ls = ll * wt;
#pragma unroll
        for (int o = 16; o; o >>= 1) Ls += __shfl_xor_sync(0xffffffffu, Ls, o);
        const bool whole = P.first >= ca && P.first + P.nt <= cb;
        const float f = whole ? inverse(Ls) : 1.f;
        const long long ci = ((long long)blockIdx.x * 2 + (P.first < ca ? 0 : 1)) * HB + h;
        float r[(HD + 127) / 128][4] = {};
        while (members) {
            const int j = __ffs(members) - 1;
            members &= members - 1;
            const float wj = __shfl_sync(0xffffffffu, wt, j);
            const float* data = pieces[j].data + h * C::HS + lane * 4;
#pragma unroll
            for (int y = 0; y < (HD + 127) / 128; ++y)
                if (lane * 4 + y * 128 < p.dim) {
                    const float4 v = *reinterpret_cast<const float4*>(data + y * 128);
                    r[y][0] = fmaf(v.x, wj, r[y][0]);
                    r[y][1] = fmaf(v.y, wj, r[y][1]);
                    r[y][2] = fmaf(v.z, wj, r[y][2]);
                    r[y][3] = fmaf(v.w, wj, r[y][3]);
                }
        }
#pragma unroll
        for (int y = 0; y < (HD + 127) / 128; ++y) {
            const int d = lane * 4 + y * 128;
            if (d >= p.dim) break;
#pragma unroll
            for (int z = 0; z < 4; ++z) r[y][z] *= f;
            if (whole)
                write4<TI>(p, P.row, kvh * p.group + h0 + h, d, r[y]);
            else
                *reinterpret_cast<float4*>(p.block_part + ci * HD + d) = make_float4(r[y][0], r[y][1], r[y][2], r[y][3]);
        }
        if (lane == 0) {
            if (!whole)
                p.block_ml[ci] = make_float2(M, Ls);
            else if (p.lse)
                p.lse[(long long)P.row * p.n_heads + kvh * p.group + h0 + h] = log_sum(M, Ls);
        }
    }
    if (tid == 0) p.meta[blockIdx.x] = make_int4(tail_row, tail_vh, (int)tail_last, 0);

    // ---- rows without a cached token ----
    for (int r = blockIdx.x; r < p.n_rows; r += gridDim.x) {
        if ((r < LENS ? slen[r] : __ldcg(p.lens + r)) > 0) continue;
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
    __shared__ float weight[MAX_CTAS];
    tc::pdl_trigger();
    tc::pdl_wait();
    const int c = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    auto at = [&](int i) { return ((long long)(c + i) * 2 + (i == 0 ? 1 : 0)) * HB + h; };
    constexpr int DG = HD / 4, PG = 128 / DG;  // threads over dims, and over pieces
    const int d = tid % DG * 4, g = tid / DG;
    // In a small grid the first pieces are loaded along with the word that says whether, and how many,
    // there are; in a large one most blocks only end here, and the loads of all would cost more than they
    // save. One row of bf16, loading early against late: 0.1 to 0.4 us less in grids of 16 to 64 blocks
    // (3000 keys of 4 heads, 63 x 1: 12.2 and 12.6 us), 0.3 to 0 less in 86 to 176, 0.3 more in 344, and 1.2
    // to 1.7 more where 148 blocks had a part (20000 keys, 148 x 1: 22.7 and 21.1; x 8: 26.0 and 24.7).
    const int4 meta = __ldcg(p.meta + c);
    if (gridDim.x * gridDim.y > 64 && meta.x < 0) return;
    const int most = gridDim.x - c;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < most) ml = __ldcg(p.block_ml + at(lane));
    float4 v0[2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
        if (d < p.dim && g + k * PG < most) v0[k] = __ldcg(reinterpret_cast<const float4*>(p.block_part + at(g + k * PG) * HD + d));
    if (meta.x < 0) return;
    const int kvh = meta.y / p.blocks_per_kv, h0 = (meta.y - kvh * p.blocks_per_kv) * HB;
    if (h0 + h >= p.group) return;
    const int n = meta.z - c + 1;
    if (lane >= n) ml = make_float2(-INFINITY, 0.f);
    float M = ml.x, L = 0.f;
    for (int i = lane + 32; i < n; i += 32) M = fmaxf(M, __ldcg(p.block_ml + at(i)).x);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ms = M == -INFINITY ? 0.f : M;
    for (int i = lane; i < n; i += 32) {
        if (i >= 32) ml = __ldcg(p.block_ml + at(i));
        const float wt = ex2(ml.x - ms);
        L += ml.y * wt;
        if ((tid >> 5) == 0) weight[i] = wt;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    __syncthreads();
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < p.dim) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (g + k * PG < n) {
                const float wt = weight[g + k * PG];
                r.x = fmaf(v0[k].x, wt, r.x);
                r.y = fmaf(v0[k].y, wt, r.y);
                r.z = fmaf(v0[k].z, wt, r.z);
                r.w = fmaf(v0[k].w, wt, r.w);
            }
#pragma unroll 4
        for (int i = g + 2 * PG; i < n; i += PG) {
            const float wt = weight[i];
            const float4 v = __ldcg(reinterpret_cast<const float4*>(p.block_part + at(i) * HD + d));
            r.x = fmaf(v.x, wt, r.x);
            r.y = fmaf(v.y, wt, r.y);
            r.z = fmaf(v.z, wt, r.z);
            r.w = fmaf(v.w, wt, r.w);
        }
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

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn tensor_map_encoder() {
    static const EncodeTiledFn fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<EncodeTiledFn>(ptr)
                   : nullptr;
    }();
    return fn;
}

constexpr size_t SMEM_LIMIT = 217 * 1024;  // dynamic; the rest for the static arrays

// A pool as a tensor [page][head][piece][slot][dim]; dims past the head's own are read as zero.
template <class C>
bool make_map(CUtensorMap* m, const PagedAttn& p, const void* base) {
    const auto encode = tensor_map_encoder();
    if (!encode) return false;
    using TC = typename C::TC;
    const auto type = C::F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                             : C::HALF ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // heads of whole pieces of 128 bytes are read with one box of all their pieces, others piece by
    // piece (a tile of several groups of keys has one piece)
    const bool merged = p.box_loads == 1;
    const cuuint64_t pieces = merged ? p.boxes : 1;
    const cuuint64_t dims[5] = {(cuuint64_t)(merged && p.boxes > 1 ? C::BOX : p.dim), (cuuint64_t)p.page, pieces, (cuuint64_t)p.n_kv,
                                (cuuint64_t)p.n_pages};
    // the stride of a dimension of one element does not matter, but may not be 0
    const cuuint64_t row = ((cuuint64_t)p.dim * sizeof(TC) + 15) / 16 * 16;
    const cuuint64_t strides[4] = {p.page == 1 ? row : p.ts16 * 16ull, 128, p.n_kv == 1 ? row : p.hs16 * 16ull,
                                   p.n_pages == 1 ? row : p.ps16 * 16ull};
    const cuuint32_t box[5] = {(cuuint32_t)C::BOX, (cuuint32_t)C::GR, (cuuint32_t)pieces, 1, 1}, step[5] = {1, 1, 1, 1, 1};
    return encode(m, type, 5, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class C, bool TMA>
cudaError_t launch_main(const PagedAttn& p, const CUtensorMap& km, const CUtensorMap& vm, int grid, int nw, size_t smem, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        e = cudaFuncSetAttribute(k_paged_attn<C, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    return launch_dependent(k_paged_attn<C, TMA>, dim3(grid), dim3(nw * 32), smem, st, p, km, vm);
}

template <class C>
cudaError_t launch(PagedAttn p, cudaStream_t st) {
    p.blocks_per_kv = (p.group + C::HB - 1) / C::HB;
    p.n_vh = p.n_kv * p.blocks_per_kv;
    p.heads_per_block = std::min(p.group, C::HB);
    size_t wb = STAGES * C::STAGE + (size_t)C::QS * p.heads_per_block * C::HD * sizeof(typename C::TI);
    if (C::F32) wb += (size_t)C::TK * C::HB * 4;
    p.warp_bytes = (int)((wb + 1023) / 1024 * 1024);
    const int nw = (int)std::min<size_t>(C::WARPS, SMEM_LIMIT / p.warp_bytes);
    // no more blocks than the longest rows the table can hold would fill
    const long long longest = p.window > 0 ? std::min(p.window, p.cap) : p.cap;
    const long long tiles = ((longest + C::TK - 1) / C::TK + (p.window > 0 ? 1 : 0)) * p.n_vh;
    const long long want = tiles > MAX_CTAS * 8LL ? MAX_CTAS : (tiles * p.n_rows + nw - 1) / nw;
    const int grid = (int)std::clamp<long long>(want, 1, MAX_CTAS);
    p.boxes = (p.dim * (int)sizeof(typename C::TC) + 127) / 128;
    p.box_loads = p.boxes > 1 && p.dim % C::BOX == 0 && C::NG == 1 ? 1 : p.boxes;
    p.group_bytes = p.boxes * C::GR * 128;
    // for the test of waits that run out: they expect 16 bytes more than are copied
    static const bool stall = std::getenv("GPT2Q_TEST_PAGED_STALL") != nullptr;
    if (stall) p.group_bytes += 16;
    CUtensorMap km{}, vm{};
    const bool tma = p.page % C::GR == 0 && make_map<C>(&km, p, p.k) && make_map<C>(&vm, p, p.v);
    const size_t smem = (size_t)nw * p.warp_bytes;
    cudaError_t e = tma ? launch_main<C, true>(p, km, vm, grid, nw, smem, st) : launch_main<C, false>(p, km, vm, grid, nw, smem, st);
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
