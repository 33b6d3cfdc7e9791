// Attention of one new token per row over a paged key/value cache (gpt2q_paged_attention), and of drafted tokens
// (gpt2q_paged_tree_attention) where they are few per row or in fp32.
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
//
// 8-bit caches: an entry is code * scale, so codes are widened to fp16, in which they are exact, on their way from shared memory
// to registers; a key's scale multiplies its scores and a value's scale its weight, relative to the largest exponent so far (in tiles
// with drafted tokens, for each query that of the keys it has a weight for), so that the product stays in fp16's range. Half the bytes leave the instructions as the bound: one row of 131071 keys in e4m3, 64
// heads on 8 of 128, 77 us (43 at the memory rate), 63 rows of 17 to 9000 in int8 67 us (30).
//
// Drafted tokens: a row's queries are its tokens times the query heads of a kv head, in blocks of HB columns; a mask or the
// position says which of the drafted keys a column sees. 8 drafted tokens behind 501, 12 heads of 64, fp32 on fp16: 17.8 us.
#pragma once
#include <cuda.h>
#include <cuda_fp8.h>

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

namespace gpt2q {
namespace {

constexpr int STAGES = 2;
constexpr int MAX_WARPS = 16;
constexpr int LENS = 512;     // rows whose lengths a block keeps in shared memory
constexpr int MAX_CTAS = 148;  // one per SM of a B200
constexpr int WAIT_TRIES = 1 << 19;  // of about 1.5 us: 0.8 s
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// Places of a segment of an 8-bit cache beside its tiles. Its queries, first copies and results cost as much as several tiles of 16
// keys, and blocks of many short rows ended last: SMs were active for 68 % of a call with 63 ragged rows, 92 us; with 2, 4 or 8 places
// 70. 16 rows of 17 to 9000 keys 34.7 to 31.3 us, 32 of 400 to 500 27.5 to 26.5, 8 of those 17.6 to 20.8, as finding tiles in
// such ranges takes 2 us. One row's segments are all alike and have none (1001 keys 13.2 us without, 15.7 with).
constexpr int PADS = 4;

// TC: cache type, TI: type of q and out, HD: head dim rounded up, HB: queries a tile is used for.
// TREE: a row has any number of queries (drafted tokens) instead of one.
template <class TC_, class TI_, int HD_, int HB_, bool TREE_>
struct Cfg {
    using TC = TC_;
    using TI = TI_;
    static constexpr int HD = HD_, HB = HB_;
    static constexpr bool TREE = TREE_;
    static constexpr bool F32 = std::is_same<TC, float>::value;
    static constexpr bool Q8 = sizeof(TC) == 1;  // codes with a scale per entry: exact in fp16, in which they are multiplied
    using CT = std::conditional_t<Q8, __half, TC>;  // type of the products' operands
    static constexpr bool HALF = std::is_same<CT, __half>::value;
    static constexpr int ROWB = Q8 && HD < 128 ? 128 : HD * (int)sizeof(TC);
    static constexpr int CHP = ROWB / 16;  // 16-byte chunks of a row
    // keys of a tile: 8 KB of keys and values (16 KB at 256 dims); of an 8-bit cache 16, half of that, as its tiles are bound
    // by their instructions and 16 warps hold more of them than 12 (ragged rows 109 to 91 us, a long row 84 to 77)
    static constexpr int TK = F32 ? (HD == 256 ? 8 : 4096 / ROWB) : (HD == 256 || Q8 ? 16 : 4096 / ROWB);
    static __device__ constexpr int lpk() { return 32 / TK; }  // lanes per key (fp32 cache)
    static_assert(!Q8 || TK == 16, "a lane's scale goes by the tile's one page lookup");
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
    // (One piece of fp16 for bf16 outputs of an 8-bit cache would be 6 % faster on a long row, but 2^-11 of the result off: a row
    // of one key would not give its value.)
    static constexpr int sp() { return SQ == 1 || HALF ? 2 : 3; }
    // queries whose range the products' type does not have: scaled by a power of two per head. bf16 ones are then exact in
    // one piece of fp16 down to 2^-24 of the head's largest element
    static constexpr bool RANGE = HALF && !std::is_same<TI, __half>::value;
    // dims of a product's operand beside one another in a register: 8-bit codes come four at a time
    static __device__ constexpr int dim_of(int t, int x) { return Q8 ? t * 4 + x * 2 : t * 2 + x * 8; }
    // dims of the results of a product of 16 dims: of fragment row r, upper half u
    static __device__ constexpr int row_dim(int r, int u) { return Q8 ? r * 2 + u : r + u * 8; }
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
    static constexpr int WARPS = !F32 && SQ * NT * KD * 2 + NT * KD * 4 > 100 ? 8 : Q8 && NT == 1 && SQ == 1 && HD <= 128 ? 16 : 12;
    static constexpr float UNSHIFT = HALF ? 1.f / 1024.f : 1.f;
    // places that a segment (a row's keys for one block of queries) has in the list beside its tiles, before them
    static constexpr int PAD = Q8 ? PADS : 0;
    static constexpr size_t SMEM_LIMIT = (PAD ? 212 : 217) * 1024;  // dynamic; the rest for the static arrays
};

struct Walk {
    int row, kvh, hb, j, nt, start, end;  // hb: block of the kv head's queries
    bool over;
    // of a tree: blocks per kv head, queries (tokens times heads) per kv head, the row's first token
    int blocks, queries, token;
};

struct Piece {
    long long first;  // index of its segment's first tile
    int nt, row, vh;  // nt = 0: none
    int blocks, queries, token;
    const float* data;
};

// The tokens of a tree's row: a malformed `first` leads to no token outside [0, n_tokens).
__device__ __forceinline__ void tokens_of(const PagedAttn& p, int row, int& first, int& n) {
    const int a = __ldcg(p.first + row), b = __ldcg(p.first + row + 1);
    first = min(max(a, 0), p.n_tokens);
    n = max(min(b, p.n_tokens) - first, 0);
}
// Where query i of a kv head's block of queries lies: its token and head.
template <class C>
__device__ __forceinline__ void query_at(const PagedAttn& p, int row, int token, int kvh, int i, int& at, int& head) {
    if constexpr (C::TREE) {
        const int t = (int)((unsigned)i / (unsigned)p.group);
        at = token + t;
        head = kvh * p.group + i - t * p.group;
    } else {
        at = row;
        head = kvh * p.group + i;
    }
}

// Row `row` of the walk; `lens` holds the first LENS rows' lengths.
template <class C>
__device__ __forceinline__ void enter(const PagedAttn& p, const int* lens, Walk& w, int row) {
    w.row = row;
    int len = row >= p.n_rows ? 0 : row < LENS ? lens[row] : __ldcg(p.lens + row);
    if constexpr (C::TREE) {
        int n = 0;
        w.token = 0;
        if (row < p.n_rows) tokens_of(p, row, w.token, n);
        w.queries = n * p.group;
        w.blocks = (w.queries + C::HB - 1) / C::HB;
        len = n > 0 ? (int)min((long long)max(len, 0) + n, (long long)INT32_MAX) : 0;
    }
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
    if (++w.hb < (C::TREE ? w.blocks : p.blocks_per_kv)) return;
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
// Four 8-bit codes as two pairs of fp16. Of neighbouring dims: bytes 0, 1 and 2, 3; of two keys (after a transposing load:
// key 0's dims, key 1's): dim 0 of both keys, dim 1 of both.
template <class TC, bool KEYS>
__device__ __forceinline__ void widen(uint32_t v, uint32_t& a, uint32_t& b) {
    if constexpr (std::is_same<TC, int8_t>::value) {
        // 0x6400 + u is the fp16 number 1024 + u; u = code + 128
        v ^= 0x80808080u;
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        uint32_t x = __byte_perm(v, 0x64646464u, KEYS ? 0x4240 : 0x4140), y = __byte_perm(v, 0x64646464u, KEYS ? 0x4341 : 0x4342);
        const __half2 hx = __hsub2(*reinterpret_cast<const __half2*>(&x), off), hy = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
        a = *reinterpret_cast<const uint32_t*>(&hx);
        b = *reinterpret_cast<const uint32_t*>(&hy);
    } else {
        if (KEYS) v = __byte_perm(v, 0, 0x3120);
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(a), "=r"(b)
            : "r"(v));
    }
}
// Whether one of 16 bytes of elements is infinite or NaN.
template <class TC>
__device__ __forceinline__ bool not_finite(uint4 v) {
    if constexpr (std::is_same<TC, int8_t>::value) return false;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(TC) == 4) {
            bad |= (w[i] & 0x7f800000u) == 0x7f800000u;
        } else if constexpr (sizeof(TC) == 2) {
            constexpr uint32_t E = std::is_same<TC, __half>::value ? 0x7c00u : 0x7f80u;
            bad |= (w[i] & E) == E || (w[i] >> 16 & E) == E;
        } else {
            bad |= __vcmpeq4(w[i] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
        }
    }
    return bad;
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
// Four elements of one head's result to the output and, when wanted, its fp16 hi/lo copies. `row`: of the output.
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

// Whether query i of the row's kv head sees the row's drafted token j: its own words say so, or it comes no later. j < 0: the
// prefix, which every query sees; false past the mask's words.
template <class C>
__device__ __forceinline__ bool sees(const PagedAttn& p, const Walk& w, int i, int j) {
    if (!C::TREE || j < 0) return true;
    const int t = (int)((unsigned)i / (unsigned)p.group);
    if (!p.mask) return j <= t;
    if (i >= w.queries || (j >> 5) >= p.mask_words) return false;
    return __ldcg(p.mask + (long long)(w.token + t) * p.mask_words + (j >> 5)) >> (j & 31) & 1;
}

template <class C, bool TMA>
__global__ void __launch_bounds__(C::WARPS * 32, 1)
    k_paged_attn(const __grid_constant__ PagedAttn p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using TC = typename C::TC;
    using CT = typename C::CT;
    using TI = typename C::TI;
    constexpr int HB = C::HB, HD = C::HD, TK = C::TK, NT = C::NT > 0 ? C::NT : 1, MT = C::MT > 0 ? C::MT : 1;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ long long cum[C::WARPS * 32 + 1];
    __shared__ long long wsum[C::WARPS];
    __shared__ long long segs[C::PAD ? C::WARPS * 32 : 1], sum_segs[C::PAD ? C::WARPS : 1], s_range[C::PAD ? 2 : 1];  // as cum and wsum, of segments
    __shared__ int slen[LENS];
    __shared__ Piece pieces[2 * C::WARPS];
    __shared__ __align__(8) uint64_t full[C::WARPS][2 * STAGES];  // per stage: keys, values
    __shared__ float pm[2 * C::WARPS][HB], pl[2 * C::WARPS][HB];
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
    const int pad = C::PAD && p.n_rows > 1 ? C::PAD : 0;  // one row's segments are all alike
    const int nc = (p.n_rows + nthr - 1) / nthr;  // rows a thread counts
    Walk w;
    long long mine = 0, mine_segs = 0;
    for (int r = tid; r < min(LENS, p.n_rows); r += nthr) slen[r] = __ldcg(p.lens + r);
    if (nc > 1) __syncthreads();
    auto row_segs = [&](const Walk& x) { return C::TREE ? p.n_kv * x.blocks : p.n_vh; };
    for (int r = tid * nc; r < min((tid + 1) * nc, p.n_rows); ++r) {
        enter<C>(p, slen, w, r);  // with nc == 1 the thread's own
        mine += C::TREE ? (long long)w.nt * (p.n_kv * w.blocks) : w.nt;
        if (pad && w.nt) mine_segs += row_segs(w);
    }
    if (!C::TREE) mine *= p.n_vh;
    if (C::PAD) mine += mine_segs * pad;
    long long inc = mine, inc_segs = mine_segs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
        if (pad) {
            const long long u = __shfl_up_sync(0xffffffffu, inc_segs, o);
            if (lane >= o) inc_segs += u;
        }
    }
    if (lane == 31) {
        wsum[warp] = inc;
        if (pad) sum_segs[warp] = inc_segs;
    }
    __syncthreads();
    long long before = 0, total = 0, before_segs = 0, all_segs = 0;
    for (int i = 0; i < nw; ++i) {
        if (i < warp) before += wsum[i];
        total += wsum[i];
        if (pad) {
            if (i < warp) before_segs += sum_segs[i];
            all_segs += sum_segs[i];
        }
    }
    if (C::TREE && total > p.most) {  // a `first` that names tokens again and again: no work rather than any amount of it
        total = all_segs = 0;
        if (tid == 0 && blockIdx.x == 0 && p.status) atomicOr(p.status, GPT2Q_STATUS_POSITION);
    }
    cum[tid] = before + inc - mine;
    if (pad) segs[tid] = before_segs + inc_segs - mine_segs;
    __syncthreads();
    const long long wper = quotient(quotient(total + gridDim.x - 1, gridDim.x) + nw - 1, nw), per = wper * nw;
    // Ranges of places are equal, of tiles they are what lies in them. `find`: w is the first tile at or behind a place of the list,
    // the result its number.
    auto find = [&](long long at) -> long long {
        int lo = 0, hi = nthr - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cum[mid] <= at)
                lo = mid;
            else
                hi = mid - 1;
        }
        long long rem = at - cum[lo], skipped = pad ? segs[lo] : 0;
        int row = lo * nc;
        enter<C>(p, slen, w, row);
        auto places = [&] { return w.nt ? w.nt + pad : 0; };
        while (rem >= (long long)places() * row_segs(w)) {
            rem -= (long long)places() * row_segs(w);
            if (pad && w.nt) skipped += row_segs(w);
            enter<C>(p, slen, w, ++row);
        }
        const int vh = (int)quotient(rem, places());
        w.j = (int)(rem - (long long)vh * places());
        w.kvh = vh / (C::TREE ? w.blocks : p.blocks_per_kv);
        w.hb = vh - w.kvh * (C::TREE ? w.blocks : p.blocks_per_kv);
        if (!pad) return at;
        const int pads = min(w.j, pad);
        w.j -= pads;
        return at - (skipped + vh) * pad - pads;
    };
    const long long end_place = min(per * (blockIdx.x + 1), total);
    long long a = per * blockIdx.x + wper * warp, b = min(a + wper, end_place);
    if (pad) {
        // two lanes: where the warp's range begins and ends
        const long long at = lane == 0 ? a : b;
        long long tile = total - all_segs * pad;
        if (lane < 2 && at < total) tile = find(at);
        __syncwarp();
        if (lane < 2 && warp == (lane ? nw - 1 : 0)) s_range[lane] = tile;  // the block's; read behind the next barrier
        a = __shfl_sync(0xffffffffu, tile, 0), b = __shfl_sync(0xffffffffu, tile, 1);
        w.row = __shfl_sync(0xffffffffu, w.row, 0), w.kvh = __shfl_sync(0xffffffffu, w.kvh, 0), w.hb = __shfl_sync(0xffffffffu, w.hb, 0);
        w.j = __shfl_sync(0xffffffffu, w.j, 0);
    }
    const int n = (int)max(0LL, b - a);

    if (n > 0) {
        if (pad)
            enter<C>(p, slen, w, w.row);
        else
            find(a);
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
        // 8-bit cache: scales of key lane % TK, of the tile worked on and of the next one
        [[maybe_unused]] float ks[2] = {}, vs[2] = {};
        [[maybe_unused]] long long s_at = -1;  // where the newest one lies
        // ... and the biased exponent that the results are held relative to, the largest of the values' scales so far: their
        // weights times scale / 2^exponent stay in the range of fp16. Of a tree one per column, as columns do not see the same
        constexpr int NE = C::TREE ? 2 * NT : 1;
        [[maybe_unused]] uint32_t vexp[NE];
        // Starts the copies of tile i's keys (and its row's queries) or values; values come second.
        // steady: the tile and the one after it lie inside the row that the loads are in.
        auto issue = [&](int i, auto values, auto steady) {
            constexpr bool V = decltype(values)::value, ST = decltype(steady)::value;
            const int stage = i % STAGES;
            if (!V && !ST && (i == 0 || L.j == 0)) {
                qload = qload + 1 == C::QS ? 0 : qload + 1;
                const int h0 = L.hb * HB;
                if constexpr (C::TREE) {
                    for (int x = lane; x < hv * (qrow / 16); x += 32) {
                        const int h = x / (qrow / 16), c = x - h * (qrow / 16);
                        int t, head;
                        query_at<C>(p, L.row, L.token, L.kvh, h0 + h, t, head);
                        const bool there = h0 + h < L.queries;
                        if (c < nqch)
                            cp16(q32 + qload * hv * qrow + x * 16,
                                 static_cast<const char*>(p.q) + (there ? ((long long)t * p.q_ts + (long long)head * p.q_hs) * (int)sizeof(TI) + c * 16 : 0),
                                 there);
                    }
                } else {
                    const char* q = static_cast<const char*>(p.q) +
                                    ((long long)L.row * p.q_ts + (long long)(L.kvh * p.group + h0) * p.q_hs) * (int)sizeof(TI);
                    for (int x = lane; x < hv * (qrow / 16); x += 32) {
                        const int h = x / (qrow / 16), c = x - h * (qrow / 16);
                        const bool there = h0 + h < p.group;
                        if (c < nqch)
                            cp16(q32 + qload * hv * qrow + x * 16, q + (there ? h * p.q_hs * (int)sizeof(TI) + c * 16 : 0), there);
                    }
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
            if constexpr (C::Q8) {
                // the scale of the lane's key; used two tiles later
                if (!V) {
                    const int key = L_key + (lane & (TK - 1));
                    s_at = -1;
                    if ((ST || (key < L.end && key >= L.start)) && (unsigned)page[0] < (unsigned)p.n_pages) {
                        const int slot = p.page_shift >= 0 ? key & (p.page - 1) : key % p.page;
                        s_at = (long long)page[0] * p.s_ps + (long long)L.kvh * p.s_hs + (long long)slot * p.s_ts;
                    }
                }
                const float f = s_at >= 0 ? __ldcg((V ? p.v_scale : p.k_scale) + s_at) : 0.f;
                if (V)
                    vs[0] = vs[1], vs[1] = f;
                else
                    ks[0] = ks[1], ks[1] = f;
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
                for (int k = 0; k < NE; ++k) vexp[k] = 1;
#pragma unroll
                for (int x = 0; x < (C::F32 ? HB : C::KD); ++x)
#pragma unroll
                    for (int y = 0; y < (C::F32 ? (HD + 127) / 128 : NT); ++y)
#pragma unroll
                        for (int z = 0; z < 4; ++z) O[x][y][z] = 0.f;
                if constexpr (!C::F32) {
                    // B fragments of the queries: head lane / 4, dims 2 (lane % 4) + {0, 1, 8, 9}, of an 8-bit cache
                    // 4 (lane % 4) + {0, 1, 2, 3}, as its codes lie
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int h = nt * 8 + (lane >> 2);
                        const TI* qh = reinterpret_cast<const TI*>(q + h * qrow);
                        const int t4 = lane & 3;
                        [[maybe_unused]] float down = 1.f, up = 1.f;  // of the queries, and back
                        if constexpr (C::RANGE) {
                            // fp16 pieces of an fp32 or bf16 query: scaled by a power of two so that the
                            // head's largest element lies in [2^10, 2^11), undone on the scores
                            float top = 0.f;
#pragma unroll
                            for (int k = 0; k < HD / 8; ++k)
                                if (h < hv) top = fmaxf(top, fmaxf(fabsf(to_f(qh[k * 8 + t4 * 2])), fabsf(to_f(qh[k * 8 + t4 * 2 + 1]))));
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
                                const TI* qd = qh + k * 16 + C::dim_of(t4, x);
                                if constexpr (C::SQ == 1 && !C::RANGE) {
                                    qf[0][nt][k][x] = h < hv ? *reinterpret_cast<const uint32_t*>(qd) : 0u;
                                    if (p.scale < 0.f) qf[0][nt][k][x] ^= 0x80008000u;
                                } else {
                                    float u = 0.f, v = 0.f;
                                    const float sd = p.scale < 0.f ? -down : down;
                                    if (h < hv) u = to_f(qd[0]) * sd, v = to_f(qd[1]) * sd;
#pragma unroll
                                    for (int s = 0; s < C::SQ; ++s) qf[s][nt][k][x] = take_pair<CT>(u, v);
                                }
                            }
                        // a score's columns are heads 2 (lane % 4) + {0, 1}
                        fac[2 * nt] = fmaxf(sl2 * __shfl_sync(0xffffffffu, up, (lane & 3) * 8), 1.17549435e-38f);
                        fac[2 * nt + 1] = fmaxf(sl2 * __shfl_sync(0xffffffffu, up, (lane & 3) * 8 + 4), 1.17549435e-38f);
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
                if constexpr (C::Q8) {
                    // a load has 32 dims of 16 keys: two steps
#pragma unroll
                    for (int k = 0; k < C::KD; k += 2) {
#pragma unroll
                        for (int x = 0; x < MT; ++x) {
                            uint32_t cf[4], af[2][4];
                            ldsm4(cf, ((kt + kat) ^ ((k & 6) * 16)) + (k >> 3) * (TK * 128) + x * 2048);
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                widen<TC, false>(cf[2 * u], af[u][0], af[u][2]);
                                widen<TC, false>(cf[2 * u + 1], af[u][1], af[u][3]);
#pragma unroll
                                for (int y = 0; y < NT; ++y)
#pragma unroll
                                    for (int t = 0; t < C::SQ; ++t)
                                        mma16816<CT>(S[x][y][t ? 2 : C::acc() > 1 ? u : 0], af[u], qf[t][y][k + u][0], qf[t][y][k + u][1]);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < C::KD; ++k) {
#pragma unroll
                        for (int x = 0; x < MT; ++x) {
                            uint32_t af[4];
                            ldsm4(af, ((kt + kat) ^ ((k & 3) * 32)) + (k >> 2) * (TK * 128) + x * 2048);
#pragma unroll
                            for (int y = 0; y < NT; ++y)
#pragma unroll
                                for (int t = 0; t < C::SQ; ++t) mma16816<CT>(S[x][y][t ? 2 : C::acc() > 1 ? k & 1 : 0], af, qf[t][y][k][0], qf[t][y][k][1]);
                        }
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
            [[maybe_unused]] const float ks_tile = ks[0];
            __syncwarp();
            if (ST || i + STAGES < n)
                issue(i + STAGES, std::false_type{}, steady);
            else if (C::Q8)
                ks[0] = ks[1];
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
            // Of a tile with drafted tokens' keys, from key `from` on: those values that are not finite, as a mask of keys. They are
            // cleared, so that a query that does not see one is not reached by it (its weight is 0, but 0 times infinity is NaN).
            auto unclean = [&](int from) -> uint32_t {
                uint32_t rows = 0;
                if constexpr (!std::is_same<TC, int8_t>::value) {
                    unsigned char* v = ring + stage * C::STAGE + TK * C::ROWB;
                    for (int x = max(from, 0) * nch + lane; x < TK * nch; x += 32)
                        if (not_finite<TC>(*reinterpret_cast<const uint4*>(v + C::at(x / nch, x % nch)))) rows |= 1u << (x / nch);
                    rows = __reduce_or_sync(0xffffffffu, rows);
                    if (rows) {
                        for (int x = lane; x < TK * nch; x += 32)
                            if (rows >> (x / nch) & 1) *reinterpret_cast<uint4*>(v + C::at(x / nch, x % nch)) = make_uint4(0, 0, 0, 0);
                        if (TMA) tc::fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                return rows;
            };
            if (ST || i >= 0) {
            // of a tree: the tile has drafted tokens' keys
            [[maybe_unused]] const int drafted0 = C::TREE ? w.end - (int)((unsigned)w.queries / (unsigned)p.group) : 0;  // the first one
            [[maybe_unused]] const int tile0 = ((unsigned)w.start / TK + w.j) * TK;
            [[maybe_unused]] const bool masked = C::TREE && tile0 + TK > drafted0;
            if constexpr (!C::F32) {
                if constexpr (C::Q8) {
                    // a score's row is a key: times its scale
#pragma unroll
                    for (int x = 0; x < MT; ++x)
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const float f = __shfl_sync(0xffffffffu, ks_tile, x * 16 + u * 8 + (lane >> 2));
#pragma unroll
                            for (int y = 0; y < NT; ++y)
#pragma unroll
                                for (int c = 0; c < C::acc(); ++c) S[x][y][c][2 * u] *= f, S[x][y][c][2 * u + 1] *= f;
                        }
                }
                if (cut || masked) {
#pragma unroll
                    for (int x = 0; x < MT; ++x)
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const int r = x * 16 + (lane >> 2) + (z >> 1) * 8;
#pragma unroll
                            for (int y = 0; y < NT; ++y)
                                if (r < klo || r >= khi || (masked && !sees<C>(p, w, w.hb * HB + y * 8 + (lane & 3) * 2 + (z & 1), tile0 + r - drafted0)))
                                    S[x][y][0][z] = S[x][y][C::acc() / 2][z] = S[x][y][C::acc() - 1][z] = -INFINITY;
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
                // queries that see one of these keys give NaN, whatever its weight
                [[maybe_unused]] auto spoil = [&](uint32_t rows) {
#pragma unroll
                    for (int i = 0; i < MT * NT * 4; ++i) {
                        const int r = i / (NT * 4) * 16 + (lane >> 2) + (i % 4 >> 1) * 8, y = i / 4 % NT;
                        if (rows >> r & 1 && r >= klo && r < khi && sees<C>(p, w, w.hb * HB + y * 8 + (lane & 3) * 2 + (i & 1), tile0 + r - drafted0))
                            l[y * 2 + (i & 1)] = NAN;
                    }
                };
                // O^T += V^T P^T: the weights, transposed 8 x 8 in registers, are the B operand. A tile's product
                // is summed by itself and then added to O with rounding to nearest: the tensor cores round a
                // running sum down, which over 600 tiles of 16 keys of values of one sign left fp32 results 2e-5
                // to 6e-5 too small (now 1e-6). It costs 0.4 % of the time on the long row, 0.9 % on ragged ones
                if constexpr (C::Q8) {
                    // weights times their values' scales, relative to the largest exponent of those so far
                    auto lower = [&](int k, uint32_t e) {  // column k's results so far, relative to exponent e
                        const uint32_t by = e - vexp[k % NE];
                        al[k] *= by > 126 ? 0.f : __uint_as_float((127 - by) << 23);
                    };
                    if (masked) {
                        const uint32_t rows = __ballot_sync(0xffffffffu, !isfinite(vs[0]));
                        if (rows) spoil(rows);
                        if (!isfinite(vs[0])) vs[0] = 0.f;
                        float f[2];  // of this lane's two keys
#pragma unroll
                        for (int u = 0; u < 2; ++u) f[u] = __shfl_sync(0xffffffffu, vs[0], u * 8 + (lane >> 2));
#pragma unroll
                        for (int k = 0; k < 2 * NT; ++k) {
                            uint32_t top = 0;
#pragma unroll
                            for (int u = 0; u < 2; ++u) top = max(top, S[0][k / 2][0][2 * u + (k & 1)] != 0.f ? __float_as_uint(fabsf(f[u])) : 0u);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                            const uint32_t e = min(max(top >> 23, vexp[k % NE]), 253u);
                            lower(k, e);
                            vexp[k % NE] = e;
                            const float down = __uint_as_float((254 - e) << 23);
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                float& w = S[0][k / 2][0][2 * u + (k & 1)];
                                w = w != 0.f ? w * (f[u] * down) : 0.f;  // (a scale without a weight may be past the range)
                            }
                        }
                    } else {
                        // (of a tree, columns differ only behind the first tile with drafted tokens, which are the row's last)
                        uint32_t e = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(vs[0]))) >> 23;
                        e = min(max(e, vexp[0]), 253u);
                        if (e != vexp[0]) {
#pragma unroll
                            for (int k = 0; k < 2 * NT; ++k) lower(k, e);
#pragma unroll
                            for (int k = 0; k < NE; ++k) vexp[k] = e;
                        }
                        const float scaled = vs[0] * __uint_as_float((254 - e) << 23);
#pragma unroll
                        for (int x = 0; x < MT; ++x)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const float f = __shfl_sync(0xffffffffu, scaled, x * 16 + u * 8 + (lane >> 2));
#pragma unroll
                                for (int y = 0; y < NT; ++y) S[x][y][0][2 * u] *= f, S[x][y][0][2 * u + 1] *= f;
                            }
                    }
                }
                uint32_t pf[C::sp()][MT][NT][2];
#pragma unroll
                for (int x = 0; x < MT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int t = 0; t < C::sp(); ++t) {
                            pf[t][x][y][0] = movm(take_pair<CT>(S[x][y][0][0], S[x][y][0][1]));
                            pf[t][x][y][1] = movm(take_pair<CT>(S[x][y][0][2], S[x][y][0][3]));
                        }
                wait(2 * stage + 1, i);
                arrived();
                if (masked) {
                    const uint32_t rows = unclean(drafted0 - tile0);
                    if (rows) spoil(rows);
                }
                constexpr int DS = C::Q8 ? 2 : 1;  // steps of 16 dims that a load has (of 8-bit codes 32 dims)
#pragma unroll
                for (int d = 0; d < C::KD; d += DS) {
                    float sum[DS][NT][4];
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        uint32_t af[DS][4];
                        if constexpr (C::Q8) {
                            // rows of the product: dims 2 r and, in the upper half, 2 r + 1
                            uint32_t cf[4];
                            ldsm4t(cf, ((kt + vat) ^ ((d & 6) * 16)) + (d >> 3) * (TK * 128) + x * 2048);
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                widen<TC, true>(cf[u], af[u][0], af[u][1]);
                                widen<TC, true>(cf[2 + u], af[u][2], af[u][3]);
                            }
                        } else {
                            ldsm4t(af[0], ((kt + vat) ^ ((d & 3) * 32)) + (d >> 2) * (TK * 128) + x * 2048);
                        }
#pragma unroll
                        for (int u = 0; u < DS; ++u)
#pragma unroll
                            for (int y = 0; y < NT; ++y)
#pragma unroll
                                for (int t = 0; t < C::sp(); ++t)
                                    if (x == 0 && t == 0)
                                        mma16816_0<CT>(sum[u][y], af[u], pf[t][x][y][0], pf[t][x][y][1]);
                                    else
                                        mma16816<CT>(sum[u][y], af[u], pf[t][x][y][0], pf[t][x][y][1]);
                    }
#pragma unroll
                    for (int u = 0; u < DS; ++u)
#pragma unroll
                        for (int y = 0; y < NT; ++y)
#pragma unroll
                            for (int z = 0; z < 4; z += 2) {
                                const float2 r = fma2(make_float2(O[d + u][y][z], O[d + u][y][z + 1]), make_float2(al[2 * y], al[2 * y + 1]),
                                                      make_float2(sum[u][y][z], sum[u][y][z + 1]));
                                O[d + u][y][z] = r.x, O[d + u][y][z + 1] = r.y;
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
                    v = key >= klo && key < khi && (!masked || sees<C>(p, w, w.hb * HB + h, tile0 + key - drafted0)) ? v * (p.scale * LOG2E) : -INFINITY;
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
                if (masked) {
                    const uint32_t rows = unclean(drafted0 - tile0);
#pragma unroll
                    for (int h = 0; h < HB; ++h)
                        if (part == 0 && rows >> key & 1 && key >= klo && key < khi && sees<C>(p, w, w.hb * HB + h, tile0 + key - drafted0)) l[h] = NAN;
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
            if (ST || i + STAGES < n)
                issue(i + STAGES, std::true_type{}, steady);
            else if (C::Q8)
                vs[0] = vs[1];
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
                const int h0 = w.hb * HB, nh = min(HB, (C::TREE ? w.queries : p.group) - h0);
                auto up = [&](int k) { return C::Q8 ? C::UNSHIFT * __uint_as_float(vexp[k % NE] << 23) : C::UNSHIFT; };  // of column k
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
                    if (lane == 0)
                        pieces[ps] = Piece{first, w.nt, w.row, w.kvh * (C::TREE ? w.blocks : p.blocks_per_kv) + w.hb,
                                           C::TREE ? w.blocks : 0, C::TREE ? w.queries : 0, C::TREE ? w.token : 0, dst};
                    __syncwarp();
                }
                if constexpr (!C::F32) {
                    // a lane has dims lane / 4 + {0, 8, 16, ...} (of an 8-bit cache 2 (lane / 4) + {0, 1, 16, 17, ...})
                    // of heads 2 (lane % 4) + {0, 1}; the addresses
                    // are one base per head and constants, as this code runs too rarely to stay in the
                    // instruction cache (a flush took 5 us with an address computed per element)
                    const int d0 = C::row_dim(lane >> 2, 0);
                    constexpr int DU = C::row_dim(0, 1);
                    auto off = [](int d) { return (d >> 1) * 16 + (d & 1) * DU; };
#pragma unroll
                    for (int y = 0; y < NT; ++y)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int h = y * 8 + (lane & 3) * 2 + c, k = 2 * y + c;
                            if (h >= nh) continue;
                            if (!whole) {
                                float* at = dst + h * C::HS + d0;  // dims past the head's own are 0, and not read
#pragma unroll
                                for (int d = 0; d < 2 * C::KD; ++d) at[off(d)] = O[d / 2][y][2 * (d & 1) + c] * up(k);
                                if (lane < 4) pm[ps][h] = m[k], pl[ps][h] = l[k];
                                continue;
                            }
                            const float f = inverse(l[k]) * up(k);
                            int to, head;
                            query_at<C>(p, w.row, w.token, w.kvh, h0 + h, to, head);
                            if (p.out) {
                                TI* at = static_cast<TI*>(p.out) + to * p.o_ts + head * p.o_hs + d0;
#pragma unroll
                                for (int d = 0; d < 2 * C::KD; ++d)
                                    if (d * 8 < p.dim) at[off(d)] = from_f<TI>(O[d / 2][y][2 * (d & 1) + c] * f);
                            }
                            if (std::is_same<TI, float>::value && p.hl.hi) {
                                const long long o = (long long)to * p.hl.ld + head * p.dim + d0;
#pragma unroll
                                for (int d = 0; d < 2 * C::KD; ++d)
                                    if (d * 8 < p.dim) {
                                        const float v = O[d / 2][y][2 * (d & 1) + c] * f;
                                        const __half hi = __float2half_rn(v);
                                        p.hl.hi[o + off(d)] = hi;
                                        p.hl.lo[o + off(d)] = __float2half_rn(v - __half2float(hi));
                                    }
                            }
                            if (p.lse && lane < 4) p.lse[(long long)to * p.n_heads + head] = log_sum(m[k], l[k]);
                        }
                } else {
#pragma unroll
                    for (int h = 0; h < HB; ++h)
                        if (h < nh) {
                            const float f = whole ? inverse(l[h]) : 1.f;
                            int to, head;
                            query_at<C>(p, w.row, w.token, w.kvh, h0 + h, to, head);
#pragma unroll
                            for (int y = 0; y < (HD + 127) / 128; ++y) {
                                const int at = (HD == 64 ? lane & 15 : lane + 32 * y) * 4;
                                float v[4];
#pragma unroll
                                for (int z = 0; z < 4; ++z) v[z] = O[h][y][z] * f;
                                if (at < p.dim && !(HD == 64 && lane > 15)) {
                                    if (whole)
                                        write4<TI>(p, to, head, at, v);
                                    else
                                        *reinterpret_cast<float4*>(dst + h * C::HS + at) = make_float4(v[0], v[1], v[2], v[3]);
                                }
                            }
                            if (lane == 0) {
                                if (!whole)
                                    pm[ps][h] = m[h], pl[ps][h] = l[h];
                                else if (p.lse)
                                    p.lse[(long long)to * p.n_heads + head] = log_sum(m[h], l[h]);
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
    const long long ca = pad ? s_range[0] : per * blockIdx.x, cb = pad ? s_range[C::PAD ? 1 : 0] : end_place;
    // lane i has piece i; pieces of one (row, head block) are neighbours and form a chain
    const bool there = lane < 2 * nw && pieces[lane].nt > 0;
    const long long of = there ? pieces[lane].first : -1 - lane;
    const unsigned mates = __match_any_sync(0xffffffffu, of);
    const unsigned heads = __ballot_sync(0xffffffffu, there && __ffs(mates) - 1 == lane);
    const int chains = __popc(heads);
    const int rank = heads >> lane & 1 ? __popc(heads & ((1u << lane) - 1)) : -1;  // which chain this lane heads
    int tail_row = -1, tail_vh = 0, tail_blocks = 0;
    long long tail_last = 0;
    if (warp == 0 && chains) {
        const Piece P = pieces[31 - __clz(heads)];  // only the last chain may go on behind the block
        if (P.first >= ca && P.first + P.nt > cb)
            tail_row = P.row, tail_vh = P.vh, tail_blocks = P.blocks, tail_last = quotient(end_place - cb + P.first + P.nt - 1, per);
    }
    for (int u = warp; u < chains * hv; u += nw) {
        const int ch = u / hv, h = u - ch * hv;
        const int i0 = __ffs(__ballot_sync(0xffffffffu, rank == ch)) - 1;  // the chain's first piece
        const Piece P = pieces[i0];
        unsigned members = __shfl_sync(0xffffffffu, mates, i0);
        const int blocks = C::TREE ? P.blocks : p.blocks_per_kv;
        const int kvh = P.vh / blocks, h0 = (P.vh - kvh * blocks) * HB;
        if (h0 + h >= (C::TREE ? P.queries : p.group)) continue;
        int to, head;
        query_at<C>(p, P.row, P.token, kvh, h0 + h, to, head);
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
                write4<TI>(p, to, head, d, r[y]);
            else
                *reinterpret_cast<float4*>(p.block_part + ci * HD + d) = make_float4(r[y][0], r[y][1], r[y][2], r[y][3]);
        }
        if (lane == 0) {
            if (!whole)
                p.block_ml[ci] = make_float2(M, Ls);
            else if (p.lse)
                p.lse[(long long)to * p.n_heads + head] = log_sum(M, Ls);
        }
    }
    if (tid == 0) p.meta[blockIdx.x] = make_int4(tail_row, tail_vh, (int)tail_last, tail_blocks);

    // ---- rows without a cached token (a tree's row with queries has some) ----
    for (int r = blockIdx.x; !C::TREE && r < p.n_rows; r += gridDim.x) {
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
template <class C>
__global__ void __launch_bounds__(128) k_paged_attn_join(const __grid_constant__ PagedAttn p) {
    using TI = typename C::TI;
    constexpr int HD = C::HD, HB = C::HB;
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
    const int blocks = C::TREE ? meta.w : p.blocks_per_kv;
    const int kvh = meta.y / blocks, h0 = (meta.y - kvh * blocks) * HB;
    int token = 0, queries = p.group;
    if constexpr (C::TREE) {
        tokens_of(p, meta.x, token, queries);
        queries *= p.group;
    }
    if (h0 + h >= queries) return;
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
    int to, head;
    query_at<C>(p, meta.x, token, kvh, h0 + h, to, head);
    if (g == 0 && d < p.dim) {
#pragma unroll
        for (int k = 1; k < PG; ++k) {
            const float4 v = part[tid + k * DG];
            r.x += v.x, r.y += v.y, r.z += v.z, r.w += v.w;
        }
        const float f = inverse(L);
        const float o[4] = {r.x * f, r.y * f, r.z * f, r.w * f};
        write4<TI>(p, to, head, d, o);
    }
    if (tid == 0 && p.lse) p.lse[(long long)to * p.n_heads + head] = log_sum(M, L);
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

// A pool as a tensor [page][head][piece][slot][dim]; dims past the head's own are read as zero.
template <class C>
bool make_map(CUtensorMap* m, const PagedAttn& p, const void* base) {
    const auto encode = tensor_map_encoder();
    if (!encode) return false;
    using TC = typename C::TC;
    const auto type = C::Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : C::F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
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
        e = cudaFuncSetAttribute(k_paged_attn<C, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM_LIMIT);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    return launch_dependent(k_paged_attn<C, TMA>, dim3(grid), dim3(nw * 32), smem, st, p, km, vm);
}

template <class C>
cudaError_t launch(PagedAttn p, cudaStream_t st) {
    p.blocks_per_kv = (p.group + C::HB - 1) / C::HB;
    p.n_vh = p.n_kv * p.blocks_per_kv;
    p.heads_per_block = C::TREE ? C::HB : std::min(p.group, C::HB);
    size_t wb = STAGES * C::STAGE + (size_t)C::QS * p.heads_per_block * C::HD * sizeof(typename C::TI);
    if (C::F32) wb += (size_t)C::TK * C::HB * 4;
    p.warp_bytes = (int)((wb + 1023) / 1024 * 1024);
    const int nw = (int)std::min<size_t>(C::WARPS, C::SMEM_LIMIT / p.warp_bytes);
    // no more blocks than the longest rows the table can hold would fill
    const long long longest = p.window > 0 ? std::min(p.window, p.cap) : p.cap;
    const long long tiles = ((longest + C::TK - 1) / C::TK + (p.window > 0 ? 1 : 0)) * p.n_vh;
    // (of a tree: every row's last block of queries may be incomplete)
    const long long rows = C::TREE ? std::min<long long>(p.n_rows, p.n_tokens) + (long long)p.n_tokens * p.group / C::HB : p.n_rows;
    const long long want = tiles > MAX_CTAS * 8LL ? MAX_CTAS : (tiles * rows + nw - 1) / nw;
    const int grid = (int)std::clamp<long long>(want, 1, MAX_CTAS);
    if (C::TREE) p.most = ((long long)p.n_tokens * p.group / C::HB + p.n_rows) * p.n_kv * (((long long)p.cap + C::TK - 1) / C::TK + C::PAD);
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
    return launch_dependent(k_paged_attn_join<C>, dim3(grid, p.heads_per_block), dim3(128), 0, st, p);
}

// Queries of a block: 8 columns of a tensor core product, or 16 where there are more and the registers allow it (of an fp32
// cache as few as there are, at most 8).
template <class TC, class TI, int HD, bool TREE>
cudaError_t by_heads(const PagedAttn& p, cudaStream_t st) {
    const long long queries = TREE ? ((long long)p.n_tokens * p.group + p.n_rows - 1) / p.n_rows : p.group;  // a kv head has per row
    if constexpr (std::is_same<TC, float>::value) {
        if (queries == 1) return launch<Cfg<TC, TI, HD, 1, TREE>>(p, st);
        if (queries == 2) return launch<Cfg<TC, TI, HD, 2, TREE>>(p, st);
        if (queries <= 4) return launch<Cfg<TC, TI, HD, 4, TREE>>(p, st);
        return launch<Cfg<TC, TI, HD, 8, TREE>>(p, st);
    } else {
        if constexpr (!std::is_same<TI, float>::value && HD <= 128)
            if (queries > 8) return launch<Cfg<TC, TI, HD, 16, TREE>>(p, st);
        return launch<Cfg<TC, TI, HD, 8, TREE>>(p, st);
    }
}

template <class TC, class TI, bool TREE>
cudaError_t by_dim(const PagedAttn& p, cudaStream_t st) {
    if (p.dim <= 64) return by_heads<TC, TI, 64, TREE>(p, st);
    if (p.dim <= 128) return by_heads<TC, TI, 128, TREE>(p, st);
    return by_heads<TC, TI, 256, TREE>(p, st);
}

}  // namespace
}  // namespace gpt2q
