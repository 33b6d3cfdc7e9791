// Attention of drafted tokens over a paged cache on tcgen05 tiles: for 16-bit queries of which a kv head has many per row.
//
//   out[t][h] = sum_j softmax_j(scale q[t][h] . K[j]) V[j], j over the prefix and what t's mask names
//
// A kv head's queries of one row (tokens times its query heads) are the rows of the products, 128 to a tile, so that what is
// read of the cache is used 128 times. The work is one flat list of tiles of 128 keys, ordered by row, kv head, block of 256
// queries and position; each block takes a range of equal length, whatever the rows' lengths are, and a second kernel joins
// what lies in several ranges. Results do not depend on the order in which blocks run.
//
// A block has two warps that start the TMA copies, one that issues the MMAs, four that prepare operands, and two streams of
// eight softmax warps, two threads per query (TMEM lane), so that one stream's exponentials run beside the other's MMAs:
//   S = Q K^T       M = 128 queries, N = 128 keys; Q and K from shared memory
//   P = 2^(S - m)   in 16 bits over half of S's own TMEM columns
//   O += P V        M = 128, N = head dim, K = 128 keys; P from TMEM, V from shared memory, O in TMEM
// With more than 128 queries each stream has its own and both use every tile of keys; with fewer both have the same
// queries, take tiles in turn, and are joined at the end. O is rescaled only when the maximum has risen by more than
// 2^8 (weights stay below that, and the sum has the same reference).
//
// 8-bit caches: the preparing warps write the codes as fp16, in which they are exact; keys' scales multiply the scores and
// values' scales the weights, both in fp32. The values' scales are held relative to the largest exponent so far of those that a query
// sees, so that weight times scale stays in fp16's range: in tiles of the prefix alone it is the same for all queries and the preparing
// warps have it, in those with drafted tokens each query finds its own. bf16 queries are scaled per row by a power of two that brings the largest
// element to [2^10, 2^11), and are exact in fp16 down to 2^-24 of it.
//
// A weight is rounded to 16 bits, once (by up to 2^-8 of itself in bf16, 2^-11 in fp16), as the output is. The sum of the weights is
// that of the rounded ones, so that a single key gives its value. Of 8-bit caches it is the product with the scale that is
// rounded: its sums before and after give a factor that returns what the rounding took on the whole (equal scales were off by
// the same 2^-12 in every key, and so was the result; 7 % of the time of wide drafts over int8, 341 to 366 us). Weights in two pieces of 16
// bits, as the warp-level kernel has them, would leave the output's own rounding (error against 64 bits on the cases below 1.7e-3 and
// not 1.9e-3 to 2.0e-3), at 114, 435 and 504 us for the three. fp32 queries and outputs, other pages and heads over 128 dims take the kernel in paged_attn.cuh.
//
// Measured (one B200): 31 drafts of 5 to 60 tokens behind 100 to 8000, 32 heads on 8 of 128 in bf16, 106 us, of 38 that the cache
// takes to read; 3 drafts of 64 tokens behind 20 to 40 thousand in int8, 64 heads on 8, 368 us (492 TFLOP/s); 2 chunks of 1100 to 2047
// tokens behind 4 to 6 thousand, 32 heads on 8 in bf16, 423 us (662 TFLOP/s). The bound of the last two is a stream's chain: read the scores, exponentials,
// weights to TMEM, product. Measured and not kept: an MMA warp per stream (the streams fall into step: chunks 489 us, of 472 then), slots
// freed by a warp of their own (607), registers moved to the softmax warps, each holding its 128 scores at once (spills).
#include <cuda.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "device_op.cuh"
#include "gpt2q.h"
#include "paged.h"

namespace gpt2q {
namespace {

constexpr int QT = 128, KT = 128;  // queries and keys of a tile
constexpr int SB = 2 * QT;         // queries of a block of queries
constexpr int CTAS = 148;          // one per SM of a B200
// Warps 0-7 and 8-15 are the two streams (the halves of the keys, four warps each), 16-19 prepare operands.
constexpr int WARPS = 23, THREADS = WARPS * 32;
constexpr int W_PREP = 16, W_MMA = 20, W_TMA = 21;  // 21 and 22: copies of keys and of values
constexpr int TILES = 4;           // of which scales and masks are kept: a tile's are read before its weights are handed on, and
                                   // its slots are written again only after that
constexpr int FLAGS = 8;           // of which page flags are kept: the copies may be four tiles ahead
constexpr int WAIT_TRIES = 1 << 26;  // of a wait that has no end in WAIT_NS either (a try takes from 20 ns to microseconds)
constexpr unsigned long long WAIT_NS = 1000000000ull;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// Places in the list: a tile of a block of at most 128 queries has one, of a block of more has two, and what a segment costs
// beside its tiles (queries, first copies, results) has EXTRA, before them. Fitted over the blocks of a call with 31 short drafts: a
// tile 2.0 us, a tile of two streams 4.1, a segment 9.0. With a place for every tile alone the blocks of many short rows took
// three times as long as the others (218 us in all, with EXTRA = 4 130).
constexpr int EXTRA = 5;
constexpr float STALE = 8.f;  // log2 of the largest weight
// Tiles of a stream whose products are summed in TMEM, before the sums go to memory and are added up there, rounded to nearest (a power of
// two). The tensor cores round a running sum towards zero, by 2^-24 of it on average for each 16 keys: a block with 131072 keys of a row
// left values of one sign 4.8e-4 too small, which is as much as an fp16 output's rounding; now 4e-5 (256 tiles 1.6e-4). 128 KB to and
// from L2 each time. Calls that cannot have more than UNFLUSHED tiles of a stream and segment in a block do without.
constexpr int FLUSH = 128, UNFLUSHED = 192;

template <class TC_, class TI_, int HD_>
struct Cfg {
    using TC = TC_;
    using TI = TI_;
    static constexpr int HD = HD_;
    static constexpr bool Q8 = sizeof(TC) == 1;
    using CT = std::conditional_t<Q8, __half, TC>;
    static constexpr bool HALF = std::is_same<CT, __half>::value;
    static constexpr bool RANGE = HALF && !std::is_same<TI, __half>::value;
    static constexpr int PIECES = HD / 64;               // of 128 bytes, of a 16-bit row
    static constexpr int PIECE = KT * 128;               // bytes of a tile's piece
    static constexpr int TILE = PIECES * PIECE;          // 16-bit tile of 128 rows
    static constexpr int SLOTS = HD == 128 && Q8 ? 3 : 4;  // 16-bit tiles of keys or values
    static constexpr int RAWS = Q8 ? (HD == 128 ? 3 : 4) : 0;              // 8-bit tiles, rows of 128 bytes
    static constexpr int OFF_KV = 2 * TILE, OFF_RAW = OFF_KV + SLOTS * TILE, SMEM = OFF_RAW + RAWS * PIECE + 1024;
    static constexpr int LOADS = Q8 ? RAWS : SLOTS;      // slots that copies go to
    static constexpr int BOXES = Q8 ? 1 : PIECES;        // of 128 bytes, that a row is copied in
    // fp16 weights are held times 2^6: 2^(8 + 6) and a scale below 2 stay in range, and small ones stay normal numbers
    static constexpr float shift() { return HALF ? 6.f : 0.f; }
};

struct Args {
    PagedAttn p;
    int box;           // keys of a TMA box
    int stall;         // for the test of waits that run out
    float4* part;      // [block][2][dims / 4][SB]
    float2* part_ml;   // [block][2][SB]
    int4* meta;        // per block: row (-1: none), kv head, block of queries, last block of its last segment
};

// ------------------------------------------------------------------ the list of tiles
struct Row {
    int row, prefix, n, token, queries, end, blocks;
    bool over;
};
struct Seg {
    Row r;
    int kvh, sb, j0, j1, nt;  // tiles j0 .. j1 - 1 of its nt
    int behind;               // places that the block has behind them
    __device__ __forceinline__ int queries() const { return min(SB, r.queries - sb * SB); }
    __device__ __forceinline__ bool pair() const { return queries() > QT; }
};

__device__ __forceinline__ Row enter(const PagedAttn& p, int row) {
    Row r{row, 0, 0, 0, 0, 0, 0, false};
    if (row >= p.n_rows) return r;
    const int a = __ldcg(p.first + row), b = __ldcg(p.first + row + 1);
    r.token = min(max(a, 0), p.n_tokens);
    r.n = max(min(b, p.n_tokens) - r.token, 0);
    if (r.n == 0) return r;
    r.prefix = max(__ldcg(p.lens + row), 0);
    r.over = (long long)r.prefix + r.n > p.cap;  // cap + 32 * KT stays below 2^31
    r.end = r.over ? p.cap : r.prefix + r.n;
    r.queries = r.n * p.group;
    r.blocks = (r.queries + SB - 1) / SB;
    return r;
}
// Tiles of blocks of queries 0 .. sb - 1 of a kv head. Under a mask every block has those of all keys. A chain's block ends with its
// last query's own key: blocks but the last have ceil((prefix + ceil(256 (x + 1) / group)) / 128) =
// floor((2 x + c) / group) tiles, whose sum goes by whole periods of `group` blocks. (A call has fewer than 2^31 places.)
__device__ __forceinline__ int tiles_of(const PagedAttn& p, const Row& r, int sb) {
    int end = r.end;
    if (!p.mask && !r.over && sb < r.blocks - 1) end = r.prefix + ((sb + 1) * SB - 1) / p.group + 1;
    return (end + KT - 1) / KT;
}
// Places of blocks 0 .. sb - 1: all but the last have more than 128 queries.
__device__ __forceinline__ int places_before(const PagedAttn& p, const Row& r, int sb) {
    const unsigned x = max(min(sb, r.blocks - 1), 0);
    unsigned sum;
    if (p.mask || r.over) {
        sum = x * tiles_of(p, r, 0);
    } else {
        const unsigned G = p.group;
        const unsigned c = (unsigned)(((unsigned long long)r.prefix * G + 2 * KT + (unsigned long long)KT * G - 1) / KT);
        const unsigned q = x / G, rest = x - q * G;
        sum = G * q * (q - 1) + 2 * q * rest;
        for (unsigned i = 0; i < (q ? G : rest); ++i) sum += (2 * i + c) / G * (q + (i < rest ? 1 : 0));
    }
    sum = 2 * sum + sb * EXTRA;
    if (sb == r.blocks && sb > 0) sum += tiles_of(p, r, sb - 1) * (r.queries - (sb - 1) * SB > QT ? 2 : 1);
    return (int)sum;
}

// Takes the places `from` .. of the block at hand that `left` covers, which it takes them from; false if they have no tile.
__device__ __forceinline__ bool cut(const PagedAttn& p, Seg& s, int from, int& left) {
    s.nt = tiles_of(p, s.r, s.sb);
    const int two = s.pair() ? 1 : 0, all = (s.nt << two) + EXTRA, to = min(all, from + left);
    left -= to - from;
    s.j0 = max(from - EXTRA, 0) >> two;
    s.j1 = max(to - EXTRA, 0) >> two;
    s.behind = all - to;
    return s.j1 > s.j0;
}
// The next segment, taken from `left`; false at the end.
__device__ __forceinline__ bool next(const PagedAttn& p, Seg& s, int& left) {
    while (left > 0) {
        if (++s.sb >= s.r.blocks) {
            s.sb = 0;
            if (++s.kvh >= p.n_kv) {
                s.kvh = 0;
                do {
                    if (s.r.row + 1 >= p.n_rows) return false;
                    s.r = enter(p, s.r.row + 1);
                } while (s.r.n == 0);
            }
        }
        if (cut(p, s, 0, left)) return true;
    }
    return false;
}
// The segment that lies `rem` places into row `row`, or behind it. By a whole warp.
__device__ __forceinline__ bool seek(const PagedAttn& p, Seg& s, int row, int rem, int& left) {
    if (left <= 0) return false;
    Row r = enter(p, row);
    int per = places_before(p, r, r.blocks);
    while (rem >= per * p.n_kv) {
        rem -= per * p.n_kv;
        if (++row >= p.n_rows) return false;
        r = enter(p, row);
        per = places_before(p, r, r.blocks);
    }
    s.r = r;
    s.kvh = (unsigned)rem / (unsigned)per;
    rem -= s.kvh * per;
    int lo = 0;
    for (int n = r.blocks; n > 1;) {  // the last block that begins at or before it, 32 candidates at once
        const int step = (n + 31) / 32, x = lo + (threadIdx.x & 31) * step;
        const int k = __popc(__ballot_sync(0xffffffffu, x < lo + n && places_before(p, r, x) <= rem)) - 1;
        n = min(step, n - k * step);
        lo += k * step;
    }
    s.sb = lo;
    return cut(p, s, rem - places_before(p, r, lo), left) || next(p, s, left);
}

// ------------------------------------------------------------------ PTX
// One lane of a warp; code behind it keeps its operands in uniform registers, which behind a comparison of the lane it does not
// (a product then took 100 cycles to issue).
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// D[tmem] (+)= A[smem desc] * B[smem desc]^T, and A[tmem] * B[smem desc]^T, kind::f16
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a_desc),
                 "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a),
                 "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}
// 32 columns of this thread's lane, which may be used after tmem_wait32 of the same registers
__device__ __forceinline__ void tmem_ask32(uint32_t at, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait32(float* v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void streams_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
__device__ __forceinline__ void half_sync(int stream) {
    if (stream)
        asm volatile("bar.sync 4, 256;" ::: "memory");
    else
        asm volatile("bar.sync 3, 256;" ::: "memory");
}

template <class CT>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    if constexpr (std::is_same<CT, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}
template <class CT>
__device__ __forceinline__ float2 unpack(uint32_t v) {
    if constexpr (std::is_same<CT, __half>::value)
        return __half22float2(*reinterpret_cast<const __half2*>(&v));
    else
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
// a += the two fp16 numbers of v
__device__ __forceinline__ void add_halves(float2& a, uint32_t v) {
    asm("{\n\t.reg .f16 x, y;\n\tmov.b32 {x, y}, %2;\n\tadd.rn.f32.f16 %0, x, %0;\n\tadd.rn.f32.f16 %1, y, %1;\n\t}" : "+f"(a.x), "+f"(a.y) : "r"(v));
}
// four neighbouring codes as two pairs of fp16
template <class TC>
__device__ __forceinline__ void widen(uint32_t v, uint32_t& a, uint32_t& b) {
    if constexpr (std::is_same<TC, int8_t>::value) {
        v ^= 0x80808080u;  // 0x6400 + u is the fp16 number 1024 + u; u = code + 128
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t x = __byte_perm(v, 0x64646464u, 0x4140), y = __byte_perm(v, 0x64646464u, 0x4342);
        const __half2 hx = __hsub2(*reinterpret_cast<const __half2*>(&x), off), hy = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
        a = *reinterpret_cast<const uint32_t*>(&hx);
        b = *reinterpret_cast<const uint32_t*>(&hy);
    } else {
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(a), "=r"(b)
            : "r"(v));
    }
}
// byte offset of 16-byte chunk c of row r in a tile of 16-bit rows: pieces of 128 bytes, chunks permuted by the row
__device__ __forceinline__ uint32_t sw(int r, int c) { return (uint32_t)((c >> 3) * (KT * 128) + r * 128 + (((c ^ r) & 7) << 4)); }

__device__ __forceinline__ uint32_t ones(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; }
// Which of keys key0 .. key0 + 31 the row's token t sees.
__device__ __forceinline__ uint32_t visible(const PagedAttn& p, const Row& r, int t, int key0) {
    if (!p.mask) return ones(r.prefix + t + 1 - key0);
    const int j = key0 - r.prefix;  // drafted token of the first key
    const int* words = p.mask + (long long)(r.token + t) * p.mask_words;
    const int w = j >> 5, sh = j & 31;
    uint32_t v = 0;
    if (w >= 0 && w < p.mask_words) v = (uint32_t)__ldcg(words + w) >> sh;
    if (sh && w + 1 >= 0 && w + 1 < p.mask_words) v |= (uint32_t)__ldcg(words + w + 1) << (32 - sh);
    return (v | ones(-j)) & ones(r.end - key0);
}

__device__ __forceinline__ unsigned long long globaltimer() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Adds `n` times 16 columns of this lane's sums in TMEM to keep times those in memory (SB float4 apart), if any are there; the result goes to memory, or
// with `back` to TMEM. Apart from the loop over tiles, which it would cost registers.
__device__ __noinline__ void carry(float4* mem, uint32_t at, int n, bool there, float keep, bool back) {
#pragma unroll 1
    for (int c = 0; c < n; ++c, at += 16) {
        uint32_t w[16];
        tmem_ld16(at, w);
#pragma unroll
        for (int k = 0; k < 4; ++k, mem += SB) {
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (there) o = *mem;
            o = make_float4(fmaf(o.x, keep, __uint_as_float(w[4 * k])), fmaf(o.y, keep, __uint_as_float(w[4 * k + 1])),
                            fmaf(o.z, keep, __uint_as_float(w[4 * k + 2])), fmaf(o.w, keep, __uint_as_float(w[4 * k + 3])));
            if (!back) *mem = o;
            w[4 * k] = __float_as_uint(o.x), w[4 * k + 1] = __float_as_uint(o.y), w[4 * k + 2] = __float_as_uint(o.z), w[4 * k + 3] = __float_as_uint(o.w);
        }
        if (back) tmem_st16(at, w);
    }
    tmem_wait_st();
}

// LONG: a stream may have more than UNFLUSHED tiles of a segment. A kernel of its own, as the code for it costs the others 2 to 4 %
// (31 short drafts 106 to 110 us, chunks 423 to 433), though it is behind one comparison.
template <class C, bool LONG>
__global__ void __launch_bounds__(THREADS, 1)
    k_paged_tree_tc(const __grid_constant__ Args a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using TC = typename C::TC;
    using TI = typename C::TI;
    using CT = typename C::CT;
    constexpr int HD = C::HD;
    constexpr bool Q8 = C::Q8;
    const PagedAttn& p = a.p;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ int cum[THREADS];
    __shared__ long long sums[WARPS];
    __shared__ uint32_t s_top[4];  // of the preparing warps
    __shared__ __align__(8) uint64_t b_load[8], b_free[8];   // copies have landed in a slot; its tile is no longer needed
    __shared__ __align__(8) uint64_t b_wide[8], b_reuse[8];  // 8-bit: a tile is there in fp16; its slot may be written again
    __shared__ __align__(8) uint64_t b_prep[TILES];          // 16-bit: a tile of values with drafted tokens is looked through
    __shared__ __align__(8) uint64_t b_q, b_s[2], b_p[2], b_o[2];
    __shared__ uint32_t tmem_slot;
    // of keys, of values (relative to 2^s_exp; as they are in tiles with drafted tokens)
    __shared__ __align__(16) float s_scale[Q8 ? TILES : 1][2][KT];
    __shared__ unsigned char s_seen[Q8 ? 2 : 1][2][Q8 ? QT : 1];  // of the streams' halves: the largest exponent of the scales that a query sees
    __shared__ uint32_t s_exp[TILES];
    __shared__ uint32_t s_spoilt[TILES][4];           // drafted tokens' values that are not finite
    __shared__ int s_bad[FLAGS];                      // a page id is out of range
    __shared__ float s_up[SB];                        // what a row's queries were scaled by, undone
    __shared__ float s_mx[2][2][QT], s_l[2][2][QT], s_m[2][QT];  // of the streams' halves: a tile's largest scores, the sums; references
    __shared__ uint32_t s_vexp[2][QT];
    __shared__ int s_stuck;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < 8; ++i) {
            tc::mbar_init(&b_load[i], 1);
            // 8-bit copies are used by the preparing warps, as are, else, those of values (odd slots): they wait for every load
            // of such a slot, as a parity cannot tell a phase from the one two before it
            tc::mbar_init(&b_free[i], Q8 ? 4 : i & 1 ? 5 : 1);
            tc::mbar_init(&b_wide[i], 4);
            tc::mbar_init(&b_reuse[i], 1);
        }
        for (int i = 0; i < TILES; ++i) tc::mbar_init(&b_prep[i], 4);
        tc::mbar_init(&b_q, 1);
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&b_s[i], 2);
            tc::mbar_init(&b_p[i], 8);
            tc::mbar_init(&b_o[i], 1);
        }
        s_stuck = 0;
        tc::fence_mbar_init();
    }
    if (warp == W_MMA) {
        tc::tmem_alloc(&tmem_slot, 512);
        tc::tmem_relinquish();
    }
    if (warp == W_TMA && lane == 0) {
        tc::prefetch_tmap(&kmap);
        tc::prefetch_tmap(&vmap);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = tmem_slot;
    tc::pdl_trigger();  // after the TMEM allocation: dependents hold no columns that this block waits for
    tc::pdl_wait();

    // ---- this block's range of tiles ----
    const int nc = (p.n_rows + THREADS - 1) / THREADS;  // rows a thread counts
    long long mine = 0;
    for (int r = tid * nc; r < min((tid + 1) * nc, p.n_rows); ++r) {
        const Row w = enter(p, r);
        mine += (long long)places_before(p, w, w.blocks) * p.n_kv;
    }
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    long long before = 0, all = 0;
    for (int i = 0; i < WARPS; ++i) {
        if (i < warp) before += sums[i];
        all += sums[i];
    }
    if (all > p.most) {  // a `first` that names tokens again and again: no work rather than any amount of it
        all = 0;
        if (tid == 0 && blockIdx.x == 0 && p.status) atomicOr(p.status, GPT2Q_STATUS_POSITION);
    }
    const int total = (int)all;
    cum[tid] = (int)(before + inc - mine);
    __syncthreads();
    const int per = max((total - 1) / (int)gridDim.x + 1, 2);  // a block inside a segment has a tile of it
    const int t_a = (int)min((long long)per * blockIdx.x, (long long)total), t_b = (int)min((long long)t_a + per, (long long)total);
    int row0 = 0, rem0 = 0;
    if (t_a < t_b) {
        int lo = 0;
        for (int n = THREADS; n > 1;) {  // the last thread whose rows begin at or before it
            const int step = (n + 31) / 32, x = lo + lane * step;
            const int k = __popc(__ballot_sync(0xffffffffu, x < lo + n && cum[x] <= t_a)) - 1;
            n = min(step, n - k * step);
            lo += k * step;
        }
        row0 = lo * nc;
        rem0 = t_a - cum[lo];
    }

    // Each thread gives up by itself and then waits for nothing more; whoever does says so to all, and results from then on are
    // NaN. The copying warps start nothing after that: a barrier that still expects bytes must not be armed again.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!ok || tc::mbar_try_wait(bar, parity)) return;
        unsigned long long began = 0;
        for (int i = 1; i < WAIT_TRIES; ++i) {
            if (tc::mbar_try_wait(bar, parity)) return;
            if (i % 256) continue;
            const unsigned long long now = globaltimer();
            if (!began) began = now;
            if (now - began > WAIT_NS) break;
        }
        ok = false;
        atomicExch(&s_stuck, 1);
    };

    Seg s;
    int left = t_b - t_a;
    int g = 0;  // tiles of this block before the segment
    if (warp < W_PREP) {
        // ------------------------------------------------------------------ softmax: two threads per query
        const int st = warp >> 3, half = warp >> 2 & 1, quarter = warp & 3, r = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t t_s = lanes + st * KT + half * (KT / 2);  // this thread's keys
        const float sl2 = fmaxf(fabsf(p.scale) * LOG2E, 1e-37f);
        uint32_t ns = 0, no = 0, specials = 0;
        if (tid == 0) a.meta[blockIdx.x] = make_int4(-1, 0, 0, 0);
        bool more = seek(p, s, row0, rem0, left);
        while (more) {
            const bool pair = s.pair();
            const int T = s.j1 - s.j0, nu = pair ? T : st ? T / 2 : (T + 1) / 2;
            const int special = max(s.r.prefix / KT, s.j0);
            const int qi = s.sb * SB + (pair ? st * QT : 0) + r;  // this thread's query of the kv head
            const bool mine_q = qi < s.r.queries;
            const int tok = (int)((unsigned)qi / (unsigned)p.group), to = s.r.token + tok, head = s.kvh * p.group + qi - tok * p.group;
            // ---- queries: neighbouring threads have neighbouring dims; the streams share one tile's ----
            {
                unsigned char* dst = smem + (pair ? st : 0) * C::TILE;
                constexpr int CPR = HD / 8;  // of 16 bytes, of a row
#pragma unroll 2
                for (int x = pair ? tid & 255 : tid; x < QT * CPR; x += pair ? 256 : 512) {
                    const int row = x / CPR, c = x % CPR, i = s.sb * SB + (pair ? st * QT : 0) + row;
                    const int tk = (int)((unsigned)i / (unsigned)p.group), hd = s.kvh * p.group + i - tk * p.group;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (i < s.r.queries && c * 8 < p.dim)
                        v = __ldcg(reinterpret_cast<const uint4*>(static_cast<const char*>(p.q) + ((s.r.token + tk) * p.q_ts + hd * p.q_hs) * 2) + c);
                    uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    float up = 1.f;
                    if constexpr (C::RANGE) {
                        uint32_t top = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, w[k] >> 16 & 0x7fffu));
#pragma unroll
                        for (int o = 1; o < CPR; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        int e = (int)(top >> 7);  // biased exponent
                        e = e == 0 || e == 255 ? 127 : min(max(e, 12), 252);
                        const float down = __uint_as_float((uint32_t)(264 - e) << 23);
                        up = __uint_as_float((uint32_t)(e - 10) << 23);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float2 f = unpack<TI>(w[k]);
                            w[k] = pack<CT>(f.x * down, f.y * down);
                        }
                    }
                    if (p.scale < 0.f) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] ^= 0x80008000u;
                    }
                    *reinterpret_cast<uint4*>(dst + sw(row, c)) = make_uint4(w[0], w[1], w[2], w[3]);
                    if (c == 0) s_up[(pair ? st * QT : 0) + row] = up;
                }
                tc::fence_proxy_async_smem();
            }
            tc::tc_fence_before();
            streams_sync();
            if (tid == 0) tc::mbar_arrive(&b_q);
            const float fac = fmaxf(sl2 * s_up[(pair ? st * QT : 0) + r], 1.17549435e-38f);  // not 0: a masked score of -inf stays one
            float m = -INFINITY, l = s.r.over ? NAN : 0.f;  // reference of the weights, in units before the factor; this half's sum
            uint32_t vexp = 1;
            // 8-bit: sums of weights times scales, before and after their rounding
            [[maybe_unused]] float exact = 0.f, rounded = 0.f;
            const bool idle = s.sb * SB + (pair ? st * QT : 0) + quarter * 32 >= s.r.queries;  // no query in this warp
            int bad = s.r.over ? GPT2Q_STATUS_POSITION : 0;
            for (int u = 0; u < nu; ++u) {
                const int t = pair ? u : 2 * u + st, j = s.j0 + t, gt = (g + t) % TILES;
                wait(&b_s[st], ns++ & 1);
                tc::tc_fence_after();
                if (s_bad[(g + t) % FLAGS]) bad |= GPT2Q_STATUS_PAGE;
                const bool look = j >= special;  // keys that not every query sees
                uint32_t vis[2] = {~0u, ~0u};
                if (look && !idle) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) vis[c] = mine_q ? visible(p, s.r, tok, j * KT + half * (KT / 2) + c * 32) : 0u;
                }
                float mx = -INFINITY;
                // Scores of a quarter of the keys, read once for the largest and once more for the weights: with 64 of them in
                // registers there would be fewer warps
                float x[32];
                auto scores = [&](int c) {
                    tmem_ask32(t_s + c * 32, x);
                    tmem_wait32(x);
                    if constexpr (Q8) {
                        const float* ks = s_scale[gt][0] + half * (KT / 2) + c * 32;
#pragma unroll
                        for (int k = 0; k < 32; k += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(ks + k);
                            const float2 y = mul2(make_float2(x[k], x[k + 1]), make_float2(f.x, f.y)), z = mul2(make_float2(x[k + 2], x[k + 3]), make_float2(f.z, f.w));
                            x[k] = y.x, x[k + 1] = y.y, x[k + 2] = z.x, x[k + 3] = z.y;
                        }
                    }
                    if (look) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) x[k] = vis[c] >> k & 1 ? x[k] : -INFINITY;
                    }
                };
                auto largest = [&](int c) {
                    scores(c);
                    float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                    for (int k = 4; k < 32; ++k) top[k & 3] = fmaxf(top[k & 3], x[k]);
                    mx = fmaxf(mx, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
                };
                __syncwarp();
                if (!idle) {
                    largest(0);
                    largest(1);
                }
                s_mx[st][half][r] = mx;
                half_sync(st);
                mx = fmaxf(mx, s_mx[st][half ^ 1][r]);
                // values' scales and what is to be known of them
                uint32_t e = vexp;
                if constexpr (Q8) {
                    const int en = 2 * (g + t) + 1;
                    wait(&b_wide[en % C::SLOTS], (en / C::SLOTS) & 1);
                    if (look) {
                        // what this query does not see must not count, however large it is
                        uint32_t top = 0;
                        if (!idle) {
                            const float* vs = s_scale[gt][1] + half * (KT / 2);
#pragma unroll 1
                            for (int c = 0; c < 2; ++c)
#pragma unroll
                                for (int k = 0; k < 32; ++k) top = max(top, vis[c] >> k & 1 ? __float_as_uint(fabsf(vs[c * 32 + k])) : 0u);
                        }
                        s_seen[st][half][r] = (unsigned char)(top >> 23);
                        half_sync(st);
                        e = min(max(max(top >> 23, (uint32_t)s_seen[st][half ^ 1][r]), vexp), 253u);
                    } else {
                        e = s_exp[gt];
                    }
                } else if (look) {
                    const uint32_t k = specials + (j - special);
                    wait(&b_prep[k % TILES], (k / TILES) & 1);
                }
                if (look) {
                    const uint32_t* sp = s_spoilt[Q8 ? gt : (specials + (j - special)) % TILES] + half * 2;
                    if ((vis[0] & sp[0]) | (vis[1] & sp[1])) l = NAN;
                }
                // a new reference, and the results so far in it
                const float mn = fmaxf(m, mx);
                const bool raise = (mn - m) * fac > STALE || (m == -INFINITY && mn > -INFINITY);
                float al = 1.f;
                if (raise) {
                    al = m == -INFINITY ? 0.f : ex2((m - mn) * fac);
                    m = mn;
                }
                l *= al;
                if constexpr (Q8) {
                    if (e != vexp) {
                        al *= e - vexp > 126 ? 0.f : __uint_as_float((127 - (e - vexp)) << 23);
                        vexp = e;
                    }
                    exact *= al, rounded *= al;
                }
                __syncwarp();
                if ((LONG ? u & (FLUSH - 1) : u) > 0 && __any_sync(0xffffffffu, al != 1.f)) {
#pragma unroll 1
                    for (int c = half * (HD / 32); c < (half + 1) * (HD / 32); ++c) {
                        uint32_t w[16];
                        const uint32_t at = lanes + 256 + st * HD + c * 16;
                        tmem_ld16(at, w);
#pragma unroll
                        for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(__uint_as_float(w[k]) * al);
                        tmem_st16(at, w);
                    }
                }
                if (!idle) {
                    const float ref = m == -INFINITY ? 0.f : m;
                    const float2 nref = make_float2(-ref, -ref), f2 = make_float2(fac, fac), sh = make_float2(C::shift(), C::shift());
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    [[maybe_unused]] float2 before = make_float2(0.f, 0.f), after = make_float2(0.f, 0.f);
                    [[maybe_unused]] const float down = __uint_as_float((254 - vexp) << 23);
                    auto weights = [&](int c, auto own) {  // own: the scales are as they are, and count where they are seen
                        scores(c);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int k = h * 16 + i * 2;
                                // (S - m) before the factor, where m's own score gives exactly 0
                                const float2 d = fma2(add2(make_float2(x[k], x[k + 1]), nref), f2, sh);
                                float2 y = make_float2(ex2(d.x), ex2(d.y));
                                if constexpr (Q8) {
                                    sum[i & 1] = add2(sum[i & 1], y);
                                    float2 f = *reinterpret_cast<const float2*>(s_scale[gt][1] + half * (KT / 2) + c * 32 + k);
                                    if constexpr (decltype(own)::value) {
                                        f = mul2(f, make_float2(down, down));
                                        f.x = vis[c] >> k & 1 ? f.x : 0.f, f.y = vis[c] >> (k + 1) & 1 ? f.y : 0.f;
                                    }
                                    y = mul2(y, f);
                                    w[i] = pack<CT>(y.x, y.y);
                                    before = add2(before, y);
                                    add_halves(after, w[i]);
                                } else {
                                    w[i] = pack<CT>(y.x, y.y);
                                    sum[i & 1] = add2(sum[i & 1], unpack<CT>(w[i]));  // of the weights that the product has
                                }
                            }
                            tmem_st8(t_s + 32 + c * 16 + h * 8, w);
                        }
                    };
                    // both quarters' weights take the columns of the later one
                    if (Q8 && look) {
                        weights(1, std::bool_constant<Q8>{});
                        weights(0, std::bool_constant<Q8>{});
                    } else {
                        weights(1, std::false_type{});
                        weights(0, std::false_type{});
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    if (Q8) exact += before.x + before.y, rounded += after.x + after.y;
                }
                tmem_wait_st();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&b_p[st]);
                if constexpr (!LONG) continue;
                const bool last = u + 1 == nu;
                if (nu <= FLUSH || (!last && ((u + 1) & (FLUSH - 1)))) continue;
                wait(&b_o[st], no++ & 1);
                tc::tc_fence_after();
                // sums in memory have the place of this segment's partial results, which come later; half 0 keeps their reference there
                const long long at = ((long long)blockIdx.x * 2 + (s.j0 > 0 ? 0 : 1)) * SB;
                float2* ref = a.part_ml + at + st * QT + r;
                float keep = 0.f;
                if (u >= FLUSH) {
                    const float2 of = *ref;
                    keep = of.x == -INFINITY ? 0.f : ex2((of.x - m) * fac);
                    if constexpr (Q8) {
                        const uint32_t by = vexp - __float_as_uint(of.y);
                        keep *= by > 126 ? 0.f : __uint_as_float((127 - by) << 23);
                    }
                }
                half_sync(st);  // both halves have the reference
                if (half == 0 && !last) *ref = make_float2(m, __uint_as_float(vexp));
                carry(a.part + (at * (HD / 4) + (long long)half * (HD / 8) * SB) + st * QT + r, lanes + 256 + st * HD + half * (HD / 2), HD / 32, u >= FLUSH, keep, last);
                tc::tc_fence_before();  // the next products take their place
            }
            if (LONG ? nu > 0 && nu <= FLUSH : nu > 0) wait(&b_o[st], no++ & 1);
            tc::tc_fence_after();
            if (!ok || *(volatile int*)&s_stuck) bad |= GPT2Q_STATUS_TIMEOUT;
            if (bad) l = NAN;
            if (bad && p.status && lane == 0) atomicOr(p.status, bad);
            // ---- results: a half of the dims each ----
            s_l[st][half][r] = l;
            if (Q8) s_mx[st][half][r] = __uint_as_float(pack<bf16>(exact, exact - rounded));  // (no thread reads a tile's maximum any more)
            if (half == 0) {
                s_m[st][r] = m;
                s_vexp[st][r] = vexp;
            }
            tc::tc_fence_before();
            streams_sync();
            tc::tc_fence_after();
            if (pair || st == 0) {
                const bool whole = s.j0 == 0 && s.j1 == s.nt;
                unsigned char* stage = smem + st * C::TILE;  // the queries' place: their products are done
                if (!idle) {
                    float wa = 1.f, wb = 0.f;  // weights of this stream's and the other's results
                    l = s_l[st][0][r] + s_l[st][1][r];
                    // 8-bit: what the rounding of all weights together took from the product is given back, so that equal scales, or a
                    // single key, do not leave their rounding in the result
                    auto back = [&](int x) {
                        const float2 a = unpack<bf16>(__float_as_uint(s_mx[x][0][r])), b = unpack<bf16>(__float_as_uint(s_mx[x][1][r]));
                        const float took = (a.y + b.y) / (a.x + b.x);
                        // (more than a rounding: sums of no sign, of weights below fp16's range, or none)
                        return fabsf(took) <= 0x1.04p-11f ? 1.f + took : 1.f;
                    };
                    if (Q8) wa = __uint_as_float(vexp << 23) * back(st);
                    if (!pair) {
                        const float o = s_m[1][r], M = fmaxf(m, o), ms = M == -INFINITY ? 0.f : M;
                        const float xa = ex2((m - ms) * fac);
                        wb = ex2((o - ms) * fac);
                        l = l * xa + (s_l[1][0][r] + s_l[1][1][r]) * wb;
                        m = M;
                        wa *= xa;
                        if (Q8) wb *= __uint_as_float(s_vexp[1][r] << 23) * back(1);
                    }
                    const int pr = (pair ? st * QT : 0) + r;
                    const long long part = (long long)blockIdx.x * 2 + (s.j0 > 0 ? 0 : 1);
                    const float f = whole ? inverse(l) : 1.f;
                    wa *= f, wb *= f;
                    const float mlog = m * fac;  // reference, as a power of two
#pragma unroll 1
                    for (int c = half * (HD / 32); c < (half + 1) * (HD / 32); ++c) {
                        uint32_t w[16];
                        float x[16];
                        tmem_ld16(lanes + 256 + st * HD + c * 16, w);
#pragma unroll
                        for (int k = 0; k < 16; ++k) x[k] = __uint_as_float(w[k]) * wa;
                        if (!pair && T > 1) {
                            tmem_ld16(lanes + 256 + HD + c * 16, w);
#pragma unroll
                            for (int k = 0; k < 16; ++k) x[k] = fmaf(__uint_as_float(w[k]), wb, x[k]);
                        }
                        if (whole) {
#pragma unroll
                            for (int k = 0; k < 2; ++k)
                                *reinterpret_cast<uint4*>(stage + sw(r, 2 * c + k)) =
                                    make_uint4(pack<TI>(x[8 * k], x[8 * k + 1]), pack<TI>(x[8 * k + 2], x[8 * k + 3]), pack<TI>(x[8 * k + 4], x[8 * k + 5]),
                                               pack<TI>(x[8 * k + 6], x[8 * k + 7]));
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                a.part[(part * (HD / 4) + c * 4 + k) * SB + pr] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                        }
                    }
                    if (mine_q && half == 0) {
                        if (!whole)
                            a.part_ml[part * SB + pr] = make_float2(mlog, l);
                        else if (p.lse)
                            p.lse[(long long)to * p.n_heads + head] = l == 0.f ? -INFINITY : (mlog + log2f(l) - C::shift()) * LN2;
                    }
                }
                if (whole) {  // rows to memory, neighbouring threads neighbouring dims
                    half_sync(st);
                    constexpr int CPR = HD / 8;
#pragma unroll 2
                    for (int x = tid & 255; x < QT * CPR; x += 256) {
                        const int row = x / CPR, c = x % CPR, i = s.sb * SB + (pair ? st * QT : 0) + row;
                        if (i >= s.r.queries || c * 8 >= p.dim) continue;
                        const int tk = (int)((unsigned)i / (unsigned)p.group), hd = s.kvh * p.group + i - tk * p.group;
                        *reinterpret_cast<uint4*>(static_cast<TI*>(p.out) + (s.r.token + tk) * p.o_ts + hd * p.o_hs + c * 8) =
                            *reinterpret_cast<const uint4*>(stage + sw(row, c));
                    }
                }
            }
            // a segment that goes on behind this block and begins in it (one that begins before is on an earlier block's list)
            if (tid == 0 && s.j1 < s.nt && s.j0 == 0) a.meta[blockIdx.x] = make_int4(s.r.row, s.kvh, s.sb, (t_b + s.behind - 1) / per);
            specials += max(s.j1 - special, 0);
            g += T;
            more = next(p, s, left);
            // nobody writes queries, sums or results before the others have read what they share
            tc::tc_fence_before();
            streams_sync();
            tc::tc_fence_after();
        }
    } else {
        if (warp >= W_TMA) {
    // ------------------------------------------------------------------ copies
            // Keys and values have a warp each, as their slots are separate (even and odd ones): the next keys do not wait
            // for the place of values that come before them. 8-bit copies have three slots, in turn.
            const int groups = KT / a.box, kind = warp - W_TMA;
            bool more = seek(p, s, row0, rem0, left);
            auto look = [&](const Seg& w, int j) {  // the page of the lane's group of keys in tile j; -1: no keys of the row, -2: out of range
                const int key = j * KT + lane * a.box;
                if (lane >= groups || key >= w.r.end) return -1;
                const int id = __ldcg(p.table + (long long)w.r.row * p.ld + (p.page_shift >= 0 ? key >> p.page_shift : key / p.page));
                return (unsigned)id < (unsigned)p.n_pages ? id : -2;
            };
            int page = more ? look(s, s.j0) : -1;
            while (more) {
                Seg n = s;
                const bool after = next(p, n, left);
                for (int j = s.j0; j < s.j1; ++j, ++g) {
                    const int key = j * KT + lane * a.box;
                    const int slot = p.page_shift >= 0 ? key & (p.page - 1) : key % p.page;
                    const int id = page;
                    page = j + 1 < s.j1 ? look(s, j + 1) : after ? look(n, n.j0) : -1;
                    const unsigned there = __ballot_sync(0xffffffffu, id >= 0), bad = __ballot_sync(0xffffffffu, id == -2);
                    for (int v = 0; v < 2; ++v) {
                        if (Q8 ? kind == 1 : v != kind) continue;
                        const int e = 2 * g + v, to = e % C::LOADS;
                        if (e >= C::LOADS) wait(&b_free[to], (e / C::LOADS - 1) & 1);
                        __syncwarp();
                        const bool go = __all_sync(0xffffffffu, ok && !*(volatile int*)&s_stuck);
                        if (lane == 0) {
                            if (v == 0) s_bad[g % FLAGS] = bad != 0;
                            if (go) tc::mbar_arrive_expect_tx(&b_load[to], __popc(there) * C::BOXES * a.box * 128 + a.stall);
                        }
                        __syncwarp();
                        if (!go) ok = false;
                        const uint32_t dst = tc::smem_u32(smem + (Q8 ? C::OFF_RAW : C::OFF_KV) + to * (Q8 ? C::PIECE : C::TILE)), bar = tc::smem_u32(&b_load[to]);
                        // one group after the other, by an elected lane: lanes that each started a box went one by one, at 100 cycles
#pragma unroll 4
                        for (int gr = 0; gr < groups; ++gr) {
                            const int pg = __shfl_sync(0xffffffffu, id, gr), sl = __shfl_sync(0xffffffffu, slot, gr);
                            if (go && pg >= 0 && elect()) {
#pragma unroll
                                for (int x = 0; x < C::BOXES; ++x)
                                    tma_load_4d(dst + x * C::PIECE + gr * a.box * 128, v ? &vmap : &kmap, x * (128 / (int)sizeof(TC)), sl, s.kvh, pg, bar);
                            }
                            __syncwarp();
                        }
                    }
                }
                s = n;
                more = after;
            }
            // copies that nobody waited for may still be on their way when a wait has run out: about as long again
            if (lane == 0 && *(volatile int*)&s_stuck) {
                const unsigned long long began = globaltimer();
                for (int i = max(0, 2 * g - C::LOADS); i < 2 * g; ++i)
                    for (int k = 0; k < WAIT_TRIES && globaltimer() - began < WAIT_NS && !tc::mbar_try_wait(&b_load[i % C::LOADS], (i / C::LOADS) & 1); ++k) {}
            }
        } else if (warp == W_MMA) {
            // ------------------------------------------------------------------ products
            constexpr uint32_t BF = C::HALF ? 0u : (1u << 7) | (1u << 10);  // operands' format: fp16 or bf16
            constexpr uint32_t idesc_s = tc::idesc_f16_f32(QT, KT) | BF, idesc_o = tc::idesc_f16_f32_bmn(QT, HD) | BF;
            bool more = seek(p, s, row0, rem0, left);
            if (elect()) {
                uint64_t* there = Q8 ? b_wide : b_load;
                const uint32_t q32 = tc::smem_u32(smem), kv32 = tc::smem_u32(smem + C::OFF_KV);
                uint32_t np[2] = {0, 0}, specials = 0;
                for (int seg = 0; more; ++seg) {
                    const bool pair = s.pair();
                    const int T = s.j1 - s.j0, n0 = pair ? T : (T + 1) / 2, n1 = pair ? T : T / 2;
                    // tiles from here on have values that are looked through
                    const int special = max(s.r.prefix / KT, s.j0);
                    auto tile = [&](int st, int u) { return g + (pair ? u : 2 * u + st); };
                    auto keys = [&](int st, int u) {
                        const int e = 2 * tile(st, u);
                        wait(&there[e % C::SLOTS], (e / C::SLOTS) & 1);
                    };
                    auto hand_back = [&](int st, int at) {
                        if (!pair || st == 1) tc::mma_commit(Q8 ? &b_reuse[at] : &b_free[at]);
                    };
                    auto scores = [&](int st, int u) {
                        const int at = 2 * tile(st, u) % C::SLOTS;
                        const uint64_t q = tc::desc_sw128(q32 + (pair ? st : 0) * C::TILE), k = tc::desc_sw128(kv32 + at * C::TILE);
                        if (ok) {
#pragma unroll
                            for (int ks = 0; ks < HD / 16; ++ks) {
                                const uint32_t o = ((ks >> 2) * C::PIECE + (ks & 3) * 32) >> 4;
                                mma_f16_ss(tmem + st * KT, q + o, k + o, idesc_s, ks > 0);
                            }
                        }
                        tc::mma_commit(&b_s[st]);
                        tc::mbar_arrive(&b_s[st]);  // what this thread has seen of the tile's flags
                        hand_back(st, at);
                    };
                    wait(&b_q, seg & 1);
                    keys(0, 0);
                    if (n1 > 0) keys(1, 0);
                    tc::tc_fence_after();
                    scores(0, 0);
                    if (n1 > 0) scores(1, 0);
                    // strictly in turn: where each stream's products came when its weights did, the streams got into step, each
                    // waiting while the other waited and working while it worked (1.3 times the time)
                    for (int u = 0; u < n0; ++u) {
                        for (int st = 0; st < 2; ++st) {
                            if (u >= (st ? n1 : n0)) continue;
                            const int e = 2 * tile(st, u) + 1, at = e % C::SLOTS, j = s.j0 + tile(st, u) - g;
                            // what is there already, usually: before the wait that is not over yet. (The next keys of a stream of
                            // its own tiles come into the slot of these values where there are three)
                            constexpr bool EARLY = C::SLOTS > 3;
                            const bool again = u + 1 < (st ? n1 : n0);
                            if (!pair || st == 0) {
                                wait(&there[at], (e / C::SLOTS) & 1);
                                if (!Q8 && j >= special) {
                                    const uint32_t k = specials + (j - special);
                                    wait(&b_prep[k % TILES], (k / TILES) & 1);
                                }
                                if (EARLY && again) keys(st, u + 1);
                            }
                            wait(&b_p[st], np[st]++ & 1);
                            tc::tc_fence_after();
                            const uint64_t v = tc::desc_sw128_mn(kv32 + at * C::TILE, C::PIECE);
                            if (ok) {
#pragma unroll
                                for (int ks = 0; ks < KT / 16; ++ks)
                                    mma_f16_ts(tmem + 256 + st * HD, tmem + st * KT + 32 + ks * 8 + (ks >> 2) * 32, v + ks * 128, idesc_o, (LONG ? u & (FLUSH - 1) : u) > 0 || ks > 0);
                            }
                            hand_back(st, at);
                            if (LONG && again && ((u + 1) & (FLUSH - 1)) == 0) tc::mma_commit(&b_o[st]);
                            if (again) {
                                if (!EARLY) {
                                    keys(st, u + 1);
                                    tc::tc_fence_after();
                                }
                                scores(st, u + 1);
                            } else {
                                tc::mma_commit(&b_o[st]);
                            }
                        }
                    }
                    specials += max(s.j1 - special, 0);
                    g += T;
                    more = next(p, s, left);
                }
            }
            __syncwarp();
        } else {
            // ------------------------------------------------------------------ operands
            const int i = tid - W_PREP * 32;
            bool more = seek(p, s, row0, rem0, left);
            if constexpr (Q8) {
                int e = 0;
                while (more) {
                    uint32_t vexp = 1;
                    for (int j = s.j0; j < s.j1; ++j, ++g) {
                        const int key = j * KT + i;
                        float sc[2] = {0.f, 0.f};
                        if (key < s.r.end) {
                            const int pg = p.page_shift >= 0 ? key >> p.page_shift : key / p.page;
                            const int id = __ldcg(p.table + (long long)s.r.row * p.ld + pg);
                            if ((unsigned)id < (unsigned)p.n_pages) {
                                const long long at = (long long)id * p.s_ps + (long long)s.kvh * p.s_hs + (long long)(key - pg * p.page) * p.s_ts;
                                sc[0] = __ldcg(p.k_scale + at);
                                sc[1] = __ldcg(p.v_scale + at);
                            }
                        }
                        const bool drafted = (j + 1) * KT > s.r.prefix;
                        for (int v = 0; v < 2; ++v, ++e) {
                            const int from = e % C::RAWS, to = e % C::SLOTS;
                            if (e >= C::SLOTS) wait(&b_reuse[to], (e / C::SLOTS - 1) & 1);
                            bool spoilt = false;
                            if (v == 0) {
                                s_scale[g % TILES][0][i] = sc[0];
                            } else {
                                spoilt = key >= s.r.prefix && !isfinite(sc[1]);
                                if (drafted) {
                                    const uint32_t b = __ballot_sync(0xffffffffu, spoilt);
                                    if (lane == 0) s_spoilt[g % TILES][warp - W_PREP] = b;
                                    s_scale[g % TILES][1][i] = spoilt ? 0.f : sc[1];
                                    asm volatile("bar.sync 2, 128;" ::: "memory");  // the masks are there
                                } else {
                                    // the largest exponent of the tile's scales, over the four warps
                                    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(sc[1])));
                                    if (lane == 0) s_top[warp - W_PREP] = m;
                                    asm volatile("bar.sync 2, 128;" ::: "memory");
                                    uint32_t x = vexp;
#pragma unroll
                                    for (int k = 0; k < 4; ++k) x = max(x, s_top[k] >> 23);
                                    vexp = min(x, 253u);
                                    s_scale[g % TILES][1][i] = sc[1] * __uint_as_float((254 - vexp) << 23);
                                    if (i == 0) s_exp[g % TILES] = vexp;
                                    asm volatile("bar.sync 2, 128;" ::: "memory");  // s_top is used again
                                }
                            }
                            wait(&b_load[from], (e / C::RAWS) & 1);
                            const unsigned char* src = smem + C::OFF_RAW + from * C::PIECE;
                            unsigned char* dst = smem + C::OFF_KV + to * C::TILE;
                            // 16 codes at a time. Eight lanes have four chunks of two rows that differ in bits 0 and 2, so that the
                            // reads and the writes of eight lanes each meet all banks once
#pragma unroll 4
                            for (int it = 0; it < HD / 16; ++it) {
                                const int x = it * 128 + i, c4 = x & 3, odd = x >> 2 & 1;
                                int c, r;
                                if constexpr (HD == 128) {
                                    c = (x >> 3 & 1) * 4 + c4;
                                    const int pr = x >> 4;  // pair of rows: 0..63
                                    r = (pr >> 2) * 8 + (pr & 3);
                                } else {
                                    c = c4;
                                    const int pr = x >> 3;
                                    r = (pr >> 2) * 8 + (pr & 3);
                                }
                                if (odd) r ^= 5;
                                uint4 w = *reinterpret_cast<const uint4*>(src + r * 128 + (((c ^ r) & 7) << 4));
                                if (v && drafted) {
                                    const int k = j * KT + r;
                                    bool drop = k >= s.r.end;
                                    if (!std::is_same<TC, int8_t>::value && k >= s.r.prefix && !drop) {
                                        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
                                        bool nan = false;
#pragma unroll
                                        for (int z = 0; z < 4; ++z) nan |= __vcmpeq4(u[z] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
                                        if (nan) {
                                            atomicOr(&s_spoilt[g % TILES][r >> 5], 1u << (r & 31));
                                            drop = true;
                                        }
                                    }
                                    if (drop) w = make_uint4(0, 0, 0, 0);
                                }
                                uint4 lo, hi;
                                widen<TC>(w.x, lo.x, lo.y);
                                widen<TC>(w.y, lo.z, lo.w);
                                widen<TC>(w.z, hi.x, hi.y);
                                widen<TC>(w.w, hi.z, hi.w);
                                *reinterpret_cast<uint4*>(dst + sw(r, 2 * c)) = lo;
                                *reinterpret_cast<uint4*>(dst + sw(r, 2 * c + 1)) = hi;
                            }
                            tc::fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                tc::mbar_arrive(&b_free[from]);
                                tc::mbar_arrive(&b_wide[to]);
                            }
                        }
                    }
                    more = next(p, s, left);
                }
            } else {
                static_assert(Q8 || C::SLOTS % 2 == 0, "keys in even slots, values in odd ones");
                uint32_t specials = 0;
                while (more) {
                    for (int j = s.j0; j < s.j1; ++j) {
                        const int e = 2 * (g + j - s.j0) + 1, at = e % C::SLOTS, key = j * KT + i;
                        wait(&b_load[at], (e / C::SLOTS) & 1);
                        if (j < s.r.prefix / KT) {
                            __syncwarp();
                            if (lane == 0) tc::mbar_arrive(&b_free[at]);
                            continue;
                        }
                        unsigned char* v = smem + C::OFF_KV + at * C::TILE;
                        bool spoilt = false;
                        if (key >= s.r.prefix && key < s.r.end) {
#pragma unroll
                            for (int c = 0; c < HD / 8; ++c) {
                                const uint4 w = *reinterpret_cast<const uint4*>(v + sw(i, c));
                                constexpr uint32_t E = C::HALF ? 0x7c00u : 0x7f80u;
                                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int z = 0; z < 4; ++z) spoilt |= (u[z] & E) == E || (u[z] >> 16 & E) == E;
                            }
                        }
                        if (spoilt || key >= s.r.end)
#pragma unroll
                            for (int c = 0; c < HD / 8; ++c) *reinterpret_cast<uint4*>(v + sw(i, c)) = make_uint4(0, 0, 0, 0);
                        const uint32_t b = __ballot_sync(0xffffffffu, spoilt);
                        if (lane == 0) s_spoilt[specials % TILES][warp - W_PREP] = b;
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tc::mbar_arrive(&b_prep[specials % TILES]);
                            tc::mbar_arrive(&b_free[at]);
                        }
                        ++specials;
                    }
                    g += s.j1 - s.j0;
                    more = next(p, s, left);
                }
            }
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == W_MMA) tc::tmem_dealloc(tmem, 512);
}

// Joins a segment that lies in several blocks' ranges: block c of the first kernel has its beginning (slot 1), the blocks after it
// up to `last` the rest (slot 0). A block takes 8 queries, whose four dims at a place lie side by side.
template <class TI, int HD>
__global__ void __launch_bounds__(HD * 2) k_paged_tree_join(const __grid_constant__ Args a, float shift) {
    tc::pdl_trigger();
    tc::pdl_wait();
    const PagedAttn& p = a.p;
    const int c = blockIdx.x, pr = blockIdx.y * 8 + (threadIdx.x & 7), d = threadIdx.x >> 3;  // d: of four dims
    const int4 meta = __ldcg(a.meta + c);
    if (meta.x < 0) return;
    const Row r = enter(p, meta.x);
    const int qi = meta.z * SB + pr;
    if (pr >= SB || qi >= r.queries) return;
    const int tok = (int)((unsigned)qi / (unsigned)p.group), to = r.token + tok, head = meta.y * p.group + qi - tok * p.group;
    const int n = meta.w - c + 1;
    auto at = [&](int i) { return (long long)(c + i) * 2 + (i == 0 ? 1 : 0); };
    float M = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < n; ++i) M = fmaxf(M, __ldcg(a.part_ml + at(i) * SB + pr).x);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
        const float2 ml = __ldcg(a.part_ml + at(i) * SB + pr);
        const float4 v = __ldcg(a.part + (at(i) * (HD / 4) + d) * SB + pr);
        const float w = ex2(ml.x - ms);
        L = fmaf(ml.y, w, L);
        o.x = fmaf(v.x, w, o.x), o.y = fmaf(v.y, w, o.y), o.z = fmaf(v.z, w, o.z), o.w = fmaf(v.w, w, o.w);
    }
    const float f = inverse(L);
    if (d * 4 < p.dim)
        *reinterpret_cast<uint2*>(static_cast<TI*>(p.out) + to * p.o_ts + head * p.o_hs + d * 4) =
            make_uint2(pack<TI>(o.x * f, o.y * f), pack<TI>(o.z * f, o.w * f));
    if (d == 0 && p.lse) p.lse[(long long)to * p.n_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L) - shift) * LN2;
}

// ------------------------------------------------------------------ host
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encoder() {
    static const EncodeTiledFn fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<EncodeTiledFn>(ptr)
                   : nullptr;
    }();
    return fn;
}

// A pool as a tensor [page][head][slot][dim], in boxes of 128 bytes of `box` slots; dims past the head's own are read as zero.
template <class C>
bool make_map(CUtensorMap* m, const PagedAttn& p, const void* base, int box) {
    using TC = typename C::TC;
    const auto encode = encoder();
    if (!encode) return false;
    const auto type = C::Q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : C::HALF ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint64_t dims[4] = {(cuuint64_t)p.dim, (cuuint64_t)p.page, (cuuint64_t)p.n_kv, (cuuint64_t)p.n_pages};
    // the stride of a dimension of one element does not matter, but may not be 0
    const cuuint64_t row = ((cuuint64_t)p.dim * sizeof(TC) + 15) / 16 * 16;
    const cuuint64_t strides[3] = {p.page == 1 ? row : p.ts16 * 16ull, p.n_kv == 1 ? row : p.hs16 * 16ull, p.n_pages == 1 ? row : p.ps16 * 16ull};
    const cuuint32_t b[4] = {(cuuint32_t)(128 / sizeof(TC)), (cuuint32_t)box, 1, 1}, step[4] = {1, 1, 1, 1};
    return encode(m, type, 4, const_cast<void*>(base), dims, strides, b, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class C, bool LONG>
cudaError_t launch_main(const Args& a, const CUtensorMap& km, const CUtensorMap& vm, int grid, cudaStream_t st) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<uint64_t> ready{0};  // devices whose shared-memory limit is raised
    if (dev >= 64 || !(ready.load() >> dev & 1)) {
        e = cudaFuncSetAttribute(k_paged_tree_tc<C, LONG>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return e;
        if (dev < 64) ready |= 1ull << dev;
    }
    return launch_dependent(k_paged_tree_tc<C, LONG>, dim3(grid), dim3(THREADS), C::SMEM, st, a, km, vm);
}

template <class C>
cudaError_t launch(const PagedAttn& p, void* work, cudaStream_t st, bool* taken) {
    Args a{};
    a.p = p;
    a.box = std::min(KT, p.page & -p.page);
    CUtensorMap km{}, vm{};
    if (!make_map<C>(&km, p, p.k, a.box) || !make_map<C>(&vm, p, p.v, a.box)) return cudaSuccess;
    *taken = true;
    static const bool stall = std::getenv("GPT2Q_TEST_PAGED_STALL") != nullptr;
    a.stall = stall ? 16 : 0;
    char* at = static_cast<char*>(work);
    a.part = reinterpret_cast<float4*>(at);
    at += (size_t)CTAS * 2 * SB * C::HD * 4;
    a.part_ml = reinterpret_cast<float2*>(at);
    at += (size_t)CTAS * 2 * SB * 8;
    a.meta = reinterpret_cast<int4*>(at);
    // no more blocks than the longest rows the table can hold would give a tile each
    const long long rows = std::min(p.n_rows, p.n_tokens), blocks = rows + (long long)p.n_tokens * p.group / SB;
    const long long tiles = (p.cap + (long long)KT - 1) / KT;
    const int grid = (int)std::clamp<long long>(tiles > CTAS ? CTAS : tiles * std::min<long long>(blocks, CTAS) * p.n_kv, 1, CTAS);
    // a stream's tiles of a segment: at most half of a block's places, and those of the longest row (half of them where both streams
    // have the same queries, which is not known here)
    const long long here = std::min<long long>((p.most / grid + 2) / 2, tiles);
    const cudaError_t e = here > UNFLUSHED ? launch_main<C, true>(a, km, vm, grid, st) : launch_main<C, false>(a, km, vm, grid, st);
    if (e != cudaSuccess || grid == 1) return e;
    const long long most = std::min<long long>(SB, (long long)p.n_tokens * p.group);
    return launch_dependent(k_paged_tree_join<typename C::TI, C::HD>, dim3(grid, (unsigned)((most + 7) / 8)), dim3(C::HD * 2), 0, st, a, C::shift());
}

template <class TC, class TI>
cudaError_t by_dim(const PagedAttn& p, void* work, cudaStream_t st, bool* taken) {
    return p.dim <= 64 ? launch<Cfg<TC, TI, 64>>(p, work, st, taken) : launch<Cfg<TC, TI, 128>>(p, work, st, taken);
}

}  // namespace

uint64_t paged_tree_tc_workspace(int dim) {
    return dim > 128 ? 0 : (uint64_t)CTAS * (2 * SB * ((dim <= 64 ? 64 : 128) * 4 + 8) + 16);
}

namespace {
// At most the places in the list (tiles_of and places_before) of a `first` that rises.
double most_places(const PagedAttn& p) {
    return ((double)p.n_tokens * p.group / SB + p.n_rows) * (2 * ((double)p.cap / KT + 1) + EXTRA) * p.n_kv;
}
}  // namespace

// From more than eight queries of a kv head per row on, on average, where the warp-level kernel reads the keys with a second set of
// columns or more than once. Measured (32 heads on 8 of 128, bf16; here against there), 32 rows of 1000 keys and one of 30000: with 16
// queries 71 to 74 us and 52 to 63, with 32 72 to 106 and 52 to 86, with 128 81 to 326 and 56 to 223. With 12 it is 71 and 52 here, with
// 8 44 and 37 there. All of equal rows: which rows have many is known on the device alone, so rows without a draft count too, and a row of 100
// tokens among 63 of none takes 125 us there, which alone takes 39 here.
bool paged_tree_tc_serves(const PagedAttn& p, int cache_dtype, int dtype) {
    return dtype != GPT2Q_F32 && cache_dtype != GPT2Q_F32 && p.dim <= 128 && p.page % 8 == 0 && p.out &&
           (long long)p.n_tokens * p.group > 8LL * p.n_rows && most_places(p) < 2147483648.0;
}

cudaError_t launch_paged_tree_tc(const PagedAttn& call, int cache_dtype, int dtype, void* work, cudaStream_t st, bool* taken) {
    PagedAttn p = call;
    p.most = (long long)most_places(p);
    if (cache_dtype == GPT2Q_F16) return by_dim<__half, __half>(p, work, st, taken);
    if (cache_dtype == GPT2Q_BF16) return by_dim<bf16, bf16>(p, work, st, taken);
    if (cache_dtype == GPT2Q_I8)
        return dtype == GPT2Q_F16 ? by_dim<int8_t, __half>(p, work, st, taken) : by_dim<int8_t, bf16>(p, work, st, taken);
    return dtype == GPT2Q_F16 ? by_dim<__nv_fp8_e4m3, __half>(p, work, st, taken) : by_dim<__nv_fp8_e4m3, bf16>(p, work, st, taken);
}

}  // namespace gpt2q
