// Paged key/value cache (gpt2q_paged_*): checks and the C-ABI; gpt2q.h states the layout.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <string>

#include "device_op.cuh"
#include "gpt2q.h"
#include "paged.h"

namespace gpt2q {
void set_global_error(const std::string& msg);  // runtime.cu
}

using namespace gpt2q;

namespace {

bool aligned16(const void* p, int64_t a, int64_t b, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a * size % 16 == 0 && b * size % 16 == 0;
}

// A term x * step of a sum, lo <= x <= hi, step >= 0.
struct Term {
    int64_t lo, hi, step;
};
// Of addresses up to 2^58: what lies beyond is no memory, and sums of six stay in 64 bits.
inline int64_t reach(int64_t n, int64_t step) { return step >> 27 ? std::min<int64_t>(n - 1, ((int64_t)1 << 58) / step) : n - 1; }

// n[0] x n[1] x n[2] runs of `bytes` bytes: run (i, j, k) begins at at + i * step[0] + j * step[1] + k * step[2].
struct Runs {
    const void* at;
    int64_t n[3], step[3], bytes;
    int64_t from, to;  // the bytes between, as addresses
    Runs() = default;
    Runs(const void* at_, int64_t n0, int64_t n1, int64_t n2, int64_t s0, int64_t s1, int64_t s2, int64_t bytes_)
        : at(at_), n{n0, n1, n2}, step{s0, s1, s2}, bytes(bytes_) {
        from = static_cast<int64_t>(reinterpret_cast<uintptr_t>(at)), to = from + bytes;
        for (int i = 0; i < 3; ++i) {
            const int64_t most = reach(n[i], std::abs(step[i])) * step[i];
            (most < 0 ? from : to) += most;
        }
    }
    bool none() const { return !at || n[0] < 1 || n[1] < 1 || n[2] < 1; }
};

// Whether a sum of terms, ordered by falling steps, lies in [low, high]. Steps that are larger than all that follows them, as
// those of nearly all tensors are, leave one or two values of each x to look at.
bool hits(const Term* t, int n, int64_t low, int64_t high) {
    if (n == 0) return low <= 0 && 0 <= high;
    int64_t least = 0, most = 0;  // of the terms that follow
    for (int i = 1; i < n; ++i) least += t[i].lo * t[i].step, most += t[i].hi * t[i].step;
    if (t->step == 0) return hits(t + 1, n - 1, low, high);
    auto below = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };  // a / b rounded down
    const int64_t from = std::max(t->lo, -below(most - low, t->step)), to = std::min(t->hi, below(high - least, t->step));
    for (int64_t x = from; x <= to; ++x)
        if (hits(t + 1, n - 1, low - x * t->step, high - x * t->step)) return true;
    return false;
}
// Orders terms by falling steps, those of one step as one (whose x is their sum or difference); returns how many there are.
int by_step(Term* t, int n) {
    std::sort(t, t + n, [](const Term& a, const Term& b) { return a.step > b.step; });
    int m = 1;
    for (int i = 1; i < n; ++i)
        if (t[i].step == t[m - 1].step)
            t[m - 1].lo += t[i].lo, t[m - 1].hi += t[i].hi;
        else
            t[m++] = t[i];
    return m;
}

// Whether two runs share a byte.
bool overlap(const Runs& r) {
    if (r.none()) return false;
    // nested, as nearly all are: each step past what the smaller ones reach
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int x, int y) { return std::abs(r.step[x]) < std::abs(r.step[y]); });
    int64_t extent = r.bytes;
    bool nested = true;
    for (int i : order)
        if (r.n[i] > 1) {
            const int64_t step = std::abs(r.step[i]);
            nested = nested && step >= extent;
            extent += reach(r.n[i], step) * step;
        }
    if (nested) return false;
    for (int i = 0; i < 3; ++i) {  // two runs whose first index that differs is i, by 1 or more
        if (r.n[i] == 1) continue;
        Term t[3];
        int n = 0;
        for (int j = i; j < 3; ++j) {
            const int64_t step = std::abs(r.step[j]), most = reach(r.n[j], step);
            t[n++] = Term{j == i ? 1 : -most, most, step};
        }
        // (the later indices take either sign, so a step's sign matters for none)
        if (hits(t, by_step(t, n), 1 - r.bytes, r.bytes - 1)) return true;
    }
    return false;
}

// Whether a run of one shares a byte with a run of the other.
bool overlap(const Runs& a, const Runs& b) {
    if (a.to <= b.from || b.to <= a.from || a.none() || b.none()) return false;
    const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.at) - reinterpret_cast<uintptr_t>(a.at));
    Term t[6];
    for (int i = 0; i < 3; ++i)
        for (int k = 0; k < 2; ++k) {
            const int64_t by = k ? b.step[i] : -a.step[i], step = std::abs(by), most = reach(k ? b.n[i] : a.n[i], step);
            t[2 * i + k] = by < 0 ? Term{-most, 0, step} : Term{0, most, step};
        }
    return hits(t, by_step(t, 6), 1 - b.bytes - off, a.bytes - 1 - off);
}

Runs runs(const gpt2q_heads* h, int64_t tokens, int64_t heads, int64_t dim, int size) {
    return Runs(h->data, tokens, heads, 1, h->token_stride * size, h->head_stride * size, 0, dim * size);
}

int refuse(std::string* why, const char* msg) {
    *why = msg;
    return GPT2Q_EARG;
}
int launched(cudaError_t e, std::string* why) {
    if (e == cudaSuccess) return GPT2Q_OK;
    *why = cudaGetErrorString(e);
    return GPT2Q_ECUDA;
}

const gpt2q_paged_kv8* scaled(const gpt2q_paged_kv* kv) { return reinterpret_cast<const gpt2q_paged_kv8*>(kv); }

// The cache's part of a call's parameters.
template <class P>
void take_cache(P* p, const gpt2q_paged_kv* kv) {
    p->kc = kv->k, p->vc = kv->v;
    p->c_ps = kv->page_stride, p->c_hs = kv->head_stride, p->c_ts = kv->token_stride;
    p->page = kv->page_size, p->n_pages = kv->n_pages, p->n_kv = kv->n_kv_heads, p->dim = kv->head_dim;
}
template <class P>
void take_scales(P* p, const gpt2q_paged_kv* kv) {
    if (!is_8bit(kv->dtype)) return;
    const gpt2q_paged_kv8* s = scaled(kv);
    p->k_scale = s->k_scale, p->v_scale = s->v_scale;
    p->s_ps = s->scale_page_stride, p->s_hs = s->scale_head_stride, p->s_ts = s->scale_token_stride;
}

// What a cache lies in: keys, values and, of 8 bits, their scales; `n` of them.
struct Parts {
    Runs part[4];
    int n;
};
Parts parts(const gpt2q_paged_kv* kv) {
    const int size = size_of(kv->dtype);
    Parts p;
    p.n = 0;
    auto add = [&](const void* at, int64_t ps, int64_t hs, int64_t ts, int64_t bytes) {
        p.part[p.n++] = Runs(at, kv->n_pages, kv->n_kv_heads, kv->page_size, ps, hs, ts, bytes);
    };
    for (const void* at : {kv->k, kv->v}) add(at, kv->page_stride * size, kv->head_stride * size, kv->token_stride * size, (int64_t)kv->head_dim * size);
    if (is_8bit(kv->dtype)) {
        const gpt2q_paged_kv8* s = scaled(kv);
        for (const void* at : {s->k_scale, s->v_scale}) add(at, s->scale_page_stride * 4, s->scale_head_stride * 4, s->scale_token_stride * 4, 4);
    }
    return p;
}
// Whether entries of a cache that is written, or their scales, share memory. `one`: keys and values may be the same pool.
bool entries_overlap(const Parts& p, bool one) {
    for (int i = 0; i < p.n; ++i) {
        if (i % 2 == 0 && overlap(p.part[i])) return true;  // (values as keys, which have the same strides)
        for (int j = 0; j < i; ++j)
            if (!(one && i == j + 1 && i % 2 && p.part[i].at == p.part[j].at) && overlap(p.part[j], p.part[i])) return true;
    }
    return false;
}
bool in_cache(const Parts& p, const Runs& r) {
    for (int i = 0; i < p.n; ++i)
        if (overlap(p.part[i], r)) return true;
    return false;
}

}  // namespace

int gpt2q::check_paged_cache(const gpt2q_paged_kv* kv, const gpt2q_page_table* t, int dtype, std::string* why) {
    if (!kv || !kv->k || !kv->v) return refuse(why, "null cache");
    const bool eight = is_8bit(kv->dtype);
    if (!eight && (kv->dtype < GPT2Q_F32 || kv->dtype > GPT2Q_BF16)) return refuse(why, "unknown cache dtype");
    if (!eight && dtype != kv->dtype && dtype != GPT2Q_F32) return refuse(why, "dtype must be the cache's or GPT2Q_F32");
    if (eight && (dtype < GPT2Q_F32 || dtype > GPT2Q_BF16))
        return refuse(why, "dtype must be GPT2Q_F32, GPT2Q_F16 or GPT2Q_BF16");
    if (kv->n_pages < 1 || kv->page_size < 1 || kv->n_kv_heads < 1) return refuse(why, "n_pages, page_size and n_kv_heads must be >= 1");
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8)
        return refuse(why, "head_dim must be a multiple of 8 in [8, 256]");
    if (eight && kv->head_dim % 16) return refuse(why, "head_dim of an 8-bit cache must be a multiple of 16");
    if (kv->page_stride < 0 || kv->head_stride < 0 || kv->token_stride < 0) return refuse(why, "negative cache stride");
    const int sz = size_of(kv->dtype);
    if (std::max({kv->page_stride, kv->head_stride, kv->token_stride}) > (int64_t)UINT32_MAX * 16 / sz)
        return refuse(why, "cache stride past 64 GB");
    if (!aligned16(kv->k, kv->page_stride, kv->head_stride, sz) || !aligned16(kv->v, kv->token_stride, 0, sz))
        return refuse(why, "the cache's addresses and strides must be multiples of 16 bytes");
    if (eight) {
        if (kv->reserved != GPT2Q_SCALED) return refuse(why, "an 8-bit cache is a gpt2q_paged_kv8, reserved GPT2Q_SCALED");
        const gpt2q_paged_kv8* s = scaled(kv);
        if (!s->k_scale || !s->v_scale) return refuse(why, "null scales");
        if (reinterpret_cast<uintptr_t>(s->k_scale) % 4 || reinterpret_cast<uintptr_t>(s->v_scale) % 4)
            return refuse(why, "unaligned scales");
        for (int64_t x : {s->scale_page_stride, s->scale_head_stride, s->scale_token_stride})
            if (x < 0 || x > (int64_t)UINT32_MAX * 16) return refuse(why, "negative scale stride, or one past 64 G elements");
    }
    if (!t || (!t->ids && t->n_rows > 0) || t->n_rows < 0 || t->width < 1 || t->ld < t->width)
        return refuse(why, "null page table, or bad n_rows / width / ld");
    return GPT2Q_OK;
}

int gpt2q::paged_append(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                        const gpt2q_heads* v, const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype, int n_q_heads,
                        int n_tokens, const int32_t* d_pos, int pos0, const int32_t* d_slot, const int32_t* d_seq,
                        const gpt2q_rotary* rot, int32_t* d_status, cudaStream_t st, std::string* why) {
    const int rc = check_paged_cache(kv, table, dtype, why);
    if (rc) return rc;
    if (n_tokens < 0) return refuse(why, "n_tokens < 0");
    if (n_tokens == 0) return GPT2Q_OK;
    if (!k || !k->data || !v || !v->data) return refuse(why, "null k or v");
    if ((q && q->data) != (q_out && q_out->data)) return refuse(why, "q and q_out come together");
    const bool with_q = q && q->data;
    if (with_q && n_q_heads < 1) return refuse(why, "n_q_heads must be >= 1");
    if (!d_pos && (d_seq || d_slot || table->n_rows < 1 || pos0 < 0)) return refuse(why, "null d_pos");
    if (d_pos && !d_seq && n_tokens > table->n_rows) return refuse(why, "more tokens than table rows, and no d_seq");
    if (rot && (rot->dim < 2 || rot->dim % 2 || rot->dim > kv->head_dim))
        return refuse(why, "the rotary dim must be even and at most head_dim");
    const int sz = size_of(dtype);
    AppendParams p{};
    p.k = k->data, p.k_ts = k->token_stride, p.k_hs = k->head_stride;
    p.v = v->data, p.v_ts = v->token_stride, p.v_hs = v->head_stride;
    bool vec = kv->head_dim % 16 == 0 && (!rot || rot->dim % 16 == 0) && aligned16(p.k, p.k_ts, p.k_hs, sz) &&
               aligned16(p.v, p.v_ts, p.v_hs, sz);
    if (with_q) {
        p.q = q->data, p.q_ts = q->token_stride, p.q_hs = q->head_stride;
        p.qo = q_out->data, p.qo_ts = q_out->token_stride, p.qo_hs = q_out->head_stride;
        p.n_q = n_q_heads;
        vec = vec && aligned16(p.q, p.q_ts, p.q_hs, sz) && aligned16(p.qo, p.qo_ts, p.qo_hs, sz);
    }
    take_cache(&p, kv);
    take_scales(&p, kv);
    p.n_tokens = n_tokens;
    p.pos = d_pos, p.pos0 = pos0, p.slot = d_slot, p.seq = d_seq, p.table = table->ids, p.n_rows = table->n_rows, p.width = table->width;
    p.ld = table->ld, p.status = d_status;
    if (rot) {
        p.rot = rot->dim, p.interleaved = rot->interleaved != 0;
        for (int i = 0; i < rot->dim / 2; ++i) p.turns[i] = rot->turns[i];
    }
    if ((long long)p.n_q + 2LL * p.n_kv > INT32_MAX / 2) return refuse(why, "too many heads");
    const Parts cache = parts(kv);
    if (with_q) {
        const Runs o = runs(q_out, n_tokens, n_q_heads, p.dim, sz);
        if (overlap(o)) return refuse(why, "the queries of q_out overlap");
        const bool same = p.qo == p.q && (n_tokens == 1 || p.qo_ts == p.q_ts) && (n_q_heads == 1 || p.qo_hs == p.q_hs);
        if ((!same && overlap(o, runs(q, n_tokens, n_q_heads, p.dim, sz))) || overlap(o, runs(k, n_tokens, p.n_kv, p.dim, sz)) ||
            overlap(o, runs(v, n_tokens, p.n_kv, p.dim, sz)))
            return refuse(why, "q_out overlaps k or v, or q in another order");
        if (in_cache(cache, o)) return refuse(why, "q_out overlaps the cache");
    }
    // (a pool that holds keys and values at once is written twice with the same bytes)
    const bool one = p.k == p.v && p.k_ts == p.v_ts && p.k_hs == p.v_hs && !rot;
    if (entries_overlap(cache, one)) return refuse(why, "the cache's entries overlap");
    const cudaError_t e = launch_append(p, kv->dtype, dtype, vec, st);
    if (e == cudaErrorInvalidConfiguration) return refuse(why, "too many tokens in one call");
    return launched(e, why);
}

int gpt2q::paged_commit(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens, const int32_t* d_accept,
                        int width, int64_t ld, int32_t* d_new_lens, int32_t* d_status, cudaStream_t st, std::string* why) {
    const int rc = check_paged_cache(kv, table, GPT2Q_F32, why);
    if (rc) return rc;
    if (width < 0 || ld < width) return refuse(why, "width < 0 or ld < width");
    if (table->n_rows == 0) return GPT2Q_OK;
    if (!d_lens || !d_new_lens || (width > 0 && !d_accept)) return refuse(why, "null d_lens, d_accept or d_new_lens");
    if (d_new_lens < d_lens + table->n_rows && d_lens < d_new_lens + table->n_rows)
        return refuse(why, "d_new_lens must not be d_lens");
    if (entries_overlap(parts(kv), false)) return refuse(why, "the cache's entries overlap");
    const Runs list(d_accept, table->n_rows, 1, 1, ld * 4, 0, 0, (int64_t)width * 4), lengths(d_new_lens, 1, 1, 1, 0, 0, 0, (int64_t)table->n_rows * 4);
    if (width > 0 && overlap(list, lengths)) return refuse(why, "d_new_lens overlaps d_accept");
    EntryParams p{};
    take_cache(&p, kv);
    take_scales(&p, kv);
    p.table = table->ids, p.n_rows = table->n_rows, p.width = table->width, p.ld = table->ld, p.status = d_status;
    p.lens = d_lens, p.accept = d_accept, p.n_accept = width, p.accept_ld = ld, p.new_lens = d_new_lens;
    return launched(launch_commit(p, kv->dtype, st), why);
}

int gpt2q::paged_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                           const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads, float scale,
                           int window, float* d_lse, int32_t* d_status, void* d_work, const HiLo& hl, cudaStream_t st,
                           std::string* why, const Tree* tree) {
    const int rc = check_paged_cache(kv, table, dtype, why);
    if (rc) return rc;
    if (tree && tree->n_tokens < 0) return refuse(why, "n_tokens < 0");
    if (table->n_rows == 0 || (tree && tree->n_tokens == 0)) return GPT2Q_OK;
    if (tree) {
        if (!tree->d_first) return refuse(why, "null d_first");
        if (tree->d_mask && tree->mask_words < 1) return refuse(why, "mask_words must be >= 1");
        if (n_heads > 0 && (long long)tree->n_tokens * n_heads > INT32_MAX / 2) return refuse(why, "too many tokens in one call");
    }
    if (!d_lens || !q || !q->data || !out || (!out->data && !hl.hi)) return refuse(why, "null d_lens, q or out");
    if (n_heads < 1 || n_heads % kv->n_kv_heads) return refuse(why, "n_heads must be a multiple of n_kv_heads");
    if (!std::isfinite(scale)) return refuse(why, "scale must be finite");
    if (window < 0) return refuse(why, "window < 0");
    if (!d_work || reinterpret_cast<uintptr_t>(d_work) % 16) return refuse(why, "null or unaligned d_work");
    const int sz = size_of(dtype);
    if (!aligned16(q->data, q->token_stride, q->head_stride, sz) ||
        !aligned16(out->data, out->token_stride, out->head_stride, sz))
        return refuse(why, "addresses and strides of q and out must be multiples of 16 bytes");
    if (out->data && overlap(runs(out, tree ? tree->n_tokens : table->n_rows, n_heads, kv->head_dim, sz)))
        return refuse(why, "the results in out overlap");
    PagedAttn p{};
    p.k = kv->k, p.v = kv->v;
    const int csz = size_of(kv->dtype);
    p.ps16 = (uint32_t)(kv->page_stride * csz / 16), p.hs16 = (uint32_t)(kv->head_stride * csz / 16);
    p.ts16 = (uint32_t)(kv->token_stride * csz / 16);
    p.page = kv->page_size, p.n_pages = kv->n_pages;
    p.q = q->data, p.q_ts = q->token_stride, p.q_hs = q->head_stride;
    p.out = out->data, p.o_ts = out->token_stride, p.o_hs = out->head_stride, p.hl = hl, p.lse = d_lse;
    p.table = table->ids, p.lens = d_lens, p.ld = table->ld, p.n_rows = table->n_rows;
    // (positions of a tile, and of a warp's 32 boxes of up to 128 keys, past a row's last stay below 2^31)
    p.cap = (int)std::min<long long>((long long)table->width * kv->page_size, INT32_MAX - (tree ? 32 * 128 : 64));
    p.n_heads = n_heads, p.n_kv = kv->n_kv_heads, p.group = n_heads / kv->n_kv_heads, p.dim = kv->head_dim;
    p.window = window, p.scale = scale, p.status = d_status;
    take_scales(&p, kv);
    if (tree) p.first = tree->d_first, p.mask = tree->d_mask, p.mask_words = tree->mask_words, p.n_tokens = tree->n_tokens;
    return launched(launch_paged_attn(p, kv->dtype, dtype, d_work, st), why);
}

// =================================================================== C-ABI
extern "C" int gpt2q_rotary_init(gpt2q_rotary* rot, int dim, int interleaved, double base) {
    if (!rot || dim < 2 || dim % 2 || dim > 256 || !(base > 0.0) || !std::isfinite(base)) {
        set_global_error("gpt2q_rotary_init: null rot, dim not even in [2, 256], or base not positive");
        return GPT2Q_EARG;
    }
    rot->dim = dim;
    rot->interleaved = interleaved != 0;
    for (int i = 0; i < 128; ++i)
        rot->turns[i] = i < dim / 2 ? std::pow(base, -2.0 * i / dim) / (2.0 * 3.14159265358979323846) : 0.0;
    return GPT2Q_OK;
}

extern "C" int gpt2q_paged_append(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                                  const gpt2q_heads* v, const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype,
                                  int n_q_heads, int n_tokens, const int32_t* d_pos, const int32_t* d_seq,
                                  const gpt2q_rotary* rot, int32_t* d_status, void* stream) {
    std::string why;
    int rc;
    if (!d_pos && n_tokens > 0)
        rc = refuse(&why, "null d_pos");
    else
        rc = paged_append(kv, table, k, v, q, q_out, dtype, n_q_heads, n_tokens, d_pos, 0, nullptr, d_seq, rot, d_status,
                          static_cast<cudaStream_t>(stream), &why);
    if (rc) set_global_error("gpt2q_paged_append: " + why);
    return rc;
}

extern "C" int gpt2q_paged_append_at(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                                     const gpt2q_heads* v, const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype,
                                     int n_q_heads, int n_tokens, const int32_t* d_pos, const int32_t* d_slot,
                                     const int32_t* d_seq, const gpt2q_rotary* rot, int32_t* d_status, void* stream) {
    std::string why;
    int rc;
    if (!d_pos && n_tokens > 0)
        rc = refuse(&why, "null d_pos");
    else
        rc = paged_append(kv, table, k, v, q, q_out, dtype, n_q_heads, n_tokens, d_pos, 0, d_slot, d_seq, rot, d_status,
                          static_cast<cudaStream_t>(stream), &why);
    if (rc) set_global_error("gpt2q_paged_append_at: " + why);
    return rc;
}

extern "C" int gpt2q_paged_read(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                                const gpt2q_heads* v, int dtype, int n_tokens, const int32_t* d_pos, const int32_t* d_seq,
                                int32_t* d_status, void* stream) {
    std::string why;
    auto call = [&]() -> int {
        const int rc = check_paged_cache(kv, table, dtype, &why);
        if (rc) return rc;
        if (n_tokens < 0) return refuse(&why, "n_tokens < 0");
        if (n_tokens == 0) return GPT2Q_OK;
        if (!k || !k->data || !v || !v->data) return refuse(&why, "null k or v");
        if (!d_pos) return refuse(&why, "null d_pos");
        if (!d_seq && n_tokens > table->n_rows) return refuse(&why, "more tokens than table rows, and no d_seq");
        const int sz = size_of(dtype);
        if (reinterpret_cast<uintptr_t>(k->data) % sz || reinterpret_cast<uintptr_t>(v->data) % sz)
            return refuse(&why, "unaligned k or v");
        const Runs ko = runs(k, n_tokens, kv->n_kv_heads, kv->head_dim, sz), vo = runs(v, n_tokens, kv->n_kv_heads, kv->head_dim, sz);
        if (overlap(ko) || overlap(vo)) return refuse(&why, "the entries of k or v overlap");
        if (overlap(ko, vo)) return refuse(&why, "k and v overlap");
        const Parts cache = parts(kv);
        if (in_cache(cache, ko) || in_cache(cache, vo)) return refuse(&why, "k or v overlaps the cache");
        EntryParams p{};
        take_cache(&p, kv);
        take_scales(&p, kv);
        p.table = table->ids, p.n_rows = table->n_rows, p.width = table->width, p.ld = table->ld, p.status = d_status;
        p.k = k->data, p.k_ts = k->token_stride, p.k_hs = k->head_stride;
        p.v = v->data, p.v_ts = v->token_stride, p.v_hs = v->head_stride;
        p.n_tokens = n_tokens, p.pos = d_pos, p.seq = d_seq;
        const bool vec = aligned16(p.k, p.k_ts, p.k_hs, sz) && aligned16(p.v, p.v_ts, p.v_hs, sz);
        const cudaError_t e = launch_read(p, kv->dtype, dtype, vec, static_cast<cudaStream_t>(stream));
        if (e == cudaErrorInvalidConfiguration) return refuse(&why, "too many tokens in one call");
        return launched(e, &why);
    };
    const int rc = call();
    if (rc) set_global_error("gpt2q_paged_read: " + why);
    return rc;
}

extern "C" int gpt2q_paged_commit(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                                  const int32_t* d_accept, int width, int64_t ld, int32_t* d_new_lens, int32_t* d_status,
                                  void* stream) {
    std::string why;
    const int rc = paged_commit(kv, table, d_lens, d_accept, width, ld, d_new_lens, d_status, static_cast<cudaStream_t>(stream), &why);
    if (rc) set_global_error("gpt2q_paged_commit: " + why);
    return rc;
}

extern "C" uint64_t gpt2q_paged_attention_workspace(const gpt2q_paged_kv* kv, int n_heads) {
    if (!kv || n_heads < 1 || kv->n_kv_heads < 1 || kv->head_dim < 8 || kv->head_dim > 256) return 0;
    return paged_attn_workspace(kv->head_dim, (n_heads + kv->n_kv_heads - 1) / kv->n_kv_heads);
}

extern "C" int gpt2q_paged_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                                     const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads, float scale,
                                     int window, float* d_lse, int32_t* d_status, void* d_work, void* stream) {
    std::string why;
    const int rc = paged_attention(kv, table, d_lens, q, out, dtype, n_heads, scale, window, d_lse, d_status, d_work,
                                   HiLo{}, static_cast<cudaStream_t>(stream), &why);
    if (rc) set_global_error("gpt2q_paged_attention: " + why);
    return rc;
}

extern "C" uint64_t gpt2q_paged_tree_attention_workspace(const gpt2q_paged_kv* kv, int n_heads, int n_tokens) {
    if (!kv || n_heads < 1 || n_tokens < 0 || kv->n_kv_heads < 1 || kv->head_dim < 8 || kv->head_dim > 256) return 0;
    return std::max(paged_attn_workspace(kv->head_dim, 16), paged_tree_tc_workspace(kv->head_dim));
}

extern "C" int gpt2q_paged_tree_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                                          const int32_t* d_first, const int32_t* d_mask, int mask_words,
                                          const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads,
                                          int n_tokens, float scale, float* d_lse, int32_t* d_status, void* d_work,
                                          void* stream) {
    std::string why;
    const Tree tree{d_first, d_mask, mask_words, n_tokens};
    const int rc = paged_attention(kv, table, d_lens, q, out, dtype, n_heads, scale, 0, d_lse, d_status, d_work, HiLo{},
                                   static_cast<cudaStream_t>(stream), &why, &tree);
    if (rc) set_global_error("gpt2q_paged_tree_attention: " + why);
    return rc;
}
