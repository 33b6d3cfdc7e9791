// Paged key/value cache (gpt2q_paged_append, gpt2q_paged_attention): gpt2q.h states the layout.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <string>
#include <utility>

#include "device_op.cuh"
#include "gpt2q.h"
#include "paged.h"

namespace gpt2q {
void set_global_error(const std::string& msg);  // runtime.cu
}

using namespace gpt2q;

namespace {

// ------------------------------------------------------------------ append
struct AppendParams {
    const void *k, *v, *q;
    void* qo;
    long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, qo_ts, qo_hs;  // elements
    void *kc, *vc;
    long long c_ps, c_hs, c_ts;
    int page, n_pages, n_tokens, n_q, n_kv, dim, rot, interleaved;
    const int *pos, *seq, *table;
    int pos0, n_rows, width;
    long long ld;
    int* status;
    int unit_shift, groups;  // threads of a token: groups * 2^unit_shift
    double turns[128];
};

// A unit is two chunks of V consecutive elements of a head, chosen so that neighbouring threads' chunks
// are neighbours: the (a, b) of V rotated pairs, or chunks that are rotated within themselves
// (interleaved pairs) or only copied; a head has dim / (2 V) of them. A thread takes one unit index of one
// token and walks over the token's heads (queries, keys, values), `groups` threads sharing a unit
// index, so that the sines and cosines of its V pairs are computed once per thread. The angle is
// the fractional part of position * turns, formed in fp64 (fp32 would lose 2^-24 * position turns:
// 0.4 rad at a position of a million), then sincospif in fp32. Bound by the memory in a prompt;
// loading four heads at a time was slower (117 against 88 us at 16 thousand tokens of 48 heads), as it
// halved the threads an SM holds.
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
    if (ti >= p.n_tokens || u * 2 * V >= p.dim) return;
    const int pos = p.pos ? __ldcg(p.pos + ti) : p.pos0 + (int)ti;
    const int row = p.pos ? (p.seq ? __ldcg(p.seq + ti) : (int)ti) : 0;
    long long at = -1;  // the token's entry in a pool, before the head
    int why = 0;
    if (pos >= 0) {
        const int pg = pos / p.page;
        if (row < 0 || row >= p.n_rows) {
            why = GPT2Q_STATUS_ROW;
        } else if (pg >= p.width) {
            why = GPT2Q_STATUS_POSITION;
        } else {
            const int id_ = __ldcg(p.table + (long long)row * p.ld + pg);
            if (id_ < 0 || id_ >= p.n_pages)
                why = GPT2Q_STATUS_PAGE;
            else
                at = (long long)id_ * p.c_ps + (long long)(pos - pg * p.page) * p.c_ts;
        }
        if (why && p.status && u == 0 && g == 0) atomicOr(p.status, why);
    }
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
    for (int h = g; h < heads; h += p.groups) {
        const bool is_q = h < p.n_q, is_v = h >= p.n_q + p.n_kv;
        if (!is_q && at < 0) continue;
        const int hk = is_q ? h : is_v ? h - p.n_q - p.n_kv : h - p.n_q;
        const TI* src = is_q ? static_cast<const TI*>(p.q) + ti * p.q_ts + hk * p.q_hs
                             : is_v ? static_cast<const TI*>(p.v) + ti * p.v_ts + hk * p.v_hs
                                    : static_cast<const TI*>(p.k) + ti * p.k_ts + hk * p.k_hs;
        const int oa = is_v ? va : ca, ob = is_v ? vb : cb;
        float a[V], b[V];
        load_vec<TI, V>(src + oa, a);
        load_vec<TI, V>(src + ob, b);
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
        } else {
            TC* dst = static_cast<TC*>(is_v ? p.vc : p.kc) + at + hk * p.c_hs;
            store_vec<TC, V>(dst + oa, a);
            store_vec<TC, V>(dst + ob, b);
        }
    }
}

template <class TI, class TC>
cudaError_t launch_append(const AppendParams& p, bool vec, unsigned blocks, cudaStream_t st) {
    return vec ? launch_dependent(k_paged_append<TI, TC, 8>, dim3(blocks), dim3(256), 0, st, p)
               : launch_dependent(k_paged_append<TI, TC, 1>, dim3(blocks), dim3(256), 0, st, p);
}

// ------------------------------------------------------------------ checks
int size_of(int dtype) { return dtype == GPT2Q_F32 ? 4 : 2; }

bool aligned16(const void* p, int64_t a, int64_t b, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && a * size % 16 == 0 && b * size % 16 == 0;
}

// Whether two of n x m runs of dim elements, starting at i * a + j * b, share an element.
bool overlap(int64_t n, int64_t a, int64_t m, int64_t b, int64_t dim) {
    if (n < 1 || m < 1) return false;
    a = std::abs(a), b = std::abs(b);
    if (a > b) std::swap(a, b), std::swap(n, m);
    if ((n > 1 && a < dim) || (m > 1 && b < dim)) return true;
    if (n == 1 || m == 1 || b >= a * (n - 1) + dim) return false;
    for (int64_t j = 1; j < m && j * b < a * (n - 1) + dim; ++j) {  // runs that lie between one another
        const int64_t i = j * b / a;  // the nearest of the a-steps on either side
        if ((i < n && j * b - i * a < dim) || (i + 1 < n && (i + 1) * a - j * b < dim)) return true;
    }
    return false;
}

int refuse(std::string* why, const char* msg) {
    *why = msg;
    return GPT2Q_EARG;
}

}  // namespace

int gpt2q::check_paged_cache(const gpt2q_paged_kv* kv, const gpt2q_page_table* t, int dtype, std::string* why) {
    if (!kv || !kv->k || !kv->v) return refuse(why, "null cache");
    if (kv->dtype < GPT2Q_F32 || kv->dtype > GPT2Q_BF16) return refuse(why, "unknown cache dtype");
    if (dtype != kv->dtype && dtype != GPT2Q_F32) return refuse(why, "dtype must be the cache's or GPT2Q_F32");
    if (kv->n_pages < 1 || kv->page_size < 1 || kv->n_kv_heads < 1) return refuse(why, "n_pages, page_size and n_kv_heads must be >= 1");
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8)
        return refuse(why, "head_dim must be a multiple of 8 in [8, 256]");
    if (kv->page_stride < 0 || kv->head_stride < 0 || kv->token_stride < 0) return refuse(why, "negative cache stride");
    const int sz = size_of(kv->dtype);
    if (std::max({kv->page_stride, kv->head_stride, kv->token_stride}) > (int64_t)UINT32_MAX * 16 / sz)
        return refuse(why, "cache stride past 64 GB");
    if (!aligned16(kv->k, kv->page_stride, kv->head_stride, sz) || !aligned16(kv->v, kv->token_stride, 0, sz))
        return refuse(why, "the cache's addresses and strides must be multiples of 16 bytes");
    if (!t || (!t->ids && t->n_rows > 0) || t->n_rows < 0 || t->width < 1 || t->ld < t->width)
        return refuse(why, "null page table, or bad n_rows / width / ld");
    return GPT2Q_OK;
}

int gpt2q::paged_append(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                        const gpt2q_heads* v, const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype, int n_q_heads,
                        int n_tokens, const int32_t* d_pos, int pos0, const int32_t* d_seq, const gpt2q_rotary* rot,
                        int32_t* d_status, cudaStream_t st, std::string* why) {
    const int rc = check_paged_cache(kv, table, dtype, why);
    if (rc) return rc;
    if (n_tokens < 0) return refuse(why, "n_tokens < 0");
    if (n_tokens == 0) return GPT2Q_OK;
    if (!k || !k->data || !v || !v->data) return refuse(why, "null k or v");
    if ((q && q->data) != (q_out && q_out->data)) return refuse(why, "q and q_out come together");
    const bool with_q = q && q->data;
    if (with_q && n_q_heads < 1) return refuse(why, "n_q_heads must be >= 1");
    if (!d_pos && (d_seq || table->n_rows < 1 || pos0 < 0)) return refuse(why, "null d_pos");
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
    p.kc = kv->k, p.vc = kv->v;
    p.c_ps = kv->page_stride, p.c_hs = kv->head_stride, p.c_ts = kv->token_stride;
    p.page = kv->page_size, p.n_pages = kv->n_pages, p.n_tokens = n_tokens, p.n_kv = kv->n_kv_heads, p.dim = kv->head_dim;
    p.pos = d_pos, p.pos0 = pos0, p.seq = d_seq, p.table = table->ids, p.n_rows = table->n_rows, p.width = table->width;
    p.ld = table->ld, p.status = d_status;
    if (rot) {
        p.rot = rot->dim, p.interleaved = rot->interleaved != 0;
        for (int i = 0; i < rot->dim / 2; ++i) p.turns[i] = rot->turns[i];
    }
    const int units = kv->head_dim / (vec ? 16 : 2);
    while ((1 << p.unit_shift) < units) ++p.unit_shift;
    // heads a thread walks over: one while the call has fewer threads than the GPU holds, so that a
    // decode step is one round of loads; up to 8 in a large call, where the angles' arithmetic
    // would otherwise be repeated for every head
    const long long heads = (long long)p.n_q + 2LL * p.n_kv;
    const long long threads = ((long long)n_tokens << p.unit_shift) * heads;
    const long long walk = std::clamp<long long>(threads / (148 * 2048), 1, 8);
    p.groups = (int)((heads + walk - 1) / walk);
    const long long blocks = ((((long long)n_tokens * p.groups) << p.unit_shift) + 255) / 256;
    if (heads > INT32_MAX / 2 || blocks > INT32_MAX) return refuse(why, "too many tokens in one call");
    if (with_q && overlap(n_tokens, p.qo_ts, n_q_heads, p.qo_hs, p.dim)) return refuse(why, "the queries of q_out overlap");
    if (overlap(p.n_pages, p.c_ps, p.n_kv, p.c_hs, p.dim) || overlap(p.n_pages, p.c_ps, p.page, p.c_ts, p.dim) ||
        overlap(p.n_kv, p.c_hs, p.page, p.c_ts, p.dim))
        return refuse(why, "the cache's entries overlap");
    cudaError_t e;
    const unsigned nb = (unsigned)blocks;
    if (kv->dtype == GPT2Q_F32)
        e = launch_append<float, float>(p, vec, nb, st);
    else if (kv->dtype == GPT2Q_F16)
        e = dtype == GPT2Q_F32 ? launch_append<float, __half>(p, vec, nb, st) : launch_append<__half, __half>(p, vec, nb, st);
    else
        e = dtype == GPT2Q_F32 ? launch_append<float, bf16>(p, vec, nb, st) : launch_append<bf16, bf16>(p, vec, nb, st);
    if (e != cudaSuccess) {
        *why = cudaGetErrorString(e);
        return GPT2Q_ECUDA;
    }
    return GPT2Q_OK;
}

int gpt2q::paged_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                           const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads, float scale,
                           int window, float* d_lse, int32_t* d_status, void* d_work, const HiLo& hl, cudaStream_t st,
                           std::string* why) {
    const int rc = check_paged_cache(kv, table, dtype, why);
    if (rc) return rc;
    if (table->n_rows == 0) return GPT2Q_OK;
    if (!d_lens || !q || !q->data || !out || (!out->data && !hl.hi)) return refuse(why, "null d_lens, q or out");
    if (n_heads < 1 || n_heads % kv->n_kv_heads) return refuse(why, "n_heads must be a multiple of n_kv_heads");
    if (!std::isfinite(scale)) return refuse(why, "scale must be finite");
    if (window < 0) return refuse(why, "window < 0");
    if (!d_work || reinterpret_cast<uintptr_t>(d_work) % 16) return refuse(why, "null or unaligned d_work");
    const int sz = size_of(dtype);
    if (!aligned16(q->data, q->token_stride, q->head_stride, sz) ||
        !aligned16(out->data, out->token_stride, out->head_stride, sz))
        return refuse(why, "addresses and strides of q and out must be multiples of 16 bytes");
    if (out->data && overlap(table->n_rows, out->token_stride, n_heads, out->head_stride, kv->head_dim))
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
    p.cap = (int)std::min<long long>((long long)table->width * kv->page_size, INT32_MAX - 64);
    p.n_heads = n_heads, p.n_kv = kv->n_kv_heads, p.group = n_heads / kv->n_kv_heads, p.dim = kv->head_dim;
    p.window = window, p.scale = scale, p.status = d_status;
    const cudaError_t e = launch_paged_attn(p, kv->dtype, dtype, d_work, st);
    if (e != cudaSuccess) {
        *why = cudaGetErrorString(e);
        return GPT2Q_ECUDA;
    }
    return GPT2Q_OK;
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
        rc = paged_append(kv, table, k, v, q, q_out, dtype, n_q_heads, n_tokens, d_pos, 0, d_seq, rot, d_status,
                          static_cast<cudaStream_t>(stream), &why);
    if (rc) set_global_error("gpt2q_paged_append: " + why);
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
