// Paged key/value cache: append with position rotation, reading back, committing drafted tokens, and attention of one new
// token or of a tree of drafted tokens per row.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <string>

#include "gpt2q.h"

namespace gpt2q {

// fp16 hi/lo copies of the attention's fp32 output (x = hi + lo), which the tensor-core linears
// read; row stride ld. Null when not wanted.
struct HiLo {
    __half* hi = nullptr;
    __half* lo = nullptr;
    int ld = 0;
};

// One attention call, checked (paged.cu); the fields after `status` are set by launch_paged_attn.
struct PagedAttn {
    const void *k, *v;
    uint32_t ps16, hs16, ts16;  // strides in units of 16 bytes
    int page, n_pages;
    const void* q;
    void* out;
    long long q_ts, q_hs, o_ts, o_hs;  // elements
    HiLo hl;
    float* lse;
    const int *table, *lens;
    long long ld;
    // 8-bit cache: scales of the entries, strides in elements
    const float *k_scale, *v_scale;
    long long s_ps, s_hs, s_ts;
    // a tree of drafted tokens per row (first != null): row r has tokens first[r] .. first[r + 1] - 1; lens are those of the prefixes
    const int *first, *mask;
    int mask_words, n_tokens;
    long long most;  // places in the list of tiles that a `first` that rises can ask for
    int n_rows, n_heads, n_kv, group, dim, window;
    int cap;  // the longest length a row of the table can hold
    float scale;
    int* status;
    int page_shift;  // page = 1 << page_shift, or -1
    // pieces of 128 bytes of a key, TMA copies of a group of keys, and its bytes in shared memory
    int boxes, box_loads, group_bytes;
    // a kv head's `group` query heads are taken in blocks_per_kv blocks of up to heads_per_block
    int blocks_per_kv, n_vh, heads_per_block;
    int warp_bytes;  // shared memory of a warp
    int4* meta;
    float *warp_part, *block_part;
    float2* block_ml;
};
uint64_t paged_attn_workspace(int dim, int group);
cudaError_t launch_paged_attn(PagedAttn p, int cache_dtype, int dtype, void* work, cudaStream_t st);
// by cache type; the workspace is laid out
cudaError_t launch_paged_attn_i8(const PagedAttn& p, int dtype, cudaStream_t st);
cudaError_t launch_paged_attn_e4m3(const PagedAttn& p, int dtype, cudaStream_t st);
// drafted tokens on tcgen05 tiles (paged_tree_tc.cu): bytes of its workspace, whether it takes a call, and the call; `taken` stays
// false where the pools cannot be described to TMA
uint64_t paged_tree_tc_workspace(int dim);
bool paged_tree_tc_serves(const PagedAttn& p, int cache_dtype, int dtype);
cudaError_t launch_paged_tree_tc(const PagedAttn& p, int cache_dtype, int dtype, void* work, cudaStream_t st, bool* taken);
cudaError_t launch_paged_tree(const PagedAttn& p, int cache_dtype, int dtype, cudaStream_t st);
cudaError_t launch_paged_tree_i8(const PagedAttn& p, int dtype, cudaStream_t st);
cudaError_t launch_paged_tree_e4m3(const PagedAttn& p, int dtype, cudaStream_t st);

inline bool is_8bit(int dtype) { return dtype == GPT2Q_I8 || dtype == GPT2Q_E4M3; }
inline int size_of(int dtype) { return dtype == GPT2Q_F32 ? 4 : is_8bit(dtype) ? 1 : 2; }

// One append, checked (paged.cu).
struct AppendParams {
    const void *k, *v, *q;
    void* qo;
    long long k_ts, k_hs, v_ts, v_hs, q_ts, q_hs, qo_ts, qo_hs;  // elements
    void *kc, *vc;
    long long c_ps, c_hs, c_ts;
    float *k_scale, *v_scale;  // 8-bit cache
    long long s_ps, s_hs, s_ts;
    int page, n_pages, n_tokens, n_q, n_kv, dim, rot, interleaved;
    const int *pos, *slot, *seq, *table;
    int pos0, n_rows, width;
    long long ld;
    int* status;
    int unit_shift, groups;  // threads of a token: groups * 2^unit_shift
    double turns[128];
};

// One read or commit, checked (paged.cu).
struct EntryParams {
    void *kc, *vc;
    long long c_ps, c_hs, c_ts;  // elements
    float *k_scale, *v_scale;
    long long s_ps, s_hs, s_ts;
    int page, n_pages, n_kv, dim;
    const int* table;
    int n_rows, width;
    long long ld;
    int* status;
    // read
    void *k, *v;
    long long k_ts, k_hs, v_ts, v_hs;
    int n_tokens;
    const int *pos, *seq;
    // commit
    const int *lens, *accept;
    int* new_lens;
    int n_accept;
    long long accept_ld;
};
cudaError_t launch_append(AppendParams p, int cache_dtype, int dtype, bool vec, cudaStream_t st);
cudaError_t launch_read(const EntryParams& p, int cache_dtype, int dtype, bool vec, cudaStream_t st);
cudaError_t launch_commit(const EntryParams& p, int cache_dtype, cudaStream_t st);

// What all calls ask of a cache and a page table; `why` receives the message. Returns a GPT2Q_* code.
int check_paged_cache(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, int dtype, std::string* why);

// The checks and launches behind gpt2q_paged_append / gpt2q_paged_attention; `why` receives the
// message of a failed call. Return GPT2Q_* codes. In paged_append a null d_pos means positions
// pos0, pos0 + 1, ... of table row 0, and a null d_slot the positions themselves.
int paged_append(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k, const gpt2q_heads* v,
                 const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype, int n_q_heads, int n_tokens,
                 const int32_t* d_pos, int pos0, const int32_t* d_slot, const int32_t* d_seq, const gpt2q_rotary* rot,
                 int32_t* d_status, cudaStream_t st, std::string* why);
struct Tree {  // what a tree's attention has beside one new token's
    const int32_t* d_first = nullptr;
    const int32_t* d_mask = nullptr;
    int mask_words = 0, n_tokens = 0;
};
int paged_commit(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens, const int32_t* d_accept,
                 int width, int64_t ld, int32_t* d_new_lens, int32_t* d_status, cudaStream_t st, std::string* why);
int paged_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                    const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads, float scale, int window,
                    float* d_lse, int32_t* d_status, void* d_work, const HiLo& hl, cudaStream_t st, std::string* why,
                    const Tree* tree = nullptr);

}  // namespace gpt2q
