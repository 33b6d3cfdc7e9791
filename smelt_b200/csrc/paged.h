// Paged key/value cache: append with position rotation, and attention of one new token per row.
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

// What both calls ask of a cache and a page table; `why` receives the message. Returns a GPT2Q_* code.
int check_paged_cache(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, int dtype, std::string* why);

// The checks and launches behind gpt2q_paged_append / gpt2q_paged_attention; `why` receives the
// message of a failed call. Return GPT2Q_* codes. In paged_append a null d_pos means positions
// pos0, pos0 + 1, ... of table row 0.
int paged_append(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k, const gpt2q_heads* v,
                 const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype, int n_q_heads, int n_tokens,
                 const int32_t* d_pos, int pos0, const int32_t* d_seq, const gpt2q_rotary* rot, int32_t* d_status,
                 cudaStream_t st, std::string* why);
int paged_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                    const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads, float scale, int window,
                    float* d_lse, int32_t* d_status, void* d_work, const HiLo& hl, cudaStream_t st, std::string* why);

}  // namespace gpt2q
