/* gpt2q — B200 (sm_100a) GPT-2 forward over group-quantized weights.
 *
 * C-ABI boundary of the smelt_b200 library (libgpt2q.so). It replaces the CUDA
 * executor of LukasParke/smelt's model-lab (experiments/model-lab/src/gpu.rs,
 * kernels in src/cu/gpt2.cu) and keeps the shape of its Rust API so a thin FFI
 * crate restores `Gpu::new / step / clear_kv`. Citations below are paths inside
 * that project.
 *
 * Conventions
 *  - Every call returns an int status: GPT2Q_OK (0) or a negative GPT2Q_E* code.
 *    Nothing aborts or panics; gpt2q_last_error() gives the message.
 *  - One handle per GPU. A handle is not thread-safe; distinct handles may be
 *    driven from distinct threads.
 *  - Host buffers are caller-owned; gpt2q_create copies every tensor, so the
 *    caller keeps ownership (gpu.rs:114-127 copies too).
 *  - Weight payloads use the SMT TENSORS layout (model-lab/src/bin/pack.rs:68-94):
 *      "core.i8.b32.f16scale"  [rows][cols/32] blocks of 34 B: f16 scale LE + 32 x int8
 *      "core.i4.b32.f16scale"  [rows][cols/32] blocks of 18 B: f16 scale LE + 16 B, byte j =
 *                              elem j (low nibble) | elem j+16 (high nibble), two's complement
 *      "core.f16"              IEEE half, little endian
 *      "core.f32"              IEEE float (fp32 weights)
 *    2-D weights are [out, in] (pack.rs transposes HF Conv1D at convert time).
 *  - Tensor names follow the HF GPT-2 names used by the pack: wte.weight,
 *    wpe.weight, ln_f.{weight,bias}, h.{L}.ln_1/ln_2.{weight,bias},
 *    h.{L}.attn.c_attn/c_proj.{weight,bias}, h.{L}.mlp.c_fc/c_proj.{weight,bias}.
 *  - Greedy argmax follows gpt2.rs:390-396: IEEE total order, ties -> LAST index.
 */
#ifndef GPT2Q_H
#define GPT2Q_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GPT2Q_OK 0
#define GPT2Q_EARG -1      /* bad argument / shape / name */
#define GPT2Q_EOOM -2      /* device allocation failed */
#define GPT2Q_ECUDA -3     /* CUDA runtime error */
#define GPT2Q_ENCCL -4     /* NCCL error (tensor-parallel handles) */
#define GPT2Q_ETIMEOUT -5  /* a bounded device-side wait gave up */
#define GPT2Q_EUNSUP -6    /* unsupported configuration */

typedef struct gpt2q_handle gpt2q_handle;

/* Model architecture (gpt2.rs:11-19 Meta) plus capacity of this handle. */
typedef struct gpt2q_config {
    int32_t n_embd;
    int32_t n_layer;
    int32_t n_head;
    int32_t n_ctx;
    int32_t vocab;
    float ln_eps;
    int32_t max_seqs;   /* KV-cache slots (sequences resident at once); >= 1 */
    int32_t max_tokens; /* tokens per prefill chunk (activation workspace); 0 = default */
} gpt2q_config;

/* One tensor record of the SMT TENSORS section (format.rs:17-28 TensorRecord). */
typedef struct gpt2q_tensor_desc {
    const char* name;
    const char* atom;
    int32_t ndim;
    int64_t shape[2];
    const void* data; /* host pointer to the payload */
    uint64_t len;     /* payload bytes */
} gpt2q_tensor_desc;

/* Replaces Gpu::new(&Engine) (gpu.rs:75-157): uploads every tensor (quantized
 * ones stay quantized in HBM), allocates the KV arena for cfg->max_seqs
 * sequences of n_ctx positions and the activation workspace. */
int gpt2q_create(const gpt2q_config* cfg, const gpt2q_tensor_desc* tensors, int n_tensors,
                 int device, gpt2q_handle** out);

/* Tensor-parallel handle (no counterpart in the reference, which is single-GPU,
 * gpu.rs:76): rank `tp_rank` of `tp_size` keeps its column slice of c_attn
 * (whole heads) and c_fc and its row slice of attn/mlp c_proj; the two c_proj
 * partial sums per layer are added by the library's own kernel from peer memory
 * when the GPUs can map each other's memory (gpt2q_info "tp_peer_mapped"), else
 * by an NCCL all-reduce. nccl_id points to the 128-byte ncclUniqueId made by
 * rank 0 and shared by the caller. */
int gpt2q_create_tp(const gpt2q_config* cfg, const gpt2q_tensor_desc* tensors, int n_tensors,
                    int device, int tp_size, int tp_rank, const void* nccl_id,
                    gpt2q_handle** out);

/* Frees everything; replaces the Drop of Gpu. Safe on NULL. */
void gpt2q_destroy(gpt2q_handle* h);

/* Last error message of this handle (or of the last failed create when h is NULL). */
const char* gpt2q_last_error(const gpt2q_handle* h);

/* Replaces Gpu::clear_kv (gpu.rs:203-209). slots == NULL clears every slot. */
int gpt2q_reset_kv(gpt2q_handle* h, const int32_t* slots, int n_slots);

/* Exactly Gpu::step (gpu.rs:212-379): batch 1, KV slot 0, token `tok` at
 * position `pos`; writes vocab fp32 logits to host `logits`. */
int gpt2q_step(gpt2q_handle* h, uint32_t tok, int32_t pos, float* logits);

/* Batched decode: one token per sequence. Sequence i feeds tok[i] at pos[i]
 * into KV slot slots[i] (slots == NULL: slot i), attends over positions
 * 0..pos[i] of that slot. Optional outputs (host, may be NULL): logits
 * [n_seq][vocab], next_tok [n_seq] (greedy argmax). Engine::step batched over
 * sequences (gpt2.rs:227-332). */
int gpt2q_decode(gpt2q_handle* h, const uint32_t* tok, const int32_t* pos, const int32_t* slots,
                 int n_seq, float* logits, uint32_t* next_tok);

/* Prefill whole prompts starting at position 0. Sequence i owns tokens
 * [seq_offsets[i], seq_offsets[i+1]) and KV slot slots[i] (NULL: slot i).
 * Optional host outputs: logits_last [n_seq][vocab] at each prompt's last
 * position, next_tok [n_seq]. Equivalent to feeding every prompt token through
 * Engine::step (gpt2.rs:373-381) but computed as one batched pass. */
int gpt2q_prefill(gpt2q_handle* h, const uint32_t* tokens, const int32_t* seq_offsets,
                  const int32_t* slots, int n_seq, float* logits_last, uint32_t* next_tok);

/* Continues the sequences of the previous gpt2q_prefill/gpt2q_decode call for
 * `steps` more greedy decode steps entirely on the device: each step feeds the
 * previous step's argmax token at position+1. Optional host output
 * out_tokens [steps][n_seq]. Fails with GPT2Q_EARG when a position would reach n_ctx. */
int gpt2q_decode_steps(gpt2q_handle* h, int steps, uint32_t* out_tokens);

/* generate_greedy (gpt2.rs:367-388) for a batch of prompts: prefill, then
 * steps-1 device-side decode steps; out [n_seq][steps]. Prompts are clipped the
 * same way (positions > n_ctx-1 stop generation; missing tokens are written as
 * UINT32_MAX). */
int gpt2q_generate_greedy(gpt2q_handle* h, const uint32_t* tokens, const int32_t* seq_offsets,
                          int n_seq, int steps, uint32_t* out);

/* Publish a plastic adapter applied to the post-ln_f hidden state of every later step and
 * prefill: h += B (A h), A [r][d] and B [d][r] fp32 row-major, 1 <= r <= 256
 * (Gpu::set_adapter gpu.rs:188-194, k_adapter_apply cu/gpt2.cu:196-215). The copy is made
 * on the handle's stream: work enqueued before the call sees the previous generation, work
 * after it the new one (RCU-style). Host buffers may be reused when the call returns. */
int gpt2q_set_adapter(gpt2q_handle* h, const float* A, const float* B, int r);
/* Remove the adapter (Gpu::clear_adapter, gpu.rs:195). */
int gpt2q_clear_adapter(gpt2q_handle* h);

/* Teacher-forced negative log-likelihood per token of ids[0..n-1]
 * (nll_per_token, gpt2.rs:347-364): the mean over positions p = 0..n-2 of
 * -(logit[ids[p+1]] - max) + ln(sum exp(logit - max)), with the log-sum-exp in f64.
 * One prefill over the sequence in cache slot `slot` (its KV cache is overwritten),
 * the head on every position, and the per-position terms on the device: logits
 * never leave the GPU; only the n-1 f64 terms are read back and summed in order.
 * 2 <= n <= min(n_ctx, max_tokens). */
int gpt2q_nll(gpt2q_handle* h, const uint32_t* ids, int n, int slot, double* out_nll);

/* Dequantize a weight tensor exactly as Engine::vec_f32 (gpt2.rs:121-142)
 * into host `out` (n floats). Computed on the device from the uploaded bytes. */
int gpt2q_dequant(gpt2q_handle* h, const char* name, float* out, uint64_t n);

/* Number of kernel launches issued so far (Gpu::launches, gpu.rs:70). A CUDA
 * graph replay counts the kernels it contains. */
uint64_t gpt2q_launches(const gpt2q_handle* h);

/* Launch on this CUDA stream (a cudaStream_t) instead of the handle's own. */
int gpt2q_set_stream(gpt2q_handle* h, void* stream);

/* Wait for all work of the handle. */
int gpt2q_sync(gpt2q_handle* h);

/* Per-launch timing (CUDA events around every kernel; disables CUDA graphs
 * while on). gpt2q_profile_read writes a JSON object
 * {"kernel": {"launches": n, "ms": t, "bytes": algorithmic bytes}, ...}. */
int gpt2q_profile(gpt2q_handle* h, int enable);
int gpt2q_profile_read(gpt2q_handle* h, char* json, size_t cap);

/* Runs one decode step of the current sequences; the first launch of every kernel
 * type (the argmax excepted) is replayed `reps` times back to back in a CUDA graph with
 * the step's own arguments and timed with CUDA events. Writes JSON
 * {"kernel": {"us": per-launch time, "bytes": algorithmic bytes per launch,
 *  "per_step": launches per decode step}, ...}. The replays repeat residual
 * additions, so decode results after this call are not meaningful until the next
 * prefill. */
int gpt2q_profile_kernels(gpt2q_handle* h, int reps, char* json, size_t cap);

/* Which execution paths this handle uses, as JSON:
 * {"persistent_decode": bool, "persistent_why": reason when false,
 *  "persistent_ctas": CTAs of the persistent launch, "tensor_core": bool}.
 * The persistent decode serves every single-sequence decode step (gpt2q_step,
 * gpt2q_decode with n_seq = 1, gpt2q_decode_steps with one sequence); the
 * environment variable GPT2Q_NO_PERSISTENT at create time turns it off.
 * No counterpart in the reference (gpu.rs has one kernel sequence). */
int gpt2q_info(gpt2q_handle* h, char* json, size_t cap);

/* Greedy argmax (IEEE total order, ties -> last index) of n_rows rows of device fp32
 * logits (row stride ld >= vocab floats) into device d_next[n_rows], on `stream` (a
 * cudaStream_t; NULL = legacy default stream). Allocates nothing: its per-row scratch is
 * a fixed array inside the library, for callers that cannot allocate device memory at
 * that point (a decode loop that must not synchronise the device, or code under another
 * framework's memory pool). No counterpart in the reference. Limit: n_rows <=
 * GPT2Q_NOALLOC_MAX_ROWS, else GPT2Q_EARG. A call looks up the scratch array's device
 * address (cudaGetSymbolAddress) unless `stream` reports an active capture, when it uses
 * the address an earlier call found; the first call on a device therefore does the set-up and
 * should come before any stream capture. All calls share the scratch, so calls that overlap on
 * the GPU race; serialise them. Errors are reported by gpt2q_last_error(NULL). */
#define GPT2Q_NOALLOC_MAX_ROWS 1024
int gpt2q_argmax_noalloc(const float* d_logits, int vocab, int ld, int n_rows, uint32_t* d_next, void* stream);

/* Workload utilities for seeded synthetic weights/tokens (no counterpart in the
 * reference's GPU API): xorshift64* Rng of model-lab/src/gpu_backward.rs:835-856
 * (Rng::new(seed) = seed ^ 0x9E3779B97F4A7C15) with the Box-Muller normal of
 * perf-lab/src/bin/atoms.rs:78-83. `state` is advanced in place. */
uint64_t gpt2q_rng_new(uint64_t seed);
/* Converter group quantisers (host, multithreaded): n % 32 == 0 values -> SMT payload.
 * q8: atoms.rs:65-78 (34 B per group); q4: perf-lab atoms.rs:89-99 math, 18 B per group. */
int gpt2q_quantize_q8(const float* x, size_t n, uint8_t* out);
int gpt2q_quantize_q4(const float* x, size_t n, uint8_t* out);
void gpt2q_rng_normal_f32(uint64_t* state, float* out, size_t n, double stdv);
void gpt2q_rng_below(uint64_t* state, uint32_t* out, size_t n, uint64_t bound);

/* SMT container loading (Engine::load, gpt2.rs:43-89, over PackReader, format.rs:94-175).
 * The file is memory-mapped; with verify != 0 the merkle content_id (format.rs:121-145: blake3
 * over the sorted BLAKE3 digests of every section) and every tensor digest (first 16 bytes of
 * blake3 of its payload, gpt2.rs:91-110) are checked on all host threads, and a mismatch fails
 * with GPT2Q_EARG and a message naming the section or tensor. META.arch supplies n_embd,
 * n_layer, n_head, n_ctx, vocab_size and ln_eps; the TENSORS records become the tensor list of
 * gpt2q_create. Errors are reported by gpt2q_last_error(NULL). */
int gpt2q_create_from_smt(const char* path, int device, int max_seqs, int max_tokens, int verify,
                          gpt2q_handle** out);

/* Parses (and with verify != 0 verifies) an SMT container without touching a GPU; writes JSON
 * {"content_id": hex, "verified": bool, "arch": {...}, "tensors": [{name, atom, len, shape}]}. */
int gpt2q_smt_inspect(const char* path, int verify, char* json, size_t cap);

/* BLAKE3 (32-byte output, unkeyed) of len bytes, the hash the SMT digests use; host threads
 * hash the subtrees of large inputs. */
int gpt2q_blake3(const void* data, uint64_t len, uint8_t* out32);

/* ---- Backward of the trunk (the reference's plasticity path: cu/backward.cu, gpu_backward.rs) ----
 *
 * Input gradient of the whole trunk for one sequence (trunk_input_grad, gpu_backward.rs:651-790,
 * over the activations of bwparity.rs forward_stash:448-580): the forward over ids[0..n-1]
 * (positions 0..n-1) keeps every activation the backward needs on the device, then
 * dlogits [n][vocab] (host) is propagated through the tied head, ln_f and every layer, all
 * positions at once. Writes dx [n][n_embd] (host): the gradient with respect to the embedding
 * output wte[ids[p]] + wpe[p] at each position. lnf_out (host, may be NULL) receives the ln_f
 * output [n][n_embd], which the tied head's weight gradient needs (dlogits[p][v] * lnf_out[p]).
 * The plastic adapter is not part of the trunk. 1 <= n <= n_ctx; single-GPU handles only. */
int gpt2q_trunk_input_grad(gpt2q_handle* h, const uint32_t* ids, int n, const float* dlogits, float* dx,
                           float* lnf_out);

/* Per-op backward kernels with the BwdOps signatures (gpu_backward.rs:69-93): host buffers,
 * uploaded and downloaded per call on `device`, like GpuBackward's methods (gpu_backward.rs:
 * 307-377). Errors are reported by gpt2q_last_error(NULL).
 * lin_input_grad: dx[i] = sum_r w[r*cols+i] * dy[r] (k_lin_input_grad); cols % 4 == 0. */
int gpt2q_bwd_lin_input_grad(int device, const float* w, const float* dy, int rows, int cols, float* dx);
/* LayerNorm backward of one n-vector (k_ln_backward); dg and db accumulate. */
int gpt2q_bwd_ln_backward(int device, const float* dy, const float* x, const float* g, const float* b, float eps,
                          int n, float* dx, float* dg, float* db);
/* dx[i] = dy[i] * gelu'(x_pre[i]) for the tanh GELU (k_gelu_bwd). */
int gpt2q_bwd_gelu(int device, const float* x_pre, const float* dy, int n, float* dx);
/* Causal training-form attention backward (k_attn_bwd_train): q/k/v/dy [t][stride], head h
 * at column h*hd, stride/hd heads; dq overwritten, dk and dv accumulate. t <= 1024, hd <= 128. */
int gpt2q_bwd_attn_train(int device, const float* q, const float* k, const float* v, const float* dy, int t, int hd,
                         int stride, float* dq, float* dk, float* dv);

/* ---- Operators on device memory: a paged key/value cache and token log probabilities ----
 *
 * Like gpt2q_argmax_noalloc these take device pointers and a cudaStream_t (NULL = the legacy
 * default stream), allocate nothing and do not synchronise, so they may be captured into a CUDA
 * graph. They launch on the current device, which has to own the memory and the stream. Calls that
 * share no output and no workspace may run at the same time. Errors found on the host are reported
 * by gpt2q_last_error(NULL); nothing is launched then. No counterpart in the reference, whose cache
 * is one [n_ctx][d] buffer per layer (gpu.rs:128-134). */
#define GPT2Q_F32 0
#define GPT2Q_F16 1
#define GPT2Q_BF16 2
/* types of a cache alone: 8-bit codes with one scale per entry (gpt2q_paged_kv8) */
#define GPT2Q_I8 8   /* int8, -127..127 */
#define GPT2Q_E4M3 9 /* 8-bit floating point, 4 exponent and 3 mantissa bits, largest 448 */

/* One layer's paged cache. Keys and values lie in two pools of n_pages pages with the same strides
 * (in elements): the entry of token slot o in page p for kv head h starts at
 * p * page_stride + h * head_stride + o * token_stride and holds head_dim elements. The pools' base
 * addresses and all strides are multiples of 16 bytes; head_dim is a multiple of 8, at most 256.
 * Entries must not overlap (an append refuses a cache in which they would), nor keys lie over values, but that an append of
 * the same k and v without a rotation takes a cache whose k and v are the same. */
typedef struct gpt2q_paged_kv {
    void* k;
    void* v;
    int32_t dtype; /* GPT2Q_F32, GPT2Q_F16 or GPT2Q_BF16; GPT2Q_I8 or GPT2Q_E4M3 in a gpt2q_paged_kv8 */
    int32_t n_pages;
    int32_t page_size; /* token slots of a page, any number >= 1 */
    int32_t n_kv_heads;
    int32_t head_dim;
    int32_t reserved; /* 0; GPT2Q_SCALED in a gpt2q_paged_kv8 */
    int64_t page_stride;
    int64_t head_stride;
    int64_t token_stride;
} gpt2q_paged_kv;

/* A paged cache of 8-bit codes: kv.reserved is GPT2Q_SCALED, kv.dtype GPT2Q_I8 or GPT2Q_E4M3, and head_dim a multiple of 16.
 * An entry (the head_dim codes of one token, kv head and pool) stands for code * scale; its scale is the fp32 number at
 * page * scale_page_stride + head * scale_head_stride + slot * scale_token_stride (elements, any strides >= 0) of k_scale or
 * v_scale. Every call that takes a gpt2q_paged_kv takes the address of `kv`; those that take one per layer take an array of
 * gpt2q_paged_kv8 where the first has 8 bits. q, k, v and outputs of such calls are GPT2Q_F32, GPT2Q_F16 or GPT2Q_BF16.
 * Written entries: scale = top / T and code = round(x * (T / top)), to nearest with ties to even, where top is the entry's
 * largest magnitude (after the rotation) and T is 127 or 448, all in fp32 (the scale at most what T times it is finite for). An
 * entry whose top is under 2^-100 has scale and codes 0; one with a NaN or an infinity has codes 0 and scale NaN.
 * Attention holds a weight times its value's scale in 16-bit numbers relative to the largest value scale among the keys that the query
 * sees. Beside its roundings each key may add an error of 2^-35 of the largest |v| seen (2^-31 where products run on wide tensor-core
 * tiles): a result that is much smaller than values of next to no weight has fewer digits for it. */
#define GPT2Q_SCALED 1
typedef struct gpt2q_paged_kv8 {
    gpt2q_paged_kv kv;
    float* k_scale;
    float* v_scale;
    int64_t scale_page_stride;
    int64_t scale_head_stride;
    int64_t scale_token_stride;
} gpt2q_paged_kv8;

/* Rows of page ids: row r's token at position p lies in page table[r * ld + p / page_size], slot
 * p % page_size. Entries past a row's last used page are never read. */
typedef struct gpt2q_page_table {
    const int32_t* ids; /* device */
    int32_t n_rows;
    int32_t width; /* pages a row can name */
    int64_t ld;    /* row stride, >= width */
} gpt2q_page_table;

/* Position rotation over the first `dim` elements of a head: pair i is turned by
 * position * 2 pi * turns[i]. Pairs are (i, i + dim/2), or (2i, 2i + 1) when interleaved != 0. */
typedef struct gpt2q_rotary {
    int32_t dim;
    int32_t interleaved;
    double turns[128];
} gpt2q_rotary;

/* turns[i] = base^(-2i/dim) / (2 pi). dim even, 2..256; a caller may write other turns afterwards. */
int gpt2q_rotary_init(gpt2q_rotary* rot, int dim, int interleaved, double base);

/* A device tensor [token][head][head_dim] with unit stride over head_dim; strides in elements. Tensors
 * that are written have entries that share no memory (a call refuses others). */
typedef struct gpt2q_heads {
    void* data;
    int64_t token_stride;
    int64_t head_stride;
} gpt2q_heads;

/* Bits of the optional device status word (int32, OR-ed into, never cleared). */
#define GPT2Q_STATUS_PAGE 1     /* a page id outside [0, n_pages) was needed */
#define GPT2Q_STATUS_POSITION 2 /* a position or length past the table's width */
#define GPT2Q_STATUS_ROW 4      /* a table row outside [0, n_rows) */
#define GPT2Q_STATUS_TIMEOUT 8  /* a bounded device-side wait gave up (results are NaN) */

/* Appends n_tokens keys and values (both or neither of k->data and v->data) to the cache. Token i
 * belongs to table row d_seq[i] (d_seq NULL: row i) and position d_pos[i]. Keys are rotated when
 * `rot` is given, rounded once to the cache's type; with `q` and `q_out` the token's n_q_heads
 * queries are rotated into q_out too (q_out may be q; it shares no other memory with q, k, v or the
 * cache). k, v, q and q_out are of type `dtype`, the
 * cache's or GPT2Q_F32. A token with d_pos[i] < 0 is padding: nothing of it is written to the
 * cache and its queries are copied unrotated. A token whose page, position or row is out of range
 * is not written either and sets its bit in d_status (may be NULL). No two tokens of a call may
 * name the same cache entry. */
int gpt2q_paged_append(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                       const gpt2q_heads* v, const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype, int n_q_heads,
                       int n_tokens, const int32_t* d_pos, const int32_t* d_seq, const gpt2q_rotary* rot,
                       int32_t* d_status, void* stream);

/* gpt2q_paged_append whose tokens lie at cache positions d_slot[i] (NULL: d_pos[i]), while the rotation is that of position
 * d_pos[i]: drafted tokens of a tree follow one another in the cache, but are as far from its root as their depth. A token with
 * d_pos[i] < 0 is padding whatever d_slot[i] is; with d_pos[i] >= 0 a negative d_slot[i] is out of range. */
int gpt2q_paged_append_at(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k,
                          const gpt2q_heads* v, const gpt2q_heads* q, const gpt2q_heads* q_out, int dtype, int n_q_heads,
                          int n_tokens, const int32_t* d_pos, const int32_t* d_slot, const int32_t* d_seq,
                          const gpt2q_rotary* rot, int32_t* d_status, void* stream);

/* Reads n_tokens entries into k and v ([token][kv head][head_dim], type `dtype`: the cache's or GPT2Q_F32, of an 8-bit cache any
 * of the three): token i is that of table row d_seq[i] (d_seq NULL: row i) at position d_pos[i]. k and v share no memory with one
 * another or the cache (a call refuses those that do). An element is rounded to `dtype` from its value, of an 8-bit cache from the
 * product code * scale in fp32, which is rounded itself. d_pos[i] < 0 gives zeros; a row, position or page out of range gives NaN and sets its bit in
 * d_status (may be NULL). */
int gpt2q_paged_read(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const gpt2q_heads* k, const gpt2q_heads* v,
                     int dtype, int n_tokens, const int32_t* d_pos, const int32_t* d_seq, int32_t* d_status, void* stream);

/* Attention of one new token per table row over that row's cached entries:
 * out[r][h] = sum_j softmax_j(scale * q[r][h] . K[j][h / (n_heads / n_kv_heads)]) V[j], j over the
 * last `window` of the positions 0..d_lens[r]-1 (window 0: all of them). q and out are of type
 * `dtype`, the cache's or GPT2Q_F32; data and strides multiples of 16 bytes. d_lse (may be NULL),
 * [n_rows][n_heads] fp32, receives the natural logarithm of each row's sum of exp. A row of length
 * <= 0 gives zeros and -inf. A row that needs a page id out of range, or whose length exceeds the
 * table, gives NaN and sets its bit in d_status (may be NULL). Scores, the running maximum and sum
 * and the output are accumulated in fp32; results do not depend on the order in which blocks run.
 * d_work: gpt2q_paged_attention_workspace(kv, n_heads) bytes of device memory, 16-byte aligned,
 * that no other call running at the same time uses; its content does not matter. */
uint64_t gpt2q_paged_attention_workspace(const gpt2q_paged_kv* kv, int n_heads);
int gpt2q_paged_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                          const gpt2q_heads* q, const gpt2q_heads* out, int dtype, int n_heads, float scale,
                          int window, float* d_lse, int32_t* d_status, void* d_work, void* stream);

/* Attention of drafted tokens over a paged cache: row r has the tokens d_first[r] .. d_first[r + 1] - 1 of q and out (d_first:
 * n_rows + 1 numbers, rising, within 0..n_tokens), which lie in its cache behind a prefix of d_lens[r] tokens, token i of the row
 * at position d_lens[r] + i. Every token sees the whole prefix, and of the row's drafted tokens those that its mask names: bit j & 31 of
 * d_mask[t * mask_words + j / 32] says whether token t (of all n_tokens) sees its row's drafted token j; tokens past the words
 * are not seen. A tree's tokens name their ancestors and themselves. d_mask NULL: a token sees itself and those before it (a
 * chain, or a chunk of a prompt). A token that sees nothing gives zeros and an lse of -inf. What a token does not see does not
 * reach it, infinities and NaN included; a drafted token's value with an infinity or NaN gives NaN in those that see it. Tokens that
 * belong to no row are left as they were. Otherwise as gpt2q_paged_attention: types, alignment, d_lse [n_tokens][n_heads],
 * status bits and NaN for a row that needs a page id out of range or is longer than the table, fp32 sums in a fixed order. Where
 * products run on wide tensor-core tiles (16-bit outputs only) each weight, of an 8-bit cache times its value's scale, is rounded once, to
 * bf16 for bf16 caches (by up to 2^-8 of itself) and to fp16 otherwise (2^-11). Sums of weights are those of the rounded ones: a result is
 * off by up to twice that part of sum w |v|, and a single key gives its value. A length <= 0 is a prefix of none. A d_first that does not
 * rise gives numbers without a meaning; where it asks for more work than one that rises could, nothing is written but
 * GPT2Q_STATUS_POSITION. A prefix and its drafted tokens are at most 2^31 - 4097 together, whatever the table's width (more give NaN
 * and the status bit).
 * d_work: gpt2q_paged_tree_attention_workspace(kv, n_heads, n_tokens) bytes, 16-byte aligned, of one call at a time. */
uint64_t gpt2q_paged_tree_attention_workspace(const gpt2q_paged_kv* kv, int n_heads, int n_tokens);
int gpt2q_paged_tree_attention(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                               const int32_t* d_first, const int32_t* d_mask, int mask_words, const gpt2q_heads* q,
                               const gpt2q_heads* out, int dtype, int n_heads, int n_tokens, float scale, float* d_lse,
                               int32_t* d_status, void* d_work, void* stream);

/* Keeps the accepted ones of each row's drafted tokens: d_accept[r * ld + i], i < width, are the row's tokens to keep, in rising
 * order (a negative one ends the list). Entry d_lens[r] + d_accept[r * ld + i] moves to position d_lens[r] + i, codes and scales as
 * they are (keys stay rotated by the position they had), and d_new_lens[r] = max(d_lens[r], 0) + the number kept. At a token that does
 * not rise, or whose page or position is out of range, the row's list ends and the bit is set in d_status (may be NULL;
 * GPT2Q_STATUS_POSITION, GPT2Q_STATUS_PAGE). Rows must not share the pages that are written. d_new_lens shares no memory with d_lens or d_accept. */
int gpt2q_paged_commit(const gpt2q_paged_kv* kv, const gpt2q_page_table* table, const int32_t* d_lens,
                       const int32_t* d_accept, int width, int64_t ld, int32_t* d_new_lens, int32_t* d_status, void* stream);

/* Log probabilities of given tokens under softmax(logits / temperature), temperature >= 1e-30, per row of n_rows rows of
 * `vocab` logits (at most 2^30; type `dtype`, row stride ld >= vocab elements, any alignment of that type):
 *   d_lp[r]       log probability of targets[r] (int32, or int64 when targets_i64 != 0). A negative
 *                 target gives 0, one >= vocab NaN.
 *   d_entropy[r]  -sum p ln p
 *   d_stats[r][3] the largest logit, ln sum exp((logit - largest) / temperature), the entropy: what
 *                 gpt2q_logprobs_grad takes
 *   d_top_ids[r][top], d_top_lp[r][top]  the `top` likeliest tokens (0 <= top <= min(vocab,
 *                 GPT2Q_TOP_MAX)) in falling order, equal logits by rising index, and their log
 *                 probabilities
 * Each output may be NULL (targets, too, when d_lp is). A logit of -inf has probability 0. A row of
 * nothing but -inf gives log probabilities of -inf and entropy 0. A row with NaN or +inf gives NaN;
 * among alternatives NaN ranks as -inf. Sums are fp32 in a fixed order. */
#define GPT2Q_TOP_MAX 64
int gpt2q_logprobs(const void* d_logits, int dtype, int64_t ld, int n_rows, int vocab, float temperature,
                   const void* d_targets, int targets_i64, int top, float* d_lp, float* d_entropy, float* d_stats,
                   int32_t* d_top_ids, float* d_top_lp, void* stream);

/* Its gradient: d_dlogits[r][j] = (d_lp[r] ([j == target] - p_j) - d_ent[r] p_j (ln p_j + H)) / temperature,
 * the sum of both outputs' gradients for the incoming gradients d_lp and d_ent (fp32 [n_rows]; either may be
 * NULL, then its term is left out). d_stats are the forward's. d_dlogits has the logits' type and row stride
 * ld_out >= vocab; it may be d_logits itself (ld_out == ld), otherwise the two must not overlap. Elements past
 * vocab are left as they are. A row of negative target has no d_lp term; a row of nothing but -inf gets zeros. */
int gpt2q_logprobs_grad(const void* d_logits, int dtype, int64_t ld, int n_rows, int vocab, float temperature,
                        const void* d_targets, int targets_i64, const float* d_stats, const float* d_lp,
                        const float* d_ent, void* d_dlogits, int64_t ld_out, void* stream);

/* ---- The model over the operators above ---- */

/* Scores ids[1..n-1] under the model, as gpt2q_nll runs it (same prefill in cache slot `slot`, same limits, the
 * published adapter applied): lp[p] is the log probability of ids[p+1] after ids[0..p], entropy[p] (may be NULL) the
 * entropy there, top_ids / top_lp [n-1][top] the `top` likeliest tokens (0 <= top <= min(vocab, GPT2Q_TOP_MAX); NULL
 * when top is 0). Host buffers of n - 1 rows; the logits stay on the device. */
int gpt2q_score(gpt2q_handle* h, const uint32_t* ids, int n, int slot, int top, float* lp, float* entropy,
                int32_t* top_ids, float* top_lp);

/* gpt2q_trunk_input_grad for the loss sum_p d_lp[p] * ln p(targets[p] | ids[0..p]) + d_entropy[p] * H_p: the logits'
 * gradient is computed on the device from the forward's own logits, so no [n][vocab] array crosses the bus. targets [n]
 * (negative: no target at that position), d_lp and d_entropy [n] (either may be NULL) and the outputs lp, entropy [n]
 * (may be NULL), dx and lnf_out [n][n_embd] (lnf_out may be NULL) are host buffers. */
int gpt2q_trunk_score_grad(gpt2q_handle* h, const uint32_t* ids, int n, const int32_t* targets, const float* d_lp,
                           const float* d_entropy, float* lp, float* entropy, float* dx, float* lnf_out);

/* Copies the first n_tokens cached keys and values of arena slot `slot` (as a prefill or decode left them) into
 * positions 0..n_tokens-1 of row `row` of `table`, in every layer's paged cache: layers[n_layer], each with the model's
 * heads and head dim, of any cache type. Single-GPU handles only. The pools and the table are device memory of the
 * handle's device, ready on the handle's stream. Returns when the copy is done. */
int gpt2q_page_out(gpt2q_handle* h, int slot, int n_tokens, const gpt2q_paged_kv* layers, const gpt2q_page_table* table,
                   int row);

/* gpt2q_decode over paged caches instead of the arena: sequence i feeds tok[i] at pos[i], its keys and values go to row
 * i of `table` (table->n_rows == n_seq), and it attends over positions 0..pos[i] of that row. n_seq is limited by the
 * activation workspace (max(max_seqs, max_tokens)), not by the arena's slots, and sequences may share pages of a common
 * prefix. Optional host outputs as in gpt2q_decode. A page id out of range, or a row too short for pos[i], fails with
 * GPT2Q_EARG after the step has run (the outputs are then not meaningful). */
int gpt2q_decode_paged(gpt2q_handle* h, const uint32_t* tok, const int32_t* pos, int n_seq, const gpt2q_paged_kv* layers,
                       const gpt2q_page_table* table, float* logits, uint32_t* next_tok);

/* Feeds drafted tokens of n_seq sequences over paged caches (table->n_rows == n_seq): sequence i has tok[first[i]] ..
 * tok[first[i + 1] - 1] (first[0] = 0; n = first[n_seq] of them in all, at most max(max_seqs, max_tokens)) behind lens[i] cached
 * tokens. parent[t] is the index of a token's parent among its sequence's earlier drafted tokens, or -1 for one that follows
 * the cached ones; a token is at its parent's position + 1 and attends over the cached tokens, its ancestors and itself. Keys and
 * values go to positions lens[i], lens[i] + 1, ... of the row, in the tokens' order. Optional host outputs: logits [n][vocab] and
 * next_tok [n], the likeliest token after each drafted one. Errors as gpt2q_decode_paged's. */
int gpt2q_verify_paged(gpt2q_handle* h, const uint32_t* tok, const int32_t* parent, const int32_t* first, const int32_t* lens,
                       int n_seq, const gpt2q_paged_kv* layers, const gpt2q_page_table* table, float* logits,
                       uint32_t* next_tok);

/* gpt2q_paged_commit in every layer: accept[i][width] names the drafted tokens of sequence i that stay, rising, ended by a
 * negative one. lens, accept and new_lens (may be NULL) are host arrays; table->n_rows sequences. A list that does not rise or
 * names a token past the table's width is refused before anything is moved. */
int gpt2q_commit_paged(gpt2q_handle* h, const int32_t* lens, const int32_t* accept, int width, int32_t* new_lens,
                       const gpt2q_paged_kv* layers, const gpt2q_page_table* table);

#ifdef __cplusplus
}
#endif
#endif /* GPT2Q_H */
