/*
 * sgl_attn.h — C ABI of the MI355X (gfx950) attention hot path.
 *
 * Every entry point takes plain device pointers, element counts and
 * strides (in elements), a hipStream_t passed as `void*`, and returns an
 * int status: 0 on success, a negative SGL_ERR_* code for an argument the
 * call rejects before launching anything, or a positive hipError_t when the
 * HIP runtime refuses the launch. No entry point allocates device memory;
 * workspaces are passed in by the caller. The pool layout is the
 * reference's MHAKVCache: one layer's K (or V) cache is [slots, Hkv, D]
 * bf16, token-granular (a "page" of page_size P is P consecutive slots).
 *
 * Each declaration names the reference interface (allen-shaw/sglang.cpp,
 * file:line) it replaces.
 */
#ifndef SGL_ATTN_H_
#define SGL_ATTN_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SGL_OK 0
#define SGL_ERR_INVALID_ARG (-1)  /* null pointer, bad size, bad stride */
#define SGL_ERR_UNSUPPORTED (-2)  /* head_dim / group size / dtype not built */
#define SGL_ERR_CAPACITY (-3)     /* workspace or plan capacity exceeded */
#define SGL_ERR_ALIGNMENT (-4)    /* pointer / stride misaligned for vector path */

#define SGL_INDEX_I32 0
#define SGL_INDEX_I64 1

#define SGL_DTYPE_BF16 0  /* 16-bit element types (norm, RoPE and residual-path kernels) */
#define SGL_DTYPE_F16 1
#define SGL_DTYPE_F32 2   /* fp32 (accepted where a declaration says so) */

/* Human-readable text for a status code (static storage). */
const char* sgl_status_string(int status);

/* Library version, to check that the loaded .so matches this header. */
int sgl_abi_version(void);
#define SGL_ABI_VERSION 18

/* ------------------------------------------------------------------ */
/* KV-cache store                                                      */
/* ------------------------------------------------------------------ */

/*
 * k_cache[out_loc[t], :] = k[t, :] and v_cache[out_loc[t], :] = v[t, :]
 * for t < num_tokens, copying elems_per_token 2-byte elements (bf16 or
 * fp16: the copy is bitwise). k/v rows are strided by k_stride_token /
 * v_stride_token elements (the narrow views of a qkv row); cache rows are
 * contiguous, elems_per_token apart. out_loc is int32 (index_dtype
 * SGL_INDEX_I32) or int64 (SGL_INDEX_I64).
 * Replaces: MHAKVCache::store_kv + store_kv_cache_kernel
 *           (src/kvcache/mha_kvcache.cu:111-155, :13-41).
 */
int sgl_store_kv(void* k_cache, void* v_cache, const void* k, const void* v,
                 const void* out_loc, int index_dtype, int64_t num_tokens,
                 int64_t elems_per_token, int64_t k_stride_token,
                 int64_t v_stride_token, void* stream);

/* ------------------------------------------------------------------ */
/* Page-table / token-pool plumbing                                    */
/* ------------------------------------------------------------------ */

/*
 * indices[kv_indptr[r] + p] = page_table[table_indices[r] * stride + p]
 * for p < kv_indptr[r+1]-kv_indptr[r] (0 where p >= cols); rows whose
 * table index is outside [0, rows) are left untouched.
 * Replaces: build_decode_indices_kernel (src/attention/flashinfer_backend.cu:43-70).
 */
int sgl_build_decode_indices(const int32_t* page_table, int64_t rows,
                             int64_t stride, int64_t cols,
                             const int32_t* table_indices,
                             const int32_t* kv_indptr, int32_t* indices,
                             int batch_size, void* stream);

/*
 * Prefill metadata gather: indices = cat_r(page_table[table_indices[r], :kv_len_r]),
 * with kv_indptr the prefix sum of kv_len. Device-side replacement of the
 * torch::cat over page-table slices.
 * Replaces: prefill branch of FlashInferBackend::prepare_metadata
 *           (src/attention/flashinfer_backend.cu:466-484).
 */
int sgl_build_prefill_indices(const int32_t* page_table, int64_t rows,
                              int64_t stride, int64_t cols,
                              const int32_t* table_indices,
                              const int32_t* kv_indptr, int32_t* indices,
                              int batch_size, void* stream);

/*
 * pool[req_indices[i] * stride + positions[i]] = tokens[i]; entries with an
 * out-of-range row or column are skipped.
 * Replaces: write_token_pool (src/kernels/token_pool.cu:53-93, kernel :10-29).
 */
int sgl_write_token_pool(int32_t* pool, int64_t rows, int64_t stride,
                         int64_t cols, const int32_t* req_indices,
                         const int32_t* positions, const int32_t* tokens,
                         int64_t count, void* stream);

/*
 * Page allocation -> token-granular page table, on the device. The
 * allocations alloc_info[a] = (table_idx, first_page, last_page), int32
 * [num_allocs, 3], take consecutive entries of page_starts (the slot of each
 * allocated page's first token, num_pages of them, in allocation order);
 * page p of allocation a writes
 *   page_table[table_idx * stride + p * page_size + i] = page_start + i,
 * i < page_size, skipping out-of-range rows and columns as
 * sgl_write_token_pool does. Pages beyond what the allocations take are
 * ignored; the caller keeps sum(last_page - first_page) == num_pages, as the
 * reference checks on the host. At most 8192 allocations per call.
 * Replaces: CacheManager::write_page_table + pages_to_tokens
 *           (src/scheduler/prefill.cc:144-187, :103-119): the host expansion
 *           loop and its three token-sized H2D copies.
 */
int sgl_write_page_table(int32_t* page_table, int64_t rows, int64_t stride,
                         int64_t cols, const int32_t* page_starts, int64_t num_pages,
                         const int32_t* alloc_info, int num_allocs, int page_size,
                         void* stream);

/*
 * out[i] = table[req_indices[i] * stride + positions[i]] (0 when out of range).
 * Replaces: gather_int32_2d (src/kernels/token_pool.cu:95-133, kernel :31-49).
 */
int sgl_gather_int32_2d(const int32_t* table, int64_t rows, int64_t stride,
                        int64_t cols, const int32_t* req_indices,
                        const int32_t* positions, int32_t* out, int64_t count,
                        void* stream);

/*
 * Up to SGL_MAX_I32_COPIES device-to-device int32 copies in one launch:
 * dst[i] = src[i] for i < count of each entry (entries must not overlap).
 * The graph-replay path refreshes every capture buffer of a step (indptrs,
 * row maps, indices) with this one call instead of one copy per buffer.
 * Replaces: the per-buffer copies of FlashInferBackend::prepare_for_replay
 *           (src/attention/flashinfer_backend.cu:267-352).
 */
typedef struct {
  const int32_t* src;
  int32_t* dst;
  int64_t count;
} sgl_i32_copy_t;
#define SGL_MAX_I32_COPIES 8
int sgl_copy_i32(const sgl_i32_copy_t* copies, int num_copies, void* stream);

/* ------------------------------------------------------------------ */
/* RoPE and q/k RMSNorm                                                */
/* ------------------------------------------------------------------ */

/*
 * cos[p, i] = cos(p * inv_freq[i]), sin likewise, for p < max_pos,
 * i < rotary_dim/2, inv_freq[i] = 1 / base^(2i / rotary_dim), fp32.
 * Replaces: RotaryEmbedding ctor cache build (src/layers/rotary_embedding.cu:75-94).
 */
int sgl_rope_cos_sin_cache(float* cos_cache, float* sin_cache, int64_t max_pos,
                           int rotary_dim, float base, void* stream);

/*
 * In-place per-(token, head) RMSNorm of q [tokens, q_heads, d] and
 * k [tokens, k_heads, d] (strided views, last dim contiguous):
 * x <- T(x * rsqrt(mean(x^2) + eps) * w), fp32 accumulation, T = bf16 or
 * fp16 (dtype SGL_DTYPE_*; q, k and the weights share it, as the reference
 * dispatches both at :346-372).
 * Pass k = NULL / k_heads = 0 to normalise q only.
 * Replaces: fused_qk_rmsnorm_inplace_3d_strided (src/layers/normalization.cu:318-384)
 *           and RMSNorm::forward_inplace_3d_strided (:271-316).
 */
int sgl_qk_rmsnorm(void* q, void* k, const void* q_weight,
                   const void* k_weight, int64_t tokens, int64_t q_heads,
                   int64_t k_heads, int64_t d, int64_t q_stride_token,
                   int64_t q_stride_head, int64_t k_stride_token,
                   int64_t k_stride_head, float eps, int dtype, void* stream);

/*
 * In-place NeoX (rotate-half) RoPE of q [nnz, q_heads, head_dim] and
 * k [nnz, kv_heads, head_dim] at positions[t] (int32), using fp32 cos/sin
 * caches of width cos_width (rotary_dim/2 or rotary_dim). Elements at
 * index >= rotary_dim pass through. q and k are bf16 or fp16 (dtype
 * SGL_DTYPE_*, the reference dispatches both at :124-168); fp32 math, one
 * rounding per element.
 * Replaces: RotaryEmbedding::forward_inplace (src/layers/rotary_embedding.cu:96-178;
 *           formula :50-66).
 */
int sgl_rope(void* q, void* k, const float* cos_cache, const float* sin_cache,
             const int32_t* positions, int64_t nnz, int64_t q_heads,
             int64_t kv_heads, int64_t rotary_dim, int64_t head_dim,
             int64_t cos_width, int64_t q_stride_token, int64_t q_stride_head,
             int64_t k_stride_token, int64_t k_stride_head, int dtype, void* stream);

/*
 * One pass over the qkv activation [T, (Hq + 2 Hkv) * D] (row stride
 * qkv_stride_token): per token, q/k heads are RMS-normalised (weights
 * q_weight / k_weight, skipped when NULL), rounded to bf16, rotated by
 * RoPE at positions[t] (full rotary, half-width fp32 cos/sin cache
 * [max_pos, D/2]), rounded to bf16 and written back in place; the rotated
 * k row and the raw v row are also written to k_cache / v_cache at slot
 * out_loc[t] (int32). Bitwise the same as running sgl_qk_rmsnorm, then
 * sgl_rope, then sgl_store_kv. flags: 0, or SGL_FUSED_NO_K_WRITEBACK to
 * leave the k part of qkv untouched (the rotated k goes to k_cache only;
 * the reference writes it back, but nothing reads it after the store).
 * Replaces the sequence AttentionLayer::forward -> qk-norm -> RoPE ->
 * store_kv (src/layers/attention_layer.cc:27-47, flashinfer_backend.cu:530-532).
 */
int sgl_fused_qknorm_rope_store(void* qkv, int64_t qkv_stride_token,
                                void* k_cache, void* v_cache,
                                const void* q_weight, const void* k_weight,
                                const float* cos_cache, const float* sin_cache,
                                const int32_t* positions, const int32_t* out_loc,
                                int64_t num_tokens, int num_qo_heads,
                                int num_kv_heads, int head_dim, float eps,
                                int flags, void* stream);
#define SGL_FUSED_NO_K_WRITEBACK 1

/*
 * cos/sin tables of a rotary embedding scaled for contexts longer than it was
 * trained on: cos[p, i] = m cos(p f_i), sin[p, i] = m sin(p f_i) for p < max_pos,
 * i < rotary_dim / 2, fp32 [max_pos, rotary_dim / 2], the angle p f_i in 64 bits
 * (sgl_rope_cos_sin_cache rounds it to fp32 as the reference does). With
 * f_i = base^(-2 i / rotary_dim), L = original_max_position, s = factor:
 *   NONE    f_i (scaling NULL too)
 *   LINEAR  f_i / s
 *   NTK     base replaced by base s^(rotary_dim / (rotary_dim - 2))
 *   YARN    f_i (g_i / s + 1 - g_i), g_i = clamp((i - lo) / (hi - lo), 0, 1), lo and hi
 *           the pairs that turn beta_fast and beta_slow times over L positions,
 *           rotary_dim ln(L / (2 pi beta)) / (2 ln base), rounded down and up and
 *           kept inside [0, rotary_dim - 1]; m = attention_factor, or, where that is 0,
 *           0.1 ln s + 1 (1 for s <= 1)
 *   BANDS   f_i ((1 - w_i) / s + w_i), w_i = clamp((L f_i / (2 pi) - low_freq_factor) /
 *           (high_freq_factor - low_freq_factor), 0, 1)
 * m is 1 for the others. rotary_dim at most 512.
 * Replaces: RotaryEmbedding ctor cache build (src/layers/rotary_embedding.cu:75-94),
 *           which has no scaling.
 */
#define SGL_ROPE_SCALING_NONE 0
#define SGL_ROPE_SCALING_LINEAR 1
#define SGL_ROPE_SCALING_NTK 2
#define SGL_ROPE_SCALING_YARN 3
#define SGL_ROPE_SCALING_BANDS 4
typedef struct {
  int32_t kind;
  int32_t original_max_position;
  double factor;
  double beta_fast, beta_slow;
  double low_freq_factor, high_freq_factor;
  double attention_factor;
} sgl_rope_scaling_t;
int sgl_rope_scaled_cache(float* cos_cache, float* sin_cache, int64_t max_pos, int rotary_dim,
                          double base, const sgl_rope_scaling_t* scaling, void* stream);

/*
 * One pass that rotates q and k and appends k and v to the paged pool, for any
 * head_dim up to 1024, rotary_dim up to it (even; elements from it on pass through)
 * and both layouts of a pair: (x[i], x[i + rotary_dim / 2]), or with
 * SGL_ROPE_INTERLEAVED (x[2 i], x[2 i + 1]). Per token t at position positions[t]:
 *   q_out[t] = rotated q[t];  k_cache[out_loc[t]] = rotated k[t];  v_cache[out_loc[t]] = v[t]
 * fp32 arithmetic, one rounding per element; cos and sin are fp32 [max_pos,
 * rotary_dim / 2] tables. q, k, v, q_out are [tokens, heads, head_dim] with strides
 * (last dim contiguous), the caches [num_slots, num_kv_heads, head_dim] likewise.
 * q_out may be q (same strides) and the cache rows k's own (rotation in place); other
 * overlaps are the caller's error. A token whose slot is outside [0, num_slots) (padding)
 * is not appended; one whose position is outside [0, max_pos) gets NaN in the rotated
 * elements. A slot listed for several tokens then holds parts of any of them. out_loc NULL:
 * token t goes to slot t. v and v_cache both NULL: no v. No q with num_qo_heads 0, no k
 * and v with num_kv_heads 0.
 * Replaces: RotaryEmbedding::forward_inplace, then MHAKVCache::store_kv
 *           (src/layers/rotary_embedding.cu:96-178, src/kvcache/mha_kvcache.cu:111-155); the
 *           reference has the half layout over the whole head only.
 */
typedef struct {
  const void* q;
  void* q_out;
  const void* k;
  const void* v;
  void* k_cache;
  void* v_cache;
  const float* cos;
  const float* sin;
  const int32_t* positions;
  const void* out_loc;
  int64_t tokens, num_slots, max_pos;
  int64_t q_stride_token, q_stride_head, q_out_stride_token, q_out_stride_head;
  int64_t k_stride_token, k_stride_head, v_stride_token, v_stride_head;
  int64_t kv_stride_slot, kv_stride_head;
  int32_t num_qo_heads, num_kv_heads, head_dim, rotary_dim;
  int32_t dtype;       /* SGL_DTYPE_BF16 or SGL_DTYPE_F16: q, k, v and the caches */
  int32_t index_dtype; /* of out_loc: SGL_INDEX_I32 or SGL_INDEX_I64 */
  int32_t flags;       /* 0 or SGL_ROPE_INTERLEAVED */
  int32_t reserved;
} sgl_rope_append_t;
#define SGL_ROPE_INTERLEAVED 1
int sgl_rope_append(const sgl_rope_append_t* args, void* stream);

/* ------------------------------------------------------------------ */
/* Paged attention                                                     */
/* ------------------------------------------------------------------ */

/* Split-KV decode plan (host). */
typedef struct {
  int32_t kv_chunk_size;  /* W_max: largest unit in tokens (multiple of 16, <= 8192) */
  int32_t min_chunk_size; /* W_min: smallest unit (64) */
  int32_t num_units;      /* work units = workgroups launched */
  int32_t split_kv;       /* 1 when a request of the planned batch spans units */
  int32_t batch_size;     /* largest batch the plan serves */
  int32_t num_qo_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int64_t max_total_tokens; /* capacity: num_units * kv_chunk_size tokens per call */
  int64_t workspace_bytes;  /* 256-byte header (status word) + fp32 partials, two per unit,
                               + one int32 per unit */
  int32_t max_request_tokens; /* longest planned request; a caller that plans a worst case it
                                 expects to stay well below (graph capture) may set it to 0:
                                 batches of few tokens then always take the one-launch kernel */
  int32_t reserved;
} sgl_decode_plan_t;

/*
 * Token-balanced schedule from the host copy of kv_indptr (kv_indptr[0] must
 * be 0): the batch's flattened token stream is cut into num_units equal
 * units, one per resident workgroup (the count comes from the device's CU
 * count, 256 when no device is visible). The launch picks the unit size on
 * the device, clamp(ceil(total / num_units), min_chunk_size, kv_chunk_size)
 * rounded to 16 tokens, from kv_indptr[batch], so a plan built from a
 * kv_indptr with every request at its maximum length stays valid and
 * balanced for any batch of at most batch_size requests and at most
 * max_total_tokens tokens, whatever the per-request lengths (graph capture /
 * replay without re-planning).
 * Replaces: FlashInfer DecodePlan as called from
 *           FlashInferBackend::initialize_decode_metadata_once
 *           (src/attention/flashinfer_backend.cu:354-397).
 */
int sgl_decode_plan(const int32_t* kv_indptr_host, int batch_size,
                    int num_qo_heads, int num_kv_heads, int head_dim,
                    sgl_decode_plan_t* plan);

/*
 * Host-side check that a batch (host kv_indptr, batch_size requests) fits a
 * plan: SGL_OK, or SGL_ERR_CAPACITY when it has more requests than
 * plan->batch_size or more tokens than plan->max_total_tokens.
 * Replaces: the batch-size / length checks of
 *           FlashInferBackend::prepare_for_replay (src/attention/flashinfer_backend.cu:267-352).
 */
int sgl_decode_plan_check(const sgl_decode_plan_t* plan, const int32_t* kv_indptr_host,
                          int batch_size);

/*
 * Paged decode: for request r (rows q[q_row(r)], q_row(r) = r, or
 * q_indptr[r] when q_indptr is non-NULL) and q head h,
 * o[q_row, h] = softmax_j(q.K[indices[kv_indptr[r] + j], h / G] * sm_scale)
 *               . V[indices[...], h / G]
 * over j < kv_indptr[r+1] - kv_indptr[r]; an empty request gets a zero row.
 * G = Hq / Hkv. q is strided (q_stride_token, q_stride_head), o likewise
 * (strides multiples of 8 elements); k_cache/v_cache are one layer's
 * [slots, Hkv, D] (slot stride kv_stride_slot, head stride kv_stride_head).
 * workspace (plan->workspace_bytes, 16-byte aligned) holds the split
 * partials and, at offset 0, an int32 status word: each call clears it, and
 * when the device kv_indptr[batch] exceeds plan->max_total_tokens the rows
 * of every request reaching past the capacity are written as NaN and the
 * word is set to SGL_ERR_CAPACITY (read it with sgl_decode_status). Two
 * kernels run on the stream (decode, then merge: one workgroup per (kv
 * head, request), or per (kv head, unit) when the batch has more requests
 * than the plan has units), or one for small batches
 * (plans at the 64-token minimum unit with batch_size x Hkv workgroups at
 * most the CU count and no request longer than 800 tokens, 896, 1024 and 1152 from
 * 8, 16 and 64 of these workgroups). Calls that share one workspace must be stream-ordered.
 * Replaces: BatchDecodeWithPagedKVCacheDispatched call in
 *           FlashInferBackend::forward (src/attention/flashinfer_backend.cu:553-595).
 */
int sgl_paged_decode(const sgl_decode_plan_t* plan, const void* q,
                     int64_t q_stride_token, int64_t q_stride_head,
                     const void* k_cache, const void* v_cache,
                     int64_t kv_stride_slot, int64_t kv_stride_head,
                     const int32_t* indices, const int32_t* kv_indptr,
                     const int32_t* q_indptr, int batch_size,
                     int num_qo_heads, int num_kv_heads, int head_dim,
                     float sm_scale, void* o, int64_t o_stride_token,
                     int64_t o_stride_head, void* workspace,
                     int64_t workspace_bytes, void* stream);

/*
 * sgl_paged_decode without a workspace argument, for callers that cannot
 * allocate device memory (code under graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). The split partials live in a file-scope
 * device array of SGL_DECODE_SCRATCH_BYTES (32 MiB) that each GPU holds
 * until the process ends; plans with workspace_bytes above it get
 * SGL_ERR_CAPACITY. Nothing is allocated. Calls on one GPU share the array
 * and must be stream-ordered: calls that overlap on one GPU race. A batch
 * past the plan's capacity gets NaN rows and the CAPACITY status word as in
 * sgl_paged_decode; sgl_decode_status(NULL, ...) reads that word from the
 * current device's scratch. sgl_decode_plan looks the scratch address up
 * for the current device, so a call captured into a graph after a plan was
 * made runs no lookup inside the capture.
 * Replaces: no counterpart in the reference; it exists for callers that
 *           cannot allocate.
 */
int sgl_paged_decode_noalloc(const sgl_decode_plan_t* plan, const void* q,
                             int64_t q_stride_token, int64_t q_stride_head,
                             const void* k_cache, const void* v_cache,
                             int64_t kv_stride_slot, int64_t kv_stride_head,
                             const int32_t* indices, const int32_t* kv_indptr,
                             const int32_t* q_indptr, int batch_size,
                             int num_qo_heads, int num_kv_heads, int head_dim,
                             float sm_scale, void* o, int64_t o_stride_token,
                             int64_t o_stride_head, void* stream);
#define SGL_DECODE_SCRATCH_BYTES (32ll << 20)

/*
 * The attention layer's decode step: sgl_fused_qknorm_rope_store (with
 * SGL_FUSED_NO_K_WRITEBACK) on the batch's tokens, token r of qkv being request
 * r's, then sgl_paged_decode of the rotated q rows over the pool (k_cache and
 * v_cache [slots, Hkv, D] contiguous), with the same results, except for
 * requests that share an out_loc (which of their tokens that slot then holds is
 * open in both). Batches of at
 * most 64 requests that sgl_paged_decode takes in one kernel run as one launch
 * here too; others as those two calls. Arguments that either call refuses are
 * refused before anything is written.
 * Replaces: AttentionLayer::forward's norm, RoPE, store and decode
 *           (src/layers/attention_layer.cc:27-47, src/attention/flashinfer_backend.cu:530-595).
 */
int sgl_decode_layer(const sgl_decode_plan_t* plan, void* qkv, int64_t qkv_stride_token,
                     void* k_cache, void* v_cache, const void* q_weight, const void* k_weight,
                     const float* cos_cache, const float* sin_cache, const int32_t* positions,
                     const int32_t* out_loc, float eps, const int32_t* indices,
                     const int32_t* kv_indptr, int batch_size, int num_qo_heads,
                     int num_kv_heads, int head_dim, float sm_scale, void* o,
                     int64_t o_stride_token, int64_t o_stride_head, void* workspace,
                     int64_t workspace_bytes, void* stream);

/*
 * Reads the status word a decode call left in its workspace (waits for the
 * stream): SGL_OK, or SGL_ERR_CAPACITY when the batch exceeded its plan.
 * workspace NULL reads the word of sgl_paged_decode_noalloc's scratch on the
 * current device.
 * Replaces: no device-side counterpart in the reference (FlashInfer's plan
 *           is host-side); pairs with sgl_paged_decode.
 */
int sgl_decode_status(const void* workspace, int32_t* status, void* stream);

/*
 * Paged causal prefill over ragged requests: query i (0-based inside
 * request r, qo_len = qo_indptr[r+1]-qo_indptr[r]) attends kv j with
 * j <= i + kv_len - qo_len (bottom-right alignment), kv_len =
 * kv_indptr[r+1]-kv_indptr[r], slots from indices[kv_indptr[r] + j].
 * Request r's query (and output) rows start at q_start[r], or at
 * qo_indptr[r] when q_start is NULL (a subset of a batch's requests can so
 * be run in place). max_qo_len bounds qo_len over the batch (sizes the grid).
 * Replaces: BatchPrefillWithPagedKVCacheDispatched<..., kCausal, ...> in
 *           FlashInferBackend::forward (src/attention/flashinfer_backend.cu:596-679).
 */
int sgl_paged_prefill(const void* q, int64_t q_stride_token,
                      int64_t q_stride_head, const void* k_cache,
                      const void* v_cache, int64_t kv_stride_slot,
                      int64_t kv_stride_head, const int32_t* indices,
                      const int32_t* qo_indptr, const int32_t* kv_indptr,
                      const int32_t* q_start, int batch_size, int max_qo_len,
                      int num_qo_heads,
                      int num_kv_heads, int head_dim, float sm_scale, void* o,
                      int64_t o_stride_token, int64_t o_stride_head,
                      void* stream);

/*
 * Prefill with the lengths known on the host, for batches with too few query
 * tiles to fill the device (a few new tokens behind long cached prefixes):
 * the kv ranges are cut into shares that run on separate workgroups and are
 * folded by a second launch.
 *   sgl_prefill_plan: from the host copies of qo_indptr and kv_indptr. Writes
 *     the launch's list into items (capacity int32 entries, at most
 *     SGL_PREFILL_PLAN_INTS are used) and its
 *     sizes into plan; num_items 0 when sgl_paged_prefill serves the batch at
 *     least as well.
 *   sgl_paged_prefill_planned: as sgl_paged_prefill for the lengths the plan
 *     was made from; items is the device copy of the list (num_items +
 *     num_merges entries of four int32), workspace (plan->workspace_bytes,
 *     16-byte aligned) holds the shares' fp32 states. Calls that share a
 *     workspace must be stream-ordered.
 * Replaces: the PrefillPlan / split-KV scheduling of FlashInfer behind
 *           BatchPrefillWithPagedKVCacheDispatched
 *           (src/attention/flashinfer_backend.cu:596-679).
 */
typedef struct {
  int32_t num_items;   /* workgroups per kv head */
  int32_t num_merges;  /* query tiles folded from several shares */
  int32_t num_qo_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t reserved;
  int64_t workspace_bytes;
} sgl_prefill_plan_t;
#define SGL_PREFILL_PLAN_INTS 4096
int sgl_prefill_plan(const int32_t* qo_indptr_host, const int32_t* kv_indptr_host,
                     int batch_size, int num_qo_heads, int num_kv_heads, int head_dim,
                     sgl_prefill_plan_t* plan, int32_t* items, int64_t capacity);
int sgl_paged_prefill_planned(const sgl_prefill_plan_t* plan, const int32_t* items, const void* q,
                              int64_t q_stride_token, int64_t q_stride_head, const void* k_cache,
                              const void* v_cache, int64_t kv_stride_slot, int64_t kv_stride_head,
                              const int32_t* indices, const int32_t* qo_indptr,
                              const int32_t* kv_indptr, const int32_t* q_start, int num_qo_heads,
                              int num_kv_heads, int head_dim, float sm_scale, void* o,
                              int64_t o_stride_token, int64_t o_stride_head, void* workspace,
                              int64_t workspace_bytes, void* stream);

/*
 * A mixed batch (decode rows beside prefill rows, the chunked-prefill step
 * of FlashInferBackend::forward's prefill phase with one-token requests) in
 * one launch plus the split merge: the first workgroups run the decode rows
 * on decode_cus CUs while the causal-prefill items run on the others, then
 * on every CU as the decode finishes (the HBM-bound decode and the
 * MFMA-bound prefill side by side). num_kv_heads must divide 8.
 *   sgl_mixed_decode_cus: the CU share for the decode rows (a multiple of
 *     8), from their K/V token count and the prefill's flops
 *     (4 D Hq sum_r sum_i (kv_r - qo_r + i + 1)).
 *   sgl_decode_plan_cus: a decode plan (as sgl_decode_plan) whose units fill
 *     decode_cus CUs, each unit short enough for the fused launch's LDS
 *     (at 1 or 2 kv heads long batches then get more units than that); like
 *     any plan it serves smaller batches on replay.
 *   sgl_paged_mixed: decode rows as sgl_paged_decode (dec_q_rows: query row
 *     of each decode request, or NULL for rows 0..dec_batch-1) and prefill
 *     rows as sgl_paged_prefill, sharing q, the caches and o. With no rows
 *     of one kind it runs the other entry point alone; with a plan whose
 *     units are too long for the fused launch (sgl_decode_plan at 1 or 2
 *     kv heads) it runs the two entry points one after the other.
 * Replaces: the decode and prefill calls of one mixed step
 *           (src/attention/flashinfer_backend.cu:553-679); the reference
 *           runs them as separate kernels.
 */
int sgl_mixed_decode_cus(int64_t decode_kv_tokens, int num_kv_heads, int head_dim,
                         double prefill_flops);
int sgl_decode_plan_cus(const int32_t* kv_indptr_host, int batch_size,
                        int num_qo_heads, int num_kv_heads, int head_dim,
                        int decode_cus, sgl_decode_plan_t* plan);
int sgl_paged_mixed(const sgl_decode_plan_t* plan, const void* q,
                    int64_t q_stride_token, int64_t q_stride_head,
                    const void* k_cache, const void* v_cache,
                    int64_t kv_stride_slot, int64_t kv_stride_head,
                    const int32_t* dec_indices, const int32_t* dec_kv_indptr,
                    const int32_t* dec_q_rows, int dec_batch,
                    const int32_t* pre_indices, const int32_t* pre_qo_indptr,
                    const int32_t* pre_kv_indptr, const int32_t* pre_q_start,
                    int pre_batch, int pre_max_qo_len, int num_qo_heads,
                    int num_kv_heads, int head_dim, float sm_scale, void* o,
                    int64_t o_stride_token, int64_t o_stride_head,
                    void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Attention of a batch whose requests share a prefix (samples of one prompt, users of
 * one system prompt, drafted tokens being verified), the prefix's K/V read once for
 * the whole batch instead of once per request. Request r's kv sequence is the
 * prefix_len slots prefix_indices[0 .. prefix_len), then its own
 * indices[kv_indptr[r] .. kv_indptr[r + 1]); its query tokens are rows
 * [qo_indptr[r], qo_indptr[r + 1]) of q, at most max_qo_len of them (qo_len), and query
 * i sees kv j with j <= i + kv_len - qo_len, kv_len = prefix_len + own length: the
 * result of sgl_paged_prefill over the joined sequences (of sgl_paged_decode for one
 * query token). A row that sees nothing is zero. K and V of tokens a row does not see
 * never reach it, whatever they hold; a V value that it sees and that is not finite makes
 * that element NaN or infinite. Rows that see less than the prefix (a request with
 * fewer own tokens than query tokens) are computed one by one: right, not fast. For one
 * request, behind a few hundred tokens, and for few requests of several query tokens behind
 * a few thousand, the paged calls over the joined sequences are faster (32q/8kv, one query
 * token: 16 requests behind 512 tokens 11.6 us here, 10.3 there; behind 1,024 13.1 and 19.8).
 *   sgl_prefix_plan: host plan for up to batch_size requests with up to max_tokens query
 *     tokens together (max_qo_len of one request at most SGL_PREFIX_MAX_QO). It does not
 *     depend on the requests' own lengths, so it serves every step of a batch (graph
 *     capture and replay) behind a prefix of prefix_len. Up to 2^29 tokens of prefix,
 *     2^25 requests, 2^24 - 1 query tokens, 2^30 of them times the heads of a kv head, 2^31
 *     times num_qo_heads.
 *   sgl_prefix_attention: q and o have max_tokens rows here (at most the plan's);
 *     rows outside [qo_indptr[0], qo_indptr[batch_size]) are left as they were. The
 *     offsets may start past 0 (a part of a larger batch); they must not decrease. A
 *     request whose own do, or leave the batch's or [0, max_tokens], or whose qo_len
 *     exceeds the plan's, gets NaN rows; where offsets decrease, the rows of the other
 *     requests are open. Slots are the caller's to keep inside the caches. sm_scale is
 *     positive. workspace: plan->workspace_bytes, 16-byte aligned, written before it is
 *     read; calls that share one must be stream-ordered.
 * q, o: bf16 [max_tokens, num_qo_heads, 128], caches one layer's bf16 [slots,
 * num_kv_heads, 128]; strides multiples of 8 elements; 1 to 64 query heads per kv head.
 * Replaces: no counterpart in the reference, whose batches walk every request's whole kv
 *           (src/attention/flashinfer_backend.cu:553-679) though its radix cache shares the
 *           slots (src/kvcache/radix_tree.cc).
 */
typedef struct {
  int32_t prefix_len;
  int32_t batch_size;
  int32_t max_tokens;
  int32_t max_qo_len;
  int32_t num_qo_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t num_blocks;   /* workgroups of the launch (two per CU) */
  int32_t max_units;    /* parts the requests' own tokens are cut into at most */
  int32_t reserved;
  int64_t prefix_rows;  /* partial rows of the prefix in the workspace */
  int64_t workspace_bytes;
} sgl_prefix_plan_t;
#define SGL_PREFIX_MAX_QO 64
int sgl_prefix_plan(int prefix_len, int batch_size, int max_tokens, int max_qo_len,
                    int num_qo_heads, int num_kv_heads, int head_dim, sgl_prefix_plan_t* plan);
int sgl_prefix_attention(const sgl_prefix_plan_t* plan, const void* q, int64_t q_stride_token,
                         int64_t q_stride_head, const void* k_cache, const void* v_cache,
                         int64_t kv_stride_slot, int64_t kv_stride_head,
                         const int32_t* prefix_indices, const int32_t* indices,
                         const int32_t* kv_indptr, const int32_t* qo_indptr, int batch_size,
                         int max_tokens, int num_qo_heads, int num_kv_heads, int head_dim,
                         float sm_scale, void* o, int64_t o_stride_token, int64_t o_stride_head,
                         void* workspace, int64_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------ */
/* Residual path: RMSNorm, fused add + RMSNorm, gated activations      */
/* ------------------------------------------------------------------ */

/*
 * out[r, :] = T(x[r, :] * rsqrt(mean(x[r, :]^2) + eps) * weight) for
 * r < rows, fp32 arithmetic, T = bf16 or fp16 (dtype SGL_DTYPE_*; weight
 * has the same type). Rows of d elements, x_stride_row / out_stride_row
 * elements apart; out may equal x (in place).
 * Replaces: RMSNorm::forward / forward_inplace
 *           (src/layers/normalization.cu:236-269).
 */
int sgl_rmsnorm(void* out, const void* x, const void* weight, int64_t rows,
                int64_t d, int64_t x_stride_row, int64_t out_stride_row,
                int dtype, float eps, void* stream);

/*
 * In place, per row: s = x + residual (fp32); residual = T(s);
 * x = T(s * rsqrt(mean(s^2) + eps) * weight). Rows longer than 8192
 * elements normalise T(s) instead of s (a second pass re-reads it).
 * Replaces: RMSNorm::fused_add_forward_inplace
 *           (src/layers/normalization.cu:386-416).
 */
int sgl_fused_add_rmsnorm(void* x, void* residual, const void* weight,
                          int64_t rows, int64_t d, int64_t x_stride_row,
                          int64_t residual_stride_row, int dtype, float eps,
                          void* stream);

/*
 * out[t, i] = T(silu(in[t, i]) * in[t, d + i]), silu(x) = x / (1 + e^-x),
 * for t < tokens, i < d; input rows hold 2 d elements (gate, then up).
 * Replaces: silu_and_mul (src/layers/activation.cu:8-10, 15-45).
 */
int sgl_silu_and_mul(void* out, const void* input, int64_t tokens, int64_t d,
                     int64_t in_stride_row, int64_t out_stride_row, int dtype,
                     void* stream);

/*
 * As sgl_silu_and_mul with the tanh GELU
 * gelu(x) = 0.5 x (1 + tanh(0.7978845608 (x + 0.044715 x^3))).
 * Replaces: gelu_and_mul (src/layers/activation.cu:12-14, 47-77).
 */
int sgl_gelu_and_mul(void* out, const void* input, int64_t tokens, int64_t d,
                     int64_t in_stride_row, int64_t out_stride_row, int dtype,
                     void* stream);

/* ------------------------------------------------------------------ */
/* Projections and experts                                             */
/* ------------------------------------------------------------------ */

/*
 * A projection and what follows it:
 *   out[t, j] = T(act(sum_i x[t, i] weight[j, i] + bias[j]) + residual[t, j]),
 * t < tokens, j < n, i < k, and for the *_AND_MUL activations, whose weight and bias have
 * 2 n rows (gate, then up),
 *   out[t, j] = T(act(g_j) u_j + residual[t, j]), g and u the biased sums of rows j, n + j.
 * fp32 sums and arithmetic, one rounding; act is off by at most (1 + |z|) 2^-21 of itself (or
 * |x| 2^-126), z what its sigmoid is taken of. x, weight, bias and residual are bf16 or fp16
 * (dtype), out that type or fp32 (out_dtype SGL_DTYPE_F32: logits). bias and residual may
 * be NULL; out may be residual (same type and strides), other overlaps are the caller's
 * error. Any sizes up to 2^31 - 256, strides and alignment; fast where k is a multiple of 8 (best
 * of 64) and rows start on 16 bytes. workspace: sgl_linear_workspace_bytes (0 where the
 * inputs are summed in one part; up to 134 MB), 16-byte aligned, written before it is
 * read; calls that share one must be stream-ordered. With NULL they are summed in one part:
 * slower, another order of the sum.
 * Replaces: Linear::forward and what the model runs on its output
 *           (src/layers/linear.cc:9-78; activation.cu:15-77).
 */
#define SGL_ACT_NONE 0
#define SGL_ACT_SILU 1
#define SGL_ACT_GELU 2 /* tanh, as sgl_gelu_and_mul */
#define SGL_ACT_SILU_AND_MUL 3
#define SGL_ACT_GELU_AND_MUL 4
typedef struct {
  const void* x;
  const void* weight;
  const void* bias;
  const void* residual;
  void* out;
  int64_t tokens, n, k;
  int64_t x_stride_row, weight_stride_row, residual_stride_row, out_stride_row;
  int32_t dtype;
  int32_t out_dtype;
  int32_t activation;
  int32_t reserved; /* 0 */
} sgl_linear_t;
int64_t sgl_linear_workspace_bytes(int64_t tokens, int64_t n, int64_t k, int activation);
int sgl_linear(const sgl_linear_t* args, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * The experts of each token from the router's logits (bf16, fp16 or fp32 [tokens,
 * num_experts], rows logits_stride_row elements apart): experts[t, j], j < top_k, are the
 * experts of the top_k largest logits, largest first, equal ones by their number;
 * weights[t, j] their probabilities in the softmax over all experts, with renormalize
 * divided by their sum. int32 and fp32 [tokens, top_k], contiguous. NaN is ranked below
 * -inf; a row with a NaN, with +inf or with nothing above -inf has NaN weights. Up to 512
 * experts, top_k 32, 2^30 tokens.
 * Replaces: the softmax, top-k and renormalisation of the router (src/moe/moe.cc:47-60).
 */
int sgl_moe_route(const void* logits, int64_t logits_stride_row, int logits_dtype, int64_t tokens,
                  int num_experts, int top_k, int renormalize, float* weights, int32_t* experts,
                  void* stream);

/*
 * The experts of a mixture-of-experts layer:
 *   out[t] = T(sum_j weights[t, j] down[e] h + residual[t]), e = experts[t, j],
 *   h = T(act(gate_up[e][:I] x[t]) * (gate_up[e][I:] x[t])), I = intermediate,
 * with x, out and residual [tokens, hidden], gate_up [num_experts, 2 I, hidden] and down
 * [num_experts, hidden, I] bf16 or fp16, weights fp32 and experts int32 [tokens, top_k]
 * contiguous. Sums and weighted terms in fp32; h is rounded to the type, as the matrix
 * instructions take it. A slot whose expert is outside [0, num_experts) adds nothing
 * (padding, experts of another device). An expert may be chosen more than once.
 * activation: SGL_ACT_SILU_AND_MUL or SGL_ACT_GELU_AND_MUL. residual may be NULL, out may
 * be residual (same strides). workspace: sgl_moe_workspace_bytes, 16-byte aligned,
 * written before it is read; calls that share one must be stream-ordered. hidden and
 * intermediate up to 2^20, 65,536 experts, 2^30 choices (tokens x top_k). Fast where hidden
 * and intermediate are multiples of 8 and rows start on 16 bytes.
 * Replaces: the loop over the experts (src/moe/moe.cc:62-98).
 */
typedef struct {
  const void* x;
  const void* gate_up;
  const void* down;
  const float* weights;
  const int32_t* experts;
  const void* residual;
  void* out;
  int64_t tokens;
  int64_t x_stride_row, residual_stride_row, out_stride_row;
  int64_t gate_up_stride_expert, gate_up_stride_row, down_stride_expert, down_stride_row;
  int32_t top_k, num_experts, hidden, intermediate;
  int32_t dtype;
  int32_t activation;
} sgl_moe_t;
int64_t sgl_moe_workspace_bytes(int64_t tokens, int top_k, int num_experts, int hidden,
                                int intermediate);
int sgl_moe_experts(const sgl_moe_t* args, void* workspace, int64_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------ */
/* Probabilities from logits, then sampling from probabilities         */
/* ------------------------------------------------------------------ */

/*
 * probs[r, i] = softmax_i(float(logits[r, i]) / t_r) over i < vocab, fp32,
 * for r < batch; t_r = temperatures[r] (fp32 [batch]) or, when temperatures
 * is NULL, the scalar temperature (> 0). logits_dtype: SGL_DTYPE_BF16,
 * SGL_DTYPE_F16 or SGL_DTYPE_F32; row strides in elements (>= vocab). One
 * workgroup per row; aligned 16-bit rows of up to 163,840 elements are
 * held in registers and read from HBM once. Small batches of long aligned rows
 * take two launches of many workgroups, with the same bits, unless probs and
 * logits overlap. Exponentials as
 * 2^(fma(x, a, -max a)) with a = log2e / t (relative error of a probability
 * below ~1e-5 against the exact softmax of float(x) / t). A row whose
 * temperature is not positive gets NaN probabilities.
 * Replaces: the probabilities of Sampler::sample, logits.to(kFloat32) /
 *           temperatures then torch::softmax (src/engine/engine.cc:306-308).
 */
int sgl_softmax_temperature(float* probs, int64_t probs_stride_row, const void* logits,
                            int64_t logits_stride_row, int logits_dtype,
                            const float* temperatures, float temperature, int64_t batch,
                            int64_t vocab, void* stream);

/*
 * probs: fp32 [batch_size, d], rows contiguous (the softmax of the
 * temperature-scaled logits). out: int32 [batch_size]. The draw with
 * uniform u is the first index i with probs[i] > 0 whose running sum of
 * such probabilities exceeds u (d - 1 if rounding leaves none). uniform is
 * fp32 [batch_size]. deterministic is accepted for the reference's
 * signature; sums here always run in a fixed order. Rows of up to 2^21
 * probabilities (SGL_ERR_UNSUPPORTED beyond). One 1024-thread workgroup
 * per row, about 153 KiB of LDS; nothing is allocated.
 * Replaces: flashinfer_sample_from_probs (src/engine/sampling.cu:65-84).
 */
int sgl_sampling_from_probs(const float* probs, const float* uniform, int32_t* out,
                            int batch_size, int d, int deterministic, void* stream);

/*
 * Top-k draw by rejection rounds: round r draws from the probabilities
 * above a pivot with u = uniform[r, row] * (their mass), the pivot rises to
 * the drawn probability, and the draw is accepted once fewer than k
 * probabilities exceed it. uniform: fp32 [max_rounds, batch_size]; k is
 * top_k_arr[row] (fp32, as the reference passes it) or top_k_val when
 * top_k_arr is NULL. success (bool bytes, optional) = accepted within
 * max_rounds; out holds the last draw either way.
 * Replaces: flashinfer_top_k_sample_from_probs (src/engine/sampling.cu:86-116).
 */
int sgl_top_k_sampling_from_probs(const float* probs, const float* uniform, int32_t* out,
                                  uint8_t* success, const float* top_k_arr,
                                  int batch_size, int top_k_val, int d, int max_rounds,
                                  int deterministic, void* stream);

/*
 * As above, accepting once the mass above the pivot is below top_p
 * (top_p_arr[row], or top_p_val when top_p_arr is NULL).
 * Replaces: flashinfer_top_p_sample_from_probs (src/engine/sampling.cu:118-148).
 */
int sgl_top_p_sampling_from_probs(const float* probs, const float* uniform, int32_t* out,
                                  uint8_t* success, const float* top_p_arr,
                                  int batch_size, float top_p_val, int d, int max_rounds,
                                  int deterministic, void* stream);

/*
 * Both filters: accepted once fewer than k probabilities exceed the pivot
 * and their mass is below top_p. top_k_arr is int32 here, as the
 * reference passes it.
 * Replaces: flashinfer_top_k_top_p_sample_from_probs
 *           (src/engine/sampling.cu:150-192).
 */
int sgl_top_k_top_p_sampling_from_probs(const float* probs, const float* uniform,
                                        const int32_t* top_k_arr, const float* top_p_arr,
                                        int32_t* out, uint8_t* success, int batch_size,
                                        int top_k_val, float top_p_val, int d,
                                        int max_rounds, int deterministic, void* stream);

/*
 * The draws above from logits instead of probabilities: row r's
 * probabilities are those sgl_softmax_temperature would write for the same
 * logits and temperature (computed on the fly, the same bits when its probs
 * buffer is 16-byte aligned), so the samples and success flags equal those
 * of sgl_softmax_temperature followed by the mode's draw; the probabilities
 * are never stored. mode: 0 plain (uniform fp32 [batch_size]), 1 top-k
 * (top_k_f fp32 [batch] or top_k_val), 2 top-p (top_p_arr or top_p_val),
 * 3 top-k + top-p (top_k_i int32 [batch] or top_k_val, and top p); modes
 * 1-3 take uniform fp32 [max_rounds, batch_size] and write success when
 * given. logits_dtype and temperatures as for sgl_softmax_temperature.
 * Replaces: Sampler::sample's probabilities and draw together
 *           (src/engine/engine.cc:306-333: torch::softmax of the scaled
 *           logits, then flashinfer_*_sample_from_probs).
 */
int sgl_sampling_from_logits(const void* logits, int64_t logits_stride_row, int logits_dtype,
                             const float* temperatures, float temperature, const float* uniform,
                             int mode, const float* top_k_f, const int32_t* top_k_i,
                             int top_k_val, const float* top_p_arr, float top_p_val,
                             int32_t* out, uint8_t* success, int batch_size, int d,
                             int max_rounds, void* stream);

/*
 * Any of the draws above with a workspace: the statistics and the first sweep
 * of a small batch's rows then run over many workgroups instead of one per
 * row, with the same samples and success flags, bit for bit. Exactly one of
 * probs (fp32 [batch_size, d], contiguous) and logits is given (an empty batch
 * may have neither: a logits_stride_row of 0 then means probs); the fields are
 * the arguments of sgl_*_sampling_from_probs and sgl_sampling_from_logits
 * (mode as there). workspace: sgl_sampling_workspace_bytes(batch_size, d)
 * bytes (room for every probability as a copy: 9.9 MB at 16 rows of 151,936,
 * 46 MB at 75, at most 338 MB, 80 rows of 2^20), 16-byte aligned, written before
 * it is read; with NULL, or where that function returns 0, each row is one
 * workgroup's. Calls that share a
 * workspace must be stream-ordered.
 * Replaces: Sampler::sample's probabilities and draws (src/engine/engine.cc:306-333).
 */
typedef struct {
  const float* probs;
  const void* logits;
  int64_t logits_stride_row;
  const float* temperatures;
  const float* uniform;
  const float* top_k_f;
  const int32_t* top_k_i;
  const float* top_p_arr;
  int32_t* out;
  uint8_t* success;
  int32_t logits_dtype;
  int32_t mode;
  float temperature;
  float top_p_val;
  int32_t top_k_val;
  int32_t batch_size;
  int32_t d;
  int32_t max_rounds;
} sgl_sampling_args_t;
int64_t sgl_sampling_workspace_bytes(int batch_size, int d);
int sgl_sampling_rows(const sgl_sampling_args_t* args, void* workspace, int64_t workspace_bytes,
                      void* stream);

/*
 * Verification of drafted tokens (speculative sampling), from given random numbers.
 * Request r's drafts are draft_tokens[i] for i in [draft_indptr[r], draft_indptr[r + 1]);
 * its target rows, one more than its drafts, are rows draft_indptr[r] + r on of
 * target_probs (fp32 [num_drafts + batch_size, vocab]; row i of a request: the
 * probabilities of the token after i drafts, as sgl_softmax_temperature writes them for a
 * batch whose q rows are the request's last token and its drafts). draft_probs: the
 * probabilities each draft was drawn from (fp32 [num_drafts, vocab]), or NULL for drafts
 * without any (n-gram lookup, greedy drafts: point masses). Drafts are accepted in order
 * while accept_uniform[i] * q(x) < p(x); the next token is the first j whose running sum
 * of max(p_j - q_j, 0) at the first rejected draft, or of p_j behind the last one, exceeds
 * sample_uniform[r] times the sum (the last j with any weight if rounding leaves none; p
 * where p <= q everywhere; vocab - 1 where p has no positive value). Products, differences
 * and sums in 64 bits; NaN weighs nothing and rejects. Uniforms are in [0, 1).
 * tokens: int32 [num_drafts + batch_size], request r's part starting at draft_indptr[r] + r:
 * the accepted drafts, the drawn token, then -1. accepted: int32 [batch_size], accepted
 * drafts, or -1 (and its tokens left as they were) for a request whose offsets decrease or
 * leave [0, num_drafts]. A draft outside [0, vocab) is rejected. workspace:
 * sgl_verify_workspace_bytes, 16-byte aligned, written before it is read; calls that share
 * one must be stream-ordered. Up to 65,535 requests and 2^24 tokens.
 * Replaces: no counterpart in the reference, whose Sampler draws one token per row
 *           (src/engine/engine.cc:300-345).
 */
typedef struct {
  const float* target_probs;
  const float* draft_probs;
  const int32_t* draft_tokens;
  const int32_t* draft_indptr; /* [batch_size + 1] */
  const float* accept_uniform; /* [num_drafts] */
  const float* sample_uniform; /* [batch_size] */
  int32_t* tokens;
  int32_t* accepted;
  int64_t target_stride_row, draft_stride_row; /* elements, >= vocab */
  int64_t num_drafts;
  int32_t batch_size;
  int32_t vocab;
} sgl_verify_args_t;
int64_t sgl_verify_workspace_bytes(int batch_size, int vocab);
int sgl_verify_drafts(const sgl_verify_args_t* args, void* workspace, int64_t workspace_bytes,
                      void* stream);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif  /* SGL_ATTN_H_ */
