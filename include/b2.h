/*
 * b2.h — C ABI of the B200-native (sm_100a) hot-path kernels.
 *
 * Every entry point takes plain device pointers, sizes and a cudaStream_t
 * passed as void*.  Nothing here allocates device memory; the caller owns
 * every buffer, including the output (the convention of the reference's
 * Metal templates, where the caller binds every buffer by index:
 * triton_metal/codegen/_msl_templates.py:2705-2712 for INT4/INT8,
 * :1625-1630 for FlashAttention, :2086-2091 for GQA decode).
 *
 * Return value: B2_OK (0) or a negative B2_ERR_* code.  The message of the
 * last failure on the calling thread is returned by b2_last_error().
 * All launches are asynchronous on the given stream; no host sync inside.
 */
#ifndef B2_H_
#define B2_H_

#include <stdint.h>
#include <stddef.h>

#if defined(__GNUC__)
#define B2_API __attribute__((visibility("default")))
#else
#define B2_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define B2_OK               0
#define B2_ERR_INVALID    (-1)  /* bad shape / argument */
#define B2_ERR_DTYPE      (-2)  /* unsupported dtype combination */
#define B2_ERR_ALIGN      (-3)  /* pointer or stride alignment */
#define B2_ERR_UNSUPPORTED (-4) /* valid but not implemented shape */
#define B2_ERR_LAUNCH     (-5)  /* CUDA launch / runtime error */
#define B2_ERR_TIMEOUT    (-6)  /* a bounded device wait ran out */

/* dtype codes for activations / scales / outputs */
#define B2_F16  0
#define B2_BF16 1
#define B2_F32  2

/* int4 weight layouts */
#define B2_LAYOUT_GPTQ 0  /* int32 [K/8, N], nibble j of a word = k%8 == j   */
#define B2_LAYOUT_REF  1  /* uint8 [N, K/2], low nibble = even k (reference) */

B2_API int         b2_version(void);
B2_API const char* b2_last_error(void);
/* Synchronise `stream`, then read and clear the device error word that the
 * kernels' bounded waits set instead of hanging.  *code (may be NULL)
 * receives the raw code.  Returns B2_OK or B2_ERR_TIMEOUT.  Counterpart of
 * the reference's command-buffer status check
 * (triton_metal/backend/driver.py:218-225). */
B2_API int b2_device_error(void* stream, unsigned int* code);

/*
 * W4A16 group-wise weight-only matmul: output[M,N] = input[M,K] @ W
 * with W[k,n] = (q[k,n] - z[k/G,n]) * scales[k/G,n].
 * Replaces the reference kernel int4_matmul
 * (triton_metal/codegen/_msl_templates.py:2682-2745, buffer order
 * input, weight, output, scales, zeros, M, N, K at :2705-2712).
 *   weight  : B2_LAYOUT_GPTQ int32 [K/8, N]
 *   scales  : dtype [K/G, N]
 *   zeros   : NULL -> symmetric zero point 8 (the layout's default);
 *             else dtype [K/G, N] zero points (asymmetric).
 *   dtype   : B2_F16 or B2_BF16 for input, scales, zeros and output: the
 *             decode GEMV (M <= 16) or the tcgen05 prefill GEMM (M > 16);
 *             B2_F32 (the reference's own dtype) for input, scales, zeros
 *             and output: the reference's arithmetic, (q - z) * s and every
 *             product in fp32 on CUDA cores (K % 8 == 0, G % 8 == 0).
 */
B2_API int b2_int4_matmul(const void* input, const void* weight, void* output,
                   const void* scales, const void* zeros,
                   int64_t M, int64_t N, int64_t K, int64_t group_size,
                   int dtype, void* stream);

/*
 * W8A16 per-channel weight-only matmul: output[M,N] = input[M,K] @ W,
 * W[k,n] = (w8[n,k] - zeros[n]) * scales[n].
 * Replaces int8_matmul (triton_metal/codegen/_msl_templates.py:2630-2679,
 * buffer order input, weight, output, scales, zeros, M, N, K at :2652-2661).
 *   weight  : int8 [N, K] (K-major, the reference layout)
 *   scales  : dtype [N];  zeros: NULL (symmetric) or dtype [N].
 *   dtype   : B2_F16 / B2_BF16 (tensor cores), or B2_F32 (the reference's
 *             dtype: fp32 (w - z) * s and fp32 products, K % 8 == 0).
 */
B2_API int b2_int8_matmul(const void* input, const void* weight, void* output,
                   const void* scales, const void* zeros,
                   int64_t M, int64_t N, int64_t K,
                   int dtype, void* stream);

/*
 * int4_matmul in the reference's own buffers and layouts, natively
 * (make_int4_matmul_kernel, _msl_templates.py:2682-2745; buffer order
 * :2705-2712): weight uint8 [N, K/2], byte j of row n = k 2j (low nibble)
 * and 2j+1 (high nibble) (:2725-2732); scales and zeros [N, K/G] in the
 * activation dtype (zeros NULL = 8); input [M, K], output [M, N].
 * 16-bit dtypes: M <= 16: K-major mma.sync GEMV (K % 128 == 0, G % 32 ==
 * 0); M > 16: the tcgen05 prefill GEMM (K % 64 == 0, G % 64 == 0); else a
 * generic kernel.  B2_F32 (the reference's buffers as they are): fp32
 * scales / zeros / output and the reference's fp32 arithmetic.
 */
B2_API int b2_int4_matmul_ref(const void* input, const void* weight, void* output,
                              const void* scales, const void* zeros,
                              int64_t M, int64_t N, int64_t K, int64_t group_size,
                              int dtype, void* stream);

/*
 * Plain bf16 GEMM on tcgen05: out[M,N] = x[M,K] @ w[N,K]^T (w K-major, the
 * nn.Linear layout), fp32 accumulate, bf16 out.  The dequantised-weight
 * path of the reference's matmuls (x @ dequant(W), _msl_templates.py:2663,
 * :2716) when W is already bf16.  Any M; needs N % 8 == 0, K % 64 == 0
 * and 16-byte aligned pointers.
 */
B2_API int b2_gemm_bf16(const void* x, const void* w, void* out,
                        int64_t M, int64_t N, int64_t K, void* stream);

/*
 * Exact int4 -> fp32 dequantisation W[k,n] = (q - z) * float(s), written
 * as fp32 [K, N].  Debug/parity export of the unpack + dequant step the
 * reference does per k inside int4_matmul (_msl_templates.py:2723-2737).
 */
B2_API int b2_int4_dequant(const void* weight, const void* scales, const void* zeros,
                    float* out, int64_t N, int64_t K, int64_t group_size,
                    int dtype, void* stream);

/*
 * Repack the reference int4 layout uint8 [N, K/2] (low nibble = even k,
 * _msl_templates.py:2725-2732) into the GPTQ layout int32 [K/8, N].
 */
B2_API int b2_int4_repack_ref_to_gptq(const void* ref_weight, void* gptq_weight,
                               int64_t N, int64_t K, void* stream);

/*
 * Host plan of the W4 decode GEMV (M <= 16) for one shape; no device work.
 * info[6] = {grid, 8-column tiles per CTA slab, CTAs with one extra tile,
 * ring stages, quantisation groups per TMA box, shared-memory bytes} for a
 * GPU with `sms` SMs.  B2_ERR_UNSUPPORTED when the streaming GEMV does not
 * take the shape (b2_int4_matmul then runs the generic kernel).
 */
B2_API int b2_w4_gemv_plan(int64_t M, int64_t N, int64_t K, int64_t group_size, int zeros, int sms,
                           int64_t* info);

/*
 * FlashAttention forward.  q [B, Hq, S, D], k/v [B, Hkv, S, D], o like q,
 * each with arbitrary element strides (b, h, s; the last dim contiguous).
 * GQA maps q head h to kv head h / (Hq/Hkv), the reference's head map
 * (_msl_templates.py:2101-2104).  Replaces flash_attention
 * (_msl_templates.py:1568-1767, buffers Q, K, V, O, seq_len, scale) and the
 * strided Triton form _flash_attn_fwd (tests/test_flash_attention.py:24-104).
 *   dtype : B2_BF16 / B2_F16 (tcgen05 path) or B2_F32 (fp32 in/out).
 */
B2_API int b2_flash_attn_fwd(const void* q, const void* k, const void* v, void* o,
                      int64_t B, int64_t Hq, int64_t Hkv,
                      int64_t Sq, int64_t Skv, int64_t D,
                      const int64_t* q_strides, const int64_t* k_strides,
                      const int64_t* v_strides, const int64_t* o_strides,
                      float scale, int causal, int dtype, void* stream);

/*
 * Causal sliding-window FlashAttention (prefill): query s attends to keys
 * s - window + 1 .. s (window > 0; Sq == Skv).  Same tensors and strides as
 * b2_flash_attn_fwd; the prefill form of sliding_window_attention
 * (_msl_templates.py:3335-3431).  tcgen05 kernel for D = 128 bf16/fp16.
 */
B2_API int b2_flash_attn_fwd_window(const void* q, const void* k, const void* v, void* o,
                                    int64_t B, int64_t Hq, int64_t Hkv,
                                    int64_t Sq, int64_t Skv, int64_t D,
                                    const int64_t* q_strides, const int64_t* k_strides,
                                    const int64_t* v_strides, const int64_t* o_strides,
                                    float scale, int64_t window, int dtype, void* stream);

/*
 * FlashAttention forward with more masks and score forms (the reference has
 * the causal mask only).  Tensors, strides and dtypes as in b2_flash_attn_fwd.
 *   s = scale q.k; softcap > 0: s = softcap tanh(s / softcap);
 *   alibi_slopes fp32 [Hq] or NULL: s -= slope[h] |query - key|.
 *   causal, window (> 0 needs causal): as in b2_flash_attn_fwd_window.
 *   doc_offsets int32 [B, n_docs + 1] ascending, or NULL (needs Sq == Skv):
 *     tokens off[d] .. off[d + 1] - 1 are document d; a query sees only keys of
 *     its document.  Tokens in no document (padding) see nothing.
 *   prefix_lens int32 [B, n_docs] (without documents [B]) or NULL (needs causal,
 *     no window): the first prefix_lens tokens of a document are seen by all
 *     of its queries, the rest causally.
 * Rows that see nothing give 0, and hidden keys do not count whatever their
 * values.  fp16 / bf16 with D = 64 or 128 and 16-byte aligned rows run on
 * tcgen05, the rest (fp32 kept in fp32) on the CUDA cores; D <= 256.
 */
B2_API int b2_flash_attn_fwd_scored(const void* q, const void* k, const void* v, void* o,
                                    int64_t B, int64_t Hq, int64_t Hkv,
                                    int64_t Sq, int64_t Skv, int64_t D,
                                    const int64_t* q_strides, const int64_t* k_strides,
                                    const int64_t* v_strides, const int64_t* o_strides,
                                    float scale, int causal, int64_t window, float softcap,
                                    const float* alibi_slopes, const int32_t* doc_offsets,
                                    int64_t n_docs, const int32_t* prefix_lens, int dtype,
                                    void* stream);

/*
 * Decode attention: one query token per head over a KV cache, split-KV.
 * Replaces kv_cache_attention, gqa_attention, batched_kv_decode,
 * paged_attention, multi_head_paged_attention and fp16_kv_attention
 * (triton_metal/codegen/_msl_templates.py:1949-2627).
 *   q [B, Hq, D] (q_dtype), o like q.
 *   page_size == 0: contiguous K/V [B, Hkv, S, D], k/v_strides = element
 *                   strides (b, h, s).
 *   page_size  > 0: paged K/V [n_pages, page_size, Hkv, D], page_table
 *                   int32 [B, max_pages] (logical -> physical page),
 *                   k/v_strides = element strides (page, token, head).
 *   seq_lens int32 [B] (<= max_seq_len); kv head of q head h = h / (Hq/Hkv).
 *   kv_dtype may differ from q_dtype (fp16 KV with fp32 queries).
 *   q_pos int32 [B] or NULL (= seq_len - 1): the query's position.
 *   window > 0: keys [max(0, q_pos + 1 - window), min(q_pos + 1, seq_len))
 *     (sliding_window_attention, _msl_templates.py:3335-3431); 0: [0, seq_len).
 *   rope_freqs fp32 [D/2] or NULL: rotate q at q_pos and key j at j, pairs
 *     (2d, 2d + 1) by pos * rope_freqs[d] (rope_attention, :1770-1887).
 *   workspace: b2_decode_attn_workspace_size(...) bytes (NULL when it is 0).
 */
B2_API size_t b2_decode_attn_workspace_size(int64_t B, int64_t Hq, int64_t Hkv,
                                            int64_t D, int64_t max_seq_len);
B2_API int b2_decode_attn(const void* q, const void* k, const void* v, void* o,
                          const int32_t* page_table, const int32_t* seq_lens,
                          void* workspace, int64_t B, int64_t Hq, int64_t Hkv,
                          int64_t D, int64_t max_seq_len, int64_t page_size,
                          int64_t max_pages, const int64_t* k_strides,
                          const int64_t* v_strides, const int32_t* q_pos,
                          int64_t window, const float* rope_freqs, float scale,
                          int q_dtype, int kv_dtype, void* stream);

/*
 * b2_decode_attn with capped and biased scores: softcap > 0: s = softcap
 * tanh(s / softcap); alibi_slopes fp32 [Hq] or NULL: s -= slope[h] |q_pos -
 * key|.  n_pages: pages of a paged cache; a page number outside [0, n_pages)
 * reads as zeros and is recorded in the device error word.
 *   workspace: b2_decode_attn_scored_workspace_size(...) bytes, 16-byte aligned,
 *   when softcap or alibi_slopes is given (else b2_decode_attn_workspace_size).
 */
B2_API size_t b2_decode_attn_scored_workspace_size(int64_t B, int64_t Hq, int64_t Hkv,
                                                   int64_t D, int64_t max_seq_len);
B2_API int b2_decode_attn_scored(const void* q, const void* k, const void* v, void* o,
                                 const int32_t* page_table, const int32_t* seq_lens,
                                 void* workspace, int64_t B, int64_t Hq, int64_t Hkv,
                                 int64_t D, int64_t max_seq_len, int64_t page_size,
                                 int64_t max_pages, int64_t n_pages,
                                 const int64_t* k_strides, const int64_t* v_strides,
                                 const int32_t* q_pos, int64_t window,
                                 const float* rope_freqs, float scale, float softcap,
                                 const float* alibi_slopes, int q_dtype, int kv_dtype,
                                 void* stream);

/*
 * repeat_kv (make_repeat_kv_kernel, _msl_templates.py:3434-3480):
 *   out[h, s, d] = in[h / n_rep, s, d]; in [n_kv_heads, seq_len, head_dim],
 *   out [n_kv_heads * n_rep, seq_len, head_dim], elements of elem_bytes.
 */
B2_API int b2_repeat_kv(const void* input, void* output, int64_t n_kv_heads,
                        int64_t seq_len, int64_t head_dim, int64_t n_rep,
                        int64_t elem_bytes, void* stream);

/*
 * Attention of a tree of drafted tokens over a KV cache (speculative
 * decoding; no counterpart in the reference).  Request b has context_lens[b]
 * tokens in the cache, then its drafted tokens, whose K/V stand behind them at
 * positions context_lens[b] + j, j < draft_lens[b] (NULL: T for every request).
 *   q [B, T, Hq, D] and o like it, element strides (b, t, h).
 *   K/V contiguous [B, Hkv, S, D] (strides b, h, s; page_size 0, max_keys = S)
 *   or paged [n_pages, page_size, Hkv, D] (strides page, token, head) with
 *   page_table int32 [B, max_pages] (max_keys = max_pages * page_size), as in
 *   b2_decode_attn.  A page number outside [0, n_pages) reads as zeros and is
 *   recorded in the device error word (b2_device_error).
 *   tree_mask uint8 [T, T] (mask_stride 0) or [B, T, T] (mask_stride T * T):
 *   drafted token t sees drafted token j iff tree_mask[t, j] != 0; every
 *   drafted token sees the whole context.
 *   scores: s = scale q.k; softcap > 0: s = softcap tanh(s / softcap).
 * Rows t >= draft_lens[b] and rows that see nothing give 0.  Lengths are
 * clamped to the cache.  workspace: b2_tree_attn_workspace_size(...) bytes
 * (may be NULL when it is 0), 16-byte aligned; one per call in flight.
 */
B2_API size_t b2_tree_attn_workspace_size(int64_t B, int64_t T, int64_t Hq, int64_t Hkv,
                                          int64_t D, int64_t max_keys, int q_dtype,
                                          int kv_dtype);
B2_API int b2_tree_attn(const void* q, const void* k, const void* v, void* o,
                        const int32_t* page_table, const int32_t* context_lens,
                        const int32_t* draft_lens, const uint8_t* tree_mask,
                        int64_t mask_stride, void* workspace, int64_t B, int64_t T,
                        int64_t Hq, int64_t Hkv, int64_t D, int64_t max_keys,
                        int64_t page_size, int64_t max_pages, int64_t n_pages,
                        const int64_t* q_strides, const int64_t* k_strides,
                        const int64_t* v_strides, const int64_t* o_strides,
                        float scale, float softcap, int q_dtype, int kv_dtype,
                        void* stream);

/*
 * Page table and slot map of one step of a paged cache, on the GPU from the
 * request lengths (no counterpart in the reference, whose host fills both).
 * Request b holds context_lens[b] tokens and gets new_lens[b] more (int32 [B];
 * negative counts as 0).  In one launch:
 *   page_table int32 [B, max_pages] (rows table_stride apart): the pages that
 *     the new tokens open are taken from free_pages (int32 [n_free]) in request
 *     order and written behind the pages the request holds; other entries stay.
 *   slots int64 [max_tokens]: page * page_size + offset of each new token, the
 *     requests' tokens one after another; -1 behind the last one, for a token
 *     whose page lies behind max_pages and for one that found no free page
 *     (its table entry is -1 as well).  max_tokens has to be at least the sum
 *     of new_lens (< 2^31): tokens behind it are dropped, with the pages that
 *     they would open.
 *   offsets int32 [B + 1]: first token of each request; offsets[B] = the sum.
 *   pages_used int32 [1]: pages wanted from free_pages (> n_free: too few).
 */
B2_API int b2_build_page_table(const int32_t* context_lens, const int32_t* new_lens,
                               const int32_t* free_pages, int32_t* page_table,
                               int64_t* slots, int32_t* offsets, int32_t* pages_used,
                               int64_t B, int64_t page_size, int64_t n_free,
                               int64_t max_pages, int64_t table_stride,
                               int64_t max_tokens, void* stream);

/*
 * New K/V rows into a paged cache by slot: k / v [N, Hkv, D] (element strides
 * row, head) to k_pages / v_pages [n_pages, page_size, Hkv, D] (element strides
 * page, token, head), row r to slot slots[r] (int64).  Slots outside
 * [0, n_pages * page_size) are passed over.  A slot may occur once: which of
 * several rows with one slot stays is not defined.  Rows and cache share one
 * dtype, or fp32 rows are rounded to nearest into an fp16 / bf16 cache.  A
 * contiguous cache [B, Hkv, S, D] is pages of size S: strides (b, s, h).
 */
B2_API int b2_store_kv(const void* k, const void* v, void* k_pages, void* v_pages,
                       const int64_t* slots, int64_t N, int64_t Hkv, int64_t D,
                       int64_t n_pages, int64_t page_size, const int64_t* k_strides,
                       const int64_t* v_strides, const int64_t* kp_strides,
                       const int64_t* vp_strides, int src_dtype, int dst_dtype,
                       void* stream);

/*
 * KDA (chunked gated delta rule) forward.  No reference counterpart: the
 * reference has no KDA code.  Layout [B, T, H, D] contiguous:
 *   q, k, v : dtype (B2_BF16) [B,T,H,Dk|Dv];  g : fp32 [B,T,H,Dk] log-decay
 *   beta    : dtype [B,T,H];  initial_state : fp32 [B,H,Dk,Dv] or NULL
 *   o       : dtype [B,T,H,Dv];  final_state : fp32 [B,H,Dk,Dv] or NULL
 *   workspace: device scratch of b2_kda_workspace_size(...) bytes
 *             (80,384 bytes per (b, h, 64-step chunk)), 16-byte aligned.
 * Two kernels: a per-chunk WY/UT transform on tcgen05 and the state +
 * output recurrence on clusters of two CTAs (one carries the state, its
 * partner computes the outputs); the state is carried in fp32.
 */
B2_API size_t b2_kda_workspace_size(int64_t B, int64_t T, int64_t H,
                             int64_t Dk, int64_t Dv, int64_t chunk);
B2_API int b2_kda_fwd(const void* q, const void* k, const void* v, const float* g,
               const void* beta, const float* initial_state,
               void* o, float* final_state, void* workspace,
               int64_t B, int64_t T, int64_t H, int64_t Dk, int64_t Dv,
               int64_t chunk, float scale, int dtype, void* stream);

/*
 * b2_kda_fwd without a workspace argument, for callers that cannot allocate
 * device memory when they run KDA (e.g. inside a custom allocator or memory
 * pool that must not be re-entered, or a plugin host that only provides the
 * input and output buffers).  No counterpart in the reference (which has no
 * KDA at all).  The workspace is a fixed 64 MiB device array inside the
 * library that every GPU loading it keeps until exit; shapes needing more
 * (B*H*(T/64) > 834 chunk-heads) are rejected with B2_ERR_INVALID.  The first call on a
 * device looks up the array's address (do it before any stream capture).
 * All calls share the array: calls overlapping on the GPU race.
 */
B2_API int b2_kda_fwd_noalloc(const void* q, const void* k, const void* v, const float* g,
                              const void* beta, const float* initial_state,
                              void* o, float* final_state,
                              int64_t B, int64_t T, int64_t H, int64_t Dk, int64_t Dv,
                              int64_t chunk, float scale, int dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* B2_H_ */
