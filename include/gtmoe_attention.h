/*
 * gtmoe_attention.h -- the decoder remainder around the MoE block for batch-1 decode (C ABI):
 * embedding lookup, the per-head q/k/v epilogue and attention over the FP32 ring KV cache.
 *
 * Replaces, for one token of ForwardRunner::produce_token (src/runner.cpp:487-533), the
 * EmbedLookup, QKVEpilogue and Attention dispatches (shaders/EmbedLookup.hlsl,
 * shaders/QKVEpilogue.hlsl, shaders/Attention.hlsl); the q/k/v/o projections stay on
 * gtm_gemv_q4 (GemvInt4). Arithmetic contract: src/cpu_reference.cpp:108-140, 322-417.
 * KV rows live where KVCacheManager puts them (src/kv_cache.cpp:36-50): position p of a layer
 * in row p % capacity, each row kv_heads * head_dim floats.
 *
 * Checked on a B200 against the reference's kernel-test known answers (EmbedLookup bit-identical,
 * QKVEpilogue and Attention with window and ring wrap within its allclose rule) and, chained with
 * the MoE block and the greedy LM head, against the reference's own generate tokens.
 */
#ifndef GTMOE_ATTENTION_H
#define GTMOE_ATTENTION_H

#include "gtmoe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* EmbedLookup (cpu_reference.cpp:322-330): out[c] = (q[token][c] * s + b) * scale, int4 MLX
 * affine rows of in_dim elements (group 64). Bit-identical to the CPU reference with
 * scale = sqrtf(in_dim). */
GTM_API int gtm_embed_lookup(uint32_t rows, uint32_t in_dim, const void* w_dev, const uint16_t* s_dev,
                             const uint16_t* b_dev, uint32_t token, float scale, float* out_dev, void* stream);

/* QKVEpilogue (cpu_reference.cpp:360-376): for each of `heads` vectors of head_dim floats, an
 * RMS norm with bf16 weight w_dev (NULL = no scale), then NeoX RoPE of the first rotated_pairs
 * pairs at `position` with base theta (rotated_pairs = 0: no rotation). in_dev and out_dev may
 * be the same buffer; out_dev may point into a KV cache row. head_dim in {128, 256, 512}. */
GTM_API int gtm_qkv_epilogue(uint32_t heads, uint32_t head_dim, const float* in_dev, const uint16_t* w_dev, float eps,
                             uint32_t rotated_pairs, uint32_t position, float theta, float* out_dev, void* stream);

/* Workspace for gtm_attention_decode with at most `max_window` attended positions. */
GTM_API size_t gtm_attention_workspace_bytes(uint32_t q_heads, uint32_t head_dim, uint32_t max_window);

/* Attention (cpu_reference.cpp:382-414): for each query head h (kv head h / (q_heads /
 * kv_heads)), scores q.k with scale 1.0 over positions [first, n_pos), softmax, and the
 * weighted sum of V into ctx_dev [q_heads * head_dim]. Position t is cache row t % capacity.
 * q_heads a multiple of kv_heads with q_heads / kv_heads <= 8; head_dim in {128, 256, 512};
 * first < n_pos; n_pos - first <= capacity. */
GTM_API int gtm_attention_decode(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n_pos,
                                 uint32_t first, uint32_t capacity, const float* q_dev, const float* k_cache_dev,
                                 const float* v_cache_dev, float* ctx_dev, void* workspace_dev, size_t workspace_bytes,
                                 void* stream);

/* ---------------------------------------------------------------------------------------
 * The same steps for n sequences at once (a batched decode step; the reference decodes one
 * sequence per produce_token call, runner.cpp:487-533). Row i of every [n][...] array belongs to
 * the i-th sequence of the step; per-row token ids, positions and sequence indices are HOST
 * arrays of n values (n <= 512), checked on the host and passed to the kernels by value. Every
 * row's result is bit-identical to the single-sequence entry on that row.
 * ------------------------------------------------------------------------------------- */
/* EmbedLookup of tokens[i] into out_dev row i ([n][in_dim]). */
GTM_API int gtm_embed_lookup_rows(uint32_t rows, uint32_t in_dim, const void* w_dev, const uint16_t* s_dev,
                                  const uint16_t* b_dev, const uint32_t* tokens, uint32_t n, float scale, float* out_dev,
                                  void* stream);
/* QKVEpilogue of in_dev row i ([n][heads * head_dim]) at positions[i]. capacity = 0: into out_dev
 * row i (out may be in). capacity > 0: into ring row positions[i] % capacity of the cache of
 * sequence seqs[i] < num_seqs, the caches laid out [num_seqs][capacity][heads * head_dim]. */
GTM_API int gtm_qkv_epilogue_rows(uint32_t heads, uint32_t head_dim, uint32_t n, const float* in_dev,
                                  const uint16_t* w_dev, float eps, uint32_t rotated_pairs, const uint32_t* positions,
                                  float theta, float* out_dev, const uint32_t* seqs, uint32_t num_seqs,
                                  uint32_t capacity, void* stream);
/* Workspace of gtm_attention_decode_rows for n rows attending at most max_window positions. */
GTM_API size_t gtm_attention_rows_workspace_bytes(uint32_t q_heads, uint32_t head_dim, uint32_t max_window,
                                                  uint32_t n);
/* Attention of q_dev row i ([n][q_heads * head_dim]) over the caches of sequence seqs[i]
 * ([num_seqs][capacity][kv_heads * head_dim]) at position positions[i]: positions
 * [first, positions[i]] with first = max(0, positions[i] + 1 - window) (window 0 = all), into
 * ctx_dev row i. The attended span must fit the ring (<= capacity). */
GTM_API int gtm_attention_decode_rows(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n,
                                      uint32_t window, uint32_t capacity, const float* q_dev, const float* k_cache_dev,
                                      const float* v_cache_dev, const uint32_t* seqs, uint32_t num_seqs,
                                      const uint32_t* positions, float* ctx_dev, void* workspace_dev,
                                      size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------------------
 * One-byte ring KV caches for serving many sequences (no counterpart in the reference, whose
 * caches are fp32): written in the pass that norms and rotates a step's queries and keys, read
 * back, and attended with one prefix shared by all rows of a step.
 *
 * A vector is head_dim values of one position and kv head, held as head_dim one-byte codes and
 * one fp32 scale; a value is code * scale. With M = 127 (GTM_KV_INT8: codes -127..127) or 448
 * (GTM_KV_E4M3: 8-bit floats with 4 exponent and 3 fraction bits, no infinity), scale =
 * fp32(max(max|y| / M, 2^-100)) and code = y / scale rounded to nearest, ties to even. A vector
 * holding an infinity or NaN has the scale NaN and codes 0, and reads back as NaN.
 * Position t of a sequence is ring row t % capacity, as in the fp32 caches.
 * ------------------------------------------------------------------------------------- */
enum { GTM_KV_INT8 = 0, GTM_KV_E4M3 = 1 };

typedef struct GtmKvCache {
    void* k_dev;                 /* codes [num_seqs][capacity][kv_heads][head_dim], 16-byte aligned */
    void* v_dev;
    float* k_scale_dev;          /* [num_seqs][kv_heads][capacity]                                  */
    float* v_scale_dev;          /* attention takes scales in [2^-100, 2^20] (and NaN)              */
    uint32_t format;             /* GTM_KV_*                                                        */
    uint32_t num_seqs, capacity, kv_heads, head_dim;   /* head_dim 128, 256 or 512                  */
    uint32_t reserved;           /* 0                                                               */
} GtmKvCache;

/* QKVEpilogue of n rows' queries, keys and values in one launch, keys and values going into the
 * cache: row i (n <= 512, i-th row of q_dev, k_dev and v_dev, whose rows are *_stride floats
 * apart) belongs to sequence seqs[i] at positions[i] (HOST arrays, as in the *_rows entries: read
 * during the call, so a captured launch keeps the values it was captured with).
 *   q: RMS norm per head with weight q_w_dev (bf16, NULL = none), rotation -> q_out_dev
 *      [n][q_heads * head_dim] (q_out_dev may be q_dev where q_stride is q_heads * head_dim; any
 *      other overlap with an input's rows is refused)
 *   k: RMS norm with k_w_dev, rotation -> cache;   v: RMS norm without a weight -> cache
 * v_dev may be k_dev. The rotation is NeoX over the first rotated_pairs pairs, angle position *
 * theta^(-2i / head_dim). Norms, angles and the codes' rounding are in 64 bits, each result
 * rounded once, so codes do not depend on the order of a sum and far positions keep their angles
 * (gtm_qkv_epilogue forms both in fp32, as the reference does). Two rows with the same ring row
 * are refused. */
GTM_API int gtm_qkv_cache_rows(const GtmKvCache* cache, uint32_t q_heads, uint32_t n, const float* q_dev,
                               const float* k_dev, const float* v_dev, uint64_t q_stride, uint64_t k_stride,
                               uint64_t v_stride, const uint16_t* q_w_dev, const uint16_t* k_w_dev, float eps,
                               uint32_t rotated_pairs, float theta, const uint32_t* positions, const uint32_t* seqs,
                               float* q_out_dev, void* stream);
/* Positions [first, first + count) of sequence `seq` as fp32 into k_out_dev and v_out_dev
 * [count][kv_heads * head_dim] (either may be NULL); count <= capacity. */
GTM_API int gtm_kv_read(const GtmKvCache* cache, uint32_t seq, uint32_t first, uint32_t count, float* k_out_dev,
                        float* v_out_dev, void* stream);
/* Workspace of gtm_attention_kv_rows for at most n rows (0 for unsupported shapes). Its first 4
 * bytes are an error word: zero them once before the first use where gtm_attention_kv_check is to
 * be called; the rest needs no initialisation. Its size depends on the current device's number of
 * SMs (a B200's where there is no device). A workspace serves one stream at a time; two captured
 * graphs may share one if their replays do not overlap. */
GTM_API size_t gtm_attention_kv_workspace_bytes(uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t n);
/* Attention of n rows (n <= 512) at positions[i] of sequences seqs[i] (HOST arrays): row i attends
 * [first, positions[i]] with first = max(0, positions[i] + 1 - window) (window 0 = all), scores
 * q.k with scale 1.0, softmax, weighted V into ctx_dev row i. Positions below prefix_len are read
 * from sequence prefix_seq of `prefix` (row t % its capacity), the others from sequence seqs[i] of
 * `cache`; a prefix long enough is read and multiplied once for all rows. prefix_len 0: no prefix
 * (`prefix` may be NULL). Rows of one sequence's prompt are attended causally by giving that
 * sequence's own cache as the prefix, with prefix_len one past the last row's position.
 * `prefix` has the cache's format, kv_heads and head_dim. A row's span must fit the rings: its
 * own positions within capacity, and prefix_len - first within the prefix's. q_heads a multiple of
 * kv_heads, at most 8 query heads per kv head. q_dev and ctx_dev [n][q_heads * head_dim], one buffer
 * or two that do not overlap. Scores are fp32, off by at most 2^-17 of the sum of |q_d k_d| over a
 * head's dims and 2^-39 of max |q| times the sum of |k_d| (q and the softmax weights are multiplied
 * as two fp16 limbs, 22 bits): |q| below 2^100, and the first sum up to 2^20 for every attended key,
 * beyond which a row may be NaN (its stabiliser's steps would pass 1/8).
 * Outputs were within 6.3e-6 of 64-bit ones (2-norm, 32,768 positions; a plain fp32 form 4.4e-6).
 * Codes that a caller brings are taken as numbers: an e4m3 0x7F or 0xFF (NaN, which gtm_kv_read
 * gives) counts as 480 here. Infinities, NaN and whatever else the rings hold outside a row's span
 * do not reach it. The waits on the device are bounded: should one run out (1 s), the rows that it
 * served are NaN, and the next gtm_attention_kv_check on the workspace says so. */
GTM_API int gtm_attention_kv_rows(const GtmKvCache* cache, const GtmKvCache* prefix, uint32_t prefix_seq,
                                  uint32_t prefix_len, uint32_t q_heads, uint32_t n, uint32_t window,
                                  const float* q_dev, const uint32_t* seqs, const uint32_t* positions, float* ctx_dev,
                                  void* workspace_dev, size_t workspace_bytes, void* stream);
/* Reads back and clears a workspace's error word after gtm_attention_kv_rows calls (synchronises
 * `stream`). Returns GTM_OK or GTM_ERR_TIMEOUT. */
GTM_API int gtm_attention_kv_check(void* workspace_dev, void* stream);
/* Test hook for the bounded waits: in the calling thread's next gtm_attention_kv_rows, where the
 * prefix is computed once for all rows, one warp of every CTA first waits for an arrival that never
 * comes, under a 2 ms limit instead of 1 s; it gives up, the other roles leave through the CTA's
 * abort flag, copies in flight are waited for and tensor memory is freed. Rows with positions in the
 * prefix are NaN, gtm_attention_kv_check reports GTM_ERR_TIMEOUT, and the workspace stays usable. */
GTM_API int gtm_attention_kv_test_wait(void);

#ifdef __cplusplus
}
#endif
#endif
