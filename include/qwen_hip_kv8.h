/*
 * K/V cache in 8 bits and the attention over it (exported by libqwen_mi355x.so).
 *
 * The reference has no counterpart: its caches are fp32 rows of 256 (llm_memory_layout.h:130-149).  A cache
 * of this format takes 1/4 of their bytes, and the decode attention, which is bound by reading the cache,
 * takes accordingly less time.
 *
 * Code.  The tokens of a sequence form blocks of QWEN_KV8_BLOCK.  Every (block, KV head) has one scale for K
 * and one for V, a power of two, and int8 codes c; a cached value is c * scale.  Storing rows into a block:
 *   need  = the least power of two >= 2^-126 with max |x| <= 127 need over the block's new rows,
 *           NaN if any of their values is not finite;
 *   scale = need if the block's first token is among the new rows, otherwise the larger of need and the
 *           block's scale so far (NaN stays NaN);
 *   c     = rint(x / scale) for the new rows (ties to even), and where the scale grew
 *           rint(c * old / scale) for the block's earlier rows.
 * So a stored value is within scale / 2 of x, and within scale (of the block as it is read) of it however
 * often the scale grows later.  A NaN scale makes every value of the block read as NaN until the block's
 * first token is stored anew: an overflow stays visible as it does in an fp32 cache.
 *
 * Layout of one layer (token t and dimension d within the block; D = head_dim, 64 or 128):
 *   codes  block j of sequence b and head h starts at byte ((b * blocks + j) * kv_heads + h) * 64 * D
 *          K: t, d at  ((d / 64) * 64 + t) * 64 + d % 64
 *          V: t, d at  d * 64 + 16 * (t / 4 % 4) + 4 * (t / 16) + t % 4
 *   scales [sequences][blocks][kv_heads] fp32
 * K and V are what one wave's loads of 1 KiB feed to the matrix cores as they are: K token-major, V
 * dimension-major with the tokens in the order in which the scores come out of the K product.
 *
 * All data pointers are DEVICE pointers; the structs are read during the call.  Work is queued on `stream`
 * (a hipStream_t of the current device, 0 for the null stream), nothing is allocated or synchronized, and
 * the calls can be captured into a graph.  Calls that use one cache (with a store among them) or one workspace
 * have to be ordered by the caller.  Return value: 0, 1 for an invalid argument, 90 for a HIP runtime
 * failure (qwen_hip_last_error() holds the message).
 */
#ifndef QWEN_HIP_KV8_H
#define QWEN_HIP_KV8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define QWEN_KV8_BLOCK 64

/* Element types of rows. */
#define QWEN_TYPE_F32 0
#define QWEN_TYPE_BF16 1

/* One layer's cache: `sequences` sequences of up to 64 * blocks tokens.  Codes 16-byte aligned. */
typedef struct qwen_kv8_cache {
  int8_t* k;
  int8_t* v;
  float* k_scale;
  float* v_scale;
  int32_t sequences;
  int32_t blocks;
  int32_t kv_heads; /* 1 .. 1024 */
  int32_t head_dim; /* 64 or 128 */
} qwen_kv8_cache;

/* Rows [sequence][token][head][head_dim] with strides in elements; the head_dim values of a row are
 * contiguous, and every row starts at a multiple of 16 bytes (base and strides). */
typedef struct qwen_kv8_rows {
  void* data;
  int64_t seq_stride;
  int64_t token_stride;
  int64_t head_stride;
} qwen_kv8_rows;

/* Stores `rows` new tokens of sequences 0..batch-1: row i of sequence b becomes token positions[b] + i.
 * positions [batch] int32: each sequence's past length.  Sequences with a negative position are left as
 * they are (inactive slots of a padded batch), and so are tokens at or behind 64 * blocks (dropped).
 * Codes behind the last new token keep their bytes.  batch 1 .. 65535, rows 1 .. 2^24 (in all calls). */
int qwen_hip_kv8_store(const qwen_kv8_cache* cache, int type, const qwen_kv8_rows* k, const qwen_kv8_rows* v, int batch,
                       int rows, const int* positions, void* stream);

/* qwen_hip_kv8_load: rows of tokens outside the cache are set to zero instead of left as they are. */
#define QWEN_KV8_ZERO_OUTSIDE 0x1

/* Reads tokens positions[b] .. positions[b] + rows - 1 of sequences 0..batch-1 back into k and v (exact in bf16
 * too: seven bits and a power of two, within bf16's range).  Rows of tokens outside 0 .. 64 * blocks - 1 are
 * left as they are unless `flags` holds QWEN_KV8_ZERO_OUTSIDE.  Tokens that were never stored read as whatever
 * the cache memory holds. */
int qwen_hip_kv8_load(const qwen_kv8_cache* cache, int type, const qwen_kv8_rows* k, const qwen_kv8_rows* v, int batch,
                      int rows, int flags, const int* positions, void* stream);

/* Bytes of workspace that qwen_hip_kv8_attention needs with these arguments (0 is possible). */
int qwen_hip_kv8_attention_workspace(const qwen_kv8_cache* cache, int type, int q_heads, int batch, int rows,
                                     int max_keys, uint64_t* bytes);

/* Causal attention of `rows` query tokens per sequence over the cache, which holds their own K/V rows
 * already (qwen_hip_kv8_store with the same positions): query i of sequence b attends tokens
 * 0 .. positions[b] + i,
 *   out[b][i][h] = sum_t softmax_t(scale * q[b][i][h] . k[t][h / group]) v[t][h / group],
 *   group = q_heads / kv_heads,
 * with fp32 statistics and sums.  QWEN_TYPE_F32 queries enter the matrix products as two fp16 terms (22
 * bits) and so do the probabilities; QWEN_TYPE_BF16 queries and their probabilities as one.  The codes are
 * exact in fp16.  A query without a token to attend (a negative position) gives zeros.
 *   q_heads    a multiple of kv_heads, at most 64 query heads a KV head
 *   rows       rows * q_heads / kv_heads and batch * kv_heads: at most 2^22 each
 *   max_keys   host int >= max(positions) + rows, at most 64 * blocks (sizes the split over the keys); tokens
 *              at or behind it are not attended
 *   workspace  16-byte aligned, qwen_hip_kv8_attention_workspace bytes; contents need not be kept
 * q and out may be the same rows. */
int qwen_hip_kv8_attention(const qwen_kv8_cache* cache, int type, const qwen_kv8_rows* q, const qwen_kv8_rows* out,
                           int q_heads, int batch, int rows, const int* positions, int max_keys, float scale,
                           void* workspace, uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QWEN_HIP_KV8_H */
