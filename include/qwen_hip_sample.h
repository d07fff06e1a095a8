/*
 * Drawing tokens from logits (exported by libqwen_mi355x.so): temperature, top-k, top-p and min-p, with the
 * random numbers given by the caller.
 *
 * The reference has no counterpart: its driver takes the argmax
 * (verification/qwen_full_model_validation.py:128,159), as qwen_hip_model_greedy does.
 *
 * Row r of logits x, with T = temperature[r], k = top_k[r], p = top_p[r], q = min_p[r], u = uniforms[r]:
 *   1. T not above 0 (NaN included), or a maximal logit that is not finite: the token is the first index of
 *      the maximum (NaN counts as the maximum), as qwen_hip_model_greedy.
 *   2. w_i = exp((x_i - max x) / T).
 *   3. Tokens in order of falling x, equal ones (-0 and +0 are equal) by rising index: the first k are kept
 *      (all, when k <= 0);
 *   4. of those, the ones before which the kept weights sum to less than p times their total, and the
 *      first in any case (all, when p >= 1 or NaN);
 *   5. of those, the ones with w_i >= min(q, 1) (all, when q <= 0 or NaN).
 *   6. The token is the lowest index i at which the sum of the kept weights up to and including i exceeds u
 *      times their total (u clamped to [0, 1], NaN as 0; the last kept token where none does).
 * exp is taken in 64 bits and each weight rounded to a multiple of 2^-min(50, 62 - ceil(log2 vocab)) (2^-44 for
 * 151936 tokens), so all sums are exact integers: the result does not depend on the order in which they are formed.
 *
 * All data pointers are DEVICE pointers; work is queued on `stream` (a hipStream_t of the current device, 0 for
 * the null stream), nothing is allocated or synchronized, and the call can be captured into a graph.  Calls
 * that use one workspace have to be ordered by the caller.  Return value: 0, 1 for an invalid argument, 90
 * for a HIP runtime failure (qwen_hip_last_error() holds the message).
 */
#ifndef QWEN_HIP_SAMPLE_H
#define QWEN_HIP_SAMPLE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of workspace that qwen_hip_sample needs. */
int qwen_hip_sample_workspace(int rows, int vocab, uint64_t* bytes);

/* logits: `rows` (1 .. 65535) rows of `vocab` (1 .. 2^24) values of `type` (QWEN_TYPE_F32 or QWEN_TYPE_BF16 of
 * qwen_hip_kv8.h), row r at r * row_stride elements.  uniforms [rows] fp32; temperature, top_p, min_p [rows]
 * fp32 and top_k [rows] int32, each may be null (1, off, off, off).  token_ids [rows] int32.  workspace
 * 16-byte aligned, contents need not be kept. */
int qwen_hip_sample(const void* logits, int type, int64_t row_stride, int rows, int vocab, const float* uniforms,
                    const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                    int* token_ids, void* workspace, uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QWEN_HIP_SAMPLE_H */
