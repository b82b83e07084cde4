/*
 * logits.h -- C ABI of the logit operators in librwkv7_hip.so (gfx950): what lies between the output head's product and the
 * next token.  logits_penalize changes the logits of running sequences (penalties for tokens they hold, per-request biases,
 * grammar masks); logits_sample chooses a token from each row (temperature, top-k, top-p, min-p, a draw by given noise).
 * They cover the reference's sampler and the penalties of its speculative step (rwkv_next/sampler.py:1-81,
 * rwkv_next/spec.py:35-84).
 *
 * Logits are [B][T][V]: T positions of B sequences (T = 1: one token each; T > 1: a block of drafted tokens).  Every
 * per-sequence parameter is a device array of B entries or, where its pointer is NULL, the scalar of the call.
 * Return codes are the WKV7_* codes of wkv7.h.  No call allocates or synchronises; all can be recorded into a HIP graph.
 */
#ifndef RWKV_NEXT_AMD_LOGITS_H
#define RWKV_NEXT_AMD_LOGITS_H

#include <stddef.h>
#include <stdint.h>

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of logits and results */
#define LOGITS_BF16 0
#define LOGITS_F16 1
#define LOGITS_F32 2

/* Element types of a count table */
#define LOGITS_COUNTS_I32 0
#define LOGITS_COUNTS_F32 1

/* Bits of the optional device status word, beside the WKV7_STATUS_* bits, so one word serves a whole step.  The kernels OR
 * them in as they meet the case, and go on as stated. */
#define LOGITS_STATUS_ROW 256    /* a slot outside the count table, or a mask row past the masks: the row went on without */
#define LOGITS_STATUS_TOKEN 512  /* a draft or bias id of V or more: ignored (negative ids are unused places) */

/* Per element, with x its logit, c = counts[slot][v] plus the number of drafts[b][0 .. t-1] equal to v:
 *   if c > 0:  x = (x > 0 ? x / repetition : x * repetition) - (frequency * c + presence)
 *   x += the sum, in order, of bias_values[b][i] with bias_ids[b][i] == v
 *   x = -infinity where bit v of the row's mask is 0
 * in fp32, rounded once to out_dtype. */
typedef struct logits_penalize_args {
    const void *logits;                      /* [B][T][V] */
    int64_t in_seq_stride, in_pos_stride;    /* elements */
    void *out;                               /* [B][T][V]; `logits` itself (same type and strides), or apart from it */
    int64_t out_seq_stride, out_pos_stride;  /* elements */
    const void *counts;                      /* NULL, or [counts_rows][V] */
    int64_t counts_stride, counts_rows;      /* elements between rows */
    const int64_t *slots;                    /* NULL (row b has counts row b), or [B] */
    const float *repetition, *presence, *frequency;  /* NULL (the scalars below), or [B] */
    const int64_t *drafts;                   /* NULL, or [B][>= T - 1]: position t has drafts[b][0 .. t-1] before it */
    int64_t drafts_stride;
    const int64_t *bias_ids;                 /* NULL, or [B][n_bias]; negative: an unused place */
    const float *bias_values;                /* [B][n_bias] */
    int64_t bias_stride;                     /* elements between rows, of both */
    const uint32_t *mask;                    /* NULL, or [mask_rows][>= ceil(V / 32)], bit v % 32 of word v / 32: allowed */
    int64_t mask_stride, mask_rows;          /* words between rows */
    const int64_t *mask_row;                 /* NULL (row b * T + t), or [B][T]; negative: no mask */
    int32_t *status;                         /* NULL, or one device word */
    float repetition_all, presence_all, frequency_all;
    int32_t B, T, V, n_bias;
    int32_t in_dtype, out_dtype, counts_dtype;
} logits_penalize_args;

/* One token for each of B * T rows.  With m the row's largest logit and d = (m - x) / temperature, w = exp(-d), tokens are
 * ordered by (d, index).  Kept are: of the first top_k of that order (all where top_k <= 0) the smallest prefix whose weights
 * reach top_p of their sum (all where top_p >= 1; always one token), and of those the ones with w >= min_p (and the first).
 * The token is the kept one with the largest w / noise, the lowest index of equals: with noise drawn from the exponential
 * distribution of rate 1 that is a draw by the kept weights.  A temperature of 0 or less (or NaN), or no noise at all: the
 * largest logit's lowest index.  NaN counts as -infinity, and tokens of -infinity are never chosen: a row of nothing else gives
 * -1 and a log-probability of -infinity.
 * logprob = -d - log(sum of w over the row), before the filters, with a temperature of 1 in greedy rows.
 * What is added up by atomics are whole numbers (of 2^-20 or less of a bin's first weight, of 2^-40): their order changes no result.
 * V is at most LOGITS_SAMPLE_MAX_V. */
#define LOGITS_SAMPLE_MAX_V 2097152
typedef struct logits_sample_args {
    const void *logits;                      /* [B][T][V] */
    int64_t seq_stride, pos_stride;          /* elements */
    const float *noise;                      /* NULL (every row greedy), or [B][T][V], positive */
    int64_t noise_seq_stride, noise_pos_stride;
    const float *temperature;                /* NULL (temperature_all), or [B] */
    const int32_t *top_k;                    /* NULL (top_k_all), or [B] */
    const float *top_p, *min_p;              /* NULL (the scalars below), or [B] */
    int64_t *token;                          /* [B][T] */
    float *logprob;                          /* NULL, or [B][T] */
    void *counts;                            /* NULL, or [counts_rows][V] (T == 1): counts[slot][token] += 1 */
    int64_t counts_stride, counts_rows;
    const int64_t *slots;                    /* NULL (row b has counts row b), or [B] */
    int32_t *status;                         /* NULL, or one device word */
    void *workspace;                         /* logits_sample_workspace_size bytes, 256-byte aligned */
    size_t workspace_bytes;
    float temperature_all, top_p_all, min_p_all;
    int32_t top_k_all;
    int32_t B, T, V;
    int32_t dtype, counts_dtype;
} logits_sample_args;

/* sizeof the structs as compiled into the library (bindings check their layout against them). */
size_t logits_penalize_args_size(void);
size_t logits_sample_args_size(void);

/* Bytes of workspace that logits_sample needs, 256-byte aligned.  The first LOGITS_SAMPLE_STATE_BYTES must be zero before the
 * workspace's first use; every completed call leaves them zero and writes nothing else into them, so one workspace serves any
 * number of calls of any shapes one after another (stream order).  Calls that can run at the same time need different ones. */
#define LOGITS_SAMPLE_STATE_BYTES 4325376
int logits_sample_workspace_size(const logits_sample_args *args, size_t *bytes);

int logits_penalize(const logits_penalize_args *args, void *stream);
int logits_sample(const logits_sample_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_NEXT_AMD_LOGITS_H */
