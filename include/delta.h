/*
 * delta.h -- C ABI of the gated delta rule in librwkv7_hip.so (gfx950), a recurrence with a state of fixed size per sequence, as
 * wkv7_run's, on the same slot pools, ragged batches and status word.
 *
 * Per sequence and value head h, with the query/key head h / (Hv / Hk) and the state S (K x V, fp32, [k][v]):
 *   S_t = a_t S_{t-1} + k_t d_t^T,   d_t = beta_t (v_t - a_t S_{t-1}^T k_t),   a_t = exp(g_t)
 *   o_t = scale S_t^T q_t
 * With qk_norm, q and k are divided by sqrt(sum of squares + 1e-6) first.  States and sums are fp32.
 * A value of token t that is not finite makes o from t on and the final state not finite, in its column (v) or head (k, g, beta); in q,
 * o of t alone.  Tokens before t, other columns, heads and sequences have the results that they have without it.
 *
 * Return codes are the WKV7_* codes of wkv7.h.  No call allocates or synchronises; all can be recorded into a HIP graph.
 */
#ifndef RWKV_NEXT_AMD_DELTA_H
#define RWKV_NEXT_AMD_DELTA_H

#include <stddef.h>
#include <stdint.h>

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bits of *status: what the kernels left out */
#define DELTA_STATUS_SLOT 2048      /* a slot outside the states: that row starts from zeros, or its state is not stored */
#define DELTA_STATUS_SEQLENS 4096   /* cu_seqlens not non-decreasing within [0, total_tokens]: clamped */
#define DELTA_STATUS_NKEEP 8192     /* negative n_keep: taken as 0 */
#define DELTA_STATUS_CLASH 16384    /* two rows store to one slot (calls of at most 1024 rows) */

/* The library's choice of token_len.  Measured, 32 heads of 128 x 128, by tokens / by chunks, us: one row of 16 tokens 23 / 21, of 12
 * 18 / 21; 16 rows of 16 37 / 61, of 24 51 / 61, of 32 66 / 61; 64 rows of 16 125 / 198, of 32 236 / 212. */
#define DELTA_TOKEN_LEN 16
#define DELTA_MAX_STRIDE (1 << 24)  /* elements between tokens of an operand */

typedef struct delta_args {
    const uint16_t *q, *k, *v;              /* bf16 [token][Hk][K], [token][Hk][K], [token][Hv][V], 16-byte aligned */
    int64_t q_stride, k_stride, v_stride;   /* elements between tokens, multiples of 8, at most DELTA_MAX_STRIDE */
    const float *g, *beta;                  /* [token][Hv] log decays (<= 0) and writing strengths, 4-byte aligned */
    int64_t g_stride, beta_stride;          /* elements between tokens */
    uint16_t *o;                            /* bf16 [token][Hv][V], 16-byte aligned, or NULL */
    int64_t o_stride;                       /* elements between tokens, a multiple of 8 */
    const float *h0;                        /* initial states [h0_rows][Hv][K][V], 16-byte aligned, or NULL: zeros */
    const int64_t *h0_idx;                  /* row of sequence n, or NULL: n */
    int64_t h0_rows;
    float *ht;                              /* final states [ht_rows][Hv][K][V], or NULL; may be h0 */
    const int64_t *ht_idx;
    int64_t ht_rows;
    const uint8_t *fresh;                   /* nonzero: sequence n starts from zeros; or NULL */
    const int32_t *cu_seqlens;              /* [num_seqs + 1] for ragged rows, or NULL: T tokens each */
    const int64_t *n_keep;                  /* sequence n runs its first n_keep[n] tokens; or NULL */
    float *snapshots;                       /* dense rows: the state after each token [num_seqs][T][Hv][K][V]; or NULL */
    int32_t *status;                        /* or NULL */
    void *workspace;                        /* delta_workspace_size bytes, 256-byte aligned; what it holds does not matter */
    size_t workspace_bytes;
    int64_t total_tokens;
    int32_t num_seqs, T;                    /* T: tokens of a dense row; ragged: 0 */
    int32_t Hk, Hv;                         /* Hv a multiple of Hk */
    int32_t K, V;                           /* K 64 or 128, V a multiple of 16 up to 256 */
    float scale;
    int32_t qk_norm;
    int32_t token_len;                      /* rows of at most this many tokens run token by token; -1: the library's choice */
} delta_args;

/* sizeof(delta_args) as compiled into the library (bindings check their struct layout against it). */
size_t delta_args_size(void);

/* Bytes of workspace that delta_run needs for this call (its pointers are not looked at, but for which are NULL). */
int delta_workspace_size(const delta_args *args, size_t *bytes);

/* The recurrence over every sequence, on `stream`.  A row of tokens run token by token gives the same bits as its tokens in calls
 * of their own, and as its snapshots. */
int delta_run(const delta_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_NEXT_AMD_DELTA_H */
