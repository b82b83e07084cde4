/*
 * dense.h -- C ABI of the products with 16-bit weights in librwkv7_hip.so (gfx950), with bias, activation and residual in the
 * epilogue: a layer's projections, its channel mix relu(x W)^2, its low-rank parts.
 *
 *   out[m][n] = act(sum_k a[m][k] w[k][n] + bias[n]) + residual[m][n]
 *
 * a and w are both bf16 or both fp16; products are exact, sums, bias, activation and residual are fp32, out is rounded once.
 * The weight is laid out once (dense_pack) in the order in which the kernels read it.
 * Return codes are the WKV7_* codes of wkv7.h.  No call allocates or synchronises; all can be recorded into a HIP graph.
 */
#ifndef RWKV_NEXT_AMD_DENSE_H
#define RWKV_NEXT_AMD_DENSE_H

#include <stddef.h>
#include <stdint.h>

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types: activations and weights (dtype: bf16, fp16), results, residuals and biases (all three) */
#define DENSE_BF16 0
#define DENSE_F16 1
#define DENSE_F32 2

/* Activations */
#define DENSE_NONE 0
#define DENSE_RELU 1
#define DENSE_RELU2 2    /* max(x, 0)^2 */
#define DENSE_TANH 3
#define DENSE_SIGMOID 4
#define DENSE_SILU 5     /* x sigmoid(x) */
#define DENSE_GELU 6     /* x (1 + erf(x / sqrt 2)) / 2 */

#define DENSE_MAX_ROW_STRIDE (1 << 24)  /* elements between rows of activations */
#define DENSE_UNSPLIT_ROWS 16           /* products of at most so many rows .. */
#define DENSE_UNSPLIT_K 6112            /* .. and of a shorter K than this need no workspace on any device */

typedef struct dense_args {
    const uint16_t *a;             /* activations [M][K], 16-byte aligned */
    int64_t a_row_stride;          /* elements, >= K, a multiple of 8, at most DENSE_MAX_ROW_STRIDE */
    const void *weight;            /* dense_pack's layout, 16-byte aligned */
    const void *bias;              /* [N], aligned to its type, or NULL */
    const void *residual;          /* [M][N], aligned to its type, or NULL; may be out, with out's strides and type */
    int64_t residual_row_stride;   /* elements, >= N */
    void *out;                     /* [M][N], aligned to its type */
    int64_t out_row_stride;        /* elements, >= N */
    int32_t M, N, K;               /* K % 32 == 0 */
    int32_t dtype, out_dtype, bias_dtype, residual_dtype;
    int32_t activation;
    void *workspace;               /* dense_workspace_size bytes, 16-byte aligned; what it holds does not matter */
    size_t workspace_bytes;
} dense_args;

/* sizeof(dense_args) as compiled into the library (bindings check their struct layout against it). */
size_t dense_args_size(void);

/* Bytes of a packed weight. */
int dense_packed_size(int32_t K, int32_t N, size_t *bytes);

/* Lays a weight of 16-bit elements [K][N] out for dense_matmul, on `stream`: element (k, n) at w + k k_stride + n n_stride (elements),
 * so either order of a matrix is taken.  packed is 16-byte aligned. */
int dense_pack(const uint16_t *w, int64_t k_stride, int64_t n_stride, int32_t K, int32_t N, void *packed, void *stream);

/* Bytes of workspace that a product of M rows needs on the current device: 0, or the sums of K's parts where it is split. */
int dense_workspace_size(int32_t M, int32_t N, int32_t K, size_t *bytes);

/* The product, on `stream`.  The order of the sums follows from M, N, K and the device's CU count: equal calls give equal bits. */
int dense_matmul(const dense_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_NEXT_AMD_DENSE_H */
