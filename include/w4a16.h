/*
 * w4a16.h -- C ABI of the 4-bit weight product in librwkv7_hip.so (gfx950): a few rows of bf16 or fp16 activations times a
 * weight of 4-bit codes with one fp16 scale per (group of rows, column).  For the output head and the projections of a
 * decode step, whose time is the reading of the weight.
 *
 * A (K, N) weight is quantised to q in [-8, 7] with w = scale * q; the stored code is u = q + 8:
 *   codes  uint8 [K/2][N]         codes[j][n] = u(row 2j) | u(row 2j + 1) << 4
 *   scales fp16  [K/group_k][N]
 * and laid out once (w4a16_pack) in the order in which the kernel reads it.
 *
 * out[m][n] = sum_g scale[g][n] * sum_{k in g} a[m][k] q[k][n]; the inner and outer sums are fp32, out is rounded once.
 * A row of `a` that holds an infinity or NaN gives NaN in every column, and so may one with elements of 1e36 and more.
 * Return codes are the WKV7_* codes of wkv7.h.  No call allocates or synchronises; all can be recorded into a HIP graph.
 */
#ifndef RWKV_NEXT_AMD_W4A16_H
#define RWKV_NEXT_AMD_W4A16_H

#include <stddef.h>
#include <stdint.h>

#include "wkv7.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Types of activations (a_dtype: bf16, fp16) and of results (out_dtype, and of w4a16_dequantize: all three) */
#define W4A16_BF16 0
#define W4A16_F16 1
#define W4A16_F32 2

#define W4A16_MAX_ROW_STRIDE (1 << 24)  /* elements between rows of activations */

typedef struct w4a16_args {
    const uint16_t *a;       /* activations [M][K], 16-byte aligned */
    int64_t a_row_stride;    /* elements, >= K, a multiple of 8, at most W4A16_MAX_ROW_STRIDE */
    const void *weight;      /* w4a16_pack's layout, 16-byte aligned */
    const uint16_t *scales;  /* w4a16_pack's layout, 16-byte aligned */
    void *out;               /* [M][N], aligned to its type */
    int64_t out_row_stride;  /* elements, >= N */
    int32_t M, N, K;         /* K % 32 == 0 */
    int32_t group_k;         /* a multiple of 32 that divides K, the one the weight was packed with */
    int32_t a_dtype, out_dtype;
} w4a16_args;

/* sizeof(w4a16_args) as compiled into the library (bindings check their struct layout against it). */
size_t w4a16_args_size(void);

/* Bytes of a packed weight and of its packed scales. */
int w4a16_packed_size(int32_t K, int32_t N, int32_t group_k, size_t *weight_bytes, size_t *scale_bytes);

/* Lays codes and scales (contiguous, as above) out for w4a16_matmul, on `stream`.  Outputs 16-byte aligned. */
int w4a16_pack(const uint8_t *codes, const uint16_t *scales, int32_t K, int32_t N, int32_t group_k, void *weight,
               uint16_t *packed_scales, void *stream);

/* w[k][n] = scale * q as bf16, fp16 or fp32 (exact in fp32), contiguous, from codes and scales. */
int w4a16_dequantize(const uint8_t *codes, const uint16_t *scales, void *w, int32_t K, int32_t N, int32_t group_k,
                     int32_t out_dtype, void *stream);

/* out = a @ dequantised weight, on `stream`.  The order of the sums follows from M, N, K, group_k and the device's CU count:
 * equal calls give equal bits. */
int w4a16_matmul(const w4a16_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* RWKV_NEXT_AMD_W4A16_H */
