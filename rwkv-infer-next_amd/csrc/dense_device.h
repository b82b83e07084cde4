// dense_device.h -- what the kernels of include/dense.h share: the operands' types, the epilogue.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dense.h"
#include "dense_plan.h"
#include "wkv7_device.h"

namespace dense {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));

struct Params {
    const uint16_t* a;
    int64_t a_row_stride;
    const uint8_t* weight;
    const void *bias, *residual;
    int64_t residual_row_stride;
    void* out;
    int64_t out_row_stride;
    float* sums;  // of split products, [part][M][kSumsRow(N)]
    int32_t M, N, K, steps, row_groups, strip_groups, strips;
    int32_t out_dtype, bias_dtype, residual_dtype, activation;
    int32_t parts, fours;  // fours: four columns of bias, residual and result are one load or store
};

template <int AT>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (AT == DENSE_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float load(const void* x, int dtype, int64_t at) {
    if (dtype == DENSE_F32) return static_cast<const float*>(x)[at];
    if (dtype == DENSE_BF16) return wkv7::bf16_to_f32(static_cast<const uint16_t*>(x)[at]);
    return (float)static_cast<const _Float16*>(x)[at];
}

__device__ __forceinline__ void store(void* out, int dtype, int64_t at, float x) {
    if (dtype == DENSE_F32)
        static_cast<float*>(out)[at] = x;
    else if (dtype == DENSE_BF16)
        static_cast<uint16_t*>(out)[at] = wkv7::f32_to_bf16(x);
    else
        static_cast<_Float16*>(out)[at] = (_Float16)x;
}

__device__ __forceinline__ float activate(float x, int activation) {
    switch (activation) {
        case DENSE_RELU: return x > 0.f ? x : x == x ? 0.f : x;  // NaN stays NaN
        case DENSE_RELU2: return x > 0.f ? x * x : x == x ? 0.f : x;
        case DENSE_TANH: return tanhf(x);
        case DENSE_SIGMOID: return 1.f / (1.f + expf(-x));
        case DENSE_SILU: return x / (1.f + expf(-x));
        case DENSE_GELU: return 0.5f * x * erfcf(x * -0.70710678118654752f);
        default: return x;
    }
}

// The sum x of (row, column n) through the epilogue.
__device__ __forceinline__ void finish(const Params& p, int64_t row, int64_t n, float x) {
    if (p.bias) x += load(p.bias, p.bias_dtype, n);
    x = activate(x, p.activation);
    if (p.residual) x += load(p.residual, p.residual_dtype, row * p.residual_row_stride + n);
    store(p.out, p.out_dtype, row * p.out_row_stride + n, x);
}

// Four columns from n on.
__device__ __forceinline__ f4 load4(const void* x, int dtype, int64_t at) {
    if (dtype == DENSE_F32) return *reinterpret_cast<const f4*>(static_cast<const float*>(x) + at);
    const u2 w = *reinterpret_cast<const u2*>(static_cast<const uint16_t*>(x) + at);
    if (dtype == DENSE_BF16)
        return f4{__uint_as_float(w[0] << 16), __uint_as_float(w[0] & 0xFFFF0000u), __uint_as_float(w[1] << 16),
                  __uint_as_float(w[1] & 0xFFFF0000u)};
    const h4 x16 = __builtin_bit_cast(h4, w);  // (of one element of w it would read the first)
    return f4{(float)x16[0], (float)x16[1], (float)x16[2], (float)x16[3]};
}
__device__ __forceinline__ void finish4(const Params& p, int64_t row, int64_t n, f4 x) {
    if (p.bias) x += load4(p.bias, p.bias_dtype, n);
    if (p.activation != DENSE_NONE)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = activate(x[r], p.activation);
    if (p.residual) x += load4(p.residual, p.residual_dtype, row * p.residual_row_stride + n);
    const int64_t at = row * p.out_row_stride + n;
    if (p.out_dtype == DENSE_F32) {
        *reinterpret_cast<f4*>(static_cast<float*>(p.out) + at) = x;
        return;
    }
    u2 w;
    if (p.out_dtype == DENSE_BF16) {
        w = u2{wkv7::pack_bf16x2(x[0], x[1]), wkv7::pack_bf16x2(x[2], x[3])};
    } else {
        w[0] = __builtin_bit_cast(uint32_t, h2{(_Float16)x[0], (_Float16)x[1]});
        w[1] = __builtin_bit_cast(uint32_t, h2{(_Float16)x[2], (_Float16)x[3]});
    }
    *reinterpret_cast<u2*>(static_cast<uint16_t*>(p.out) + at) = w;
}

hipError_t launch_tiles(const Params& p, const Plan& pl, int32_t dtype, hipStream_t stream);

}  // namespace dense
