// logits_device.h -- loads and stores shared by the logit kernels.  Rows begin anywhere their type allows (an odd vocabulary
// leaves none aligned), so eight elements are read and written as words of the type's alignment; the hardware takes 16-byte
// accesses at such addresses.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "logits.h"
#include "wkv7_device.h"

namespace lg {

typedef uint32_t u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f4a4 __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

__host__ __device__ constexpr int element_bytes(int dtype) { return dtype == LOGITS_F32 ? 4 : 2; }

__device__ __forceinline__ float from16(int dtype, uint32_t bits) {
    return dtype == LOGITS_BF16 ? __uint_as_float(bits << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

// x[0 .. n-1] = row[at ..] in fp32 (n = 8: two or one 16-byte loads); the rest is `fill`.
template <int DT>
__device__ __forceinline__ void load8(const void* row, int64_t at, int n, float fill, float (&x)[8]) {
    const char* const p = static_cast<const char*>(row) + at * element_bytes(DT);
    if (n == 8) {
        if constexpr (DT == LOGITS_F32) {
            const f4a4 a = *reinterpret_cast<const f4a4*>(p), b = *reinterpret_cast<const f4a4*>(p + 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
        } else {
            const u4a2 a = *reinterpret_cast<const u4a2*>(p);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[2 * j] = from16(DT, a[j] & 0xFFFFu), x[2 * j + 1] = from16(DT, a[j] >> 16);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = fill;
            if (j < n) {
                if constexpr (DT == LOGITS_F32)
                    x[j] = reinterpret_cast<const float*>(p)[j];
                else
                    x[j] = from16(DT, reinterpret_cast<const uint16_t*>(p)[j]);
            }
        }
    }
}

__device__ __forceinline__ uint16_t to16(int dtype, float x) {
    return dtype == LOGITS_BF16 ? wkv7::f32_to_bf16(x) : __builtin_bit_cast(uint16_t, (_Float16)x);
}

__device__ __forceinline__ void store8(void* row, int dtype, int64_t at, int n, const float (&x)[8]) {
    char* const p = static_cast<char*>(row) + at * element_bytes(dtype);
    if (dtype == LOGITS_F32) {
        if (n == 8) {
            *reinterpret_cast<f4a4*>(p) = f4a4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f4a4*>(p + 16) = f4a4{x[4], x[5], x[6], x[7]};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) reinterpret_cast<float*>(p)[j] = x[j];
        }
    } else {
        if (n == 8) {
            u4a2 w;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = (uint32_t)to16(dtype, x[2 * j]) | (uint32_t)to16(dtype, x[2 * j + 1]) << 16;
            *reinterpret_cast<u4a2*>(p) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) reinterpret_cast<uint16_t*>(p)[j] = to16(dtype, x[j]);
        }
    }
}

}  // namespace lg
