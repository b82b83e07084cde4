// dense.hip -- products of bf16 / fp16 activations with 16-bit weights, bias, activation and residual in the epilogue
// (include/dense.h), on the matrix cores (16x16x32, fp32 accumulation).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dense.h"
#include "dense_plan.h"
#include "wkv7_device.h"
#include "wkv7_launch.h"

namespace dense {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

struct Params {
    const uint16_t* a;
    int64_t a_row_stride;
    const uint8_t* weight;
    const void *bias, *residual;
    int64_t residual_row_stride;
    void* out;
    int64_t out_row_stride;
    int32_t M, N, K, steps, row_groups, strip_groups, strips;
    int32_t out_dtype, bias_dtype, residual_dtype, activation;
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

// Strips: a workgroup's wavefronts take the 128-row chunks of K in turn, each with sums of its own for 16 rows by 16 NT columns; they
// are added in LDS in the wavefronts' order.
template <int AT, int NT>
__global__ __launch_bounds__(512) void dense_strip_kernel(const Params p) {
    extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][16][16 * NT]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const uint32_t on_xcd = blockIdx.x >> 3;
    const uint32_t group = on_xcd / (uint32_t)p.row_groups * 8 + (blockIdx.x & 7);
    const int row0 = (int)(on_xcd % (uint32_t)p.row_groups) * 16;
    if (group >= (uint32_t)p.strip_groups) return;
    const int strip0 = (int)group * NT, col = lane & 15, quad = lane >> 4;

    const uint8_t* wp[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)  // past the last strip: that strip again, not stored
        wp[t] = p.weight + (int64_t)min(strip0 + t, p.strips - 1) * p.steps * kBlockBytes + lane * 16;
    const uint16_t* const ap = p.a + (int64_t)min(row0 + col, p.M - 1) * p.a_row_stride + quad * 8;  // past the last row: it again

    f4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = wave * 4; s0 < p.steps; s0 += waves * 4) {
        u4 w[4][NT], a[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = min(s0 + k, p.steps - 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) w[k][t] = *reinterpret_cast<const u4*>(wp[t] + (int64_t)s * kBlockBytes);
            a[k] = *reinterpret_cast<const u4*>(ap + s * kStep);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (s0 + k < p.steps)
#pragma unroll
                for (int t = 0; t < NT; ++t) acc[t] = mfma<AT>(a[k], w[k][t], acc[t]);
    }
    float* const mine = part + wave * (NT * 256);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) mine[(quad * 4 + r) * (16 * NT) + 16 * t + col] = acc[t][r];
    __syncthreads();
    for (int e = threadIdx.x; e < NT * 256; e += blockDim.x) {
        float x = 0.f;
        for (int v = 0; v < waves; ++v) x += part[v * (NT * 256) + e];
        const int64_t row = row0 + e / (16 * NT), n = (int64_t)strip0 * kStrip + e % (16 * NT);
        if (row < p.M && n < p.N) finish(p, row, n, x);
    }
}

// One 16-byte piece of the packed weight a thread: lane l of (strip, step) holds column l % 16, rows 8 (l / 16) + 0..7 of the step;
// zeros past the last column.
__global__ __launch_bounds__(256) void dense_pack_kernel(const uint16_t* w, int64_t k_stride, int64_t n_stride, uint8_t* packed,
                                                         int32_t N, int64_t steps, int64_t pieces) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= pieces) return;
    const int lane = (int)(id & 63);
    const int64_t k = (id >> 6) % steps * kStep + 8 * (lane >> 4), n = (id >> 6) / steps * kStrip + (lane & 15);
    u4 x = {0, 0, 0, 0};
    if (n < N)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j / 2] |= (uint32_t)w[(k + j) * k_stride + n * n_stride] << (16 * (j & 1));
    *reinterpret_cast<u4*>(packed + id * 16) = x;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool good_weight(int32_t K, int32_t N) { return K >= kStep && N >= 1 && K % kStep == 0; }
uintptr_t size_of(int32_t dtype) { return dtype == DENSE_F32 ? 4 : 2; }
bool good_type(int32_t dtype) { return dtype >= DENSE_BF16 && dtype <= DENSE_F32; }
constexpr int64_t kMaxGrid = 0x7FFFFF;  // workgroups of one launch: with 512 threads below 2^32 work-items

template <int AT>
void launch(const Params& p, const Plan& pl, hipStream_t s) {
    const dim3 grid((unsigned)pl.grid), block(64 * pl.waves);
    const size_t lds = (size_t)pl.waves * pl.nt * 256 * sizeof(float);
    if (pl.nt == 1)
        hipLaunchKernelGGL((dense_strip_kernel<AT, 1>), grid, block, lds, s, p);
    else if (pl.nt == 2)
        hipLaunchKernelGGL((dense_strip_kernel<AT, 2>), grid, block, lds, s, p);
    else
        hipLaunchKernelGGL((dense_strip_kernel<AT, 4>), grid, block, lds, s, p);
}

}  // namespace
}  // namespace dense

extern "C" {

size_t dense_args_size(void) { return sizeof(dense_args); }

int dense_packed_size(int32_t K, int32_t N, size_t* bytes) {
    if (!bytes) return WKV7_ERR_NULL;
    if (!dense::good_weight(K, N)) return WKV7_ERR_SHAPE;
    *bytes = dense::weight_bytes(K, N);
    return WKV7_OK;
}

int dense_pack(const uint16_t* w, int64_t k_stride, int64_t n_stride, int32_t K, int32_t N, void* packed, void* stream) {
    if (!dense::good_weight(K, N)) return WKV7_ERR_SHAPE;
    if (!w || !packed) return WKV7_ERR_NULL;
    if (!dense::aligned(w, 2) || !dense::aligned(packed, 16)) return WKV7_ERR_ALIGN;
    const int64_t pieces = (int64_t)dense::weight_bytes(K, N) / 16, blocks = (pieces + 255) / 256;
    if (blocks > 2 * dense::kMaxGrid) return WKV7_ERR_SHAPE;
    hipLaunchKernelGGL(dense::dense_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream), w,
                       k_stride, n_stride, static_cast<uint8_t*>(packed), N, dense::steps(K), pieces);
    return static_cast<int>(hipGetLastError());
}

int dense_matmul(const dense_args* x, void* stream) {
    if (!x) return WKV7_ERR_NULL;
    if (!dense::good_weight(x->K, x->N) || x->M < 0) return WKV7_ERR_SHAPE;
    if (x->dtype < DENSE_BF16 || x->dtype > DENSE_F16 || !dense::good_type(x->out_dtype) ||
        (x->bias && !dense::good_type(x->bias_dtype)) || (x->residual && !dense::good_type(x->residual_dtype)) ||
        x->activation < DENSE_NONE || x->activation > DENSE_GELU)
        return WKV7_ERR_ARG;
    if (x->M == 0) return WKV7_OK;
    if (!x->a || !x->weight || !x->out) return WKV7_ERR_NULL;
    if (!dense::aligned(x->a, 16) || !dense::aligned(x->weight, 16) || x->a_row_stride % 8 ||
        !dense::aligned(x->out, dense::size_of(x->out_dtype)) || (x->bias && !dense::aligned(x->bias, dense::size_of(x->bias_dtype))) ||
        (x->residual && !dense::aligned(x->residual, dense::size_of(x->residual_dtype))))
        return WKV7_ERR_ALIGN;
    if (x->M > 1 && (x->a_row_stride < x->K || x->a_row_stride > DENSE_MAX_ROW_STRIDE || x->out_row_stride < x->N ||
                     (x->residual && x->residual_row_stride < x->N)))
        return WKV7_ERR_SHAPE;
    const dense::Plan pl = dense::plan(x->M, x->N, x->K, wkv7::device_cu_count());
    if (pl.grid > dense::kMaxGrid) return WKV7_ERR_SHAPE;
    dense::Params p;
    p.a = x->a, p.a_row_stride = x->M > 1 ? x->a_row_stride : x->K, p.weight = static_cast<const uint8_t*>(x->weight);
    p.bias = x->bias, p.residual = x->residual, p.residual_row_stride = x->residual_row_stride;
    p.out = x->out, p.out_row_stride = x->out_row_stride;
    p.M = x->M, p.N = x->N, p.K = x->K;
    p.steps = (int32_t)dense::steps(x->K), p.strips = (int32_t)dense::strips(x->N);
    p.row_groups = (int32_t)pl.row_groups, p.strip_groups = (int32_t)pl.strip_groups;
    p.out_dtype = x->out_dtype, p.bias_dtype = x->bias_dtype, p.residual_dtype = x->residual_dtype, p.activation = x->activation;
    const auto s = static_cast<hipStream_t>(stream);
    if (x->dtype == DENSE_BF16)
        dense::launch<DENSE_BF16>(p, pl, s);
    else
        dense::launch<DENSE_F16>(p, pl, s);
    return static_cast<int>(hipGetLastError());
}

}  // extern "C"
