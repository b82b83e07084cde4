// dense.hip -- products of bf16 / fp16 activations with 16-bit weights, bias, activation and residual in the epilogue
// (include/dense.h), on the matrix cores (16x16x32, fp32 accumulation).
#include "dense_device.h"
#include "wkv7_launch.h"

namespace dense {
namespace {

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

int dense_workspace_size(int32_t M, int32_t N, int32_t K, size_t* bytes) {
    if (!bytes) return WKV7_ERR_NULL;
    if (!dense::good_weight(K, N) || M < 0) return WKV7_ERR_SHAPE;
    *bytes = M == 0 ? 0 : dense::plan(M, N, K, wkv7::device_cu_count()).workspace;
    return WKV7_OK;
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
    if (pl.workspace && (!x->workspace || x->workspace_bytes < pl.workspace)) return WKV7_ERR_WORKSPACE;
    if (pl.workspace && !dense::aligned(x->workspace, 16)) return WKV7_ERR_ALIGN;
    dense::Params p;
    p.a = x->a, p.a_row_stride = x->M > 1 ? x->a_row_stride : x->K, p.weight = static_cast<const uint8_t*>(x->weight);
    p.bias = x->bias, p.residual = x->residual, p.residual_row_stride = x->residual_row_stride;
    p.out = x->out, p.out_row_stride = x->out_row_stride;
    p.sums = static_cast<float*>(x->workspace), p.parts = pl.parts;
    // four columns at once: bias, residual and result in steps of four elements, aligned to them
    p.fours = x->N % 4 == 0 && dense::aligned(x->out, 4 * dense::size_of(x->out_dtype)) && (x->M == 1 || x->out_row_stride % 4 == 0) &&
              (!x->bias || dense::aligned(x->bias, 4 * dense::size_of(x->bias_dtype))) &&
              (!x->residual || (dense::aligned(x->residual, 4 * dense::size_of(x->residual_dtype)) &&
                                (x->M == 1 || x->residual_row_stride % 4 == 0)));
    p.M = x->M, p.N = x->N, p.K = x->K;
    p.steps = (int32_t)dense::steps(x->K), p.strips = (int32_t)dense::strips(x->N);
    p.row_groups = (int32_t)pl.row_groups, p.strip_groups = (int32_t)pl.strip_groups;
    p.out_dtype = x->out_dtype, p.bias_dtype = x->bias_dtype, p.residual_dtype = x->residual_dtype, p.activation = x->activation;
    return static_cast<int>(dense::launch_tiles(p, pl, x->dtype, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
