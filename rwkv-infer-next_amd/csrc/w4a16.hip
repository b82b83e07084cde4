// w4a16.hip -- products of bf16 / fp16 activations with 4-bit weights (include/w4a16.h).
//
//   out[m][n] = sum_g s[g][n] sum_{k in g} a[m][k] q[k][n],   q = u - 8,  u the stored code in 0 .. 15
//
// The inner sums run on the matrix cores (16x16x32, fp32 accumulation).  A code becomes an operand without a conversion: put
// into mantissa bits 3..6 (bf16) or 6..9 (fp16) of the pattern of 16.0, it reads as exactly 16 + u, two codes to one shift and
// one and-or.  The 24 that this is too much is taken out once per sum: a product with a tile of ones gives sum_k a[m][k] in the
// same lanes as the result, so   sum a q = sum a (16 + u) - 24 sum a.   All three are fp32 sums of exact products; of the
// offsets that give whole numbers 16 is the smallest, so the subtraction cancels least.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "w4a16.h"
#include "w4a16_plan.h"
#include "wkv7_device.h"
#include "wkv7_launch.h"

namespace w4 {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

struct Params {
    const uint16_t* a;
    int64_t a_row_stride;
    const uint8_t* weight;
    const uint16_t* scales;
    void* out;
    int64_t out_row_stride;
    int32_t M, N, K, chunks, row_groups, strip_groups, strips;
    int32_t out_dtype;
};

template <int AT>
__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    if constexpr (AT == W4A16_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Eight codes (k = 2j in bits 4j.., k = 2j + 1 in bits 16 + 4j..) as eight operands of value 16 + u.
template <int AT>
__device__ __forceinline__ u4 operands(uint32_t w) {
    u4 r;
    if constexpr (AT == W4A16_BF16) {  // bf16 of 16: 0x4180, the code's place is bit 3
        r[0] = ((w << 3) & 0x00780078u) | 0x41804180u;
        r[1] = ((w >> 1) & 0x00780078u) | 0x41804180u;
        r[2] = ((w >> 5) & 0x00780078u) | 0x41804180u;
        r[3] = ((w >> 9) & 0x00780078u) | 0x41804180u;
    } else {  // fp16 of 16: 0x4C00, the code's place is bit 6
        r[0] = ((w << 6) & 0x03C003C0u) | 0x4C004C00u;
        r[1] = ((w << 2) & 0x03C003C0u) | 0x4C004C00u;
        r[2] = ((w >> 2) & 0x03C003C0u) | 0x4C004C00u;
        r[3] = ((w >> 6) & 0x03C003C0u) | 0x4C004C00u;
    }
    return r;
}

__device__ __forceinline__ float f16_to_f32(uint32_t bits) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

__device__ __forceinline__ void store(void* out, int dtype, int64_t at, float x) {
    if (dtype == W4A16_F32)
        static_cast<float*>(out)[at] = x;
    else if (dtype == W4A16_BF16)
        static_cast<uint16_t*>(out)[at] = wkv7::f32_to_bf16(x);
    else
        static_cast<_Float16*>(out)[at] = (_Float16)x;
}

// A workgroup's wavefronts take the 128-row chunks of K in turn, each with sums of its own; they are added in LDS in the
// wavefronts' order.
template <int AT, int MT, int NT, int SPC>
__global__ __launch_bounds__(512) void w4a16_kernel(const Params p) {
    extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][MT * 16][NT * 16]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const uint32_t on_xcd = blockIdx.x >> 3;
    const uint32_t group = on_xcd / (uint32_t)p.row_groups * 8 + (blockIdx.x & 7);
    const int row0 = (int)(on_xcd % (uint32_t)p.row_groups) * 16 * MT;
    if (group >= (uint32_t)p.strip_groups) return;
    const int strip0 = (int)group * NT, col = lane & 15, quad = lane >> 4;

    const uint8_t* wp[NT];
    const uint16_t* sp[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {  // past the last strip: that strip again, not stored
        const int64_t s = min(strip0 + t, p.strips - 1);
        wp[t] = p.weight + s * p.chunks * kBlockBytes + lane * 16;
        sp[t] = p.scales + (s * p.chunks * kStrip + col) * SPC;
    }
    const uint16_t* ap[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)  // past the last row: that row again, not stored
        ap[i] = p.a + (int64_t)min(row0 + 16 * i + col, p.M - 1) * p.a_row_stride;

    f4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};
    const uint32_t one = AT == W4A16_BF16 ? 0x3F803F80u : 0x3C003C00u;
    const u4 ones = {one, one, one, one};

    for (int c = wave; c < p.chunks; c += waves) {
        u4 w[NT], a[MT][4];
        float s[NT][SPC];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            w[t] = *reinterpret_cast<const u4*>(wp[t] + (int64_t)c * kBlockBytes);
#pragma unroll
            for (int j = 0; j < SPC; ++j) s[t][j] = f16_to_f32(sp[t][(int64_t)c * kStrip * SPC + j]);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int at = c * kChunk + k * 32 + quad * 8;
                a[i][k] = u4{0, 0, 0, 0};
                if (at < p.K) a[i][k] = *reinterpret_cast<const u4*>(ap[i] + at);
            }
        const f4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < SPC; ++j) {
            f4 sum[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                sum[i] = zero;
#pragma unroll
                for (int k = j * 4 / SPC; k < (j + 1) * 4 / SPC; ++k) sum[i] = mfma<AT>(a[i][k], ones, sum[i]);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f4 d[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) d[i] = zero;
#pragma unroll
                for (int k = j * 4 / SPC; k < (j + 1) * 4 / SPC; ++k) {
                    const u4 b = operands<AT>(w[t][k]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) d[i] = mfma<AT>(a[i][k], b, d[i]);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        acc[i][t][r] = fmaf(s[t][j], fmaf(-24.f, sum[i][r], d[i][r]), acc[i][t][r]);
            }
        }
    }

    float* const mine = part + wave * (MT * NT * 256);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) mine[(16 * i + quad * 4 + r) * (16 * NT) + 16 * t + col] = acc[i][t][r];
    __syncthreads();
    for (int e = threadIdx.x; e < MT * NT * 256; e += blockDim.x) {
        float x = 0.f;
        for (int v = 0; v < waves; ++v) x += part[v * (MT * NT * 256) + e];
        const int row = row0 + e / (16 * NT);
        const int64_t n = (int64_t)strip0 * kStrip + e % (16 * NT);
        if (row < p.M && n < p.N) store(p.out, p.out_dtype, row * p.out_row_stride + n, x);
    }
}

// One 16-byte piece of the packed weight a thread: lane l of (strip, chunk) holds column l % 16, and in word k the rows
// 32 k + 8 (l / 16) + 0..7 of the chunk, row 2j in bits 4j.., row 2j + 1 in bits 16 + 4j...  Rows and columns past the weight's
// are code 8 (q = 0).
__global__ __launch_bounds__(256) void w4a16_pack_kernel(const uint8_t* codes, uint8_t* weight, int32_t K, int32_t N,
                                                         int64_t chunks, int64_t pieces) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= pieces) return;
    const int lane = (int)(id & 63);
    const int64_t c = (id >> 6) % chunks, n = (id >> 6) / chunks * kStrip + (lane & 15);
    u4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t x = 0;
        const int64_t row = c * kChunk + 32 * k + 8 * (lane >> 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t two = row + 2 * j < K && n < N ? codes[(row / 2 + j) * N + n] : 0x88u;
            x |= (two & 15u) << (4 * j) | (two >> 4) << (16 + 4 * j);
        }
        w[k] = x;
    }
    *reinterpret_cast<u4*>(weight + id * 16) = w;
}

// packed[strip][chunk][column][j] = the scale of the chunk's j-th of `spc` equal parts (0 past the weight)
__global__ __launch_bounds__(256) void w4a16_pack_scales_kernel(const uint16_t* scales, uint16_t* packed, int32_t K, int32_t N,
                                                                int32_t group_k, int64_t chunks, int spc, int64_t total) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const int j = (int)(id % spc), col = (int)(id / spc % kStrip);
    const int64_t c = id / (spc * kStrip) % chunks, n = id / (spc * kStrip) / chunks * kStrip + col;
    const int64_t row = c * kChunk + j * (kChunk / spc);
    packed[id] = row < K && n < N ? scales[row / group_k * N + n] : 0;
}

__global__ __launch_bounds__(256) void w4a16_dequantize_kernel(const uint8_t* codes, const uint16_t* scales, void* w, int32_t N,
                                                               int32_t group_k, int32_t dtype, int64_t total) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;  // one byte of codes: rows 2j, 2j + 1 of column n
    if (id >= total) return;
    const int64_t j = id / N, n = id % N;
    const uint32_t two = codes[id];
    const float s = f16_to_f32(scales[2 * j / group_k * N + n]);
    store(w, dtype, 2 * j * N + n, s * (float)((int)(two & 15) - 8));
    store(w, dtype, (2 * j + 1) * N + n, s * (float)((int)(two >> 4) - 8));
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool good_weight(int32_t K, int32_t N, int32_t g) {
    return K >= 32 && N >= 1 && K % 32 == 0 && g >= 32 && g % 32 == 0 && K % g == 0;
}
constexpr int64_t kMaxGrid = 0x7FFFFF;  // workgroups of one launch: with 512 threads below 2^32 work-items

template <int AT, int MT, int NT>
void launch(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    const dim3 grid((unsigned)pl.grid), block(64 * pl.waves);
    const size_t lds = (size_t)pl.waves * MT * NT * 256 * sizeof(float);
    if (spc == 1)
        hipLaunchKernelGGL((w4a16_kernel<AT, MT, NT, 1>), grid, block, lds, s, p);
    else if (spc == 2)
        hipLaunchKernelGGL((w4a16_kernel<AT, MT, NT, 2>), grid, block, lds, s, p);
    else
        hipLaunchKernelGGL((w4a16_kernel<AT, MT, NT, 4>), grid, block, lds, s, p);
}

template <int AT, int MT>
void launch(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    if (pl.nt == 1)
        launch<AT, MT, 1>(p, pl, spc, s);
    else if (pl.nt == 2)
        launch<AT, MT, 2>(p, pl, spc, s);
    else
        launch<AT, MT, 4>(p, pl, spc, s);
}

template <int AT>
void launch(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    if (pl.mt == 1)
        launch<AT, 1>(p, pl, spc, s);
    else if (pl.mt == 2)
        launch<AT, 2>(p, pl, spc, s);
    else
        launch<AT, 4>(p, pl, spc, s);
}

}  // namespace
}  // namespace w4

extern "C" {

size_t w4a16_args_size(void) { return sizeof(w4a16_args); }

int w4a16_packed_size(int32_t K, int32_t N, int32_t group_k, size_t* weight_bytes, size_t* scale_bytes) {
    if (!weight_bytes || !scale_bytes) return WKV7_ERR_NULL;
    if (!w4::good_weight(K, N, group_k)) return WKV7_ERR_SHAPE;
    *weight_bytes = w4::weight_bytes(K, N);
    *scale_bytes = w4::scale_bytes(K, N, group_k);
    return WKV7_OK;
}

int w4a16_pack(const uint8_t* codes, const uint16_t* scales, int32_t K, int32_t N, int32_t group_k, void* weight,
               uint16_t* packed_scales, void* stream) {
    if (!w4::good_weight(K, N, group_k)) return WKV7_ERR_SHAPE;
    if (!codes || !scales || !weight || !packed_scales) return WKV7_ERR_NULL;
    if (!w4::aligned(weight, 16) || !w4::aligned(packed_scales, 16) || !w4::aligned(scales, 2)) return WKV7_ERR_ALIGN;
    const int64_t pieces = (int64_t)w4::weight_bytes(K, N) / 16;
    const int64_t total = (int64_t)w4::scale_bytes(K, N, group_k) / 2;  // less than the pieces: 16 to 64 to a block's 64
    const int64_t blocks = (std::max(pieces, total) + 255) / 256;
    if (blocks > 2 * w4::kMaxGrid) return WKV7_ERR_SHAPE;
    const auto s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(w4::w4a16_pack_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, s, codes,
                       static_cast<uint8_t*>(weight), K, N, w4::chunks(K), pieces);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return static_cast<int>(e);
    hipLaunchKernelGGL(w4::w4a16_pack_scales_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, s, scales,
                       packed_scales, K, N, group_k, w4::chunks(K), w4::scales_per_chunk(group_k), total);
    return static_cast<int>(hipGetLastError());
}

int w4a16_dequantize(const uint8_t* codes, const uint16_t* scales, void* w, int32_t K, int32_t N, int32_t group_k,
                     int32_t out_dtype, void* stream) {
    if (!w4::good_weight(K, N, group_k)) return WKV7_ERR_SHAPE;
    if (out_dtype < W4A16_BF16 || out_dtype > W4A16_F32) return WKV7_ERR_ARG;
    if (!codes || !scales || !w) return WKV7_ERR_NULL;
    if (!w4::aligned(scales, 2) || !w4::aligned(w, out_dtype == W4A16_F32 ? 4 : 2)) return WKV7_ERR_ALIGN;
    const int64_t total = (int64_t)K / 2 * N;
    if ((total + 255) / 256 > 2 * w4::kMaxGrid) return WKV7_ERR_SHAPE;
    hipLaunchKernelGGL(w4::w4a16_dequantize_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0,
                       static_cast<hipStream_t>(stream), codes, scales, w, N, group_k, out_dtype, total);
    return static_cast<int>(hipGetLastError());
}

int w4a16_matmul(const w4a16_args* x, void* stream) {
    if (!x) return WKV7_ERR_NULL;
    if (!w4::good_weight(x->K, x->N, x->group_k) || x->M < 0) return WKV7_ERR_SHAPE;
    if (x->a_dtype < W4A16_BF16 || x->a_dtype > W4A16_F16 || x->out_dtype < W4A16_BF16 || x->out_dtype > W4A16_F32)
        return WKV7_ERR_ARG;
    if (x->M == 0) return WKV7_OK;
    if (!x->a || !x->weight || !x->scales || !x->out) return WKV7_ERR_NULL;
    if (!w4::aligned(x->a, 16) || !w4::aligned(x->weight, 16) || !w4::aligned(x->scales, 16) || x->a_row_stride % 8 ||
        !w4::aligned(x->out, x->out_dtype == W4A16_F32 ? 4 : 2))
        return WKV7_ERR_ALIGN;
    if ((x->M > 1 && (x->a_row_stride < x->K || x->out_row_stride < x->N))) return WKV7_ERR_SHAPE;
    const w4::Plan pl = w4::plan(x->M, x->N, x->K, wkv7::device_cu_count());
    if (pl.grid > w4::kMaxGrid) return WKV7_ERR_SHAPE;
    w4::Params p;
    p.a = x->a;
    p.a_row_stride = x->a_row_stride;
    p.weight = static_cast<const uint8_t*>(x->weight);
    p.scales = x->scales;
    p.out = x->out;
    p.out_row_stride = x->out_row_stride;
    p.M = x->M, p.N = x->N, p.K = x->K;
    p.chunks = (int32_t)w4::chunks(x->K), p.strips = (int32_t)w4::strips(x->N);
    p.row_groups = (int32_t)pl.row_groups, p.strip_groups = (int32_t)pl.strip_groups;
    p.out_dtype = x->out_dtype;
    const int spc = w4::scales_per_chunk(x->group_k);
    const auto s = static_cast<hipStream_t>(stream);
    if (x->a_dtype == W4A16_BF16)
        w4::launch<W4A16_BF16>(p, pl, spc, s);
    else
        w4::launch<W4A16_F16>(p, pl, spc, s);
    return static_cast<int>(hipGetLastError());
}

}  // extern "C"
