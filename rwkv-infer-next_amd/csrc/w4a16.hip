// w4a16.hip -- products of bf16 / fp16 activations with 4-bit weights (include/w4a16.h).
//
//   out[m][n] = sum_g s[g][n] sum_{k in g} a[m][k] q[k][n],   q = u - 8,  u the stored code in 0 .. 15
//
// The inner sums run on the matrix cores (16x16x32, fp32 accumulation).  A code becomes an operand without a conversion: put
// into mantissa bits 3..6 (bf16) or 6..9 (fp16) of the pattern of 16.0, it reads as exactly 16 + u, two codes to one shift and
// one and-or.  The 24 that this is too much comes off once for all columns: a product with a tile of -24 gives -24 sum_k a[m][k] in
// the lanes of the result, where each strip's sum begins:   sum a q = -24 sum a + sum a (16 + u).   All are fp32 sums of exact
// products; of the offsets that give whole numbers 16 is the smallest, so the difference cancels least.
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

// The codes' bits in an operand pair, and the pattern of (16, 16).  Kept in vector registers: v_and_or_b32 takes one constant.
struct Patterns {
    uint32_t mask, sixteen;
};
template <int AT>
__device__ __forceinline__ Patterns patterns() {
    Patterns p = AT == W4A16_BF16 ? Patterns{0x00780078u, 0x41804180u}   // bf16 of 16: the code's place is bit 3
                                  : Patterns{0x03C003C0u, 0x4C004C00u};  // fp16 of 16: bit 6
    asm("" : "+v"(p.mask), "+v"(p.sixteen));
    return p;
}

// Eight codes (k = 2j in bits 4j.., k = 2j + 1 in bits 16 + 4j..) as eight operands of value 16 + u.
template <int AT>
__device__ __forceinline__ u4 operands(uint32_t w, const Patterns& p) {
    u4 r;
    if constexpr (AT == W4A16_BF16) {
        r[0] = ((w << 3) & p.mask) | p.sixteen;
        r[1] = ((w >> 1) & p.mask) | p.sixteen;
        r[2] = ((w >> 5) & p.mask) | p.sixteen;
        r[3] = ((w >> 9) & p.mask) | p.sixteen;
    } else {
        r[0] = ((w << 6) & p.mask) | p.sixteen;
        r[1] = ((w << 2) & p.mask) | p.sixteen;
        r[2] = ((w >> 2) & p.mask) | p.sixteen;
        r[3] = ((w >> 6) & p.mask) | p.sixteen;
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

// Strips, for up to 16 rows and for narrow products of more: a workgroup's wavefronts take the 128-row chunks of K in turn, each with
// sums of its own; they are added in LDS in the wavefronts' order.  A wavefront reads A in operand order by itself, so 16 rows of A go
// with up to 64 columns.  Measured (graph replays; weights cycled past the 256 MB cache, in brackets three weights in turn):
// 4096 x 65536, one row 30.6 us = 4.5 TB/s where a large copy moves 4.9, bound by memory; 4096 x 4096, one row 6.0 us (4.2) and
// 2560 x 10240, five rows 7.4 us (6.5), bound by the trips to memory of a wavefront's two to four chunks, one after another.  Asked
// for a chunk ahead, the first and the last of these took twice the registers and were slower (three weights 33 and 7.8 us, then by
// 16 columns a workgroup for the last); for 4096 x 4096, whose 256 workgroups leave registers free, that was not tried.  Workgroups of 32
// and 64 rows, whose wavefronts use a weight's operands two and four times, were slower than more workgroups: 64 rows, 4096 x 4096
// 19 us against 9.2.
template <int AT, int NT, int SPC>
__global__ __launch_bounds__(512) void w4a16_strip_kernel(const Params p) {
    extern __shared__ __attribute__((aligned(16))) float part[];  // [waves][16][16 * NT]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const uint32_t on_xcd = blockIdx.x >> 3;
    const uint32_t group = on_xcd / (uint32_t)p.row_groups * 8 + (blockIdx.x & 7);
    const int row0 = (int)(on_xcd % (uint32_t)p.row_groups) * 16;
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
    const uint16_t* const ap = p.a + (int64_t)min(row0 + col, p.M - 1) * p.a_row_stride;  // past the last row: it again, not stored

    f4 acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f4{0.f, 0.f, 0.f, 0.f};
    const uint32_t m24 = AT == W4A16_BF16 ? 0xC1C0C1C0u : 0xCE00CE00u;  // -24
    const u4 minus24 = {m24, m24, m24, m24};
    const Patterns pat = patterns<AT>();

    for (int c = wave; c < p.chunks; c += waves) {
        u4 w[NT], a[4];
        float s[NT][SPC];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            w[t] = *reinterpret_cast<const u4*>(wp[t] + (int64_t)c * kBlockBytes);
#pragma unroll
            for (int j = 0; j < SPC; ++j) s[t][j] = f16_to_f32(sp[t][(int64_t)c * kStrip * SPC + j]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = c * kChunk + k * 32 + quad * 8;
            a[k] = u4{0, 0, 0, 0};
            if (at < p.K) a[k] = *reinterpret_cast<const u4*>(ap + at);
        }
        constexpr int kSteps = 4 / SPC;
#pragma unroll
        for (int j = 0; j < SPC; ++j) {
            f4 bias = {0.f, 0.f, 0.f, 0.f};  // -24 sum a, where each strip's sum begins
#pragma unroll
            for (int k = 0; k < kSteps; ++k) bias = mfma<AT>(a[j * kSteps + k], minus24, bias);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f4 d = bias;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) d = mfma<AT>(a[j * kSteps + k], operands<AT>(w[t][j * kSteps + k], pat), d);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[t][r] = fmaf(s[t][j], d[r], acc[t][r]);
            }
        }
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
        const int row = row0 + e / (16 * NT);
        const int64_t n = (int64_t)strip0 * kStrip + e % (16 * NT);
        if (row < p.M && n < p.N) store(p.out, p.out_dtype, row * p.out_row_stride + n, x);
    }
}

template <int MT, int WK>
constexpr int kPanelStride = WK * kChunk * 2 + 16;  // bytes of a row of A's panel in LDS: 16 more, so 16 rows lie in different banks
template <int MT, int WK>
constexpr int kPanelBytes = 16 * MT * kPanelStride<MT, WK>;
// Blocks, from 17 rows on: a workgroup's WN WK wavefronts are WN groups of columns by WK groups of chunks.  They share A, a panel of
// WK chunks at a time, through LDS, which loads of whole lines fill (in operand order a load of A takes four times as long, and
// every wavefront would read all of it); weights come two panels ahead into registers.  Measured: 64 rows, 4096 x 65536 57.7 us (93 by
// strips; 61.3 with weights cycled past the caches), 203 rows, 2560 x 8191, groups of 32 25 us (33).  In the first the matrix cores
// work 37 % of the time, the vector units 31 % and LDS 28 %, hardly at once: two wavefronts a SIMD is what registers and 256
// workgroups leave.  A two panels ahead as well, and four strips a wavefront at one wavefront a SIMD, were not faster (62 to 82 us).
template <int AT, int MT, int NT, int SPC, int WN, int WK>
__global__ __launch_bounds__(64 * WN * WK, 2) void w4a16_block_kernel(const Params p) {
    constexpr int kThreads = 64 * WN * WK;
    constexpr int kStride = kPanelStride<MT, WK>, kBuffers = 3;
    constexpr int kSums = (WK - 1) * WN * MT * NT * 1024;
    constexpr int kLds = kBuffers * kPanelBytes<MT, WK> > kSums ? kBuffers * kPanelBytes<MT, WK> : kSums;
    constexpr int kPieces = 16 * MT * WK * 16 / kThreads;  // 16-byte pieces of a panel to a thread
    static_assert(kPieces >= 1, "");
    __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave % WN, wk = wave / WN, col = lane & 15, quad = lane >> 4;
    const uint32_t on_xcd = blockIdx.x >> 3;
    const uint32_t group = on_xcd / (uint32_t)p.row_groups * 8 + (blockIdx.x & 7);
    const int row0 = (int)(on_xcd % (uint32_t)p.row_groups) * 16 * MT;
    if (group >= (uint32_t)p.strip_groups) return;
    const int strip0 = ((int)group * WN + wn) * NT;

    const uint8_t* wp[NT];
    const uint8_t* sp[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {  // past the last strip: that strip again, not stored
        const int64_t s = min(strip0 + t, p.strips - 1);
        wp[t] = wkv7::uniform_ptr(p.weight + s * p.chunks * kBlockBytes);
        sp[t] = wkv7::uniform_ptr(reinterpret_cast<const uint8_t*>(p.scales) + s * p.chunks * (kStrip * SPC * 2));
    }
    const int panels = (p.chunks + WK - 1) / WK;

    // A's pieces of a thread: rows past the last are that row again (not stored), columns past K zeros
    const uint8_t* const ap = reinterpret_cast<const uint8_t*>(p.a) + (int64_t)row0 * p.a_row_stride * 2;
    uint32_t at_a[kPieces];
    int at_k[kPieces], at_lds[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int e = tid + kThreads * i, row = e / (WK * 16), piece = e % (WK * 16);
        at_a[i] = (uint32_t)min(row, p.M - 1 - row0) * (uint32_t)(p.a_row_stride * 2);
        at_k[i] = piece * 8;
        at_lds[i] = row * kStride + piece * 16;
    }
    u4 next[kPieces];
    // No branch around a load, here and below: what lies past the end is read from the end and then not used.
    const auto load_a = [&](int panel) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            next[i] = *reinterpret_cast<const u4*>(ap + at_a[i] + (int64_t)min(panel * (WK * kChunk) + at_k[i], p.K - 8) * 2);
    };
    const auto store_a = [&](int panel, int buffer) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const bool in = panel * (WK * kChunk) + at_k[i] < p.K;
            u4 x = next[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = in ? x[j] : 0;
            *reinterpret_cast<u4*>(lds + buffer * kPanelBytes<MT, WK> + at_lds[i]) = x;
        }
    };
    struct Weights {
        u4 w[NT];
        uint32_t s[NT][(SPC + 1) / 2];
    };
    const auto load_w = [&](int panel, Weights& w) {
        const int64_t c = min(panel * WK + wk, p.chunks - 1);  // past the last chunk A is zero
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            w.w[t] = *reinterpret_cast<const u4*>(wp[t] + c * kBlockBytes + (uint32_t)lane * 16);
            const uint8_t* const s = sp[t] + c * (kStrip * SPC * 2) + (uint32_t)col * (SPC * 2);
            if constexpr (SPC == 1)
                w.s[t][0] = *reinterpret_cast<const uint16_t*>(s);
            else
#pragma unroll
                for (int j = 0; j < SPC / 2; ++j) w.s[t][j] = reinterpret_cast<const uint32_t*>(s)[j];
        }
    };

    f4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};
    const uint32_t m24 = AT == W4A16_BF16 ? 0xC1C0C1C0u : 0xCE00CE00u;  // -24
    const u4 minus24 = {m24, m24, m24, m24};
    const Patterns pat = patterns<AT>();

    // A chunk in parts of kSteps MFMA steps, at least two: the operands of one are read from LDS while the one before multiplies.
    constexpr int kParts = SPC > 2 ? SPC : 2, kSteps = 4 / kParts;
    struct Operands {
        u4 a[MT][kSteps];
    };
    const auto read = [&](int buffer, int part, Operands& o) {
        const uint8_t* const at =
            lds + buffer * kPanelBytes<MT, WK> + col * kStride + wk * (kChunk * 2) + quad * 16 + part * (kSteps * 64);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int k = 0; k < kSteps; ++k) o.a[i][k] = *reinterpret_cast<const u4*>(at + i * (16 * kStride) + k * 64);
    };
    const auto multiply = [&](int part, const Operands& o, const Weights& w) {
        f4 bias[MT];  // -24 sum a, where each strip's sum begins
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int i = 0; i < MT; ++i)
                bias[i] = mfma<AT>(o.a[i][k], minus24, k == 0 ? f4{0.f, 0.f, 0.f, 0.f} : bias[i]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int js = part * SPC / kParts;
            const float s = f16_to_f32(SPC == 1 ? w.s[t][0] : js & 1 ? w.s[t][js / 2] >> 16 : w.s[t][js / 2] & 0xFFFFu);
            f4 d[MT];
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const u4 b = operands<AT>(w.w[t][part * kSteps + k], pat);
#pragma unroll
                for (int i = 0; i < MT; ++i) d[i] = mfma<AT>(o.a[i][k], b, k == 0 ? bias[i] : d[i]);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][t][r] = fmaf(s, d[i][r], acc[i][t][r]);
        }
    };

    Weights w0, w1, w2;
    Operands even, odd;
    load_a(0);
    load_w(0, w0);
    load_w(1, w1);
    store_a(0, 0);
    load_a(1);
    store_a(1, 1);
    __syncthreads();
    read(0, 0, even);
    // Step p multiplies panel p, in LDS buffer `now`; the next panel is in LDS already, the one after it goes there.
    const auto step = [&](int panel, int now, int next_one, int after, const Weights& w, Weights& later) {
        load_a(panel + 2);
        load_w(panel + 2, later);
        __builtin_amdgcn_sched_barrier(0);  // the loads go out before the products, not beside their uses
        wkv7::unroll<kParts>([&](auto q) {
            constexpr int part = decltype(q)::value;
            Operands& mine = part % 2 == 0 ? even : odd;
            Operands& other = part % 2 == 0 ? odd : even;
            if (part + 1 < kParts)
                read(now, part + 1, other);
            else
                read(next_one, 0, other);
            multiply(part, mine, w);
        });
        __builtin_amdgcn_sched_barrier(0);
        store_a(panel + 2, after);
        __syncthreads();
    };
    int panel = 0;
    for (; panel + 3 <= panels; panel += 3) {
        step(panel, 0, 1, 2, w0, w2);
        step(panel + 1, 1, 2, 0, w1, w0);
        step(panel + 2, 2, 0, 1, w2, w1);
    }
    if (panel < panels) step(panel, 0, 1, 2, w0, w2);
    if (panel + 1 < panels) step(panel + 1, 1, 2, 0, w1, w0);

    // chunk groups 1 .. put their sums into LDS, group 0 adds them to its own in their order and stores
    if constexpr (WK > 1) {
        float* const sums = reinterpret_cast<float*>(lds);
        if (wk > 0)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    *reinterpret_cast<f4*>(sums + ((((wk - 1) * WN + wn) * MT + i) * NT + t) * 256 + lane * 4) = acc[i][t];
        __syncthreads();
        if (wk > 0) return;
        for (int g = 0; g < WK - 1; ++g)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    acc[i][t] += *reinterpret_cast<const f4*>(sums + (((g * WN + wn) * MT + i) * NT + t) * 256 + lane * 4);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + 16 * i + quad * 4 + r;
            if (row < p.M)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const int64_t n = (int64_t)(strip0 + t) * kStrip + col;
                    if (n < p.N) store(p.out, p.out_dtype, row * p.out_row_stride + n, acc[i][t][r]);
                }
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

template <int AT, int MT, int NT, int WN, int WK>
void launch_block(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    const dim3 grid((unsigned)pl.grid), block(64 * WN * WK);
    if (spc == 1)
        hipLaunchKernelGGL((w4a16_block_kernel<AT, MT, NT, 1, WN, WK>), grid, block, 0, s, p);
    else if (spc == 2)
        hipLaunchKernelGGL((w4a16_block_kernel<AT, MT, NT, 2, WN, WK>), grid, block, 0, s, p);
    else
        hipLaunchKernelGGL((w4a16_block_kernel<AT, MT, NT, 4, WN, WK>), grid, block, 0, s, p);
}

template <int AT, int MT>
void launch_block(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    if (pl.shape == kBlock256)
        launch_block<AT, MT, 2, 8, 1>(p, pl, spc, s);
    else if (pl.shape == kBlock128)
        launch_block<AT, MT, 2, 4, 2>(p, pl, spc, s);
    else
        launch_block<AT, MT, 1, 4, 2>(p, pl, spc, s);
}

template <int AT, int NT>
void launch_strips(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    const dim3 grid((unsigned)pl.grid), block(64 * pl.waves);
    const size_t lds = (size_t)pl.waves * NT * 256 * sizeof(float);
    if (spc == 1)
        hipLaunchKernelGGL((w4a16_strip_kernel<AT, NT, 1>), grid, block, lds, s, p);
    else if (spc == 2)
        hipLaunchKernelGGL((w4a16_strip_kernel<AT, NT, 2>), grid, block, lds, s, p);
    else
        hipLaunchKernelGGL((w4a16_strip_kernel<AT, NT, 4>), grid, block, lds, s, p);
}

template <int AT>
void launch(const Params& p, const Plan& pl, int spc, hipStream_t s) {
    if (pl.shape != kStrips)
        pl.mt == 2 ? launch_block<AT, 2>(p, pl, spc, s) : launch_block<AT, 4>(p, pl, spc, s);
    else
        pl.nt == 1   ? launch_strips<AT, 1>(p, pl, spc, s)
        : pl.nt == 2 ? launch_strips<AT, 2>(p, pl, spc, s)
                     : launch_strips<AT, 4>(p, pl, spc, s);
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
    if ((x->M > 1 && (x->a_row_stride < x->K || x->a_row_stride > W4A16_MAX_ROW_STRIDE || x->out_row_stride < x->N))) return WKV7_ERR_SHAPE;
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
