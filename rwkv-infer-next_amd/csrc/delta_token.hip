// delta_token.hip -- the gated delta rule token by token: decode, verification, replay, short rows (include/delta.h).
//
// A wavefront holds 32 columns of one head's state in registers, K / 8 rows by 4 columns a lane, and walks the row's tokens.  With
// r = S_{t-1}^T k and u = S_{t-1}^T q from one pass over the state,
//     d = beta (v - a r),   S_t = a S_{t-1} + k d^T,   o = scale (a u + (q . k) d)
// so a token costs one sum over the lanes.  For one token the reading and writing of the states, 8 K V bytes a head, bounds it: 64
// sequences, 32 heads of 128 x 128, 49 us with states from memory (eight pools in turn), 5.5 TB/s in place where a large copy moves 4.9;
// 44 to 47 with one pool, half of which the caches hold; one sequence 5.3 to 5.6 us.  Blocks of 2, 4, 8 tokens 51, 56, 70 us; with a
// snapshot of each token 78, 138, 253 (4.8 TB/s).  Each
// lane has its 16-byte pieces of 16 rows in flight at once, so nothing needs LDS or a barrier.
#include "delta_device.h"

namespace delta {
namespace {

constexpr int kCols = 32;  // columns of a wavefront

// x + the x of lane ^ 8, ^ 16, ^ 32, in this order
__device__ __forceinline__ float sum_groups(float x) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));  // row_ror:8
    const u2 a = __builtin_bit_cast(u2, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const u2 b = __builtin_bit_cast(u2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <int K>
__global__ __launch_bounds__(256) void delta_token_kernel(const Params p, int blocks, int64_t units) {
    constexpr int R = K / 8;  // rows of the state a lane holds: kg R .. kg R + R - 1
    const int lane = threadIdx.x & 63, kg = lane >> 3;
    const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (unit >= units) return;
    const int block = (int)(unit % blocks);
    const int h = (int)(unit / blocks % p.Hv), n = (int)(unit / blocks / p.Hv);
    int64_t first;
    int len;
    extent(p, n, first, len);
    if (p.cu && len > p.token_len) return;  // runs by chunks
    const int col = block * kCols + (lane & 7) * 4;
    const bool on = col < p.V;  // V is a multiple of 16: the last block may have 16 columns
    const int64_t at = (int64_t)kg * R * p.V + col;

    const float* const from = initial(p, n, h);
    f4 S[R];
#pragma unroll
    for (int j = 0; j < R; ++j)
        S[j] = from && on ? __builtin_nontemporal_load(reinterpret_cast<const f4*>(from + at + (int64_t)j * p.V)) : f4{0.f, 0.f, 0.f, 0.f};

    const int hk = h / p.share;
    const uint16_t* qp = p.q + first * p.q_stride + hk * K + kg * R;
    const uint16_t* kp = p.k + first * p.k_stride + hk * K + kg * R;
    const uint16_t* vp = p.v + first * p.v_stride + (int64_t)h * p.V + (on ? col : 0);
    const float* gp = p.g + first * p.g_stride + h;
    const float* bp = p.beta + first * p.beta_stride + h;
    for (int t = 0; t < len; ++t) {
        u4 qw[R / 8], kw[R / 8];
#pragma unroll
        for (int i = 0; i < R / 8; ++i) {
            qw[i] = *reinterpret_cast<const u4*>(qp + 8 * i);
            kw[i] = *reinterpret_cast<const u4*>(kp + 8 * i);
        }
        const u2 vw = *reinterpret_cast<const u2*>(vp);
        const float a = expf(*gp), beta = *bp;
        qp += p.q_stride, kp += p.k_stride, vp += p.v_stride, gp += p.g_stride, bp += p.beta_stride;
        f4 r = {0.f, 0.f, 0.f, 0.f}, u = {0.f, 0.f, 0.f, 0.f};
        float qk = 0.f, qq = 0.f, kk = 0.f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float kj = bf16_at(kw[j / 8], j % 8), qj = bf16_at(qw[j / 8], j % 8);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                r[c] = fmaf(kj, S[j][c], r[c]);
                u[c] = fmaf(qj, S[j][c], u[c]);
            }
            qk = fmaf(qj, kj, qk);
            if (p.qk_norm) {
                qq = fmaf(qj, qj, qq);
                kk = fmaf(kj, kj, kk);
            }
        }
        float rq = p.scale, rk = 1.f;
        if (p.qk_norm) {
            rq = p.scale / sqrtf(sum_groups(qq) + kNormEps);
            rk = 1.f / sqrtf(sum_groups(kk) + kNormEps);
        }
        qk = sum_groups(qk) * rk;
        f4 o, d;
        const float v[4] = {__uint_as_float(vw[0] << 16), __uint_as_float(vw[0] & 0xFFFF0000u), __uint_as_float(vw[1] << 16),
                            __uint_as_float(vw[1] & 0xFFFF0000u)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float rc = sum_groups(r[c]) * rk, uc = sum_groups(u[c]);
            const float dc = beta * fmaf(-a, rc, v[c]);
            o[c] = rq * fmaf(qk, dc, a * uc);
            d[c] = rk * dc;
        }
#pragma unroll
        for (int j = 0; j < R; ++j) {
            const float kj = bf16_at(kw[j / 8], j % 8);
#pragma unroll
            for (int c = 0; c < 4; ++c) S[j][c] = fmaf(kj, d[c], a * S[j][c]);
        }
        if (p.o && kg == 0 && on) {
            u2 w;
            w[0] = wkv7::pack_bf16x2(o[0], o[1]);
            w[1] = wkv7::pack_bf16x2(o[2], o[3]);
            *reinterpret_cast<u2*>(p.o + (first + t) * p.o_stride + (int64_t)h * p.V + col) = w;
        }
        if (p.snapshots && on) {
            float* const to = p.snapshots + (((int64_t)n * p.T + t) * p.Hv + h) * ((int64_t)K * p.V) + at;
#pragma unroll
            for (int j = 0; j < R; ++j) __builtin_nontemporal_store(S[j], reinterpret_cast<f4*>(to + (int64_t)j * p.V));
        }
    }
    float* const to = final_state(p, n, h);
    if (to && on)
#pragma unroll
        for (int j = 0; j < R; ++j) __builtin_nontemporal_store(S[j], reinterpret_cast<f4*>(to + at + (int64_t)j * p.V));
}

}  // namespace

hipError_t launch_tokens(const Params& p, hipStream_t stream) {
    const int blocks = (p.V + kCols - 1) / kCols;
    const int64_t units = (int64_t)p.num_seqs * p.Hv * blocks;
    const dim3 grid((unsigned)((units + 3) / 4)), block(256);
    if (p.K == 64)
        hipLaunchKernelGGL(delta_token_kernel<64>, grid, block, 0, stream, p, blocks, units);
    else
        hipLaunchKernelGGL(delta_token_kernel<128>, grid, block, 0, stream, p, blocks, units);
    return hipGetLastError();
}

}  // namespace delta
