// delta_chunk.hip -- the gated delta rule by chunks of 64 tokens, on the matrix cores (include/delta.h).
//
// With c_i the sum of g up to token i of a chunk, k and q normalised and q scaled, S the state before the chunk:
//     A_ij = beta_i (k_i . k_j) e^(c_i - c_j), i > j           T = (1 + A)^-1, lower triangular
//     R_i = beta_i (v_i - e^c_i S^T k_i)                       D = T R           (what each token writes)
//     B_ij = (q_i . k_j) e^(c_i - c_j), i >= j                 o_i = e^c_i S^T q_i + sum_j B_ij D_j
//     S <- e^c_63 S + sum_j e^(c_63 - c_j) k_j D_j^T
// Two launches: one makes T, B and the tokens' factors of every chunk, all chunks at once; the other goes through a row's chunks in
// order.  Norms, decays and beta are factors of rows, kept apart from the products, whose one operand is so the caller's bf16, exact.
// The other, fp32, is split into three bf16 parts, 24 bits, wherever it leads to the state; the outputs, bf16, take two parts.
// A product with a triangle multiplies the zeros above its diagonal too, and 0 times an infinity or NaN of a later token is NaN for an
// earlier one.  So on the way to T 0 goes in the place of what is out of range, and from the first token that had such a value, R is
// NaN.  In the scan the state of R's column is then NaN, as it is token by token; outputs that came out of range are made again, by the
// wavefronts which make them, without the tokens that cannot have a part in them.
// Measured, 4096 tokens, 16 query/key and 32 value heads of 128: 31 to 34 us and 95 us (token by token 5.4 ms).
#include "delta_device.h"

namespace delta {
namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f4 mfma(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Waits for this wavefront's LDS traffic and then for the workgroup; global loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kRow = 68;           // floats between rows of a matrix in LDS: 16-byte reads of 16 rows meet no bank twice
constexpr float kMost = 3.3895314e38f;  // the largest bf16: no part of what is within is infinite
constexpr float kLeast = -1e4f;    // decays below e^-10000 are 0 all the same, and differences of their sums stay finite

// Of a 64 x 64 lower triangle in blocks of 16 x 32: tile t = 0, 1 has one, tile 2, 3 have two.
__device__ __forceinline__ constexpr int block_of(int tile, int half) { return tile < 2 ? tile : 2 * tile - 2 + half; }
// Token of row `row` of tile t.  Rows are dealt out so that the four rows which a lane holds of tile 2b and the four of tile 2b + 1
// are eight tokens in a row: a result is the next product's operand without an exchange between lanes.  Rows of the state too.
__device__ __forceinline__ int token_of(int tile, int row) { return 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3); }

// Which row and chunk a slot of the workspace holds; false for a slot that holds none.
__device__ __forceinline__ int64_t first_slot(const Params& p, const Work& w, int n, int64_t first) {
    return p.cu ? ragged_slot(w.shift, w.rows, n, first) : (int64_t)n * ((p.T + kChunk - 1) / kChunk);
}
__device__ __forceinline__ bool locate(const Params& p, const Work& w, int64_t slot, int& n, int64_t& first, int& len, int& chunk) {
    if (p.cu) {
        int lo = 0, hi = p.num_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            int64_t s = p.cu[mid];
            s = s < 0 ? 0 : s > p.total_tokens ? p.total_tokens : s;
            if (ragged_slot(w.shift, w.rows, mid, s) <= slot) lo = mid; else hi = mid;
        }
        n = lo;
    } else {
        n = (int)(slot / ((p.T + kChunk - 1) / kChunk));
    }
    extent(p, n, first, len);
    const int64_t c = slot - first_slot(p, w, n, first);
    chunk = (int)c;
    return c >= 0 && c * kChunk < len && !(p.cu && len <= p.token_len);
}

// x as three bf16 parts (24 bits), for two values at a time
__device__ __forceinline__ void split3(float x0, float x1, uint32_t& a, uint32_t& b, uint32_t& c) {
    typedef wkv7::f2_t f2;
    const f2 x = {x0, x1};
    const wkv7::bf16x2_t h = __builtin_convertvector(x, wkv7::bf16x2_t);
    const wkv7::bf16x2_t m0 = wkv7::bf16_pair_in_register(0x0000BF80u), m1 = wkv7::bf16_pair_in_register(0xBF800000u);
    const f2 y = {__builtin_amdgcn_fdot2_f32_bf16(h, m0, x0, false), __builtin_amdgcn_fdot2_f32_bf16(h, m1, x1, false)};
    a = __builtin_bit_cast(uint32_t, h);
    wkv7::split_pair(y[0], y[1], b, c);
}

// split3 of two tokens' values, of which the later, x1, reaches no part of x0: where it is infinite or NaN, split3's products with 0 do.
__device__ __forceinline__ void split3_in_order(float x0, float x1, uint32_t& a, uint32_t& b, uint32_t& c) {
    typedef wkv7::f2_t f2;
    const wkv7::bf16x2_t m1 = wkv7::bf16_pair_in_register(0xBF800000u);
    const auto rest = [&](f2 x, uint32_t& part) {
        const wkv7::bf16x2_t h = __builtin_convertvector(x, wkv7::bf16x2_t);
        part = __builtin_bit_cast(uint32_t, h);
        return f2{x[0] - __uint_as_float(part << 16), __builtin_amdgcn_fdot2_f32_bf16(h, m1, x[1], false)};
    };
    const f2 z = rest(rest(f2{x0, x1}, a), b);
    c = wkv7::pack_bf16x2(z[0], z[1]);
}

__device__ __forceinline__ bool within(float x) { return fabsf(x) <= kMost; }  // false for NaN
__device__ __forceinline__ bool within(f4 x) { return within(x[0]) && within(x[1]) && within(x[2]) && within(x[3]); }
// x, whose elements belong to the tokens from `token` on, with 0 for what is not within, whose first token *first learns.
__device__ __forceinline__ f4 kept(f4 x, int token, int* first) {
    if (!within(x)) {
        atomicMin(first, token + (!within(x[0]) ? 0 : !within(x[1]) ? 1 : !within(x[2]) ? 2 : 3));
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = within(x[r]) ? x[r] : 0.f;
    }
    return x;
}

// x of the lane that DPP control `kCtrl` names, 0 where there is none or the row of 16 lanes is not in `kRows`
template <int kCtrl, int kRows>
__device__ __forceinline__ double moved(double x) {
    const u2 w = __builtin_bit_cast(u2, x);
    const uint32_t lo = w[0], hi = w[1];
    return __builtin_bit_cast(double, u2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)lo, kCtrl, kRows, 0xF, false),
                                         (uint32_t)__builtin_amdgcn_update_dpp(0, (int)hi, kCtrl, kRows, 0xF, false)});
}

// The ragged rows that run by chunks into w.order, longest first (to a chunk, and up to kOrders of them): a scan that begins with its
// longest rows ends together, and workgroups without a row come last, where they hold nothing up.  Which of two rows as long comes
// first is left to chance; results do not depend on it.
constexpr int kOrders = 256;
__device__ void order_rows(const Params& p, const Work& w, int32_t* count) {
    const int tid = threadIdx.x;
    const auto place = [&](int n) {  // -1: runs by tokens
        int64_t first;
        int len;
        extent(p, n, first, len);
        return len <= p.token_len ? -1 : kOrders - 1 - min(kOrders - 1, len / kChunk);
    };
    for (int i = tid; i < kOrders; i += 256) count[i] = 0;
    __syncthreads();
    for (int n = tid; n < p.num_seqs; n += 256) {
        const int at = place(n);
        if (at >= 0) atomicAdd(&count[at], 1);
    }
    __syncthreads();
    if (tid == 0) {
        int sum = 0;
        for (int i = 0; i < kOrders; ++i) {
            const int c = count[i];
            count[i] = sum;
            sum += c;
        }
        w.order[0] = sum;
    }
    __syncthreads();
    for (int n = tid; n < p.num_seqs; n += 256) {
        const int at = place(n);
        if (at >= 0) w.order[1 + atomicAdd(&count[at], 1)] = n;
    }
}

// One workgroup: a chunk of a query/key head, then each of the value heads that share it.  Bound by its bytes: 48 KiB of operands a
// query/key head and 31 KiB a value head are written for each chunk, 139 MB with what is read for 4096 tokens in 31 to 34 us.
template <int K>
__global__ __launch_bounds__(256, 3) void delta_prep_kernel(const Params p, const Work w) {
    constexpr int kSteps = K / 32, kPitch = K + 8;
    __shared__ __attribute__((aligned(16))) float am[64 * kRow];   // K's tile, then A, then T
    __shared__ __attribute__((aligned(16))) float bm[64 * kRow];   // Q's tile, then products on the way to T
    __shared__ __attribute__((aligned(16))) double cs[64];
    __shared__ __attribute__((aligned(16))) float rk[64], rq[64], be[64];
    __shared__ int lost;  // the first token whose row of A or T is not within
    float* const mm = bm;
    static_assert(64 * kPitch * 2 <= (int)sizeof(bm), "");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int row = lane & 15, quad = lane >> 4;
    if (p.cu && blockIdx.x == gridDim.x - 1) {
        order_rows(p, w, reinterpret_cast<int32_t*>(am));
        return;
    }
    const int64_t slot = blockIdx.x / (uint32_t)p.Hk;
    const int hk = (int)(blockIdx.x % (uint32_t)p.Hk);
    int n, len, chunk;
    int64_t first;
    if (!locate(p, w, slot, n, first, len, chunk)) return;
    first += (int64_t)chunk * kChunk;
    len = min(len - chunk * kChunk, kChunk);  // tokens of this chunk

    // K and Q by whole rows into LDS, zeros past the last token, and from there in operand order
    constexpr int kRowPieces = K / 8, kPieces = 64 * kRowPieces / 256;
    uint16_t* const k_tile = reinterpret_cast<uint16_t*>(am);
    uint16_t* const q_tile = reinterpret_cast<uint16_t*>(bm);
    {
        u4 x[kPieces], y[kPieces];
        const int at = tid / kRowPieces, piece = tid % kRowPieces * 8;
        const uint16_t* const kp = p.k + first * p.k_stride + hk * K + piece;
        const uint16_t* const qp = p.q + first * p.q_stride + hk * K + piece;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int t = at + i * (256 / kRowPieces), from = min(t, len - 1);
            x[i] = *reinterpret_cast<const u4*>(kp + from * p.k_stride);
            y[i] = *reinterpret_cast<const u4*>(qp + from * p.q_stride);
            if (t >= len) x[i] = y[i] = u4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int t = at + i * (256 / kRowPieces);
            *reinterpret_cast<u4*>(k_tile + t * kPitch + piece) = x[i];
            *reinterpret_cast<u4*>(q_tile + t * kPitch + piece) = y[i];
        }
    }
    __syncthreads();
    const auto rows = [&](const uint16_t* x, int token, u4* f) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) f[s] = *reinterpret_cast<const u4*>(x + token * kPitch + 32 * s + 8 * quad);
    };
    const bool two = wave >= 2;
    f4 kk[4], kq[4];  // K K^T by rows of this wavefront's 16 tokens in a row; K Q^T by columns of its dealt out ones
    char* const operands = w.kq + (slot * p.Hk + hk) * (3 * K * kChunk * 2);
    {
        u4 kf[kSteps], of[kSteps];
        rows(k_tile, 16 * wave + row, kf);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kk[j] = kq[j] = f4{0.f, 0.f, 0.f, 0.f};
            if (j <= wave) {
                rows(k_tile, 16 * j + row, of);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) kk[j] = mfma(kf[s], of[s], kk[j]);
            }
        }
        u4 qf[kSteps];
        const int mine = token_of(wave, row);
        rows(q_tile, mine, qf);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < 2 || two) {
                rows(k_tile, token_of(j, row), of);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) kq[j] = mfma(of[s], qf[s], kq[j]);
            }
        rows(k_tile, mine, kf);
        float nk = 0.f, nq = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = bf16_at(kf[s], i), y = bf16_at(qf[s], i);
                nk = fmaf(x, x, nk);
                nq = fmaf(y, y, nq);
            }
            *reinterpret_cast<u4*>(operands + ((wave * kSteps + s) * 64 + lane) * 16) = kf[s];
            *reinterpret_cast<u4*>(operands + K * kChunk * 2 + ((wave * kSteps + s) * 64 + lane) * 16) = qf[s];
        }
        nk += __shfl_xor(nk, 16), nq += __shfl_xor(nq, 16);
        nk += __shfl_xor(nk, 32), nq += __shfl_xor(nq, 32);
        if (quad == 0) {
            rk[mine] = p.qk_norm ? 1.f / sqrtf(nk + kNormEps) : 1.f;
            rq[mine] = p.qk_norm ? p.scale / sqrtf(nq + kNormEps) : p.scale;
        }
    }
    // K^T in operand order: tile of 16 rows of the state, half of the tokens, lane
    u4* const kt = reinterpret_cast<u4*>(operands + 2 * K * kChunk * 2);
    for (int e = tid; e < K / 16 * 2 * 64; e += 256) {
        const int l = e & 63, half = (e >> 6) & 1, t = e >> 7, d = token_of(t, l & 15);
        u4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint16_t* const at = k_tile + (32 * half + 8 * (l >> 4) + 2 * j) * kPitch + d;
            x[j] = (uint32_t)at[0] | (uint32_t)at[kPitch] << 16;
        }
        kt[e] = x;
    }

#pragma unroll 1
    for (int h = hk * p.share; h < (hk + 1) * p.share; ++h) {
        // (without this the addresses of a head's work are kept from head to head, in more registers than there are)
        asm("" : "+v"(row), "+v"(quad));
        char* const rec = w.rec + (slot * p.Hv + h) * kRecord;
        // The sums of g log2(e), in 64 bits: differences of far tokens' sums lose nothing, and the hardware's exp2, good to one unit in
        // the last place, takes them as they are.
        const int64_t token = first + min(lane, len - 1);
        const float g = p.g[token * p.g_stride + h], b = p.beta[token * p.beta_stride + h];
        double c = lane < len ? (double)(g < kLeast ? kLeast : g) * 1.4426950408889634 : 0.0;
        c += moved<0x111, 0xF>(c);  // row_shr by 1, 2, 4, 8
        c += moved<0x112, 0xF>(c);
        c += moved<0x114, 0xF>(c);
        c += moved<0x118, 0xF>(c);
        c += moved<0x142, 0xA>(c);  // the rows' sums: lane 15 to row 1, 47 to row 3, then 31 to rows 2 and 3
        c += moved<0x143, 0xC>(c);
        const double last = __shfl(c, 63);
        const float beta = lane < len ? b : 0.f;
        __syncthreads();  // the tiles are read; the head before is written
        if (wave == 0) {
            cs[lane] = c;
            be[lane] = beta;
            float* const f = reinterpret_cast<float*>(rec + kRecordFactors);
            const float gamma = __builtin_amdgcn_exp2f((float)c);
            f[lane] = beta;
            f[64 + lane] = beta * gamma * rk[lane];
            f[128 + lane] = __builtin_amdgcn_exp2f((float)(last - c)) * rk[lane];
            f[192 + lane] = gamma * rq[lane];
            if (lane == 0) f[256] = __builtin_amdgcn_exp2f((float)last), lost = kChunk;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j <= wave) {
                const int col = 16 * j + row, i0 = 16 * wave + 4 * quad;
                f4 x;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = i0 + r;
                    const float decay = i > col ? __builtin_amdgcn_exp2f((float)(cs[i] - cs[col])) * rk[col] : 0.f;
                    x[r] = i > col ? kk[j][r] * (be[i] * rk[i]) * decay : 0.f;
                }
                x = kept(x, i0, &lost);
#pragma unroll
                for (int r = 0; r < 4; ++r) am[(i0 + r) * kRow + col] = x[r];
            }
        {  // B, in two bf16 parts: the rows of a K Q^T that a lane has are its operand of B D
            const int i = token_of(wave, row);
            const double ci = cs[i];
            const float scale = rq[i];
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (half == 0 || two) {
                    u4 hi, lo;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        float x[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int j = 32 * half + 8 * quad + 2 * m + e;
                            const float decay = __builtin_amdgcn_exp2f((float)(ci - cs[j])) * rk[j];
                            x[e] = i >= j ? kq[2 * half + (m >> 1)][2 * (m & 1) + e] * scale * decay : 0.f;
                        }
                        uint32_t a, b;
                        wkv7::split_pair(x[0], x[1], a, b);
                        hi[m] = a, lo[m] = b;
                    }
                    char* const to = rec + kRecordB + block_of(wave, half) * 2048 + lane * 16;
                    *reinterpret_cast<u4*>(to) = hi;
                    *reinterpret_cast<u4*>(to + 1024) = lo;
                }
        }
        wkv7::wave_lds_sync();
        // the inverse of this wavefront's 16 x 16 block, a column a lane, by forward substitution
        {
            const float* const a = am + 16 * wave * (kRow + 1);
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s0 = i == row ? 1.f : 0.f, s1 = 0.f;
#pragma unroll
                for (int m = 0; m < (i + 3) / 4; ++m) {
                    const f4 y = *reinterpret_cast<const f4*>(a + i * kRow + 4 * m);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (4 * m + r < i) (r & 1 ? s1 : s0) = fmaf(-y[r], x[4 * m + r], r & 1 ? s1 : s0);
                }
                x[i] = s0 + s1;
                if (i == 7 || i == 11) __builtin_amdgcn_sched_barrier(0);  // a few rows of A at a time: all of them are 144 registers
            }
            if (!within(x[15])) {  // an infinity or NaN makes all rows behind it so too
                int first = 16 * wave + 15;
#pragma unroll
                for (int i = 15; i >= 0; --i)
                    if (!within(x[i])) x[i] = 0.f, first = 16 * wave + i;
                atomicMin(&lost, first);
            }
            wkv7::wave_lds_sync();
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i >> 2 == quad) am[(16 * wave + i) * kRow + 16 * wave + row] = x[i];
        }
        __syncthreads();
        // Products of 16 x 16 blocks in fp32: of the second operand lane `quad` holds rows 4 quad .., which are then the ones that
        // step s of the sum takes (4 quad + s), as they lie in a result.
        const auto left = [&](const float* m, int i, int k) {
            return *reinterpret_cast<const f4*>(m + (16 * i + row) * kRow + 16 * k + 4 * quad);
        };
        const auto right = [&](const float* m, int k, int j) {
            f4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = m[(16 * k + 4 * quad + r) * kRow + 16 * j + row];
            return x;
        };
        const auto times = [&](f4 a, f4 b, f4 c) {
#pragma unroll
            for (int s = 0; s < 4; ++s) c = mfma4(a[s], b[s], c);
            return c;
        };
        const auto put = [&](float* m, int i, int j, f4 x) {
#pragma unroll
            for (int r = 0; r < 4; ++r) m[(16 * i + 4 * quad + r) * kRow + 16 * j + row] = x[r];
        };
        const f4 zero = {0.f, 0.f, 0.f, 0.f};
        // [[P, 0], [X, Q]]^-1 = [[P^-1, 0], [-Q^-1 X P^-1, Q^-1]], for blocks of 16, then of 32
        if (wave < 2) {
            const int token0 = 16 * (2 * wave + 1) + 4 * quad;
            const f4 m = kept(times(left(am, 2 * wave + 1, 2 * wave), right(am, 2 * wave, 2 * wave), zero), token0, &lost);
            const f4 x = kept(times(left(am, 2 * wave + 1, 2 * wave + 1), m, zero), token0, &lost);
            put(am, 2 * wave + 1, 2 * wave, -x);
        }
        __syncthreads();
        const int i = wave >> 1, j = wave & 1, token0 = 16 * (2 + i) + 4 * quad;
        {
            f4 m = zero;
            for (int k = j; k < 2; ++k) m = times(left(am, 2 + i, k), right(am, k, j), m);
            put(mm, i, j, kept(m, token0, &lost));
        }
        __syncthreads();
        {
            f4 x = zero;
            for (int k = 0; k <= i; ++k) x = times(left(am, 2 + i, 2 + k), right(mm, k, j), x);
            put(am, 2 + i, j, -kept(x, token0, &lost));
        }
        __syncthreads();
        // R of the tokens from `lost` on is NaN by its factor
        if (wave == 0 && lane >= lost) reinterpret_cast<float*>(rec + kRecordFactors)[lane] = __builtin_nanf("");
        // T in three bf16 parts, in operand order
        for (int e = tid; e < 6 * 64; e += 256) {
            const int block = e >> 6, l = e & 63;
            const int t = block < 2 ? block : (block + 2) >> 1, half = block < 2 ? 0 : block & 1;
            const int i = token_of(t, l & 15), at = 32 * half + 8 * (l >> 4);
            u4 part[3];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                f4 x = *reinterpret_cast<const f4*>(am + i * kRow + at + 4 * m);
#pragma unroll
                for (int r = 0; r < 4; ++r)  // above the diagonal nothing was computed
                    if (at + 4 * m + r > i) x[r] = 0.f;
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    uint32_t a, b, c;
                    split3(x[2 * o], x[2 * o + 1], a, b, c);
                    part[0][2 * m + o] = a, part[1][2 * m + o] = b, part[2][2 * m + o] = c;
                }
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) *reinterpret_cast<u4*>(rec + kRecordT + ((block * 3 + m) * 64 + l) * 16) = part[m];
        }
    }
}

// One workgroup: 16 NT columns of a head's state, through a row's chunks.  Wavefronts 0 to 3 carry the state, a quarter of its rows
// each; the chain from one state to the next is what a long row waits for, so that nothing else is on it:
//     its rows' share of S^T k for all tokens, from registers | summed over the wavefronts, R, for its tokens | D for them | S
// with barriers between.  Wavefronts 4 to 7 have a quarter of the tokens each and make the outputs beside it.  Operands of the next
// chunk are asked for as soon as those of this one are used, while LDS is waited for, so the loads, 78 KiB a chunk, are spread over
// it: asked for together, at its begin, they held the chain up for a third of its time (4096 tokens 133 us then, 95 now, 1.5 us a chunk).
// By 32 columns a chunk takes 2.8 us, half the loads for each: taken where 16 would leave every CU two workgroups or more, were all rows
// to run by chunks (8 rows of 1276 tokens on average 227 us; by 16 columns 359).  Which of a ragged call's rows do is the device's
// knowledge, and little hangs on it: one row of 2048 tokens among 63 of one, 32 heads of 128, 76 us by 32 columns, 75 by 16.
template <int K, int NT>
__global__ __launch_bounds__(512, 2) void delta_scan_kernel(const Params p, const Work w) {
    constexpr int kSteps = K / 32, kTiles = K / 64;  // of the state's rows: MFMA steps, tiles of a wavefront
    __shared__ f4 pf[4][4][NT][64];                  // S^T k: [wavefront][tile of tokens]
    __shared__ u4 sf[kSteps][2][NT][64];             // the state, two parts
    __shared__ u4 rf[2][3][NT][64];                  // R
    __shared__ u4 df[2][2][NT][64];                  // D, two parts
    __shared__ u4 ef[2][3][NT][64];                  // D with the decay to the chunk's end
    const int tid = threadIdx.x, lane = tid & 63, role = __builtin_amdgcn_readfirstlane(tid >> 8),
              wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;
    const int col = lane & 15, quad = lane >> 4;
    // the columns of `together` heads follow each other on one XCD, whose L2 they share
    const uint32_t slices = (uint32_t)(p.V / (16 * NT)), each = slices * (uint32_t)w.together;
    const uint32_t group = blockIdx.x / 8 / each * 8 + blockIdx.x % 8, in = blockIdx.x / 8 % each;
    const int64_t unit = (int64_t)group * w.together + in / slices;
    if (unit >= (int64_t)(p.cu ? w.order[0] : p.num_seqs) * p.Hv) return;
    const int n = p.cu ? w.order[1 + (int)(unit / p.Hv)] : (int)(unit / p.Hv), h = (int)(unit % p.Hv), hk = h / p.share;
    const int col0 = (int)(in % slices) * 16 * NT;
    int64_t first;
    int len;
    extent(p, n, first, len);
    const int chunks = (len + kChunk - 1) / kChunk;
    const int64_t slot = first_slot(p, w, n, first);
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    const char* const records = wkv7::uniform_ptr(w.rec + (slot * p.Hv + h) * kRecord);
    const char* const operands = wkv7::uniform_ptr(w.kq + (slot * p.Hk + hk) * (3 * K * kChunk * 2));
    const int64_t record_size = p.Hv * kRecord, operand_size = (int64_t)p.Hk * (3 * K * kChunk * 2);
    const bool two = wave >= 2;  // these rows of the lower triangles have a second half
    const int token0 = token_of(wave, 4 * quad);     // the first of a lane's four
    const uint32_t at = lane * 16u, tokens_at = token0 * 4u;

    if (role == 1) {
        u4 q[kSteps], b[2][2];
        f4 gamma;
        const char *x = operands + (4 + wave) * (kSteps * 1024), *rec = records;
        const auto fetch_q = [&] {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[s] = *reinterpret_cast<const u4*>(x + s * 1024 + at);
        };
        const auto fetch_b = [&] {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int m = 0; m < 2; ++m)
                    b[half][m] = *reinterpret_cast<const u4*>(rec + kRecordB + (block_of(wave, two ? half : 0) * 2 + m) * 1024 + at);
            gamma = *reinterpret_cast<const f4*>(rec + kRecordFactors + 768 + tokens_at);
        };
        if (chunks > 0 && p.o) {
            fetch_q();
            fetch_b();
        }
        for (int c = 0; c < chunks; ++c) {
            x += c + 1 < chunks ? operand_size : 0;  // behind the last chunk: it again
            rec += c + 1 < chunks ? record_size : 0;
            lds_barrier();
            f4 O[NT][2];
            if (p.o) {
#pragma unroll
                for (int x = 0; x < NT; ++x) O[x][0] = O[x][1] = zero;
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    u4 a[kSteps][2];
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) a[s][0] = sf[s][0][x][lane], a[s][1] = sf[s][1][x][lane];
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) {
                        O[x][0] = mfma(q[s], a[s][0], O[x][0]);
                        O[x][1] = mfma(q[s], a[s][1], O[x][1]);
                    }
                }
                fetch_q();
            }
            lds_barrier();
            lds_barrier();
            if (p.o) {
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    u4 d[2][2];
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        if (half == 0 || two) d[half][0] = df[half][0][x][lane], d[half][1] = df[half][1][x][lane];
                    const auto output = [&] {
                        f4 y = (O[x][0] + O[x][1]) * gamma;
#pragma unroll
                        for (int half = 0; half < 2; ++half)
                            if (half == 0 || two) {
                                y = mfma(b[half][1], d[half][0], y);
                                y = mfma(b[half][0], d[half][1], y);
                                y = mfma(b[half][0], d[half][0], y);
                            }
                        return y;
                    };
                    f4 y = output();
                    if (__ballot(!within(y))) {  // D once more, from R and of D what is within; NaN from the first token that is not
                        int lost = kChunk;
                        const char* const t = records + c * record_size + kRecordT + at;
                        u4 r[2][3];
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
#pragma unroll
                            for (int m = 0; m < 3; ++m) r[half][m] = rf[half][m][x][lane];
#pragma unroll
                            for (int i = 7; i >= 0; --i)
                                if (!within(bf16_at(r[half][0], i)) || !within(bf16_at(r[half][1], i)) || !within(bf16_at(r[half][2], i))) {
                                    lost = min(lost, 32 * half + 8 * quad + i);
#pragma unroll
                                    for (int m = 0; m < 3; ++m) r[half][m][i / 2] &= i & 1 ? 0xFFFFu : 0xFFFF0000u;
                                }
                        }
#pragma unroll
                        for (int tile = 0; tile < 4; ++tile) {
                            f4 D[3] = {zero, zero, zero};
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                if (half == 0 || tile >= 2) {
                                    u4 tri[3];
#pragma unroll
                                    for (int m = 0; m < 3; ++m)
                                        tri[m] = *reinterpret_cast<const u4*>(t + (block_of(tile, half) * 3 + m) * 1024);
                                    D[2] = mfma(tri[2], r[half][0], D[2]);
                                    D[1] = mfma(tri[1], r[half][0], D[1]);
                                    D[0] = mfma(tri[0], r[half][0], D[0]);
                                    D[2] = mfma(tri[0], r[half][2], D[2]);
                                    D[1] = mfma(tri[0], r[half][1], D[1]);
                                    D[2] = mfma(tri[1], r[half][1], D[2]);
                                }
                            f4 z = D[0] + (D[1] + D[2]);
#pragma unroll
                            for (int i = 3; i >= 0; --i)
                                if (!within(z[i])) z[i] = 0.f, lost = min(lost, token_of(tile, 4 * quad) + i);
#pragma unroll
                            for (int m = 0; m < 2; ++m) {
                                uint32_t i, j;
                                wkv7::split_pair(z[2 * m], z[2 * m + 1], i, j);
                                d[tile >> 1][0][2 * (tile & 1) + m] = i, d[tile >> 1][1][2 * (tile & 1) + m] = j;
                            }
                        }
                        lost = min(lost, __shfl_xor(lost, 16));
                        lost = min(lost, __shfl_xor(lost, 32));
                        y = output();
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (token0 + i >= lost) y[i] = __builtin_nanf("");
                    }
                    const int t0 = c * kChunk + token0;
                    uint16_t* const to = p.o + (first + t0) * p.o_stride + ((int64_t)h * p.V + col0 + 16 * x + col);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (t0 + r < len) to[r * p.o_stride] = wkv7::f32_to_bf16(y[r]);
                }
                fetch_b();
            }
        }
        return;
    }

    __builtin_amdgcn_s_setprio(2);  // the chain goes first where both have something to issue
    // rows of the state in tile 2b + j, row r of a lane: 32 b + 8 quad + 4 j + r
    const float* const from = initial(p, n, h);
    float* const to = final_state(p, n, h);
    const auto state_at = [&](int tile, int r) {
        const int t = wave * kTiles + tile;
        return (int64_t)(32 * (t >> 1) + 8 * quad + 4 * (t & 1) + r) * p.V + col0 + col;
    };
    f4 S[kTiles][NT];
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][x][r] = from ? from[state_at(t, r) + 16 * x] : 0.f;

    constexpr bool kHalf = kTiles == 1;  // its rows are half an MFMA step: the other half is zeros
    const int my_step = kHalf ? wave >> 1 : wave;
    u4 k[4], tri[2][3], kt[kTiles][2];
    f4 beta, seen, left;
    float keep;
    uint16_t v[NT][4];
    const char *head = operands, *rec = records;
    const uint16_t* vp = wkv7::uniform_ptr(p.v + first * p.v_stride + (int64_t)h * p.V + col0);
    uint32_t v_at[4];
    const auto tokens_of_v = [&](int most) {  // past the last token: it again, with factors of 0
#pragma unroll
        for (int r = 0; r < 4; ++r) v_at[r] = (uint32_t)min(token_of(wave, 4 * quad + r), most) * (uint32_t)p.v_stride + col;
    };
    const auto fetch_k = [&] {
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const u4*>(head + (my_step + i * kSteps) * 1024 + at);
    };
    const auto fetch_v = [&] {
        beta = *reinterpret_cast<const f4*>(rec + kRecordFactors + tokens_at);
        seen = *reinterpret_cast<const f4*>(rec + kRecordFactors + 256 + tokens_at);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int x = 0; x < NT; ++x) v[x][r] = vp[v_at[r] + 16 * x];
    };
    const auto fetch_t = [&] {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int m = 0; m < 3; ++m)
                tri[half][m] = *reinterpret_cast<const u4*>(rec + kRecordT + (block_of(wave, two ? half : 0) * 3 + m) * 1024 + at);
        left = *reinterpret_cast<const f4*>(rec + kRecordFactors + 512 + tokens_at);
    };
    const auto fetch_kt = [&] {
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                kt[t][half] = *reinterpret_cast<const u4*>(head + (8 * kSteps + 2 * kTiles * wave + t * 2 + half) * 1024 + at);
        keep = *reinterpret_cast<const float*>(rec + kRecordFactors + 1024);
    };
    // the state to the other wavefronts (two parts), and this one's share of S^T k (all three)
    const auto hand_on = [&] {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            u4 part[3] = {u4{0, 0, 0, 0}, u4{0, 0, 0, 0}, u4{0, 0, 0, 0}};
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    uint32_t i, j, l;
                    split3(S[t][x][2 * m], S[t][x][2 * m + 1], i, j, l);
                    part[0][2 * t + m] = i, part[1][2 * t + m] = j, part[2][2 * t + m] = l;
                }
            if constexpr (kHalf) {
#pragma unroll
                for (int m = 0; m < 2; ++m) reinterpret_cast<u2*>(&sf[my_step][m][x][lane])[wave & 1] = u2{part[m][0], part[m][1]};
                if (wave & 1)
#pragma unroll
                    for (int m = 0; m < 3; ++m) part[m] = u4{0, 0, part[m][0], part[m][1]};
            } else {
#pragma unroll
                for (int m = 0; m < 2; ++m) sf[my_step][m][x][lane] = part[m];
            }
            f4 P[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) P[i] = mfma(k[i], part[2], zero);
#pragma unroll
            for (int i = 0; i < 4; ++i) P[i] = mfma(k[i], part[1], P[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) P[i] = mfma(k[i], part[0], P[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) pf[wave][i][x][lane] = P[i];
        }
    };
    if (chunks > 0) {
        tokens_of_v(min(len, kChunk) - 1);
        fetch_k();
        fetch_v();
        fetch_t();
        fetch_kt();
        hand_on();
    }
    for (int c = 0; c < chunks; ++c) {
        const bool more = c + 1 < chunks;
        head += more ? operand_size : 0;  // behind the last chunk: it again
        rec += more ? record_size : 0;
        vp += more ? kChunk * p.v_stride : 0;
        if (more && len - (c + 1) * kChunk < kChunk) tokens_of_v(len - (c + 1) * kChunk - 1);
        lds_barrier();
        // Operands that were used last before are asked for here and below while the answers of LDS are awaited.
        f4 share[4][NT];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int x = 0; x < NT; ++x) share[i][x] = pf[i][wave][x][lane];
        fetch_k();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const f4 P = (share[0][x] + share[1][x]) + (share[2][x] + share[3][x]);
            f4 R;
            u2 a, b, d;
#pragma unroll
            for (int r = 0; r < 4; ++r) R[r] = fmaf(-seen[r], P[r], beta[r] * wkv7::bf16_to_f32(v[x][r]));
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t i, j, l;
                split3_in_order(R[2 * m], R[2 * m + 1], i, j, l);
                a[m] = i, b[m] = j, d[m] = l;
            }
            reinterpret_cast<u2*>(&rf[wave >> 1][0][x][lane])[wave & 1] = a;
            reinterpret_cast<u2*>(&rf[wave >> 1][1][x][lane])[wave & 1] = b;
            reinterpret_cast<u2*>(&rf[wave >> 1][2][x][lane])[wave & 1] = d;
        }
        lds_barrier();
        f4 D[NT][3];
#pragma unroll
        for (int x = 0; x < NT; ++x) D[x][0] = D[x][1] = D[x][2] = zero;
        u4 y[2][3][NT];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int m = 0; m < 3; ++m)
#pragma unroll
                for (int x = 0; x < NT; ++x) y[half][m][x] = rf[half][m][x][lane];
        fetch_v();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int half = 0; half < 2; ++half)
            if (half == 0 || two)
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    D[x][2] = mfma(tri[half][2], y[half][0][x], D[x][2]);
                    D[x][1] = mfma(tri[half][1], y[half][0][x], D[x][1]);
                    D[x][0] = mfma(tri[half][0], y[half][0][x], D[x][0]);
                    D[x][2] = mfma(tri[half][0], y[half][2][x], D[x][2]);
                    D[x][1] = mfma(tri[half][0], y[half][1][x], D[x][1]);
                    D[x][2] = mfma(tri[half][1], y[half][1][x], D[x][2]);
                }
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const f4 d = D[x][0] + (D[x][1] + D[x][2]);
            u2 part[5];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t i, j, l;
                split3(d[2 * m] * left[2 * m], d[2 * m + 1] * left[2 * m + 1], i, j, l);
                part[0][m] = i, part[1][m] = j, part[2][m] = l;
                wkv7::split_pair(d[2 * m], d[2 * m + 1], i, j);
                part[3][m] = i, part[4][m] = j;
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) reinterpret_cast<u2*>(&ef[wave >> 1][m][x][lane])[wave & 1] = part[m];
#pragma unroll
            for (int m = 0; m < 2; ++m) reinterpret_cast<u2*>(&df[wave >> 1][m][x][lane])[wave & 1] = part[3 + m];
        }
        lds_barrier();
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int x = 0; x < NT; ++x) y[half][part][x] = ef[half][part][x][lane];
        fetch_t();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int x = 0; x < NT; ++x) S[t][x] *= keep;
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) S[t][x] = mfma(kt[t][half], y[half][part][x], S[t][x]);
        fetch_kt();
        if (more) hand_on();
    }
    if (to)
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int r = 0; r < 4; ++r) to[state_at(t, r) + 16 * x] = S[t][x][r];
}

template <int K>
hipError_t launch(const Params& p, const Work& w, int64_t slots, bool wide, hipStream_t stream) {
    hipLaunchKernelGGL(delta_prep_kernel<K>, dim3((unsigned)(slots * p.Hk + (p.cu ? 1 : 0))), dim3(256), 0, stream, p, w);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t rows = p.cu ? long_rows(p.num_seqs, p.total_tokens, p.token_len) : p.num_seqs;
    const int64_t groups = (rows * p.Hv / w.together + 7) / 8 * 8;
    if (wide)
        hipLaunchKernelGGL((delta_scan_kernel<K, 2>), dim3((unsigned)(groups * w.together * (p.V / 32))), dim3(512), 0, stream, p, w);
    else
        hipLaunchKernelGGL((delta_scan_kernel<K, 1>), dim3((unsigned)(groups * w.together * (p.V / 16))), dim3(512), 0, stream, p, w);
    return hipGetLastError();
}

}  // namespace

Slots chunk_slots(int32_t num_seqs, int32_t T, int64_t total_tokens, int32_t token_len, bool ragged) {
    return ragged ? ragged_slots(num_seqs, total_tokens, token_len) : row_slots(num_seqs, T);
}
int64_t chunk_groups(int64_t rows, int32_t Hv, int32_t V) { return (rows + 7) / 8 * 8 * Hv * (V / 16); }
size_t chunk_workspace(int64_t slots, int32_t num_seqs, int32_t Hk, int32_t Hv, int32_t K) {
    return (size_t)slots * (Hk * (size_t)(3 * K * kChunk * 2) + Hv * (size_t)kRecord) + (size_t)(num_seqs + 1) * 4;
}

hipError_t launch_chunks(const Params& p, int cus, hipStream_t stream) {
    const Slots of = chunk_slots(p.num_seqs, p.T, p.total_tokens, p.token_len, p.cu != nullptr);
    const int64_t slots = of.count;
    Work w;
    w.shift = of.shift, w.rows = of.rows;
    w.kq = p.workspace;
    w.rec = p.workspace + slots * p.Hk * (int64_t)(3 * p.K * kChunk * 2);
    w.order = reinterpret_cast<int32_t*>(w.rec + slots * p.Hv * kRecord);
    w.together = (int64_t)p.num_seqs * p.Hk >= 8 ? p.share : 1;
    const bool wide = p.V % 32 == 0 && (int64_t)p.num_seqs * p.Hv * (p.V / 32) >= 2 * cus;
    return p.K == 64 ? launch<64>(p, w, slots, wide, stream) : launch<128>(p, w, slots, wide, stream);
}

}  // namespace delta
