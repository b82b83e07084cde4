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
constexpr float kLeast = -1e4f;    // decays below e^-10000 are 0 all the same, and differences of their sums stay finite

// Of a 64 x 64 lower triangle in blocks of 16 x 32: tile t = 0, 1 has one, tile 2, 3 have two.
__device__ __forceinline__ constexpr int block_of(int tile, int half) { return tile < 2 ? tile : 2 * tile - 2 + half; }
// Token of row `row` of tile t.  Rows are dealt out so that the four rows which a lane holds of tile 2b and the four of tile 2b + 1
// are eight tokens in a row: a result is the next product's operand without an exchange between lanes.  Rows of the state too.
__device__ __forceinline__ int token_of(int tile, int row) { return 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (tile & 1) + (row & 3); }

// Which row and chunk a slot of the workspace holds; false for a slot that holds none.  Ragged rows begin at slot
// cu[n] / 64 + n, which leaves each one room enough.
__device__ __forceinline__ int64_t first_slot(const Params& p, int n, int64_t first) {
    return p.cu ? first / kChunk + n : (int64_t)n * ((p.T + kChunk - 1) / kChunk);
}
__device__ __forceinline__ bool locate(const Params& p, int64_t slot, int& n, int64_t& first, int& len, int& chunk) {
    if (p.cu) {
        int lo = 0, hi = p.num_seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            int64_t s = p.cu[mid];
            s = s < 0 ? 0 : s > p.total_tokens ? p.total_tokens : s;
            if (s / kChunk + mid <= slot) lo = mid; else hi = mid;
        }
        n = lo;
    } else {
        n = (int)(slot / ((p.T + kChunk - 1) / kChunk));
    }
    extent(p, n, first, len);
    const int64_t c = slot - first_slot(p, n, first);
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

// One workgroup: a chunk of a query/key head, then each of the value heads that share it.
template <int K>
__global__ __launch_bounds__(256, 3) void delta_prep_kernel(const Params p, const Work w) {
    constexpr int kSteps = K / 32, kPitch = K + 8;
    __shared__ __attribute__((aligned(16))) float am[64 * kRow];   // K's tile, then A, then T
    __shared__ __attribute__((aligned(16))) float bm[64 * kRow];   // Q's tile, then B
    __shared__ __attribute__((aligned(16))) float mm[32 * kRow];
    __shared__ double cs[64];
    __shared__ float rk[64], rq[64], be[64];
    static_assert(64 * kPitch * 2 <= (int)sizeof(bm), "");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int row = lane & 15, quad = lane >> 4;
    const int64_t slot = blockIdx.x / (uint32_t)p.Hk;
    const int hk = (int)(blockIdx.x % (uint32_t)p.Hk);
    int n, len, chunk;
    int64_t first;
    if (!locate(p, slot, n, first, len, chunk)) return;
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
    const auto rows = [&](const uint16_t* x, int block, u4* f) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) f[s] = *reinterpret_cast<const u4*>(x + (16 * block + row) * kPitch + 32 * s + 8 * quad);
    };
    f4 kk[4], qk[4];
    char* const operands = w.kq + (slot * p.Hk + hk) * (3 * K * kChunk * 2);
    {
        u4 kf[kSteps], qf[kSteps];
        rows(k_tile, wave, kf);
        rows(q_tile, wave, qf);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            kk[j] = qk[j] = f4{0.f, 0.f, 0.f, 0.f};
            if (j <= wave) {
                u4 of[kSteps];
                rows(k_tile, j, of);
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    kk[j] = mfma(kf[s], of[s], kk[j]);
                    qk[j] = mfma(qf[s], of[s], qk[j]);
                }
            }
        }
        float nk = 0.f, nq = 0.f;
        const int t = 16 * wave + row, tile = 2 * (t >> 5) + (t >> 2 & 1), to = 16 * quad + 4 * (t >> 3 & 3) + (t & 3);  // token_of(tile, to) = t
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = bf16_at(kf[s], i), y = bf16_at(qf[s], i);
                nk = fmaf(x, x, nk);
                nq = fmaf(y, y, nq);
            }
            *reinterpret_cast<u4*>(operands + ((tile * kSteps + s) * 64 + to) * 16) = kf[s];
            *reinterpret_cast<u4*>(operands + K * kChunk * 2 + ((tile * kSteps + s) * 64 + to) * 16) = qf[s];
        }
        nk += __shfl_xor(nk, 16), nq += __shfl_xor(nq, 16);
        nk += __shfl_xor(nk, 32), nq += __shfl_xor(nq, 32);
        if (quad == 0) {
            rk[16 * wave + row] = p.qk_norm ? 1.f / sqrtf(nk + kNormEps) : 1.f;
            rq[16 * wave + row] = p.qk_norm ? p.scale / sqrtf(nq + kNormEps) : p.scale;
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
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double other = __shfl_up(c, d);
            c += lane >= d ? other : 0.0;
        }
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
            if (lane == 0) f[256] = __builtin_amdgcn_exp2f((float)last);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j <= wave) {
                const int col = 16 * j + row;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = 16 * wave + 4 * quad + r;
                    const float decay = i >= col ? __builtin_amdgcn_exp2f((float)(cs[i] - cs[col])) * rk[col] : 0.f;
                    am[i * kRow + col] = i > col ? kk[j][r] * (be[i] * rk[i]) * decay : 0.f;
                    bm[i * kRow + col] = qk[j][r] * rq[i] * decay;
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
            const f4 m = times(left(am, 2 * wave + 1, 2 * wave), right(am, 2 * wave, 2 * wave), zero);
            const f4 x = times(left(am, 2 * wave + 1, 2 * wave + 1), m, zero);
            put(am, 2 * wave + 1, 2 * wave, -x);
        }
        __syncthreads();
        const int i = wave >> 1, j = wave & 1;
        {
            f4 m = zero;
            for (int k = j; k < 2; ++k) m = times(left(am, 2 + i, k), right(am, k, j), m);
            put(mm, i, j, m);
        }
        __syncthreads();
        {
            f4 x = zero;
            for (int k = 0; k <= i; ++k) x = times(left(am, 2 + i, 2 + k), right(mm, k, j), x);
            put(am, 2 + i, j, -x);
        }
        __syncthreads();
        // T in three bf16 parts and B in two, in operand order
        for (int e = tid; e < 6 * 64; e += 256) {
            const int block = e >> 6, l = e & 63;
            const int t = block < 2 ? block : (block + 2) >> 1, half = block < 2 ? 0 : block & 1;
            const int i = token_of(t, l & 15), at = 32 * half + 8 * (l >> 4);
            f4 x[2], y[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                x[m] = *reinterpret_cast<const f4*>(am + i * kRow + at + 4 * m);
                y[m] = *reinterpret_cast<const f4*>(bm + i * kRow + at + 4 * m);
#pragma unroll
                for (int r = 0; r < 4; ++r)  // above the diagonal nothing was computed
                    if (at + 4 * m + r > i) x[m][r] = y[m][r] = 0.f;
            }
            u4 hi, lo, part[3];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                uint32_t a, b, c;
                wkv7::split_pair(y[m >> 1][2 * (m & 1)], y[m >> 1][2 * (m & 1) + 1], a, b);
                hi[m] = a, lo[m] = b;
                split3(x[m >> 1][2 * (m & 1)], x[m >> 1][2 * (m & 1) + 1], a, b, c);
                part[0][m] = a, part[1][m] = b, part[2][m] = c;
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) *reinterpret_cast<u4*>(rec + kRecordT + ((block * 3 + m) * 64 + l) * 16) = part[m];
            *reinterpret_cast<u4*>(rec + kRecordB + ((block * 2) * 64 + l) * 16) = hi;
            *reinterpret_cast<u4*>(rec + kRecordB + ((block * 2 + 1) * 64 + l) * 16) = lo;
        }
    }
}

// What a wavefront reads of a chunk: one of those that carry the state ..
template <int K, int NT>
struct StateOperands {
    u4 k[K / 32];            // its 16 tokens
    u4 kt[K / 64][2];        // its rows of the state
    u4 t[2][3];              // its rows of T, in halves, three parts
    f4 beta, seen, left;     // the factors of its tokens' four rows of a lane
    float keep;
    uint16_t v[NT][4];
};
// .. and one of those that make the outputs.
template <int K>
struct OutputOperands {
    u4 q[K / 32];
    u4 b[2][2];
    f4 gamma;
};

// One workgroup: 16 NT columns of a head's state, through a row's chunks.  Wavefronts 0 to 3 carry the state, a quarter of the chunk's
// tokens and of the state's rows each, and hand each other operands through LDS: the state, R, D; the chain from one state to the
// next is what a long row waits for, so that nothing else is on it.  Wavefronts 4 to 7 have a quarter of the tokens each and make the outputs beside it.
template <int K, int NT>
__global__ __launch_bounds__(512, 2) void delta_scan_kernel(const Params p, const Work w) {
    constexpr int kSteps = K / 32, kTiles = K / 64;  // of the state's rows: MFMA steps, tiles of a wavefront
    __shared__ u4 sf[kSteps][3][NT][64];             // the state, three parts
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
    if (unit >= (int64_t)p.num_seqs * p.Hv) return;
    const int n = (int)(unit / p.Hv), h = (int)(unit % p.Hv), hk = h / p.share, col0 = (int)(in % slices) * 16 * NT;
    int64_t first;
    int len;
    extent(p, n, first, len);
    if (p.cu && len <= p.token_len) return;
    const int chunks = (len + kChunk - 1) / kChunk;
    const int64_t slot = first_slot(p, n, first);
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    const auto record = [&](int chunk) { return wkv7::uniform_ptr(w.rec + ((slot + chunk) * p.Hv + h) * kRecord); };
    const auto heads = [&](int chunk) { return wkv7::uniform_ptr(w.kq + ((slot + chunk) * p.Hk + hk) * (3 * K * kChunk * 2)); };
    const bool two = wave >= 2;  // these rows of the lower triangles have a second half

    if (role == 1) {
        const auto fetch = [&](int chunk, OutputOperands<K>& o) {
            const char* const rec = record(chunk);
            const char* const q = heads(chunk) + (4 + wave) * (kSteps * 1024);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                o.q[s] = *reinterpret_cast<const u4*>(q + s * 1024 + lane * 16u);
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int m = 0; m < 2; ++m)
                    o.b[half][m] = *reinterpret_cast<const u4*>(rec + kRecordB + (block_of(wave, two ? half : 0) * 2 + m) * 1024 + lane * 16u);
            o.gamma = *reinterpret_cast<const f4*>(rec + kRecordFactors + 768 + token_of(wave, 4 * quad) * 4u);
        };
        const auto step = [&](int chunk, const OutputOperands<K>& o) {
            f4 O[NT][2];
#pragma unroll
            for (int x = 0; x < NT; ++x) O[x][0] = O[x][1] = zero;
            if (p.o)
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        O[x][0] = mfma(o.q[s], sf[s][0][x][lane], O[x][0]);
                        O[x][1] = mfma(o.q[s], sf[s][1][x][lane], O[x][1]);
                    }
            lds_barrier();
            lds_barrier();
            if (p.o) {
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    f4 y = (O[x][0] + O[x][1]) * o.gamma;
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        if (half == 0 || two) {
                            const u4 a = df[half][0][x][lane], b = df[half][1][x][lane];
                            y = mfma(o.b[half][1], a, y);
                            y = mfma(o.b[half][0], b, y);
                            y = mfma(o.b[half][0], a, y);
                        }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int t = chunk * kChunk + token_of(wave, 4 * quad + r);
                        if (t < len) p.o[(first + t) * p.o_stride + (int64_t)h * p.V + col0 + 16 * x + col] = wkv7::f32_to_bf16(y[r]);
                    }
                }
            }
            lds_barrier();
        };
        lds_barrier();
        OutputOperands<K> even, odd;
        if (chunks > 0) fetch(0, even);
        for (int c = 0; c < chunks; c += 2) {
            fetch(min(c + 1, chunks - 1), odd);
            step(c, even);
            if (c + 1 < chunks) {
                fetch(min(c + 2, chunks - 1), even);
                step(c + 1, odd);
            }
        }
        return;
    }

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

    const auto fetch = [&](int chunk, StateOperands<K, NT>& o) {
        const int64_t t0 = first + (int64_t)chunk * kChunk;
        const int most = min(len - chunk * kChunk, kChunk) - 1;
        const char* const rec = record(chunk);
        const char *const k = heads(chunk) + wave * (kSteps * 1024), *const kt = heads(chunk) + (8 * kSteps + 2 * kTiles * wave) * 1024;
        const uint16_t* const vp = wkv7::uniform_ptr(p.v + t0 * p.v_stride + (int64_t)h * p.V + col0);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
            o.k[s] = *reinterpret_cast<const u4*>(k + s * 1024 + lane * 16u);
        const char* const f = rec + kRecordFactors;
        const uint32_t at = token_of(wave, 4 * quad) * 4u;
        o.beta = *reinterpret_cast<const f4*>(f + at);
        o.seen = *reinterpret_cast<const f4*>(f + 256 + at);
        o.left = *reinterpret_cast<const f4*>(f + 512 + at);
        o.keep = *reinterpret_cast<const float*>(f + 1024);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t v_at = (uint32_t)min(token_of(wave, 4 * quad + r), most) * (uint32_t)p.v_stride + col;
#pragma unroll
            for (int x = 0; x < NT; ++x) o.v[x][r] = vp[v_at + 16 * x];
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int m = 0; m < 3; ++m)
                o.t[half][m] = *reinterpret_cast<const u4*>(rec + kRecordT + (block_of(wave, two ? half : 0) * 3 + m) * 1024 + lane * 16u);
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int half = 0; half < 2; ++half) o.kt[t][half] = *reinterpret_cast<const u4*>(kt + (t * 2 + half) * 1024 + lane * 16u);
    };
    const auto share_state = [&] {
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                const int tile = wave * kTiles + t;
                u2 a, b, c;
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    uint32_t i, j, k;
                    split3(S[t][x][2 * m], S[t][x][2 * m + 1], i, j, k);
                    a[m] = i, b[m] = j, c[m] = k;
                }
                reinterpret_cast<u2*>(&sf[tile >> 1][0][x][lane])[tile & 1] = a;
                reinterpret_cast<u2*>(&sf[tile >> 1][1][x][lane])[tile & 1] = b;
                reinterpret_cast<u2*>(&sf[tile >> 1][2][x][lane])[tile & 1] = c;
            }
    };
    const auto step = [&](const StateOperands<K, NT>& o) {
        f4 P[NT][3];
#pragma unroll
        for (int x = 0; x < NT; ++x) P[x][0] = P[x][1] = P[x][2] = zero;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int m = 0; m < 3; ++m) P[x][m] = mfma(o.k[s], sf[s][m][x][lane], P[x][m]);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            f4 R;
            u2 a, b, c;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                R[r] = fmaf(-o.seen[r], P[x][0][r] + (P[x][1][r] + P[x][2][r]), o.beta[r] * wkv7::bf16_to_f32(o.v[x][r]));
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t i, j, k;
                split3(R[2 * m], R[2 * m + 1], i, j, k);
                a[m] = i, b[m] = j, c[m] = k;
            }
            reinterpret_cast<u2*>(&rf[wave >> 1][0][x][lane])[wave & 1] = a;
            reinterpret_cast<u2*>(&rf[wave >> 1][1][x][lane])[wave & 1] = b;
            reinterpret_cast<u2*>(&rf[wave >> 1][2][x][lane])[wave & 1] = c;
        }
        lds_barrier();
        f4 D[NT][3];
#pragma unroll
        for (int x = 0; x < NT; ++x) D[x][0] = D[x][1] = D[x][2] = zero;
#pragma unroll
        for (int half = 0; half < 2; ++half)
            if (half == 0 || two)
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    const u4 a = rf[half][0][x][lane], b = rf[half][1][x][lane], c = rf[half][2][x][lane];
                    D[x][2] = mfma(o.t[half][2], a, D[x][2]);
                    D[x][1] = mfma(o.t[half][1], a, D[x][1]);
                    D[x][0] = mfma(o.t[half][0], a, D[x][0]);
                    D[x][2] = mfma(o.t[half][0], c, D[x][2]);
                    D[x][1] = mfma(o.t[half][0], b, D[x][1]);
                    D[x][2] = mfma(o.t[half][1], b, D[x][2]);
                }
#pragma unroll
        for (int x = 0; x < NT; ++x) {
            const f4 d = D[x][0] + (D[x][1] + D[x][2]);
            u2 a, b, c, g, e;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                uint32_t i, j, k;
                split3(d[2 * m] * o.left[2 * m], d[2 * m + 1] * o.left[2 * m + 1], i, j, k);
                c[m] = i, g[m] = j, e[m] = k;
                wkv7::split_pair(d[2 * m], d[2 * m + 1], i, j);
                a[m] = i, b[m] = j;
            }
            reinterpret_cast<u2*>(&ef[wave >> 1][0][x][lane])[wave & 1] = c;
            reinterpret_cast<u2*>(&ef[wave >> 1][1][x][lane])[wave & 1] = g;
            reinterpret_cast<u2*>(&ef[wave >> 1][2][x][lane])[wave & 1] = e;
            reinterpret_cast<u2*>(&df[wave >> 1][0][x][lane])[wave & 1] = a;
            reinterpret_cast<u2*>(&df[wave >> 1][1][x][lane])[wave & 1] = b;
        }
        lds_barrier();
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int x = 0; x < NT; ++x) S[t][x] *= o.keep;
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    const u4 e = ef[half][part][x][lane];
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) S[t][x] = mfma(o.kt[t][half], e, S[t][x]);
                }
        share_state();
        lds_barrier();
    };
    share_state();
    StateOperands<K, NT> even, odd;
    if (chunks > 0) fetch(0, even);
    lds_barrier();
    for (int c = 0; c < chunks; c += 2) {
        fetch(min(c + 1, chunks - 1), odd);
        step(even);
        if (c + 1 < chunks) {
            fetch(min(c + 2, chunks - 1), even);
            step(odd);
        }
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
    hipLaunchKernelGGL(delta_prep_kernel<K>, dim3((unsigned)(slots * p.Hk)), dim3(256), 0, stream, p, w);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t groups = ((int64_t)p.num_seqs * p.Hv / w.together + 7) / 8 * 8;
    if (wide)
        hipLaunchKernelGGL((delta_scan_kernel<K, 2>), dim3((unsigned)(groups * w.together * (p.V / 32))), dim3(512), 0, stream, p, w);
    else
        hipLaunchKernelGGL((delta_scan_kernel<K, 1>), dim3((unsigned)(groups * w.together * (p.V / 16))), dim3(512), 0, stream, p, w);
    return hipGetLastError();
}

}  // namespace

int64_t chunk_slots(int32_t num_seqs, int32_t T, int64_t total_tokens, bool ragged) {
    return ragged ? total_tokens / kChunk + num_seqs : (int64_t)num_seqs * ((T + kChunk - 1) / kChunk);
}
int64_t chunk_groups(int32_t num_seqs, int32_t Hv, int32_t V) { return ((int64_t)num_seqs + 7) / 8 * 8 * Hv * (V / 16); }
size_t chunk_workspace(int64_t slots, int32_t Hk, int32_t Hv, int32_t K) {
    return (size_t)slots * (Hk * (size_t)(3 * K * kChunk * 2) + Hv * (size_t)kRecord);
}

hipError_t launch_chunks(const Params& p, int cus, hipStream_t stream) {
    const int64_t slots = chunk_slots(p.num_seqs, p.T, p.total_tokens, p.cu != nullptr);
    Work w;
    w.kq = p.workspace;
    w.rec = p.workspace + slots * p.Hk * (int64_t)(3 * p.K * kChunk * 2);
    w.together = (int64_t)p.num_seqs * p.Hk >= 8 ? p.share : 1;
    const bool wide = p.V % 32 == 0 && (int64_t)p.num_seqs * p.Hv * (p.V / 32) >= 2 * cus;
    return p.K == 64 ? launch<64>(p, w, slots, wide, stream) : launch<128>(p, w, slots, wide, stream);
}

}  // namespace delta
