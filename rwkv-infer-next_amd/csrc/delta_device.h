// delta_device.h -- what the kernels of the gated delta rule share (include/delta.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "delta.h"
#include "delta_plan.h"
#include "wkv7_device.h"

namespace delta {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

constexpr float kNormEps = 1e-6f;

struct Params {
    const uint16_t *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *g, *beta;
    int64_t g_stride, beta_stride;
    uint16_t* o;
    int64_t o_stride;
    const float* h0;
    const int64_t* h0_idx;
    int64_t h0_rows;
    float* ht;
    const int64_t* ht_idx;
    int64_t ht_rows;
    const uint8_t* fresh;
    const int32_t* cu;
    const int64_t* n_keep;
    float* snapshots;
    int32_t* status;
    char* workspace;
    int64_t total_tokens;
    int32_t num_seqs, T, Hk, Hv, K, V, share;  // share = Hv / Hk
    float scale;
    int32_t qk_norm;
    int32_t token_len;  // rows of at most this many tokens run token by token
};

// First token and length of sequence n: clamped, so that no cu_seqlens or n_keep leads outside the operands.
__device__ __forceinline__ void extent(const Params& p, int n, int64_t& first, int& len) {
    int64_t s = (int64_t)n * p.T, e = s + p.T;
    if (p.cu) {
        s = p.cu[n], e = p.cu[n + 1];
        s = s < 0 ? 0 : s > p.total_tokens ? p.total_tokens : s;
        e = e < s ? s : e > p.total_tokens ? p.total_tokens : e;
    }
    if (p.n_keep) {
        const int64_t nk = p.n_keep[n];
        if (nk < e - s) e = s + (nk < 0 ? 0 : nk);
    }
    first = s;
    len = (int)(e - s);
}

// State of (sequence n, value head h), NULL for zeros.
__device__ __forceinline__ const float* initial(const Params& p, int n, int h) {
    if (!p.h0 || (p.fresh && p.fresh[n])) return nullptr;
    const int64_t s = p.h0_idx ? p.h0_idx[n] : n;
    if (s < 0 || s >= p.h0_rows) return nullptr;
    return p.h0 + (s * p.Hv + h) * ((int64_t)p.K * p.V);
}
__device__ __forceinline__ float* final_state(const Params& p, int n, int h) {
    if (!p.ht) return nullptr;
    const int64_t s = p.ht_idx ? p.ht_idx[n] : n;
    if (s < 0 || s >= p.ht_rows) return nullptr;
    return p.ht + (s * p.Hv + h) * ((int64_t)p.K * p.V);
}

__device__ __forceinline__ float bf16_at(u4 x, int i) {  // element i of eight
    const uint32_t w = x[i / 2];
    return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
}

// The workspace of the chunks' kernels.  For each slot (a chunk's place) and query/key head K, Q and K^T in operand order, and for each slot and
// value head a record: T (three bf16 parts) and B (two) of the lower triangle's blocks, six each, and the tokens' factors.
constexpr int64_t kRecordT = 0, kRecordB = 18 * 1024, kRecordFactors = 30 * 1024, kRecord = 30 * 1024 + 1280;
struct Work {
    char *kq, *rec;
    int32_t* order;    // ragged rows: how many run by chunks, then their numbers
    int32_t shift, rows;  // ragged rows: where their slots begin (ragged_slot)
    int32_t together;  // heads whose workgroups follow each other on one XCD
};
Slots chunk_slots(int32_t num_seqs, int32_t T, int64_t total_tokens, int32_t token_len, bool ragged);
int64_t chunk_groups(int64_t rows, int32_t Hv, int32_t V);  // most workgroups of the chunks' scan
size_t chunk_workspace(int64_t slots, int32_t num_seqs, int32_t Hk, int32_t Hv, int32_t K);

// All rows (ragged: those longer than token_len) by chunks; by tokens (ragged: those up to token_len).
hipError_t launch_chunks(const Params& p, int cus, hipStream_t stream);
hipError_t launch_tokens(const Params& p, hipStream_t stream);

}  // namespace delta
