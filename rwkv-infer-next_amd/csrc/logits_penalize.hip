// logits_penalize.hip -- penalties, biases and grammar masks on logits (include/logits.h), one pass over the logits.
//
// A workgroup owns 2048 columns of one sequence, eight to a thread, for all T positions: the columns' counts are read once and
// carried from position to position, each draft adding one where it falls.  A bias list belongs to a whole row: every workgroup
// picks the entries of its columns out of it, 256 at a time, and adds them up in LDS.  Entries of one column are added in their order:
// of those that are left the first takes the column, adds and leaves, until none is left (mostly after one turn).  One entry after
// another, looked at by all threads, took 33 us a call where this takes 12.4 (16 sequences of two positions, V = 1500, 300
// biases each).
//
// Bound by memory where there is enough of it: V = 65536, 64 sequences of five positions, fp32 with counts and masks, 187 MB in
// 42.0 us = 4.5 TB/s (a large copy moves 4.9); 64 sequences bf16, 33.6 MB in 9.7 us = 3.5 TB/s, a workgroup's three dependent
// reads and the biases' barriers counting; one sequence 4.0 us, a launch.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "logits.h"
#include "logits_device.h"

namespace lg {
namespace {

constexpr int kThreads = 256;
constexpr int kColumns = kThreads * 8;

// BLOCK: more than one position; the next one's logits are asked for while this one's are worked on.
template <int DT, bool BLOCK>
__global__ __launch_bounds__(kThreads) void penalize_kernel(const logits_penalize_args p, uint32_t segments) {
    __shared__ float sums[kColumns];
    __shared__ uint32_t turn[kColumns];  // of the entries of a column that are left, the first one's thread
    const int tid = threadIdx.x;
    const int64_t b = blockIdx.x / segments, first = (int64_t)(blockIdx.x % segments) * kColumns, v0 = first + 8 * tid;
    const int n = v0 >= p.V ? 0 : p.V - v0 < 8 ? (int)(p.V - v0) : 8;
    const bool reports = p.status && first == 0 && tid == 0;  // one thread a sequence

    // The first position's logits and its mask are asked for before the parameters and the biases are known: a workgroup's time is
    // its loads', one after another.
    const char* in = static_cast<const char*>(p.logits) + b * p.in_seq_stride * element_bytes(DT);
    char* out = static_cast<char*>(p.out) + b * p.out_seq_stride * element_bytes(p.out_dtype);
    float x[8];
    load8<DT>(in, v0, n, 0.f, x);
    const auto mask_of = [&](int t) -> uint32_t {  // eight bits; all set without a mask
        if (!p.mask) return 0xFF;
        const int64_t row = b * p.T + t, m = p.mask_row ? p.mask_row[row] : row;
        if (m >= p.mask_rows && reports) atomicOr(p.status, LOGITS_STATUS_ROW);
        return m >= 0 && m < p.mask_rows && n > 0 ? reinterpret_cast<const uint8_t*>(p.mask + m * p.mask_stride)[v0 >> 3] : 0xFF;
    };
    uint32_t allowed = mask_of(0);

    const float rep = p.repetition ? p.repetition[b] : p.repetition_all;
    const float pres = p.presence ? p.presence[b] : p.presence_all;
    const float freq = p.frequency ? p.frequency[b] : p.frequency_all;
    const bool penalised = rep != 1.f || pres != 0.f || freq != 0.f;

    float c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = 0.f;
    if (p.counts) {
        const int64_t s = p.slots ? p.slots[b] : b;
        if (s < 0 || s >= p.counts_rows) {
            if (reports) atomicOr(p.status, LOGITS_STATUS_ROW);
        } else if (penalised) {
            load8<LOGITS_F32>(p.counts, s * p.counts_stride + v0, n, 0.f, c);
            if (p.counts_dtype == LOGITS_COUNTS_I32)
#pragma unroll
                for (int j = 0; j < 8; ++j) c[j] = (float)__float_as_int(c[j]);
        }
    }

    float bias[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) bias[j] = 0.f;
    if (p.n_bias > 0) {
        for (int e = tid; e < kColumns; e += kThreads) sums[e] = 0.f, turn[e] = ~0u;
        for (int i0 = 0; i0 < p.n_bias; i0 += kThreads) {
            const int i = i0 + tid;
            const int64_t id = i < p.n_bias ? p.bias_ids[b * p.bias_stride + i] : -1;
            if (p.status && first == 0 && id >= p.V) atomicOr(p.status, LOGITS_STATUS_TOKEN);
            bool left = id >= first && id < first + kColumns && id < p.V;
            const int column = left ? (int)(id - first) : 0;
            const float add = left ? p.bias_values[b * p.bias_stride + i] : 0.f;
            while (__syncthreads_or(left)) {
                if (left) atomicMin(&turn[column], (uint32_t)tid);
                __syncthreads();
                const bool mine = left && turn[column] == (uint32_t)tid;
                if (mine) sums[column] += add, left = false;
                __syncthreads();
                if (mine) turn[column] = ~0u;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) bias[j] = sums[8 * tid + j];
    }

    for (int t = 0; t < (BLOCK ? p.T : 1); ++t) {
        if (BLOCK && t > 0 && p.drafts) {
            const int64_t id = p.drafts[b * p.drafts_stride + t - 1];
            if (reports && id >= p.V) atomicOr(p.status, LOGITS_STATUS_TOKEN);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (id == v0 + j) c[j] += 1.f;
        }
        float next[8];
        uint32_t next_allowed = 0xFF;
        if (BLOCK && t + 1 < p.T) {
            load8<DT>(in + (t + 1) * p.in_pos_stride * element_bytes(DT), v0, n, 0.f, next);
            next_allowed = mask_of(t + 1);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (penalised && c[j] > 0.f) x[j] = (x[j] > 0.f ? x[j] / rep : x[j] * rep) - (freq * c[j] + pres);
            x[j] += bias[j];
            if (!(allowed >> j & 1)) x[j] = -__builtin_inff();
        }
        store8(out + t * p.out_pos_stride * element_bytes(p.out_dtype), p.out_dtype, v0, n, x);
        if (BLOCK) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = next[j];
            allowed = next_allowed;
        }
    }
}

template <int DT>
void launch(const logits_penalize_args& p, dim3 grid, uint32_t segments, hipStream_t s) {
    if (p.T > 1)
        hipLaunchKernelGGL((penalize_kernel<DT, true>), grid, dim3(kThreads), 0, s, p, segments);
    else
        hipLaunchKernelGGL((penalize_kernel<DT, false>), grid, dim3(kThreads), 0, s, p, segments);
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace lg

extern "C" {

size_t logits_penalize_args_size(void) { return sizeof(logits_penalize_args); }

int logits_penalize(const logits_penalize_args* a, void* stream) {
    if (!a) return WKV7_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->V < 1 || a->n_bias < 0) return WKV7_ERR_SHAPE;
    if (a->in_dtype < LOGITS_BF16 || a->in_dtype > LOGITS_F32 || a->out_dtype < LOGITS_BF16 || a->out_dtype > LOGITS_F32 ||
        (a->counts && a->counts_dtype != LOGITS_COUNTS_I32 && a->counts_dtype != LOGITS_COUNTS_F32))
        return WKV7_ERR_ARG;
    if (a->B == 0 || a->T == 0) return WKV7_OK;
    if (!a->logits || !a->out || (a->n_bias && (!a->bias_ids || !a->bias_values))) return WKV7_ERR_NULL;
    if (a->counts && (a->counts_rows < 0 || a->counts_stride < a->V)) return WKV7_ERR_SHAPE;
    if (a->drafts && a->T > 1 && a->B > 1 && a->drafts_stride < a->T - 1) return WKV7_ERR_SHAPE;
    if (a->n_bias && a->B > 1 && a->bias_stride < a->n_bias) return WKV7_ERR_SHAPE;
    if (a->mask && (a->mask_rows < 0 || a->mask_stride < ((int64_t)a->V + 31) / 32)) return WKV7_ERR_SHAPE;
    if (!lg::aligned(a->logits, lg::element_bytes(a->in_dtype)) || !lg::aligned(a->out, lg::element_bytes(a->out_dtype)) ||
        !lg::aligned(a->counts, 4) || !lg::aligned(a->mask, 4))
        return WKV7_ERR_ALIGN;
    const int64_t segments = ((int64_t)a->V + lg::kColumns - 1) / lg::kColumns;
    if (segments * a->B > 0xFFFFFF) return WKV7_ERR_SHAPE;  // 256 threads each: below 2^32 work-items
    logits_penalize_args p = *a;
    if (!p.counts && !p.drafts) {  // nothing is counted
        p.repetition = p.presence = p.frequency = nullptr;
        p.repetition_all = 1.f;
        p.presence_all = p.frequency_all = 0.f;
    }
    const dim3 grid((unsigned)(segments * a->B));
    const auto s = static_cast<hipStream_t>(stream);
    if (a->in_dtype == LOGITS_BF16)
        lg::launch<LOGITS_BF16>(p, grid, (uint32_t)segments, s);
    else if (a->in_dtype == LOGITS_F16)
        lg::launch<LOGITS_F16>(p, grid, (uint32_t)segments, s);
    else
        lg::launch<LOGITS_F32>(p, grid, (uint32_t)segments, s);
    return static_cast<int>(hipGetLastError());
}

}  // extern "C"
