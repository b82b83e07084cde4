// logits_sample.hip -- the choice of a token from each row of logits (include/logits.h).
//
// A workgroup of 1024 threads has a row and goes over it a few times (the first from memory, the others mostly from L2): the
// maximum, the sum of the weights w = exp(-d), d = (max - x) / T, a search for the last kept place in the order of (d, index),
// and the draw among what is kept.  Nothing is sorted but a bin of that search: a histogram over d in steps of 1/32 holds
// the tokens' number and their weights as whole numbers of 2^-40 (so no order of the atomics shows in a result); the bin in which
// the wanted number or weight is reached is gathered in LDS, sorted by (d, index) and scanned.  A bin of more tokens than fit
// (equal logits) is first cut into 1024 parts by its (d, index), again and again.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "logits.h"
#include "logits_device.h"

namespace lg {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 1024;        // one per thread
constexpr float kPerUnit = 32.f;   // bins to a unit of d; the last one holds all from 1023/32 on
constexpr int kGather = 4096;      // tokens of a bin that are sorted in LDS
constexpr float kOne = 1099511627776.f;  // 2^40: a weight of 1
constexpr uint32_t kInfBits = 0x7F800000u;

struct Shared {
    uint64_t list[kGather];
    uint64_t weight[kBins];
    uint32_t count[kBins];
    uint64_t wave[kWaves];
    float wave_f[kWaves];
    uint64_t found, base;
    uint32_t gathered, bin;
};

__device__ __forceinline__ uint64_t shuffle(uint64_t x, int from) {
    const uint32_t lo = __shfl((int)(uint32_t)x, from), hi = __shfl((int)(uint32_t)(x >> 32), from);
    return (uint64_t)hi << 32 | lo;
}

template <typename F>
__device__ __forceinline__ float block_reduce(Shared& s, float x, F&& f) {
    for (int o = 32; o; o >>= 1) x = f(x, __shfl_xor(x, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave_f[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s.wave_f[0];
    for (int w = 1; w < kWaves; ++w) x = f(x, s.wave_f[w]);
    return x;
}

template <typename F>
__device__ __forceinline__ uint64_t block_reduce64(Shared& s, uint64_t x, F&& f) {
    for (int o = 32; o; o >>= 1) x = f(x, shuffle(x, (threadIdx.x & 63) ^ o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s.wave[0];
    for (int w = 1; w < kWaves; ++w) x = f(x, s.wave[w]);
    return x;
}

// The sum over the threads before this one.
__device__ __forceinline__ uint64_t block_before(Shared& s, uint64_t x) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t sum = x;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = shuffle(sum, (lane - o) & 63);
        if (lane >= o) sum += y;
    }
    __syncthreads();
    if (lane == 63) s.wave[wave] = sum;
    __syncthreads();
    uint64_t before = sum - x;
    for (int w = 0; w < wave; ++w) before += s.wave[w];
    return before;
}

// What a row's passes need to know of it.
struct Row {
    const void* x;
    int V;
    float max, inv;  // inv = 1 / temperature
};

// (max - x) / temperature; 0 for the maximum (an infinite one too), infinity for -infinity.
__device__ __forceinline__ float distance(const Row& r, float x) {
    const float d = (r.max - x) * r.inv;
    return x == r.max ? 0.f : d >= 0.f ? d : __builtin_inff();
}
__device__ __forceinline__ float weight(float d) { return __builtin_amdgcn_exp2f(d * -1.44269504088896341f); }
__device__ __forceinline__ uint64_t whole(float w) { return (uint64_t)(w * kOne); }
__device__ __forceinline__ uint32_t bin_of(float d) { return (uint32_t)(int)fminf(d * kPerUnit, (float)(kBins - 1)); }

// f(index, x) for every element of the row, NaN as -infinity; four 8-element pieces of it in flight to a thread.
template <int DT, typename F>
__device__ __forceinline__ void each(const Row& r, F&& f) {
    constexpr int kAhead = 4;
    for (int64_t i0 = 8 * (int64_t)threadIdx.x; i0 < r.V; i0 += (int64_t)kAhead * kThreads * 8) {
        float x[kAhead][8];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int64_t i = i0 + (int64_t)a * kThreads * 8;
            load8<DT>(r.x, i, i >= r.V ? 0 : r.V - i < 8 ? (int)(r.V - i) : 8, -__builtin_inff(), x[a]);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = x[a][j];
                f((uint32_t)(i0 + (int64_t)a * kThreads * 8 + j), v == v ? v : -__builtin_inff());
            }
    }
}

__device__ __forceinline__ uint64_t key_of(float d, uint32_t i) { return (uint64_t)__float_as_uint(d) << 32 | i; }
__device__ __forceinline__ float d_of(uint64_t key) { return __uint_as_float((uint32_t)(key >> 32)); }

// Sorts list[0 .. n-1] upwards; the threads' own, n <= kGather.
__device__ void sort_list(Shared& s, uint32_t n) {
    uint32_t size = 64;
    while (size < n) size *= 2;
    for (uint32_t i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = ~0ull;
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j; j /= 2) {
            __syncthreads();
            for (uint32_t e = threadIdx.x; e < size / 2; e += kThreads) {
                const uint32_t a = (e & ~(j - 1)) * 2 + (e & (j - 1)), b = a + j;
                const uint64_t x = s.list[a], y = s.list[b];
                if ((x > y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
            }
        }
    __syncthreads();
}

// The key of the last token of the smallest prefix, in the order of keys up to `limit`, whose number (COUNT) or weight reaches
// `target`; `limit` where all together do not.  Tokens without weight in 64 bits (d infinite) are in no prefix.
template <int DT, bool COUNT>
__device__ uint64_t last_kept(Shared& s, const Row& r, uint64_t limit, uint64_t target) {
    const int tid = threadIdx.x;
    uint64_t lo = 0, hi = (uint64_t)kInfBits << 32, base = 0;  // keys of the part that is searched
    int shift = -1;                                             // -1: by bins of d
    for (;;) {
        s.count[tid] = 0;
        s.weight[tid] = 0;
        if (tid == 0) s.bin = kBins, s.gathered = 0;
        __syncthreads();
        each<DT>(r, [&](uint32_t i, float x) {
            const float d = distance(r, x);
            const uint64_t key = key_of(d, i);
            if (key >= lo && key < hi && key <= limit) {
                const uint32_t b = shift < 0 ? bin_of(d) : (uint32_t)((key - lo) >> shift);
                atomicAdd(&s.count[b], 1u);
                if (!COUNT) atomicAdd((unsigned long long*)&s.weight[b], (unsigned long long)whole(weight(d)));
            }
        });
        __syncthreads();
        const uint64_t mine = COUNT ? s.count[tid] : s.weight[tid], before = base + block_before(s, mine);
        if (before < target && before + mine >= target) s.bin = tid, s.base = before;  // one thread at most
        __syncthreads();
        const uint32_t b = s.bin;
        if (b == kBins) return limit;
        const uint32_t n = s.count[b];
        base = s.base;
        if (shift < 0) {
            lo = (uint64_t)__float_as_uint((float)b / kPerUnit) << 32;
            if (b < kBins - 1) hi = (uint64_t)__float_as_uint((float)(b + 1) / kPerUnit) << 32;
        } else {
            lo += (uint64_t)b << shift;
            hi = min(hi, lo + (1ull << shift));
        }
        __syncthreads();
        if (n <= kGather) break;
        shift = 0;
        while (((hi - lo - 1) >> shift) >= kBins) ++shift;
    }
    each<DT>(r, [&](uint32_t i, float x) {
        const uint64_t key = key_of(distance(r, x), i);
        if (key >= lo && key < hi && key <= limit) {
            const uint32_t at = atomicAdd(&s.gathered, 1u);
            if (at < kGather) s.list[at] = key;  // as many as were counted, unless someone writes the logits meanwhile
        }
    });
    __syncthreads();
    const uint32_t n = min(s.gathered, (uint32_t)kGather);
    sort_list(s, n);
    if (COUNT) return s.list[min((uint32_t)(target - base - 1), (uint32_t)kGather - 1)];
    uint64_t w[kGather / kThreads], sum = 0;
#pragma unroll
    for (int j = 0; j < kGather / kThreads; ++j) {
        const uint32_t e = tid * (kGather / kThreads) + j;
        w[j] = e < n ? whole(weight(d_of(s.list[e]))) : 0;
        sum += w[j];
    }
    uint64_t before = base + block_before(s, sum);
#pragma unroll
    for (int j = 0; j < kGather / kThreads; ++j) {
        if (before < target && before + w[j] >= target) s.found = s.list[tid * (kGather / kThreads) + j];
        before += w[j];
    }
    __syncthreads();
    return s.found;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void sample_kernel(const logits_sample_args p) {
    __shared__ Shared s;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x, b = row / p.T, t = row % p.T;
    const auto largest = [](float a, float c) { return fmaxf(a, c); };
    const auto plus = [](float a, float c) { return a + c; };
    const auto lowest64 = [](uint64_t a, uint64_t c) { return a < c ? a : c; };
    const auto plus64 = [](uint64_t a, uint64_t c) { return a + c; };

    Row r;
    r.x = static_cast<const char*>(p.logits) + (b * p.seq_stride + t * p.pos_stride) * element_bytes(DT);
    r.V = p.V;
    const float temperature = p.temperature ? p.temperature[b] : p.temperature_all;
    const bool greedy = !p.noise || !(temperature > 0.f);
    r.inv = temperature > 0.f ? fminf(fmaxf(1.f / temperature, 1e-30f), 3e38f) : 1.f;

    float m = -__builtin_inff();
    each<DT>(r, [&](uint32_t, float x) { m = fmaxf(m, x); });
    r.max = m = block_reduce(s, m, largest);
    if (m == -__builtin_inff()) {  // nothing is allowed
        if (tid == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = m;
        }
        return;
    }
    float total = 0.f;
    uint64_t first = ~0ull;  // the maximum's lowest index
    each<DT>(r, [&](uint32_t i, float x) {
        const float d = distance(r, x);
        total += weight(d);
        if (x == r.max && i < first) first = i;
    });
    total = block_reduce(s, total, plus);
    uint32_t token = (uint32_t)block_reduce64(s, first, lowest64);

    if (!greedy) {
        const int k = p.top_k ? p.top_k[b] : p.top_k_all;
        const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
        const float min_p = fminf(p.min_p ? p.min_p[b] : p.min_p_all, 1.f);
        uint64_t limit = ((uint64_t)kInfBits << 32) - 1;
        if (k > 0 && k < p.V) limit = last_kept<DT, true>(s, r, limit, (uint64_t)k);
        if (top_p < 1.f) {
            uint64_t sum = 0;
            each<DT>(r, [&](uint32_t i, float x) {
                const float d = distance(r, x);
                if (key_of(d, i) <= limit) sum += whole(weight(d));
            });
            sum = block_reduce64(s, sum, plus64);
            const double want = (double)top_p * (double)sum;
            limit = last_kept<DT, false>(s, r, limit, want >= 1.0 ? (uint64_t)ceil(want) : 1);
        }
        const float* const noise = p.noise + b * p.noise_seq_stride + t * p.noise_pos_stride;
        float best = 0.f;  // of this thread: its largest w / noise and where; indexes go up, so the first of equals stays
        uint32_t at = ~0u;
        each<DT>(r, [&](uint32_t i, float x) {
            const float d = distance(r, x), w = weight(d);
            if (key_of(d, i) <= limit && w > 0.f && (w >= min_p || i == token)) {
                const float score = w / noise[i];
                if (score > best) best = score, at = i;
            }
        });
        // positive floats order as their bits; the lowest index of the largest
        uint64_t won = ~(uint64_t)__float_as_uint(best) << 32 | at;
        won = block_reduce64(s, won, lowest64);
        if ((uint32_t)won != ~0u) token = (uint32_t)won;  // else no noise was a number: the most likely token
    }

    if (tid == 0) {
        p.token[row] = token;
        if (p.logprob) {
            float x[8];
            load8<DT>(r.x, token, 1, 0.f, x);
            p.logprob[row] = -distance(r, x[0]) - logf(total);
        }
        if (p.counts) {
            const int64_t slot = p.slots ? p.slots[b] : b;
            if (slot < 0 || slot >= p.counts_rows) {
                if (p.status) atomicOr(p.status, LOGITS_STATUS_ROW);
            } else if (p.counts_dtype == LOGITS_COUNTS_I32) {
                atomicAdd(static_cast<int*>(p.counts) + slot * p.counts_stride + token, 1);
            } else {
                atomicAdd(static_cast<float*>(p.counts) + slot * p.counts_stride + token, 1.f);
            }
        }
    }
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace lg

extern "C" {

size_t logits_sample_args_size(void) { return sizeof(logits_sample_args); }

int logits_sample(const logits_sample_args* a, void* stream) {
    if (!a) return WKV7_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->V < 1) return WKV7_ERR_SHAPE;
    if (a->dtype < LOGITS_BF16 || a->dtype > LOGITS_F32 ||
        (a->counts && ((a->counts_dtype != LOGITS_COUNTS_I32 && a->counts_dtype != LOGITS_COUNTS_F32) || a->T > 1)))
        return WKV7_ERR_ARG;
    if (a->B == 0 || a->T == 0) return WKV7_OK;
    if (!a->logits || !a->token) return WKV7_ERR_NULL;
    if (a->counts && (a->counts_rows < 0 || a->counts_stride < a->V)) return WKV7_ERR_SHAPE;
    if (!lg::aligned(a->logits, lg::element_bytes(a->dtype)) || !lg::aligned(a->noise, 4) || !lg::aligned(a->counts, 4))
        return WKV7_ERR_ALIGN;
    const int64_t rows = (int64_t)a->B * a->T;
    if (rows > 0x3FFFFF) return WKV7_ERR_SHAPE;  // 1024 threads each: below 2^32 work-items
    const dim3 grid((unsigned)rows), block(lg::kThreads);
    const auto s = static_cast<hipStream_t>(stream);
    if (a->dtype == LOGITS_BF16)
        hipLaunchKernelGGL((lg::sample_kernel<LOGITS_BF16>), grid, block, 0, s, *a);
    else if (a->dtype == LOGITS_F16)
        hipLaunchKernelGGL((lg::sample_kernel<LOGITS_F16>), grid, block, 0, s, *a);
    else
        hipLaunchKernelGGL((lg::sample_kernel<LOGITS_F32>), grid, block, 0, s, *a);
    return static_cast<int>(hipGetLastError());
}

}  // extern "C"
