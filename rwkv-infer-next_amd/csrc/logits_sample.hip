// logits_sample.hip -- the choice of a token from each row of logits (include/logits.h), in three launches:
//
//   max     segments of 8192 elements, a workgroup each: the row's maximum and its lowest index
//   weigh   the same segments: with d = (max - x) / T, w = exp(-d) the sum of w; in rows without top-k and top-p the draw among
//           their elements; in the others a histogram over d in steps of 1/32, of the tokens' number and of their weights
//   choose  a workgroup a row: where the histogram reaches the wanted number or weight the threshold lies in that bin; one pass
//           over the row gathers the bin in LDS (and draws among the tokens before it); sorted by (d, index) and scanned, it gives
//           the last kept token
//
// A row's maximum must be known before its weights are, and its weights before a threshold: hence the launches.  Sums are
// of whole numbers of 2^-40, so no order of the atomics shows in a result.  A bin of more tokens than the list in LDS holds (equal
// logits, or a top-k of thousands) goes the long way: the workgroup cuts it into 1024 parts by (d, index), again and again.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "logits.h"
#include "logits_device.h"

namespace lg {
namespace {

constexpr int kThreads = 1024;     // of the choosing workgroup
constexpr int kWaves = kThreads / 64;
constexpr int kSegThreads = 256;   // of a segment's workgroup
constexpr int kSegPieces = 4;      // eight elements each to a thread
constexpr int kSegment = kSegThreads * kSegPieces * 8;
constexpr int kRowsAtOnce = 512;   // rows of one set of launches: the workspace holds as many
constexpr int kBins = 1024;        // one per thread
constexpr float kPerUnit = 32.f;   // bins to a unit of d; the last one holds all from 1023/32 on
constexpr int kGather = 4096;      // tokens of a bin that are sorted in LDS
constexpr float kOne = 1099511627776.f;  // 2^40: a weight of 1
constexpr uint32_t kInfBits = 0x7F800000u;

// A row's part of the workspace: all zero between calls.
struct RowState {
    unsigned long long max_key;     // order_bits(max) << 32 | ~index
    unsigned long long total;       // sum of the weights
    unsigned long long won;         // order of w / noise << 32 | ~index, rows without top-k and top-p
    unsigned long long unused[29];
    unsigned long long weight[kBins];
    uint32_t count[kBins];
};

struct Shared {
    uint64_t list[kGather];
    uint64_t weight[kBins];
    uint32_t count[kBins];
    uint64_t wave[kWaves];
    uint64_t found, base;
    uint32_t gathered, bin;
};

__device__ __forceinline__ uint64_t shuffle(uint64_t x, int from) {
    const uint32_t lo = __shfl((int)(uint32_t)x, from), hi = __shfl((int)(uint32_t)(x >> 32), from);
    return (uint64_t)hi << 32 | lo;
}

template <typename F>
__device__ __forceinline__ uint64_t wave_reduce(uint64_t x, F&& f) {
    for (int o = 32; o; o >>= 1) x = f(x, shuffle(x, (threadIdx.x & 63) ^ o));
    return x;
}
template <typename F>
__device__ __forceinline__ uint64_t block_reduce(Shared& s, uint64_t x, F&& f) {
    x = wave_reduce(x, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = x;
    __syncthreads();
    x = s.wave[0];
    for (int w = 1; w < kWaves; ++w) x = f(x, s.wave[w]);
    return x;
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t plus(uint64_t a, uint64_t b) { return a + b; }

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

// Bits of a float that order as the numbers do (-0 as 0), and back.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u); }

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

// A row's parameters, the same in every launch.
struct Choice {
    int64_t b, t;
    Row row;
    const float* noise;
    int k;              // 0: no top-k
    float top_p, min_p;
    bool greedy, searches;  // searches: top-k or top-p
};

template <int DT>
__device__ __forceinline__ Choice choice_of(const logits_sample_args& p, int64_t row) {
    Choice c;
    c.b = row / p.T, c.t = row % p.T;
    const float temperature = p.temperature ? p.temperature[c.b] : p.temperature_all;
    c.greedy = !p.noise || !(temperature > 0.f);
    c.row.x = static_cast<const char*>(p.logits) + (c.b * p.seq_stride + c.t * p.pos_stride) * element_bytes(DT);
    c.row.V = p.V;
    c.row.max = 0.f;
    c.row.inv = temperature > 0.f ? fminf(fmaxf(1.f / temperature, 1e-30f), 3e38f) : 1.f;
    c.noise = p.noise + c.b * p.noise_seq_stride + c.t * p.noise_pos_stride;
    c.k = p.top_k ? p.top_k[c.b] : p.top_k_all;
    if (c.k < 0 || c.k >= p.V) c.k = 0;
    c.top_p = p.top_p ? p.top_p[c.b] : p.top_p_all;
    c.min_p = fminf(p.min_p ? p.min_p[c.b] : p.min_p_all, 1.f);
    c.searches = !c.greedy && (c.k > 0 || c.top_p < 1.f);
    return c;
}

// This thread's pieces of a segment, NaN as -infinity; fill past the row.
template <int DT>
__device__ __forceinline__ void load_segment(const Row& r, int64_t first, float (&x)[kSegPieces][8]) {
#pragma unroll
    for (int a = 0; a < kSegPieces; ++a) {
        const int64_t i = first + (a * kSegThreads + threadIdx.x) * 8;
        load8<DT>(r.x, i, i >= r.V ? 0 : r.V - i < 8 ? (int)(r.V - i) : 8, -__builtin_inff(), x[a]);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[a][j] = x[a][j] == x[a][j] ? x[a][j] : -__builtin_inff();
    }
}

template <int DT>
__global__ __launch_bounds__(kSegThreads) void max_kernel(const logits_sample_args p, int64_t row0, uint32_t segments,
                                                          RowState* states) {
    const uint32_t at = blockIdx.x / segments;
    const int64_t first = (int64_t)(blockIdx.x % segments) * kSegment;
    const Choice c = choice_of<DT>(p, row0 + at);
    float x[kSegPieces][8];
    load_segment<DT>(c.row, first, x);
    float m = x[0][0];
#pragma unroll
    for (int a = 0; a < kSegPieces; ++a)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, x[a][j]);
    uint32_t where = 0;
#pragma unroll
    for (int a = kSegPieces - 1; a >= 0; --a)
#pragma unroll
        for (int j = 7; j >= 0; --j)
            if (x[a][j] == m) where = (uint32_t)(first + (a * kSegThreads + threadIdx.x) * 8 + j);
    const uint64_t key = wave_reduce((uint64_t)order_bits(m) << 32 | (uint32_t)~where, larger);
    if ((threadIdx.x & 63) == 0) atomicMax(&states[at].max_key, (unsigned long long)key);
}

// The noise of eight elements from i on, where any of them may be drawn.
__device__ __forceinline__ void load_noise(const float* noise, int64_t i, int V, bool any, float (&e)[8]) {
    load8<LOGITS_F32>(noise, i, !any || i >= V ? 0 : V - i < 8 ? (int)(V - i) : 8, 1.f, e);
}

// The better of a draw so far and of element i: the largest w / noise, NaN never; indexes come upwards, so the first of equals
// stays.
__device__ __forceinline__ void draw(float w, float noise, uint32_t i, float& best, uint32_t& where) {
    const float score = w / noise;
    if (score > best) best = score, where = i;
}
__device__ __forceinline__ uint64_t draw_key(float best, uint32_t where) {  // 0: nothing drawn
    return best > 0.f ? (uint64_t)__float_as_uint(best) << 32 | (uint32_t)~where : 0;
}

template <int DT>
__global__ __launch_bounds__(kSegThreads) void weigh_kernel(const logits_sample_args p, int64_t row0, uint32_t segments,
                                                            RowState* states) {
    __shared__ uint64_t weights[kBins];
    __shared__ uint32_t counts[kBins];
    const int tid = threadIdx.x;
    const uint32_t at = blockIdx.x / segments;
    const int64_t first = (int64_t)(blockIdx.x % segments) * kSegment;
    RowState& state = states[at];
    Choice c = choice_of<DT>(p, row0 + at);
    float x[kSegPieces][8];
    load_segment<DT>(c.row, first, x);
    c.row.max = from_order((uint32_t)(state.max_key >> 32));
    if (c.row.max == -__builtin_inff()) return;
    const bool draws = !c.greedy && !c.searches, weighs = c.top_p < 1.f;
    if (c.searches) {
        for (int b = tid; b < kBins; b += kSegThreads) weights[b] = 0, counts[b] = 0;
        __syncthreads();
    }
    uint64_t total = 0, far_weight = 0;
    uint32_t far = 0, where = 0;
    float best = 0.f;
#pragma unroll
    for (int a = 0; a < kSegPieces; ++a) {
        const int64_t i = first + (a * kSegThreads + tid) * 8;
        float e[8];
        if (draws) load_noise(c.noise, i, p.V, true, e);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = distance(c.row, x[a][j]), w = weight(d);
            const uint64_t u = whole(w);
            total += u;
            if (draws && w >= c.min_p && w > 0.f) draw(w, e[j], (uint32_t)(i + j), best, where);
            if (c.searches && d < __builtin_inff()) {
                const uint32_t b = bin_of(d);
                if (b == kBins - 1) {  // a long tail's tokens all fall here: counted in registers
                    ++far, far_weight += u;
                } else {
                    atomicAdd(&counts[b], 1u);
                    if (weighs) atomicAdd((unsigned long long*)&weights[b], (unsigned long long)u);
                }
            }
        }
    }
    total = wave_reduce(total, plus);
    if ((tid & 63) == 0) atomicAdd(&state.total, (unsigned long long)total);
    if (draws) {
        const uint64_t key = wave_reduce(draw_key(best, where), larger);
        if ((tid & 63) == 0 && key) atomicMax(&state.won, (unsigned long long)key);
    }
    if (c.searches) {
        far_weight = wave_reduce(far_weight, plus);
        const uint64_t n = wave_reduce((uint64_t)far, plus);
        if ((tid & 63) == 0 && n) {
            atomicAdd(&counts[kBins - 1], (uint32_t)n);
            if (weighs) atomicAdd((unsigned long long*)&weights[kBins - 1], (unsigned long long)far_weight);
        }
        __syncthreads();
        for (int b = tid; b < kBins; b += kSegThreads)
            if (counts[b]) {
                atomicAdd(&state.count[b], counts[b]);
                if (weighs && weights[b]) atomicAdd(&state.weight[b], (unsigned long long)weights[b]);
            }
    }
}

// The first bin at whose end the running sum of `mine` reaches `target`, and the sum before it; kBins where none does.
__device__ __forceinline__ uint32_t reaching_bin(Shared& s, uint64_t mine, uint64_t target, uint64_t& base) {
    if (threadIdx.x == 0) s.bin = kBins, s.base = 0;
    const uint64_t before = block_before(s, mine);  // its barriers order the line above
    if (before < target && before + mine >= target) s.bin = threadIdx.x, s.base = before;
    __syncthreads();
    const uint32_t b = s.bin;
    base = s.base;
    __syncthreads();
    return b;
}

// Keys of d below a bin's end; every finite d for the last bin.
__device__ __forceinline__ uint64_t end_of_bin(uint32_t b) {
    return b >= kBins - 1 ? (uint64_t)kInfBits << 32 : (uint64_t)__float_as_uint((float)(b + 1) / kPerUnit) << 32;
}

constexpr int kOwn = kGather / kThreads;  // entries of the sorted list to a thread

// Draws among what top-k, top-p and min-p keep.  `total`: the row's sum of weights; `top`: its most likely token, which min-p
// always keeps.  Returns draw_key of the chosen, 0 for none.
template <int DT>
__device__ uint64_t draw_kept(Shared& s, const Choice& c, RowState& state, uint64_t total, uint32_t top) {
    const int tid = threadIdx.x;
    const Row& r = c.row;
    const uint32_t count = state.count[tid];
    const uint64_t weights = state.weight[tid];
    state.count[tid] = 0;
    state.weight[tid] = 0;
    float best = 0.f;
    uint32_t where = 0;
    const auto want = [&](uint64_t sum) {  // the weight that a top-p prefix has to reach
        const double x = (double)c.top_p * (double)sum;
        return x >= 1.0 ? (uint64_t)ceil(x) : 1;
    };

    uint64_t base = 0, lo = 0, hi;
    bool listed = false;  // the list holds every candidate (top-k), not the threshold's bin alone
    uint32_t n;
    if (c.k > 0) {
        const uint32_t b = reaching_bin(s, count, (uint64_t)c.k, base);
        // fewer than k tokens can be drawn at all: all of them are candidates
        n = (uint32_t)block_reduce(s, (uint32_t)tid <= b ? count : 0, plus);
        hi = end_of_bin(b);
        base = 0;
        listed = true;
    } else {
        const uint32_t b = reaching_bin(s, weights, want(total), base);
        n = (uint32_t)block_reduce(s, (uint32_t)tid == b ? count : 0, plus);
        if (b == kBins) n = kGather + 1;  // not reached: only if someone writes the logits meanwhile
        hi = end_of_bin(b);
        lo = b > 0 && b < kBins ? end_of_bin(b - 1) : 0;
    }

    if (n > kGather) {  // the long way
        uint64_t limit = ((uint64_t)kInfBits << 32) - 1;
        if (c.k > 0) limit = last_kept<DT, true>(s, r, limit, (uint64_t)c.k);
        if (c.top_p < 1.f) {
            uint64_t sum = 0;
            each<DT>(r, [&](uint32_t i, float x) {
                const float d = distance(r, x);
                if (key_of(d, i) <= limit) sum += whole(weight(d));
            });
            limit = last_kept<DT, false>(s, r, limit, want(block_reduce(s, sum, plus)));
        }
        each<DT>(r, [&](uint32_t i, float x) {
            const float d = distance(r, x), w = weight(d);
            if (key_of(d, i) <= limit && w > 0.f && (w >= c.min_p || i == top)) draw(w, c.noise[i], i, best, where);
        });
        return block_reduce(s, draw_key(best, where), larger);
    }

    if (tid == 0) s.gathered = 0;
    __syncthreads();
    const float d_lo = d_of(lo), d_hi = d_of(hi);  // whole bins: d alone decides
    for (int64_t i0 = 8 * (int64_t)tid; i0 < r.V; i0 += 4 * (int64_t)kThreads * 8) {
        float x[4][8], e[4][8];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int64_t i = i0 + (int64_t)a * kThreads * 8;
            load8<DT>(r.x, i, i >= r.V ? 0 : r.V - i < 8 ? (int)(r.V - i) : 8, -__builtin_inff(), x[a]);
        }
        bool any[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            float m = x[a][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) m = fmaxf(m, x[a][j]);
            const float d = distance(r, m);
            any[a] = d < d_hi;
            load_noise(c.noise, i0 + (int64_t)a * kThreads * 8, r.V, d < d_lo, e[a]);
        }
#pragma unroll
        for (int a = 0; a < 4; ++a)
            if (any[a])
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t i = (uint32_t)(i0 + (int64_t)a * kThreads * 8 + j);
                    const float v = x[a][j];
                    const float d = v == v ? distance(r, v) : __builtin_inff();
                    if (d < d_lo) {
                        const float w = weight(d);
                        if (w > 0.f && (w >= c.min_p || i == top)) draw(w, e[a][j], i, best, where);
                    } else if (d < d_hi) {
                        const uint32_t g = atomicAdd(&s.gathered, 1u);
                        if (g < kGather) s.list[g] = key_of(d, i);  // as many as were counted, unless someone writes the logits
                    }
                }
    }
    __syncthreads();
    n = min(s.gathered, (uint32_t)kGather);
    sort_list(s, n);
    if (listed) n = min(n, (uint32_t)c.k);
    uint64_t key[kOwn], w[kOwn], sum = 0;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        const uint32_t e = tid * kOwn + j;
        key[j] = e < n ? s.list[e] : ~0ull;
        w[j] = e < n ? whole(weight(d_of(key[j]))) : 0;
        sum += w[j];
    }
    uint64_t target = ~0ull;
    if (c.top_p < 1.f) target = want(listed ? block_reduce(s, sum, plus) : total);
    uint64_t before = base + block_before(s, sum);
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        if (key[j] != ~0ull && before < target) {
            const float x = weight(d_of(key[j]));
            const uint32_t i = (uint32_t)key[j];
            if (x > 0.f && (x >= c.min_p || i == top)) {
                const float score = x / c.noise[i];  // in the list's order: of equals the lowest index
                if (score > best || (score == best && score > 0.f && i < where)) best = score, where = i;
            }
        }
        before += w[j];
    }
    return block_reduce(s, draw_key(best, where), larger);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void choose_kernel(const logits_sample_args p, int64_t row0, RowState* states) {
    __shared__ Shared s;
    const int tid = threadIdx.x;
    const int64_t row = row0 + blockIdx.x;
    RowState& state = states[blockIdx.x];
    Choice c = choice_of<DT>(p, row);
    const uint64_t max_key = state.max_key, total = state.total;
    uint64_t won = state.won;
    uint32_t token = ~(uint32_t)max_key;
    c.row.max = from_order((uint32_t)(max_key >> 32));
    const bool none = c.row.max == -__builtin_inff();  // nothing is allowed
    if (c.searches && !none) won = draw_kept<DT>(s, c, state, total, token);
    if (won) token = ~(uint32_t)won;  // else greedy, or no noise was a number: the most likely token
    __syncthreads();
    if (tid == 0) {
        state.max_key = state.total = state.won = 0;
        p.token[row] = none ? -1 : (int64_t)token;
        if (p.logprob) {
            float x[8];
            load8<DT>(c.row.x, token, 1, 0.f, x);
            p.logprob[row] = none ? c.row.max : -distance(c.row, x[0]) - logf((float)total * (1.f / kOne));
        }
        if (p.counts && !none) {
            const int64_t slot = p.slots ? p.slots[c.b] : c.b;
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

template <int DT>
hipError_t launch(const logits_sample_args& a, hipStream_t s) {
    const int64_t rows = (int64_t)a.B * a.T;
    const uint32_t segments = (uint32_t)(((int64_t)a.V + kSegment - 1) / kSegment);
    RowState* const states = static_cast<RowState*>(a.workspace);
    for (int64_t row0 = 0; row0 < rows; row0 += kRowsAtOnce) {
        const uint32_t n = (uint32_t)(rows - row0 < kRowsAtOnce ? rows - row0 : kRowsAtOnce);
        hipLaunchKernelGGL((max_kernel<DT>), dim3(n * segments), dim3(kSegThreads), 0, s, a, row0, segments, states);
        hipLaunchKernelGGL((weigh_kernel<DT>), dim3(n * segments), dim3(kSegThreads), 0, s, a, row0, segments, states);
        hipLaunchKernelGGL((choose_kernel<DT>), dim3(n), dim3(kThreads), 0, s, a, row0, states);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace lg

extern "C" {

size_t logits_sample_args_size(void) { return sizeof(logits_sample_args); }

int logits_sample_workspace_size(const logits_sample_args* a, size_t* bytes) {
    if (!a || !bytes) return WKV7_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->V < 1) return WKV7_ERR_SHAPE;
    const int64_t rows = (int64_t)a->B * a->T;
    *bytes = sizeof(lg::RowState) * (size_t)(rows < lg::kRowsAtOnce ? rows : lg::kRowsAtOnce);
    return WKV7_OK;
}

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
    size_t bytes = 0;
    const int rc = logits_sample_workspace_size(a, &bytes);
    if (rc != WKV7_OK) return rc;
    if (!a->workspace || a->workspace_bytes < bytes) return WKV7_ERR_WORKSPACE;
    if (!lg::aligned(a->workspace, 256)) return WKV7_ERR_ALIGN;
    const auto s = static_cast<hipStream_t>(stream);
    if (a->dtype == LOGITS_BF16) return static_cast<int>(lg::launch<LOGITS_BF16>(*a, s));
    if (a->dtype == LOGITS_F16) return static_cast<int>(lg::launch<LOGITS_F16>(*a, s));
    return static_cast<int>(lg::launch<LOGITS_F32>(*a, s));
}

}  // extern "C"
