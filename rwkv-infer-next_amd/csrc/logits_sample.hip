// logits_sample.hip -- the choice of a token from each row of logits (include/logits.h), in four launches:
//
//   max     a row's segments, a workgroup each: the row's maximum and its lowest index
//   weigh   the same segments: with d = (max - x) / T, w = exp(-d), in rows without top-k and top-p the sum of w and the draw
//           among their elements; in the others a histogram over d in steps of 1/32, of the tokens' number and of their weights
//   gather  the same segments: where the histogram reaches the wanted number or weight, the last kept token is in that bin.  The
//           tokens before it are kept, and drawn among; the bin's own (top-k: all up to its end) go into the row's list
//   choose  a workgroup a row: the last kept token of the list, by histograms over ever finer parts of (d, index), and the draw
//
// A row's maximum must be known before its weights, its weights before a threshold, and the threshold before the draw: hence the
// launches; no row and no list is sorted.  What atomics add up are whole numbers, so their order shows in no result.  A bin of
// more tokens than the list holds (equal logits, a top-k of thousands) goes the long way: its row's workgroup cuts the row itself
// into finer parts.
//
// d is kept as 32 d (bins are its whole part), which the scaling by a power of two leaves as exact as d.  A bin's weights are
// added up as whole numbers of 2^-24 of the weight at its start (the last place of an fp32 weight; 2^-23 .. 2^-20 where there are more
// than 2^17 tokens), beside its tokens' number in one 64-bit word: one atomic to a token.
//
// Measured, V = 65536, us of max / weigh / gather / choose: one row fp32 with top-p 3.5 / 4.3 / 5.7 / 6.8 (18.1 together in a graph),
// each bound by its chain of dependent reads; 64 rows with top-k and top-p 5.6 / 8.5 / 6.6 / 10.4 (28.3); 320 rows bf16 with a wide
// nucleus 12.0 / 19.0 / 24.0 / 14.7 (65.7): max by memory (42 MB, 3.5 TB/s), weigh and gather by vector instructions (46 and 45 % of
// the time) and the histogram's reading by every gathering workgroup.  A workgroup a row doing all took 78, 111 and 183 us.  Gather
// and choose in one launch, the last workgroup of a row going on, took 20, 39 and 81 us together: its four wavefronts are too few for
// the choosing rounds.  The long way takes 0.75 ms for a row of 65536 equal logits, or for 64 of them at once.
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include <algorithm>

#include "logits.h"
#include "logits_device.h"
#include "wkv7_launch.h"

namespace lg {
namespace {

constexpr int kThreads = 512;      // of the choosing workgroup
constexpr int kSegThreads = 256;   // of a segment's workgroup: 8 elements, or 4 x 8, to a thread
constexpr int kBins = 1024;        // the last one holds all from 1023/32 on
constexpr float kPerUnit = 32.f;   // bins to a unit of d
constexpr int kList = 4096;        // tokens that a row's list holds
constexpr int kOwn = kList / kThreads;
constexpr int kRowsAtOnce = 512;   // rows of one set of launches
constexpr float kOne = 1099511627776.f;  // 2^40: a weight of 1
constexpr uint32_t kInfBits = 0x7F800000u;
constexpr float kExp2PerBin = -1.44269504088896341f / kPerUnit;  // w = 2^(32 d * this)
// A bin's word: its tokens' number above their weights, each at most 2^weight_bits(V), V of them below 2^42.
constexpr int kCountAt = 42;
constexpr int weight_bits(int V) {
    int bits = 24;
    while ((int64_t)V << bits > (int64_t)1 << (kCountAt - 1)) --bits;
    return bits;
}
static_assert(weight_bits(1 << 17) == 24 && weight_bits((1 << 17) + 1) == 23 && weight_bits(LOGITS_SAMPLE_MAX_V) == 20 &&
              LOGITS_SAMPLE_MAX_V < 1 << (64 - kCountAt), "");

// A row's part of the workspace: all zero between calls.  The rows' lists, which need not be, follow the kRowsAtOnce of them.
struct RowState {
    unsigned long long max_key;  // order_bits(max) << 32 | ~index
    unsigned long long total;    // sum of the weights, of whole()s
    unsigned long long won;      // the draw so far: w / noise as an integer << 32 | ~index
    uint32_t gathered;           // entries of the list
    uint32_t bin;                // a Part's bin, target and n, written by the gathering workgroup of the row's first segment
    unsigned long long target;
    uint32_t n;
    uint32_t unused[53];
    unsigned long long bins[kBins];
};
static_assert(sizeof(RowState) * kRowsAtOnce == LOGITS_SAMPLE_STATE_BYTES, "include/logits.h");

// The value of the lane that DPP control CTRL selects, 0 in lanes of rows outside ROWS or without such a lane.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t from_lane(uint64_t x) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T plus(T a, T b) { return a + b; }

// f over the lanes up to this one; bits 0 are f's identity.  Rows of 16 lanes by shifts, then a row's end to the rows after it
// (without the LDS crossbar's round trips).
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T x, F&& f) {
    const auto bits = [](T v) { return __builtin_bit_cast(uint64_t, v); };
    x = f(x, __builtin_bit_cast(T, from_lane<0x111, 0xF>(bits(x))));  // row_shr:1, 2, 4, 8
    x = f(x, __builtin_bit_cast(T, from_lane<0x112, 0xF>(bits(x))));
    x = f(x, __builtin_bit_cast(T, from_lane<0x114, 0xF>(bits(x))));
    x = f(x, __builtin_bit_cast(T, from_lane<0x118, 0xF>(bits(x))));
    x = f(x, __builtin_bit_cast(T, from_lane<0x142, 0xA>(bits(x))));  // row_bcast:15 into rows 1 and 3
    x = f(x, __builtin_bit_cast(T, from_lane<0x143, 0xC>(bits(x))));  // row_bcast:31 into rows 2 and 3
    return x;
}

// f over all lanes of the wavefront.
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T x, F&& f) {
    const uint64_t all = __builtin_bit_cast(uint64_t, wave_scan(x, f));
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)all, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(all >> 32), 63);
    return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}

template <int THREADS>
struct Scratch {
    uint64_t wave[THREADS / 64];
    uint64_t base, found;
    uint32_t bin, n;
};

template <int THREADS, typename T, typename F>
__device__ __forceinline__ T block_reduce(Scratch<THREADS>& s, T x, F&& f) {
    x = wave_reduce(x, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s.wave[threadIdx.x >> 6] = __builtin_bit_cast(uint64_t, x);
    __syncthreads();
    x = __builtin_bit_cast(T, s.wave[0]);
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) x = f(x, __builtin_bit_cast(T, s.wave[w]));
    return x;
}

// The sum over the threads before this one, always added in the same order; `all`: over all threads.
template <int THREADS, typename T>
__device__ __forceinline__ T block_before(Scratch<THREADS>& s, T x, T& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T sum = wave_scan(x, plus<T>);
    // of the lane before, in the row and at a row's start
    uint64_t bits = from_lane<0x111, 0xF>(__builtin_bit_cast(uint64_t, sum));
    const uint64_t bits15 = from_lane<0x142, 0xA>(__builtin_bit_cast(uint64_t, sum));
    const uint64_t bits31 = from_lane<0x143, 0xC>(__builtin_bit_cast(uint64_t, sum));
    if (lane == 16 || lane == 48) bits = bits15;
    if (lane == 32) bits = bits31;
    __syncthreads();
    if (lane == 63) s.wave[wave] = __builtin_bit_cast(uint64_t, sum);
    __syncthreads();
    T others = T(0);
    all = T(0);
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w == wave) others = all;
        all += __builtin_bit_cast(T, s.wave[w]);
    }
    return others + __builtin_bit_cast(T, bits);
}

// The first of kBins bins at whose end the running sum reaches `target`, with the sum before it (s.base) and its `counts` (s.n);
// kBins where none does.  A thread has kBins / THREADS of them.
template <int THREADS, typename T>
__device__ __forceinline__ uint32_t reaching_bin(Scratch<THREADS>& s, const T (&sums)[kBins / THREADS],
                                                 const uint32_t (&counts)[kBins / THREADS], T target, T& base, uint32_t& n) {
    if (threadIdx.x == 0) s.bin = kBins, s.base = 0, s.n = 0;
    T mine = sums[0];
#pragma unroll
    for (int j = 1; j < kBins / THREADS; ++j) mine += sums[j];
    T all, before = block_before(s, mine, all);  // its barriers order the first line
#pragma unroll
    for (int j = 0; j < kBins / THREADS; ++j) {
        // sums before two neighbours may be rounded apart in floating point: the lowest bin of those that fit
        if (before < target && before + sums[j] >= target) atomicMin(&s.bin, threadIdx.x * (kBins / THREADS) + j);
        before += sums[j];
    }
    __syncthreads();
    const uint32_t b = s.bin;
#pragma unroll
    for (int j = kBins / THREADS - 1; j >= 0; --j) {
        before -= sums[j];
        if (b == threadIdx.x * (kBins / THREADS) + j) s.base = __builtin_bit_cast(uint64_t, before), s.n = counts[j];
    }
    __syncthreads();
    base = __builtin_bit_cast(T, s.base), n = s.n;
    __syncthreads();
    return b;
}

// What a row's passes need to know of it.
struct Row {
    const void* x;
    int V;
    float max, inv;  // inv = 32 / temperature
};

// A logit as the kernels take it: NaN as -infinity, infinity as the largest number (so that no difference is NaN).
__device__ __forceinline__ float logit(float x) { return fminf(fmaxf(x, -__builtin_inff()), FLT_MAX); }

// Bits of a float that order as the numbers do (-0 as 0), and back.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t u) { return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u); }

__device__ __forceinline__ float distance(const Row& r, float x) { return (r.max - x) * r.inv; }  // 32 d >= 0
// 2^(32 d c): the product is rounded by up to 2^-19 for the rarest weights that matter, c itself by 2^-26 of it.  What both leave
// out is `lo`, and 2^lo = 1 + lo ln 2.  (NaN for infinity: no weight, or kFar in its place.)
constexpr float kFar = 8192.f;  // of weight 0
__device__ __forceinline__ float weight(float d32) {
    constexpr float kRest = (float)(-1.44269504088896340736 / kPerUnit - (double)kExp2PerBin);
    const float hi = d32 * kExp2PerBin, lo = fmaf(d32, kRest, fmaf(d32, kExp2PerBin, -hi));
    const float w = __builtin_amdgcn_exp2f(hi);
    return fmaf(w, lo * 0.693147181f, w);
}
// Whole numbers are the nearest ones: what is cut off would lean all sums to one side.
__device__ __forceinline__ uint64_t whole(float w) { return (uint64_t)rintf(w * kOne); }
// A weight in its bin's units, `units` = 2^weight_bits(V) of them to the bin's first weight, and the unit.
__device__ __forceinline__ uint32_t in_bin(float d32, float units) {
    return (uint32_t)rintf(__builtin_amdgcn_exp2f(__builtin_amdgcn_fractf(d32) * kExp2PerBin) * units);
}
__device__ __forceinline__ double unit_of_bin(uint32_t b, float units) { return (double)weight((float)b) * (1.0 / units); }
// The first 32 d past a bin; every finite one lies before the last bin's.
__device__ __forceinline__ float end_of_bin(uint32_t b) { return b >= kBins - 1 ? __builtin_inff() : (float)(b + 1); }

__device__ __forceinline__ uint64_t key_of(float d32, uint32_t i) { return (uint64_t)__float_as_uint(d32) << 32 | i; }
__device__ __forceinline__ float d_of(uint64_t key) { return __uint_as_float((uint32_t)(key >> 32)); }

// A row's parameters, the same in every launch.
struct Choice {
    int64_t b, t;
    Row row;
    const float* noise;
    int k;                  // 0: no top-k
    float top_p, min_p;
    float units;            // of a bin's first weight
    bool greedy, searches;  // searches: top-k or top-p
    __device__ uint64_t want(uint64_t sum) const {  // the weight that a top-p prefix has to reach, of whole()s
        const double x = (double)top_p * (double)sum;
        return x >= 1.0 ? (uint64_t)ceil(x) : 1;
    }
};

template <int DT>
__device__ __forceinline__ Choice choice_of(const logits_sample_args& p, int64_t row, float units) {
    Choice c;
    c.b = row / p.T, c.t = row % p.T;
    const float temperature = p.temperature ? p.temperature[c.b] : p.temperature_all;
    c.greedy = !p.noise || !(temperature > 0.f);
    c.row.x = static_cast<const char*>(p.logits) + (c.b * p.seq_stride + c.t * p.pos_stride) * element_bytes(DT);
    c.row.V = p.V;
    c.row.max = 0.f;
    c.row.inv = kPerUnit * (c.greedy ? 1.f : fminf(fmaxf(1.f / temperature, 1e-25f), 1e30f));
    c.noise = p.noise + c.b * p.noise_seq_stride + c.t * p.noise_pos_stride;
    c.k = p.top_k ? p.top_k[c.b] : p.top_k_all;
    if (c.k < 0 || c.k >= p.V) c.k = 0;
    c.top_p = p.top_p ? p.top_p[c.b] : p.top_p_all;
    c.min_p = fminf(p.min_p ? p.min_p[c.b] : p.min_p_all, 1.f);
    c.units = units;
    c.searches = !c.greedy && (c.k > 0 || c.top_p < 1.f);
    return c;
}

__device__ __forceinline__ int piece(int64_t i, int V) { return i >= V ? 0 : V - i < 8 ? (int)(V - i) : 8; }

// This thread's pieces of a segment; -infinity past the row.
template <int DT, int PIECES>
__device__ __forceinline__ void load_segment(const Row& r, int64_t first, float (&x)[PIECES][8]) {
#pragma unroll
    for (int a = 0; a < PIECES; ++a) {
        const int64_t i = first + (a * kSegThreads + threadIdx.x) * 8;
        load8<DT>(r.x, i, piece(i, r.V), -__builtin_inff(), x[a]);
    }
#pragma unroll
    for (int a = 0; a < PIECES; ++a)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[a][j] = logit(x[a][j]);
}

template <int DT, int PIECES>
__global__ __launch_bounds__(kSegThreads) void max_kernel(const logits_sample_args p, int64_t row0, float units, uint32_t segments,
                                                          RowState* states) {
    const uint32_t at = blockIdx.x / segments;
    const int64_t first = (int64_t)(blockIdx.x % segments) * (kSegThreads * PIECES * 8);
    const Choice c = choice_of<DT>(p, row0 + at, units);
    float x[PIECES][8];
    load_segment<DT, PIECES>(c.row, first, x);
    float m = x[0][0];
#pragma unroll
    for (int a = 0; a < PIECES; ++a)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, x[a][j]);
    uint32_t where = 0;
#pragma unroll
    for (int a = PIECES - 1; a >= 0; --a)
#pragma unroll
        for (int j = 7; j >= 0; --j)
            if (x[a][j] == m) where = (uint32_t)(first + (a * kSegThreads + threadIdx.x) * 8 + j);
    const uint64_t key = wave_reduce((uint64_t)order_bits(m) << 32 | (uint32_t)~where, larger);
    if ((threadIdx.x & 63) == 0) atomicMax(&states[at].max_key, (unsigned long long)key);
}

// The best of a draw so far: the largest w / noise, of equals the first that was offered; nothing to begin with, and never an
// element whose noise is negative or no number.  Quotients are compared as the products of one's weight and the other's noise: equal ones
// are then equal, and an element costs no division (weights are at most 1, so no product is too large).
struct Draw {
    float w = 0.f, noise = 1.f;
    uint32_t where = 0;
    __device__ __forceinline__ void offer(float w1, float noise1, uint32_t i) {
        if (w1 * noise > w * noise1 && noise1 >= 0.f) w = w1, noise = noise1, where = i;
    }
    __device__ __forceinline__ void offer_in_any_order(float w1, float noise1, uint32_t i) {
        const float mine = w1 * noise, best = w * noise1;
        if ((mine > best || (mine == best && i < where)) && noise1 >= 0.f) w = w1, noise = noise1, where = i;
    }
    __device__ __forceinline__ uint64_t key() const {  // 0: nothing drawn
        const float score = w / noise;
        return score > 0.f ? (uint64_t)__float_as_uint(score) << 32 | (uint32_t)~where : 0;
    }
};

template <int DT, int PIECES>
__global__ __launch_bounds__(kSegThreads) void weigh_kernel(const logits_sample_args p, int64_t row0, float units, uint32_t segments,
                                                            RowState* states) {
    __shared__ uint64_t bins[kBins];
    const int tid = threadIdx.x;
    const uint32_t at = blockIdx.x / segments;
    const int64_t first = (int64_t)(blockIdx.x % segments) * (kSegThreads * PIECES * 8);
    RowState& state = states[at];
    Choice c = choice_of<DT>(p, row0 + at, units);
    float x[PIECES][8];
    load_segment<DT, PIECES>(c.row, first, x);
    c.row.max = from_order((uint32_t)(state.max_key >> 32));
    if (c.row.max == -__builtin_inff()) return;
    if (c.searches) {
        for (int b = tid; b < kBins; b += kSegThreads) bins[b] = 0;
        __syncthreads();
        // A long tail's tokens all fall into the last bin: counted in registers, their weights left out (e^-32 each, 2^21 of them 2.7e-8).
        uint32_t far = 0;
#pragma unroll
        for (int a = 0; a < PIECES; ++a)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = distance(c.row, x[a][j]);
                if (d < (float)(kBins - 1))
                    atomicAdd((unsigned long long*)&bins[(uint32_t)fmaxf(d, 0.f)], 1ull << kCountAt | in_bin(d, c.units));
                else
                    far += d < __builtin_inff();
            }
        far = (uint32_t)wave_reduce((uint64_t)far, plus<uint64_t>);
        if ((tid & 63) == 0 && far) atomicAdd((unsigned long long*)&bins[kBins - 1], (unsigned long long)far << kCountAt);
        __syncthreads();
        for (int b = tid; b < kBins; b += kSegThreads)
            if (bins[b]) atomicAdd(&state.bins[b], (unsigned long long)bins[b]);
    } else {
        const bool draws = !c.greedy;
        // Eight neighbours' weights are added in order and then taken as a whole number: the same sum whatever the segments' length,
        // which follows from the number of rows.
        uint64_t total = 0;
        Draw best;
        float e[PIECES][8];
        if (draws)
#pragma unroll
            for (int a = 0; a < PIECES; ++a) {
                const int64_t i = first + (a * kSegThreads + tid) * 8;
                load8<LOGITS_F32>(c.noise, i, piece(i, p.V), 1.f, e[a]);
            }
#pragma unroll
        for (int a = 0; a < PIECES; ++a) {
            float eight = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float w = weight(fminf(distance(c.row, x[a][j]), kFar));
                eight += w;
                if (draws && w >= c.min_p && w > 0.f)
                    best.offer(w, e[a][j], (uint32_t)(first + (a * kSegThreads + tid) * 8 + j));
            }
            total += whole(eight);
        }
        if (draws) {
            const uint64_t key = wave_reduce(best.key(), larger);
            if ((tid & 63) == 0 && key) atomicMax(&state.won, (unsigned long long)key);
        }
        const uint64_t sum = wave_reduce(total, plus<uint64_t>);
        if ((tid & 63) == 0) atomicAdd(&state.total, (unsigned long long)sum);
    }
}

// Where a row's last kept token lies, from its histogram: in bin [from, to) of 32 d, where the prefix that ends with it has to
// reach `target` tokens (top-k) or units of the bin (top-p) beside what lies before the bin.  The candidates' list begins at d_lo:
// with top-k at 0, since top-p looks at them all again; with top-p alone at the bin, what lies before it being kept.
// All gathering workgroups of a row make it of the same sums in the same order, and the choosing one takes it from the first of
// them: sums in another order may be a last place apart, and so a bin.
struct Part {
    uint32_t bin, n;  // n: candidates
    uint64_t target;
    __device__ float from() const { return bin > 0 ? end_of_bin(bin - 1) : 0.f; }
    __device__ float to() const { return end_of_bin(bin); }
    __device__ float d_lo(const Choice& c) const { return c.k > 0 ? 0.f : from(); }
};

// `total`: of the row's weights, where the part needs it or wants_total.
__device__ __forceinline__ Part part_of(Scratch<kSegThreads>& s, const Choice& c, const RowState& state, bool wants_total,
                                        double& total) {
    constexpr int kEach = kBins / kSegThreads;
    uint32_t counts[kEach], n;
    uint64_t numbers[kEach];
    double sums[kEach], all = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const uint32_t b = threadIdx.x * kEach + j;
        const uint64_t word = state.bins[b];
        numbers[j] = counts[j] = (uint32_t)(word >> kCountAt);
        sums[j] = (double)(word & ((1ull << kCountAt) - 1)) * unit_of_bin(b, c.units);
        all += sums[j];
    }
    Part part;
    total = 0;
    if (c.k <= 0 || wants_total) total = block_reduce(s, all, plus<double>);
    if (c.k > 0) {
        uint64_t base;
        const uint32_t b = reaching_bin(s, numbers, counts, (uint64_t)c.k, base, n);
        if (b == kBins) {  // less than k tokens can be drawn at all: all of them are candidates
            uint64_t mine = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) mine += numbers[j];
            base = block_reduce(s, mine, plus<uint64_t>);
        }
        part.bin = b;
        part.target = (uint64_t)c.k - (b == kBins ? 0 : base);
        part.n = (uint32_t)base + n;
    } else {
        double base;
        const uint32_t b = reaching_bin(s, sums, counts, fmax((double)c.top_p * total, 1e-300), base, n);
        part.bin = b;
        const double rest = ceil(((double)c.top_p * total - base) / unit_of_bin(b, c.units));
        part.target = rest >= 1.0 ? (uint64_t)rest : 1;
        part.n = b == kBins ? kList + 1 : n;  // past all bins only if someone writes the logits meanwhile
    }
    return part;
}

template <int DT, int PIECES>
__global__ __launch_bounds__(kSegThreads) void gather_kernel(const logits_sample_args p, int64_t row0, float units, uint32_t segments,
                                                             RowState* states, uint64_t* lists) {
    __shared__ Scratch<kSegThreads> s;
    const int tid = threadIdx.x;
    const uint32_t at = blockIdx.x / segments;
    const int64_t first = (int64_t)(blockIdx.x % segments) * (kSegThreads * PIECES * 8);
    RowState& state = states[at];
    Choice c = choice_of<DT>(p, row0 + at, units);
    if (!c.searches) return;
    float x[PIECES][8];
    load_segment<DT, PIECES>(c.row, first, x);
    const uint64_t max_key = state.max_key;
    const uint32_t top = ~(uint32_t)max_key;
    c.row.max = from_order((uint32_t)(max_key >> 32));
    if (c.row.max == -__builtin_inff()) return;
    double total;
    const Part part = part_of(s, c, state, first == 0, total);
    if (first == 0 && tid == 0) {
        state.bin = part.bin, state.n = part.n, state.target = part.target;
        state.total = (unsigned long long)(total * (double)kOne);
    }
    if (part.n > kList) return;  // the choosing workgroup's work
    const float d_lo = part.d_lo(c);

    float nearest[PIECES];  // x becomes 32 d, nearest a piece's smallest
#pragma unroll
    for (int a = 0; a < PIECES; ++a) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[a][j] = distance(c.row, x[a][j]);
        nearest[a] = x[a][0];
#pragma unroll
        for (int j = 1; j < 8; ++j) nearest[a] = fminf(nearest[a], x[a][j]);
    }
    if (d_lo > 0.f) {  // kept for sure
        Draw best;
        float e[PIECES][8];
#pragma unroll
        for (int a = 0; a < PIECES; ++a) {
            const int64_t i = first + (a * kSegThreads + tid) * 8;
            load8<LOGITS_F32>(c.noise, i, nearest[a] < d_lo ? piece(i, p.V) : 0, 1.f, e[a]);
        }
#pragma unroll
        for (int a = 0; a < PIECES; ++a)
            if (nearest[a] < d_lo)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t i = (uint32_t)(first + (a * kSegThreads + tid) * 8 + j);
                    const float w = weight(x[a][j]);
                    if (x[a][j] < d_lo && w > 0.f && (w >= c.min_p || i == top)) best.offer(w, e[a][j], i);
                }
        const uint64_t key = wave_reduce(best.key(), larger);
        if ((tid & 63) == 0 && key) atomicMax(&state.won, (unsigned long long)key);
    }
    // bits of non-negative floats order as they do
    const uint32_t from = __float_as_uint(d_lo), span = __float_as_uint(part.to()) - from;
    uint32_t hits = 0;  // a bit for each of the 8 PIECES elements, the first the highest
#pragma unroll
    for (int a = 0; a < PIECES; ++a)
#pragma unroll
        for (int j = 0; j < 8; ++j) hits = hits + hits + (__float_as_uint(x[a][j]) - from < span);
    const uint32_t mine = __popc(hits);
    uint64_t all;
    uint32_t to = (uint32_t)block_before(s, (uint64_t)mine, all);
    if (tid == kSegThreads - 1) s.n = to + mine ? atomicAdd(&state.gathered, to + mine) : 0;
    __syncthreads();
    to += s.n;
    uint64_t* const list = lists + (int64_t)at * kList;
    while (hits) {  // few: read again rather than picked out of registers
        const int bit = 31 - __clz(hits), e = 8 * PIECES - 1 - bit;
        hits ^= 1u << bit;
        const int64_t i = first + ((e >> 3) * kSegThreads + tid) * 8 + (e & 7);
        float y[8];
        load8<DT>(c.row.x, i, 1, 0.f, y);
        // as many as were counted, unless someone writes the logits meanwhile
        if (to < kList) list[to] = key_of(distance(c.row, logit(y[0])), (uint32_t)i);
        ++to;
    }
}

struct Shared {
    uint64_t weight[kBins];
    uint32_t count[kBins];
    Scratch<kThreads> scratch;
};

// f(index, 32 d) for every element of the row; four 8-element pieces in flight to a thread.
template <int DT, typename F>
__device__ __forceinline__ void each(const Row& r, F&& f) {
    constexpr int kAhead = 4;
    for (int64_t i0 = 8 * (int64_t)threadIdx.x; i0 < r.V; i0 += (int64_t)kAhead * kThreads * 8) {
        float x[kAhead][8];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int64_t i = i0 + (int64_t)a * kThreads * 8;
            load8<DT>(r.x, i, piece(i, r.V), -__builtin_inff(), x[a]);
        }
#pragma unroll 1
        for (int a = 0; a < kAhead; ++a) {
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = a == 0 ? x[0][j] : a == 1 ? x[1][j] : a == 2 ? x[2][j] : x[3][j];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                f((uint32_t)(i0 + (int64_t)a * kThreads * 8 + j), distance(r, logit(y[j])));
        }
    }
}

enum Measure { kNumber, kUnits, kWhole };  // of a prefix: its tokens, their weights in their bin's units, or in whole()s

// The key of the last token of the smallest prefix, in the order of keys, whose measure reaches `target`, among the tokens of
// `all(f)` (f(key) for each) with keys in [lo, hi); `none` where all do not reach it.  [lo, hi) is cut into 1024 parts, first
// (BINS) by bins of d, until the part in which the target is reached has one token.
template <Measure M, bool BINS, typename All>
__device__ uint64_t last_kept(Shared& s, float units, All&& all, uint64_t lo, uint64_t hi, uint64_t target, uint64_t none) {
    constexpr int kEach = kBins / kThreads;
    const int tid = threadIdx.x;
    bool bins = BINS;
    for (;;) {
        const uint64_t last = hi - lo - 1;
        const int shift = max(0, 54 - (int)__clzll(last | 1));  // last >> shift < kBins
#pragma unroll
        for (int j = 0; j < kEach; ++j) s.count[tid * kEach + j] = 0, s.weight[tid * kEach + j] = 0;
        __syncthreads();
        all([&](uint64_t key) {
            if (key >= lo && key < hi) {
                const float d = d_of(key);
                const uint32_t b = bins ? (uint32_t)fminf(d, (float)(kBins - 1)) : (uint32_t)((key - lo) >> shift);
                atomicAdd(&s.count[b], 1u);
                if (M != kNumber)
                    atomicAdd((unsigned long long*)&s.weight[b],
                              (unsigned long long)(M == kUnits ? in_bin(d, units) : whole(weight(d))));
            }
        });
        __syncthreads();
        uint32_t counts[kEach], n;
        uint64_t sums[kEach], before;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            counts[j] = s.count[tid * kEach + j];
            sums[j] = M == kNumber ? counts[j] : s.weight[tid * kEach + j];
        }
        const uint32_t b = reaching_bin(s.scratch, sums, counts, target, before, n);
        if (b == kBins) return none;
        target -= before;
        if (bins) {
            const uint64_t from = key_of(b > 0 ? end_of_bin(b - 1) : 0.f, 0), to = key_of(end_of_bin(b), 0);
            lo = lo > from ? lo : from;
            hi = hi < to ? hi : to;
            bins = false;
        } else {
            lo += (uint64_t)b << shift;
            const uint64_t to = lo + (uint64_t(1) << shift);
            hi = hi < to ? hi : to;
        }
        if (n <= 1 || hi - lo <= 1) break;
    }
    if (hi - lo <= 1) return lo;
    all([&](uint64_t key) {
        if (key >= lo && key < hi) s.scratch.found = key;
    });
    __syncthreads();
    const uint64_t found = s.scratch.found;
    __syncthreads();
    return found;
}

constexpr uint64_t kEveryKey = (uint64_t)kInfBits << 32;  // past every token that can be drawn

// The choice in a row with top-k or top-p, as draw_key; `won`: the draw among the tokens that the gathering workgroups kept.
template <int DT>
__device__ uint64_t choose(Shared& s, const Choice& c, RowState& state, const uint64_t* list, uint32_t top, uint64_t won) {
    const int tid = threadIdx.x;
    uint64_t mine[kOwn];  // asked for before it is known how many of them are there
#pragma unroll
    for (int j = 0; j < kOwn; ++j) mine[j] = list[tid + j * kThreads];
    const uint32_t n = min(state.gathered, (uint32_t)kList);
    const Part part = {state.bin, state.n, state.target};
    for (int b = tid; b < kBins; b += kThreads) state.bins[b] = 0;
    Draw best;

    if (part.n > kList) {  // the long way
        uint64_t limit = kEveryKey - 1;
        const auto all = [&](auto&& f) {
            each<DT>(c.row, [&](uint32_t i, float d) {
                const uint64_t key = key_of(d, i);
                if (key <= limit) f(key);
            });
        };
        if (c.k > 0) limit = last_kept<kNumber, true>(s, c.units, all, 0, kEveryKey, (uint64_t)c.k, limit);
        if (c.top_p < 1.f) {
            uint64_t sum = 0;
            all([&](uint64_t key) { sum += whole(weight(d_of(key))); });
            limit = last_kept<kWhole, true>(s, c.units, all, 0, kEveryKey, c.want(block_reduce(s.scratch, sum, plus<uint64_t>)), limit);
        }
        all([&](uint64_t key) {
            const float w = weight(d_of(key));
            const uint32_t i = (uint32_t)key;
            if (w > 0.f && (w >= c.min_p || i == top)) best.offer(w, c.noise[i], i);
        });
        return block_reduce(s.scratch, best.key(), larger);
    }

    uint64_t key[kOwn];
#pragma unroll
    for (int j = 0; j < kOwn; ++j) key[j] = tid + j * kThreads < n ? mine[j] : ~0ull;
    float noise[kOwn];  // of all candidates, asked for before it is known which are kept
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
        noise[j] = 1.f;
        if (key[j] != ~0ull) noise[j] = c.noise[min((uint32_t)key[j], (uint32_t)c.row.V - 1)];
    }
    uint64_t limit = kEveryKey - 1;
    const auto all = [&](auto&& f) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j)
            if (key[j] <= limit) f(key[j]);
    };
    const uint64_t lo = key_of(part.from(), 0), hi = key_of(part.to(), 0);
    if (c.k > 0) {
        if (n > (uint32_t)c.k) limit = last_kept<kNumber, false>(s, c.units, all, lo, hi, part.target, limit);
        if (c.top_p < 1.f) {
            uint64_t sum = 0;
            all([&](uint64_t k) { sum += whole(weight(d_of(k))); });
            limit = last_kept<kWhole, true>(s, c.units, all, 0, hi, c.want(block_reduce(s.scratch, sum, plus<uint64_t>)), limit);
        }
    } else {
        limit = last_kept<kUnits, false>(s, c.units, all, lo, hi, part.target, limit);
    }
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
        if (key[j] <= limit) {
            const float w = weight(d_of(key[j]));
            const uint32_t i = (uint32_t)key[j];
            if (w > 0.f && (w >= c.min_p || i == top)) best.offer_in_any_order(w, noise[j], i);
        }
    return larger(won, block_reduce(s.scratch, best.key(), larger));
}

template <int DT>
__global__ __launch_bounds__(kThreads, 4) void choose_kernel(const logits_sample_args p, int64_t row0, float units, RowState* states,
                                                          const uint64_t* lists) {
    __shared__ Shared s;
    const int64_t row = row0 + blockIdx.x;
    RowState& state = states[blockIdx.x];
    Choice c = choice_of<DT>(p, row, units);
    const uint64_t max_key = state.max_key;
    uint64_t won = state.won;
    const double total = (double)state.total * (1.0 / kOne);
    uint32_t token = ~(uint32_t)max_key;
    c.row.max = from_order((uint32_t)(max_key >> 32));
    const bool none = c.row.max == -__builtin_inff();  // nothing is allowed
    if (c.searches && !none) won = choose<DT>(s, c, state, lists + (int64_t)blockIdx.x * kList, token, won);
    if (won) token = ~(uint32_t)won;  // else greedy, or no noise was a number: the most likely token
    // A token past the row comes only out of a workspace that calls used at the same time: no memory is touched for it.
    const bool chosen = !none && token < (uint32_t)p.V;
    __syncthreads();
    if (threadIdx.x == 0) {
        state.max_key = state.total = state.won = state.target = 0;
        state.gathered = state.bin = state.n = 0;
        p.token[row] = chosen ? (int64_t)token : -1;
        if (p.logprob) {
            float x[8];
            load8<DT>(c.row.x, chosen ? token : 0, 1, 0.f, x);
            p.logprob[row] =
                chosen ? -distance(c.row, logit(x[0])) * (1.f / kPerUnit) - logf((float)total) : -__builtin_inff();
        }
        if (p.counts && chosen) {
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

template <int DT, int PIECES>
hipError_t launch(const logits_sample_args& a, hipStream_t s) {
    constexpr int kSegment = kSegThreads * PIECES * 8;
    const int64_t rows = (int64_t)a.B * a.T, segments = ((int64_t)a.V + kSegment - 1) / kSegment;
    RowState* const states = static_cast<RowState*>(a.workspace);
    uint64_t* const lists = reinterpret_cast<uint64_t*>(static_cast<char*>(a.workspace) + LOGITS_SAMPLE_STATE_BYTES);
    // rows' own parameters decide what the gathering kernel does; where one for all says that nothing is searched, it is left out
    const bool searches = a.noise && (a.top_k || a.top_p || (a.top_k_all > 0 && a.top_k_all < a.V) || a.top_p_all < 1.f);
    const float units = (float)(1 << weight_bits(a.V));
    const int64_t at_once = std::min<int64_t>(kRowsAtOnce, 0xFFFFFF / segments);  // 256 threads each: below 2^32 work-items
    for (int64_t row0 = 0; row0 < rows; row0 += at_once) {
        const int64_t n = std::min(rows - row0, at_once);
        const dim3 grid((unsigned)(n * segments)), block(kSegThreads);
        const uint32_t seg = (uint32_t)segments;
        hipLaunchKernelGGL((max_kernel<DT, PIECES>), grid, block, 0, s, a, row0, units, seg, states);
        hipLaunchKernelGGL((weigh_kernel<DT, PIECES>), grid, block, 0, s, a, row0, units, seg, states);
        if (searches) hipLaunchKernelGGL((gather_kernel<DT, PIECES>), grid, block, 0, s, a, row0, units, seg, states, lists);
        hipLaunchKernelGGL((choose_kernel<DT>), dim3((unsigned)n), dim3(kThreads), 0, s, a, row0, units, states, lists);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Short segments while long ones would leave CUs without two workgroups.
template <int DT>
hipError_t launch(const logits_sample_args& a, hipStream_t s) {
    const int64_t long_ones = (int64_t)a.B * a.T * (((int64_t)a.V + 8191) / 8192);
    return long_ones < 2 * wkv7::device_cu_count() ? launch<DT, 1>(a, s) : launch<DT, 4>(a, s);
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace lg

extern "C" {

size_t logits_sample_args_size(void) { return sizeof(logits_sample_args); }

int logits_sample_workspace_size(const logits_sample_args* a, size_t* bytes) {
    if (!a || !bytes) return WKV7_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->V < 1 || a->V > LOGITS_SAMPLE_MAX_V) return WKV7_ERR_SHAPE;
    const int64_t rows = std::min<int64_t>((int64_t)a->B * a->T, lg::kRowsAtOnce);
    *bytes = LOGITS_SAMPLE_STATE_BYTES + (size_t)rows * lg::kList * sizeof(uint64_t);
    return WKV7_OK;
}

int logits_sample(const logits_sample_args* a, void* stream) {
    if (!a) return WKV7_ERR_NULL;
    if (a->B < 0 || a->T < 0 || a->V < 1 || a->V > LOGITS_SAMPLE_MAX_V) return WKV7_ERR_SHAPE;
    if (a->dtype < LOGITS_BF16 || a->dtype > LOGITS_F32 ||
        (a->counts && ((a->counts_dtype != LOGITS_COUNTS_I32 && a->counts_dtype != LOGITS_COUNTS_F32) || a->T > 1)))
        return WKV7_ERR_ARG;
    if (a->B == 0 || a->T == 0) return WKV7_OK;
    if (!a->logits || !a->token) return WKV7_ERR_NULL;
    if (a->counts && (a->counts_rows < 0 || a->counts_stride < a->V)) return WKV7_ERR_SHAPE;
    if (!lg::aligned(a->logits, lg::element_bytes(a->dtype)) || !lg::aligned(a->noise, 4) || !lg::aligned(a->counts, 4) ||
        !lg::aligned(a->workspace, 256))
        return WKV7_ERR_ALIGN;
    size_t bytes = 0;
    const int rc = logits_sample_workspace_size(a, &bytes);
    if (rc != WKV7_OK) return rc;
    if (!a->workspace || a->workspace_bytes < bytes) return WKV7_ERR_WORKSPACE;
    const auto s = static_cast<hipStream_t>(stream);
    if (a->dtype == LOGITS_BF16) return static_cast<int>(lg::launch<LOGITS_BF16>(*a, s));
    if (a->dtype == LOGITS_F16) return static_cast<int>(lg::launch<LOGITS_F16>(*a, s));
    return static_cast<int>(lg::launch<LOGITS_F32>(*a, s));
}

}  // extern "C"
