// slots.hip -- copies, compaction and freeing of the slots of several cache tensors in one launch (include/slots.h).
//
// All three move bytes: rows are read once and written once, and HBM bounds them.  A workgroup owns a range of a row's bytes in one
// layer of one cache, for all the slots that the call names, so that sources which are also destinations are read before they are
// written, and a source that goes to many slots comes from memory once.  Measured, where a large copy moves 4.9 TB/s: four states of 2.7 MB
// to 28 slots 19.9 us, 4.3 TB/s; 17 slots of 21 MB moved 148 us, 4.9 TB/s.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "slots.h"

namespace slots {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kUnits = 16;  // units of a copy that a thread holds in registers
constexpr int kTable = 2 * SLOTS_MAX_PAIRS;

struct Cache {
    const char* from;
    char* to;
    int64_t from_layer, from_slot, to_layer, to_slot;
    int64_t units;       // of a row
    int32_t unit;        // bytes: 16, 4, 2 or 1
    uint32_t ranges;     // of a row
    uint32_t end;        // workgroups of this and the caches before it
};

struct Call {
    Cache c[SLOTS_MAX_CACHES];
    const int64_t *src, *dst;
    const uint8_t* live;
    int64_t* where;
    int32_t* count;
    int32_t* status;
    int64_t from_slots, to_slots;
    int32_t n, num_caches;
    int32_t shift;   // copy: a range has 2^shift units; free, compact: kThreads * kUnits units
    int32_t groups;  // compact, free: workgroups that share a range's moves or slots
};

// The cache, layer and range of workgroup `b`.
struct Place {
    int cache;
    int64_t layer;
    uint32_t range;
};
__device__ __forceinline__ Place place(const Call& p, uint32_t b) {
    int i = 0;
    while (i + 1 < p.num_caches && b >= p.c[i].end) ++i;
    const uint32_t at = b - (i ? p.c[i - 1].end : 0u);
    return {i, (int64_t)(at / p.c[i].ranges), at % p.c[i].ranges};
}

template <typename F>
__device__ __forceinline__ void with_unit(int unit, F&& f) {
    if (unit == 16)
        f(u4{});
    else if (unit == 4)
        f(uint32_t{});
    else if (unit == 2)
        f(uint16_t{});
    else
        f(uint8_t{});
}

__device__ __forceinline__ void report(int32_t* status) { atomicOr(status, SLOTS_STATUS_SLOT); }

__global__ __launch_bounds__(kThreads) void slots_copy_kernel(const Call p) {
    __shared__ int32_t from[SLOTS_MAX_PAIRS], to[SLOTS_MAX_PAIRS];
    __shared__ int32_t key[kTable], last[kTable];
    const int tid = threadIdx.x;
    if (p.num_caches == 0) {  // the indices alone
        for (int i = tid; i < p.n; i += kThreads)
            if (p.src[i] >= p.from_slots || p.dst[i] >= p.to_slots) report(p.status);
        return;
    }
    const Place at = place(p, blockIdx.x);
    const Cache c = p.c[at.cache];
    int table = 2;  // at most half full
    while (table < 2 * p.n) table *= 2;
    for (int i = tid; i < table; i += kThreads) key[i] = -1, last[i] = -1;
    __syncthreads();
    const auto hash = [&](int32_t d) { return (int)((uint32_t)d * 2654435761u >> 16) & (table - 1); };
    for (int i = tid; i < p.n; i += kThreads) {
        const int64_t s = p.src[i], d = p.dst[i];
        const bool in = s >= 0 && s < p.from_slots && d >= 0 && d < p.to_slots;
        if (p.status && blockIdx.x == 0 && (s >= p.from_slots || d >= p.to_slots)) report(p.status);
        from[i] = (int32_t)s;
        to[i] = in ? (int32_t)d : -1;
        if (!in) continue;
        for (int h = hash((int32_t)d);; h = (h + 1) & (table - 1)) {
            const int32_t was = atomicCAS(&key[h], -1, (int32_t)d);
            if (was == -1 || was == (int32_t)d) {
                atomicMax(&last[h], i);
                break;
            }
        }
    }
    __syncthreads();
    for (int i = tid; i < p.n; i += kThreads) {  // its own entries
        const int32_t d = to[i];
        if (d < 0) continue;
        int h = hash(d);
        while (key[h] != d) h = (h + 1) & (table - 1);
        if (last[h] != i || (c.from == c.to && from[i] == d)) to[i] = -1;
    }
    __syncthreads();

    const char* const src = c.from + at.layer * c.from_layer;
    char* const dst = c.to + at.layer * c.to_layer;
    const int64_t first = (int64_t)at.range << p.shift;
    const int total = p.n << p.shift;  // at most kThreads * kUnits
    with_unit(c.unit, [&](auto zero) {
        typedef decltype(zero) T;
        T x[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int e = u * kThreads + tid, i = e >> p.shift;
            const int64_t q = first + (e & ((1 << p.shift) - 1));
            if (e < total && q < c.units && to[i] >= 0)
                x[u] = reinterpret_cast<const T*>(src + from[i] * c.from_slot)[q];
        }
        __syncthreads();  // every source is read
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int e = u * kThreads + tid, i = e >> p.shift;
            const int64_t q = first + (e & ((1 << p.shift) - 1));
            if (e < total && q < c.units && to[i] >= 0)
                __builtin_nontemporal_store(x[u], reinterpret_cast<T*>(dst + to[i] * c.to_slot) + q);
        }
    });
}

// Workgroup (x, y): range x for slots idx[y], idx[y + groups], ..
__global__ __launch_bounds__(kThreads) void slots_free_kernel(const Call p) {
    if (p.num_caches == 0) {  // the indices alone
        for (int i = threadIdx.x; i < p.n; i += kThreads)
            if (p.dst[i] >= p.to_slots) report(p.status);
        return;
    }
    const Place at = place(p, blockIdx.x);
    const Cache c = p.c[at.cache];
    const int64_t first = (int64_t)at.range * (kThreads * kUnits);
    for (int i = blockIdx.y; i < p.n; i += p.groups) {
        const int64_t s = p.dst[i];
        if (p.status && blockIdx.x == 0 && threadIdx.x == 0 && s >= p.to_slots) report(p.status);
        if (s < 0 || s >= p.to_slots) continue;
        char* const row = c.to + at.layer * c.to_layer + s * c.to_slot;
        with_unit(c.unit, [&](auto zero) {
            typedef decltype(zero) T;
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int64_t q = first + u * kThreads + threadIdx.x;
                if (q < c.units) __builtin_nontemporal_store(T{}, reinterpret_cast<T*>(row) + q);
            }
        });
    }
}

// Workgroup (x, y): range x for the moves y, y + groups, ..  Each makes the plan for itself: it is a scan of `slots` bytes.
__global__ __launch_bounds__(kThreads) void slots_compact_kernel(const Call p) {
    extern __shared__ int32_t list[];  // [holes of slots / 2][movers of slots / 2]
    __shared__ int32_t sums[kThreads / 64], before_k;
    const int tid = threadIdx.x, lane = tid & 63, slots = (int)p.to_slots, most = slots / 2 + 1;
    const int each = (slots + kThreads - 1) / kThreads, s0 = min(slots, tid * each), s1 = min(slots, s0 + each);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += p.live[s] != 0;
    int run = mine;  // inclusive scan over the wavefront
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int other = __shfl_up(run, d);
        run += lane >= d ? other : 0;
    }
    if (lane == 63) sums[tid >> 6] = run;
    __syncthreads();
    int k = 0, base = run - mine;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < (tid >> 6)) base += sums[w];
        k += sums[w];
    }
    if (tid == 0) before_k = k;  // where every live slot lies before k
    __syncthreads();
    int live = base;
    for (int s = s0; s < s1; ++s) {
        if (s == k) before_k = live;
        live += p.live[s] != 0;
    }
    __syncthreads();
    const int moves = k - before_k;
    const bool tell = blockIdx.x == 0 && blockIdx.y == 0;
    live = base;
    for (int s = s0; s < s1; ++s) {
        const bool on = p.live[s] != 0;
        if (s < k && !on) list[s - live] = s;
        if (s >= k && on) list[most + live - before_k] = s;
        live += on;
    }
    __syncthreads();
    if (tell) {
        live = base;
        for (int s = s0; s < s1; ++s) {
            const bool on = p.live[s] != 0;
            if (p.where) p.where[s] = !on ? -1 : s < k ? s : list[live - before_k];
            live += on;
        }
        if (p.count && tid == 0) *p.count = k;
    }
    if (p.num_caches == 0) return;

    const Place at = place(p, blockIdx.x);
    const Cache c = p.c[at.cache];
    char* const rows = c.to + at.layer * c.to_layer;
    constexpr int kPer = 4, kAhead = kUnits / kPer;  // units of a move, moves in flight
    const int64_t first = (int64_t)at.range * (kThreads * kPer);
    with_unit(c.unit, [&](auto zero) {
        typedef decltype(zero) T;
        for (int j0 = blockIdx.y; j0 < moves; j0 += kAhead * p.groups) {
            T x[kAhead][kPer];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int j = j0 + a * p.groups;
                if (j < moves)
#pragma unroll
                    for (int u = 0; u < kPer; ++u) {
                        const int64_t q = first + u * kThreads + tid;
                        if (q < c.units)
                            x[a][u] = __builtin_nontemporal_load(
                                reinterpret_cast<const T*>(rows + list[most + j] * c.to_slot) + q);
                    }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int j = j0 + a * p.groups;
                if (j < moves)
#pragma unroll
                    for (int u = 0; u < kPer; ++u) {
                        const int64_t q = first + u * kThreads + tid;
                        if (q < c.units)
                            __builtin_nontemporal_store(x[a][u], reinterpret_cast<T*>(rows + list[j] * c.to_slot) + q);
                    }
            }
        }
    });
}

constexpr int64_t kMaxGrid = 0x7FFFFF;  // workgroups of one launch: with 256 threads below 2^32 work-items

// The caches that hold something (in `slots` slots), with their units and workgroups; a range has `range` units.  A negative code for
// what is refused.
int fill(Call& p, const slots_cache* caches, int32_t num, bool copies, int64_t slots, int64_t range, int64_t* blocks) {
    if (num < 0 || num > SLOTS_MAX_CACHES) return WKV7_ERR_SHAPE;
    if (num && !caches) return WKV7_ERR_NULL;
    *blocks = 0;
    p.num_caches = 0;
    for (int i = 0; i < num; ++i) {
        const slots_cache& x = caches[i];
        if (x.row_bytes < 0 || x.layers < 0) return WKV7_ERR_SHAPE;
        if (x.row_bytes == 0 || x.layers == 0 || slots == 0) continue;
        if (!x.to || (copies && !x.from)) return WKV7_ERR_NULL;
        if (x.to_slot_stride < x.row_bytes || x.to_layer_stride < 0 ||
            (copies && (x.from_slot_stride < x.row_bytes || x.from_layer_stride < 0)))
            return WKV7_ERR_SHAPE;
        uint64_t all = reinterpret_cast<uintptr_t>(x.to) | x.to_slot_stride | x.to_layer_stride | x.row_bytes;
        if (copies) all |= reinterpret_cast<uintptr_t>(x.from) | x.from_slot_stride | x.from_layer_stride;
        Cache& c = p.c[p.num_caches++];
        c.unit = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
        c.units = x.row_bytes / c.unit;
        const int64_t ranges = (c.units + range - 1) / range;
        if (ranges > kMaxGrid || x.layers > kMaxGrid) return WKV7_ERR_SHAPE;
        *blocks += ranges * x.layers;
        if (*blocks > kMaxGrid) return WKV7_ERR_SHAPE;
        c.from = static_cast<const char*>(x.from);
        c.to = static_cast<char*>(x.to);
        c.from_layer = x.from_layer_stride, c.from_slot = x.from_slot_stride;
        c.to_layer = x.to_layer_stride, c.to_slot = x.to_slot_stride;
        c.ranges = (uint32_t)ranges;
        c.end = (uint32_t)*blocks;
    }
    return WKV7_OK;
}

}  // namespace
}  // namespace slots

extern "C" {

size_t slots_cache_size(void) { return sizeof(slots_cache); }

int slots_copy(const slots_cache* caches, int32_t num_caches, const int64_t* src, const int64_t* dst, int32_t n,
               int64_t from_slots, int64_t to_slots, int32_t* status, void* stream) {
    if (n < 0 || n > SLOTS_MAX_PAIRS || from_slots < 0 || to_slots < 0 || from_slots > 0x7FFFFFFF || to_slots > 0x7FFFFFFF)
        return WKV7_ERR_SHAPE;
    slots::Call p{};
    int shift = 0;  // as many units of a row as the registers hold for n slots
    while (shift < 12 && (n << (shift + 1)) <= slots::kThreads * slots::kUnits) ++shift;
    int64_t blocks;
    const int rc = slots::fill(p, caches, num_caches, true, std::min(from_slots, to_slots), (int64_t)1 << shift, &blocks);
    if (rc != WKV7_OK) return rc;
    if (n == 0 || (blocks == 0 && !status)) return WKV7_OK;
    if (!src || !dst) return WKV7_ERR_NULL;
    if (blocks == 0) blocks = 1;  // looks at the indices alone
    p.src = src, p.dst = dst, p.n = n, p.from_slots = from_slots, p.to_slots = to_slots, p.status = status, p.shift = shift;
    hipLaunchKernelGGL(slots::slots_copy_kernel, dim3((unsigned)blocks), dim3(slots::kThreads), 0,
                       static_cast<hipStream_t>(stream), p);
    return static_cast<int>(hipGetLastError());
}

int slots_free(const slots_cache* caches, int32_t num_caches, const int64_t* idx, int32_t n, int64_t slots, int32_t* status,
               void* stream) {
    if (n < 0 || n > 65535 || slots < 0) return WKV7_ERR_SHAPE;
    slots::Call p{};
    int64_t blocks;
    const int rc = slots::fill(p, caches, num_caches, false, slots, slots::kThreads * slots::kUnits, &blocks);
    if (rc != WKV7_OK) return rc;
    if (n == 0 || (blocks == 0 && !status)) return WKV7_OK;
    if (!idx) return WKV7_ERR_NULL;
    // a slot each where a launch holds them; without caches one workgroup looks at the indices alone
    p.groups = blocks == 0 ? 1 : (int32_t)std::min<int64_t>(n, std::max<int64_t>(1, slots::kMaxGrid / blocks));
    if (blocks == 0) blocks = 1;
    p.dst = idx, p.n = n, p.to_slots = slots, p.status = status;
    hipLaunchKernelGGL(slots::slots_free_kernel, dim3((unsigned)blocks, (unsigned)p.groups), dim3(slots::kThreads), 0,
                       static_cast<hipStream_t>(stream), p);
    return static_cast<int>(hipGetLastError());
}

int slots_compact(const slots_cache* caches, int32_t num_caches, const uint8_t* live, int64_t slots, int64_t* where,
                  int32_t* count, void* stream) {
    if (slots < 0 || slots > SLOTS_MAX_COMPACT) return WKV7_ERR_SHAPE;
    slots::Call p{};
    int64_t blocks;
    const int rc = slots::fill(p, caches, num_caches, false, slots, slots::kThreads * 4, &blocks);
    if (rc != WKV7_OK) return rc;
    if (slots > 0 && !live) return WKV7_ERR_NULL;
    if (blocks == 0) blocks = 1;  // the plan alone
    // few ranges: several workgroups share the moves of one
    p.groups = (int32_t)std::max<int64_t>(1, std::min<int64_t>(slots / 8, 4096 / blocks));
    if (blocks * p.groups > slots::kMaxGrid) return WKV7_ERR_SHAPE;
    p.live = live, p.where = where, p.count = count, p.to_slots = slots;
    hipLaunchKernelGGL(slots::slots_compact_kernel, dim3((unsigned)blocks, (unsigned)p.groups), dim3(slots::kThreads),
                       (size_t)(slots / 2 + 1) * 2 * sizeof(int32_t), static_cast<hipStream_t>(stream), p);
    return static_cast<int>(hipGetLastError());
}

}  // extern "C"
