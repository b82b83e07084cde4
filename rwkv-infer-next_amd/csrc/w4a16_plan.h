// w4a16_plan.h -- the packed layout of a 4-bit weight, and in what shape a product runs.  Host arithmetic on sizes alone.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace w4 {

constexpr int kStrip = 16;        // columns of an MFMA tile: the unit of the layout along N
constexpr int kChunk = 128;       // rows of a weight that one 16-byte load per lane covers (four MFMA steps of 32)
constexpr int kBlockBytes = 1024; // of a (strip, chunk)

// Scales a chunk and column: one where a group holds whole chunks, two where it holds whole half chunks, else four.
inline int scales_per_chunk(int group_k) { return group_k % 128 == 0 ? 1 : group_k % 64 == 0 ? 2 : 4; }

inline int64_t strips(int32_t N) { return ((int64_t)N + kStrip - 1) / kStrip; }
inline int64_t chunks(int32_t K) { return ((int64_t)K + kChunk - 1) / kChunk; }

inline size_t weight_bytes(int32_t K, int32_t N) { return (size_t)(strips(N) * chunks(K)) * kBlockBytes; }
inline size_t scale_bytes(int32_t K, int32_t N, int32_t group_k) {
    return (size_t)(strips(N) * chunks(K)) * kStrip * scales_per_chunk(group_k) * 2;
}

// How a product runs: a workgroup computes 16 mt rows by 16 nt columns, its `waves` wavefronts share K.
struct Plan {
    int mt, nt, waves;
    int64_t row_groups, strip_groups, grid;
};

inline Plan plan(int32_t M, int32_t N, int32_t K, int cus) {
    Plan p;
    p.mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    p.row_groups = ((int64_t)M + 16 * p.mt - 1) / (16 * p.mt);
    p.nt = 4;
    while (p.nt > 1 && (strips(N) + p.nt - 1) / p.nt * p.row_groups < 2 * cus) p.nt /= 2;
    p.strip_groups = (strips(N) + p.nt - 1) / p.nt;
    p.waves = (int)std::min<int64_t>(p.mt == 4 && p.nt == 4 ? 4 : 8, chunks(K));
    // strip groups are dealt to the eight XCDs in turn, the row groups of one of them following each other on one XCD
    p.grid = (p.strip_groups + 7) / 8 * 8 * p.row_groups;
    return p;
}

}  // namespace w4
