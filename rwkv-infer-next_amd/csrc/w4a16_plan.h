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

// How a product runs: by strips (a workgroup's wavefronts share K, each reading A for itself) or by blocks of 256, 128 or 64
// columns (they share A in LDS).
enum Shape { kStrips, kBlock256, kBlock128, kBlock64 };
struct Plan {
    Shape shape;
    int mt, nt, waves;  // 16 mt rows; kStrips: 16 nt columns, shared by `waves` wavefronts
    int64_t row_groups, strip_groups, grid;
};

inline int64_t groups(int32_t N, int columns) { return ((int64_t)N + columns - 1) / columns; }

// Up to 16 rows strips, as wide as leaves every CU two workgroups: A is little, and 16 columns read it as fast as 256 (4096 x
// 65536, one row: 28.5 us, blocks of 256 columns 36).  From 17 rows on A's share of the reading decides: the widest blocks of
// which every CU gets one, and the narrowest while every second CU does (64 rows, K = 4096, strips / blocks: N = 65536 93 / 62 us,
// 16384 40 / 24.3; K = 2560, N = 10240 34 / 15.6; but N = 4096, 64 blocks, 19.1 / 21.5).
inline Plan plan(int32_t M, int32_t N, int32_t K, int cus) {
    Plan p;
    p.mt = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    p.row_groups = ((int64_t)M + 16 * p.mt - 1) / (16 * p.mt);
    p.nt = 1;
    p.waves = 8;
    p.shape = M <= 16                                          ? kStrips
              : groups(N, 256) * p.row_groups >= cus           ? kBlock256
              : groups(N, 128) * p.row_groups >= cus           ? kBlock128
              : 2 * groups(N, 64) * p.row_groups >= cus        ? kBlock64
                                                               : kStrips;
    if (p.shape == kStrips) {
        if (M <= 16)
            for (p.nt = 4; p.nt > 1 && groups(N, kStrip * p.nt) < 2 * cus;) p.nt /= 2;
        p.waves = (int)std::min<int64_t>(8, chunks(K));
    }
    p.strip_groups = groups(N, p.shape == kBlock256 ? 256 : p.shape == kBlock128 ? 128 : p.shape == kBlock64 ? 64 : kStrip * p.nt);
    // column groups are dealt to the eight XCDs in turn, the row groups of one of them following each other on one XCD
    p.grid = (p.strip_groups + 7) / 8 * 8 * p.row_groups;
    return p;
}

}  // namespace w4
