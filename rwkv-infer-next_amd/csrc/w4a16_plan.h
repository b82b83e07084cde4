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

// How a product runs: by strips (16 rows by 16 nt columns to a workgroup, whose wavefronts share K, each reading A for itself) or by
// blocks (32 or 64 rows by 256, 128 or 64 columns, whose wavefronts share A in LDS).
enum Shape { kStrips, kBlock256, kBlock128, kBlock64 };
struct Plan {
    Shape shape;
    int mt, nt, waves;  // 16 mt rows; kStrips: 16 nt columns, K shared by `waves` wavefronts
    int64_t row_groups, strip_groups, grid;
};

inline int64_t groups(int32_t N, int columns) { return ((int64_t)N + columns - 1) / columns; }

// Blocks once there are more than 16 rows and enough of them for every CU, the widest first: A is then read once a block.  Below
// that, strips of 16 rows: more workgroups, and as many columns to each as leave three CUs in five one.  us, K = 4096, strips /
// blocks: 64 rows N = 65536 97 / 62, 16384 26.6 / 24.3, 4096 9.0 / 21.5; 256 rows N = 4096 24.1 / 22.6; 203 rows, K = 2560, N = 8191
// 30.8 / 25.2; but N = 10240 64 rows, 160 blocks, 14.3 / 16.5.  Strips of 64 / 32 / 16 columns: 64 rows, K = N = 2560 (160, 320, 640
// workgroups) 7.1 / 8.9 / 10.8; 24 rows, N = 4096 (128, 256, 512) 8.7 / 7.7 / 10.7; one row, N = 4096 (64, 128, 256) 8.0 / 6.2 / 5.4:
// the bound lies between 128 and 160 workgroups, where nothing else was measured.
inline Plan plan(int32_t M, int32_t N, int32_t K, int cus) {
    Plan p;
    const int rows = M <= 32 ? 32 : 64;
    const int64_t blocks = ((int64_t)M + rows - 1) / rows;
    p.shape = M <= 16                          ? kStrips
              : groups(N, 256) * blocks >= cus ? kBlock256
              : groups(N, 128) * blocks >= cus ? kBlock128
              : groups(N, 64) * blocks >= cus  ? kBlock64
                                               : kStrips;
    p.mt = p.shape == kStrips ? 1 : rows / 16;
    p.row_groups = ((int64_t)M + 16 * p.mt - 1) / (16 * p.mt);
    p.nt = 1;
    p.waves = 8;
    if (p.shape == kStrips) {
        for (p.nt = 4; p.nt > 1 && 5 * groups(N, kStrip * p.nt) * p.row_groups < 3 * cus;) p.nt /= 2;
        p.waves = (int)std::min<int64_t>(8, chunks(K));
    }
    p.strip_groups = groups(N, p.shape == kBlock256 ? 256 : p.shape == kBlock128 ? 128 : p.shape == kBlock64 ? 64 : kStrip * p.nt);
    // column groups are dealt to the eight XCDs in turn, the row groups of one of them following each other on one XCD
    p.grid = (p.strip_groups + 7) / 8 * 8 * p.row_groups;
    return p;
}

}  // namespace w4
