// dense_plan.h -- the packed layout of a 16-bit weight, and in what shape a product runs.  Host arithmetic on sizes alone.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace dense {

constexpr int kStrip = 16;         // columns of an MFMA tile: the unit of the layout along N
constexpr int kStep = 32;          // rows of a weight that an MFMA step takes
constexpr int kBlockBytes = 1024;  // of a (strip, step): 16 bytes a lane, in operand order

inline int64_t strips(int32_t N) { return ((int64_t)N + kStrip - 1) / kStrip; }
inline int64_t steps(int32_t K) { return K / kStep; }
inline size_t weight_bytes(int32_t K, int32_t N) { return (size_t)(strips(N) * steps(K)) * kBlockBytes; }

constexpr int64_t sums_row(int32_t N) { return ((int64_t)N + 3) / 4 * 4; }  // floats of a row of a split product's sums

// How a product runs: by strips (16 rows by 16 nt columns to a workgroup, whose wavefronts share K) or by tiles.
enum Shape { kStrips, kTile256, kTile128x256, kTile128 };
struct Plan {
    Shape shape;
    int nt, waves, parts;
    int64_t row_groups, strip_groups, grid;
    size_t workspace;
};

inline Plan plan(int32_t M, int32_t N, int32_t K, int cus, int shape = -1, int parts = 0) {
    Plan p{};
    p.shape = shape >= 0 ? (Shape)shape : M <= 64 ? kStrips : kTile256;
    p.parts = 1;
    if (p.shape != kStrips) {
        const int rows = p.shape == kTile256 ? 256 : 128, columns = p.shape == kTile128 ? 128 : 256;
        p.row_groups = ((int64_t)M + rows - 1) / rows;
        p.strip_groups = ((int64_t)N + columns - 1) / columns;
        if (parts) p.parts = parts;
        if (p.parts > 1) p.workspace = (size_t)p.parts * M * sums_row(N) * sizeof(float);
        p.grid = (p.row_groups * p.strip_groups * p.parts + 7) / 8 * 8;
        return p;
    }
    p.row_groups = ((int64_t)M + 15) / 16;
    for (p.nt = 4; p.nt > 1 && 5 * ((strips(N) + p.nt - 1) / p.nt) * p.row_groups < 3 * cus;) p.nt /= 2;
    p.waves = (int)std::min<int64_t>(8, (steps(K) + 3) / 4);
    p.strip_groups = (strips(N) + p.nt - 1) / p.nt;
    // column groups are dealt to the eight XCDs in turn, the row groups of one of them following each other on one XCD
    p.grid = (p.strip_groups + 7) / 8 * 8 * p.row_groups;
    return p;
}

}  // namespace dense
