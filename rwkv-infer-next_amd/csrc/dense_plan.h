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

// The tile of a workgroup, rows x columns, and among how many groups of wavefronts it shares K.
enum Shape { k16x16, k32x16, k64x16, k16x64, k32x64, k64x64, k128x128, k128x256, kShapes };
struct Tile {
    int rows, columns, k_groups, threads;
};
constexpr Tile kTiles[kShapes] = {{16, 16, 8, 512}, {32, 16, 8, 512}, {64, 16, 6, 384}, {16, 64, 4, 512},
                                  {32, 64, 4, 512}, {64, 64, 4, 512}, {128, 128, 1, 256}, {128, 256, 1, 256}};
constexpr int kPanelSteps = 2;  // K is shared in panels of so many steps

struct Plan {
    Shape shape;
    int parts;  // of K, among workgroups; more than one are added by a second launch
    int64_t row_groups, strip_groups, grid;
    size_t workspace;
};

inline Plan plan_of(int32_t M, int32_t N, int32_t K, Shape shape, int64_t parts) {
    Plan p{};
    const int64_t panels = (steps(K) + kPanelSteps - 1) / kPanelSteps;
    p.shape = shape;
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({parts, panels / (4 * kTiles[shape].k_groups), 16}));
    p.row_groups = ((int64_t)M + kTiles[shape].rows - 1) / kTiles[shape].rows;
    p.strip_groups = ((int64_t)N + kTiles[shape].columns - 1) / kTiles[shape].columns;
    p.workspace = p.parts > 1 ? (size_t)p.parts * M * sums_row(N) * sizeof(float) : 0;
    p.grid = (p.row_groups * p.strip_groups * p.parts + 7) / 8 * 8;
    return p;
}

// Measured with weights cycled past the caches, bf16, us.
// Up to 16 rows bytes count: columns of 16 while two workgroups a CU hold them all (one row, K = N = 4096 9.5 against 10.4 by columns of 64
// in four parts; N = 8192 15.0 / 16.9), else of 64 (N = 16384 26 / 36 by 32 x 16).
// Up to 64 rows: columns of 16 while every CU gets one tile at most, their rows 32 where that holds, else 64 (K = N = 4096, 32 rows 10.3 /
// 13.3 by 32 x 64 in four parts; 64 rows 12.8 / 15.5, by 32 x 16 18.7; 64 rows, N = 6144 22.3 / 19.3); else of 64, K in as many parts as
// CUs are left for (N = 16384, 64 rows 33 / 37 by 128 x 256 in three parts).
// More rows: the same while tiles are that few and, for those of 64, K is short (192 rows, K = N = 2560 13.7 / 17.3 by 128 x 128; K = 4096
// 25.7 / 21.7), else the cheaper of 128 x 128 and 128 x 256 by what a step of one takes and what adding the parts does (K = N = 4096, 256 rows
// 23.1 / 25.5, 1000 rows 49 / 44.6; K = 10240, N = 2560, 500 rows 45 / 41).
inline Plan plan(int32_t M, int32_t N, int32_t K, int cus) {
    const auto tiles = [&](Shape s) {
        return ((int64_t)M + kTiles[s].rows - 1) / kTiles[s].rows * (((int64_t)N + kTiles[s].columns - 1) / kTiles[s].columns);
    };
    if (M <= 16) return plan_of(M, N, K, tiles(k16x16) <= 2 * cus ? k16x16 : k16x64, 1);
    for (Shape s : {k32x16, k64x16})
        if (tiles(s) <= cus) return plan_of(M, N, K, s, 1);
    if (M <= 64) {
        const Shape s = M <= 32 ? k32x64 : k64x64;
        return plan_of(M, N, K, s, cus / tiles(s));
    }
    if (K <= 2560)
        for (Shape s : {k32x64, k64x64})
            if (tiles(s) <= cus) return plan_of(M, N, K, s, 1);
    Plan best{};
    double least = 0;
    for (Shape s : {k128x128, k128x256}) {
        const Plan p = plan_of(M, N, K, s, cus / tiles(s));
        const int64_t rounds = (tiles(s) * p.parts + cus - 1) / cus;
        const double us = (double)rounds * steps(K) / p.parts * (s == k128x128 ? 0.36 : 0.45) +
                          (p.parts > 1 ? 3 + 8e-6 * p.parts * M * N / 6 : 0);
        if (s == k128x128 || us < least) best = p, least = us;
    }
    return best;
}

}  // namespace dense
