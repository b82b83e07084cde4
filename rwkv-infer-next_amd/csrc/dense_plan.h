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
enum Shape { k16x16, k16x64, k32x64, k64x64, k128x128, k128x256, kShapes };
struct Tile {
    int rows, columns, k_groups, threads;
};
constexpr Tile kTiles[kShapes] = {{16, 16, 8, 512}, {16, 64, 4, 512}, {32, 64, 4, 512},
                                  {64, 64, 4, 512}, {128, 128, 1, 256}, {128, 256, 1, 256}};
constexpr int kPanelSteps = 2;  // K is shared in panels of so many steps
constexpr int kPartPanels = 6;  // the least of a part's panels that a group has
// Weights of so many bytes that one row of tiles reads pass by the caches: 64 rows, 4096 x 16384, 31.2 us against 32.6, 16 rows 25.3
// against 26.8; but 13 MB, 2560 x 2560, 7.7 against 7.1.
constexpr size_t kStreamBytes = (size_t)64 << 20;

constexpr int64_t kShortTiles = (int64_t)9 << 18;  // tiles x K of 16 x 16, 64 bytes each: 150 MB of reads

struct Plan {
    Shape shape;
    int parts;    // of K, among workgroups; more than one are added by a second launch
    bool stream;  // weights by loads that leave nothing in the caches
    int64_t row_groups, strip_groups, grid;
    size_t workspace;
};

inline Plan plan_of(int32_t M, int32_t N, int32_t K, Shape shape, int64_t parts) {
    Plan p{};
    const int64_t panels = (steps(K) + kPanelSteps - 1) / kPanelSteps;
    p.shape = shape;
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({parts, panels / (kPartPanels * kTiles[shape].k_groups), 16}));
    p.row_groups = ((int64_t)M + kTiles[shape].rows - 1) / kTiles[shape].rows;
    p.strip_groups = ((int64_t)N + kTiles[shape].columns - 1) / kTiles[shape].columns;
    p.stream = kTiles[shape].columns == 64 && p.row_groups == 1 && weight_bytes(K, N) >= kStreamBytes;
    p.workspace = p.parts > 1 ? (size_t)p.parts * M * sums_row(N) * sizeof(float) : 0;
    p.grid = (p.row_groups * p.strip_groups * p.parts + 7) / 8 * 8;
    return p;
}

// Measured with weights cycled past the caches, bf16, us.
// Little work, of any number of rows: tiles of 16 x 16 while two workgroups a CU hold them all (and, of more than 16 rows, read little),
// in parts where there are fewer and K is long (one row, K = N = 4096 10.7 / 12.3 by 32 x 64 in parts; 16 rows, N = 8192 16.3 / 18.3 by
// 16 x 64; 64 rows, K = N = 768 4.3 / 5.5; 256 rows, K = 4096, N = 320 8.5 / 9.6; but 16 rows, K = 2560, N = 10240, 640 tiles, 16.2 /
// 14.2; 64 rows, K = 10240, N = 2560 36.9 / 20.0 by 64 x 64).
// Up to 64 rows: of the tiles of 64 columns the one of fewest rows of which every CU gets one at most (32 rows, K = 4096, N = 8192 17.8
// by 16 / 19.2 by 32; N = 16384 30.9 / 29.0; 64 rows 37.2 by 32 / 32.4 by 64); of long K, where A's and the weight's bytes count for
// more, as many rows as there are, in parts (K = 10240, N = 2560, 64 rows 20.0 by 64 / 26.6 by 16).
// More rows, short K, few tiles: the same (192 rows, K = N = 2560 13.3 / 17.1 by 128 x 128; but K = N = 4096 25.2 / 21.8).
// Else 128 x 128 or 128 x 256, and 64 x 64 for narrow products of long K (75 rows, K = 7872, N = 1003 19.4 / 21.7 by 128 x 128): up to 128
// rows or K = 1024 not 128 x 256 (K = 4096, N = 16384, 128 rows 38.0 / 41.1; K = 768, 512 rows 26.9 / 33.7), else the cheapest by what a
// step of one takes, alone on a CU or not, and what adding the parts does (K = N = 4096, 256 rows 23.2 / 25.7, 1000 rows 49.0 / 44.1;
// K = 5952, N = 1588, 2459 rows 97.7 whole, 65.6 in three parts; K = 10240, N = 2560, 512 rows 45.1 / 40.5; K = 2560, N = 10240, 2048
// rows 107 / 127; K = 4096, N = 16384, 2048 rows 253 / 240).
inline Plan plan(int32_t M, int32_t N, int32_t K, int cus) {
    const auto tiles = [&](Shape s) {
        return ((int64_t)M + kTiles[s].rows - 1) / kTiles[s].rows * (((int64_t)N + kTiles[s].columns - 1) / kTiles[s].columns);
    };
    if (tiles(k16x16) <= 2 * cus && (M <= 16 || tiles(k16x16) * K <= kShortTiles)) return plan_of(M, N, K, k16x16, 2 * cus / tiles(k16x16));
    if (M <= 16) return plan_of(M, N, K, k16x64, cus / tiles(k16x64));
    if (M <= 64 && K > 4096) {
        const Shape s = M <= 32 ? k32x64 : k64x64;
        return plan_of(M, N, K, s, cus / tiles(s));
    }
    for (Shape s : {k16x64, k32x64, k64x64})
        if (tiles(s) <= cus && (M <= 64 || K <= 2560 || (s == k16x64 && K <= 4096))) return plan_of(M, N, K, s, cus / tiles(s));
    if (M <= 64) return plan_of(M, N, K, M <= 32 ? k32x64 : k64x64, 1);
    Plan best{};
    double least = 0;
    for (Shape s : {k128x256, k128x128, k64x64})
        for (int per_cu : {1, 2}) {  // parts for one or two workgroups a CU
            const Plan p = plan_of(M, N, K, s, per_cu * cus / tiles(s));
            const int64_t rounds = (tiles(s) * p.parts + cus - 1) / cus;
            const double step = s == k128x256 ? (rounds > 1 ? 0.48 : 0.53) : s == k128x128 ? (rounds > 1 ? 0.255 : 0.36) : 0.163;
            const double us = rounds * (steps(K) * step / p.parts + 3) + (p.parts > 1 ? 3 + 1e-6 * p.parts * M * N : 0);
            if (least == 0 || us < least || ((M <= 128 || K <= 1024) && s == k128x128 && per_cu == 1)) best = p, least = us;
        }
    return best;
}

}  // namespace dense
