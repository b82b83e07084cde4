// dense_tile.hip -- products of many rows (include/dense.h): tiles of a workgroup in registers, on the matrix cores.
//
// A wavefront has 16 MT rows by 16 NT columns of sums, a workgroup WM x WN wavefronts.  A comes through LDS, a panel of 64 columns at a
// time, three panels in turn; the weight, packed in operand order, goes from memory to registers.  Within a panel the operands of
// a row tile are read for the step after as soon as its products of this step are out, so that neither LDS nor the barrier between
// panels is waited for.  Products are taken as out^T = w^T a^T: a lane then holds four columns of a row.
#include "dense_device.h"

namespace dense {
namespace {

constexpr int kPanelSteps = 2;

template <int AT, int MT, int NT, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2) void dense_tile_kernel(const Params p) {
    constexpr int kThreads = 64 * WM * WN, kTiles = MT * WM;  // row tiles of a workgroup
    constexpr int kPanel = kTiles * kPanelSteps * 1024;       // bytes
    constexpr int kAhead = 4;                                 // row tiles whose operands are read ahead
    constexpr int kPieces = kPanel / 16 / kThreads;
    static_assert(kPieces * 16 * kThreads == kPanel, "");
    __shared__ __attribute__((aligned(16))) char lds[3 * kPanel];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM, col = lane & 15, quad = lane >> 4;
    // Workgroup b runs on XCD b % 8.  Each XCD has an equal share of the tiles, in an order in which 32 that follow each other are
    // eight row groups by four column groups.
    const uint32_t tiles = (uint32_t)p.row_groups * (uint32_t)p.strip_groups, units = tiles * (uint32_t)p.parts;
    const uint32_t share = (units + 7) / 8, unit = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= share || unit >= units) return;
    const int part = (int)(unit / tiles);
    const uint32_t tile = unit % tiles, band = tile / (4 * (uint32_t)p.row_groups), in = tile % (4 * (uint32_t)p.row_groups);
    const uint32_t width = min(4u, (uint32_t)p.strip_groups - 4 * band);
    const int row0 = (int)(in / width) * (16 * kTiles);
    const int strip0 = (int)(((4 * band + in % width) * WN + wn) * NT);
    // this part's steps
    const int panels = (p.steps + kPanelSteps - 1) / kPanelSteps;
    const int first = (int)((int64_t)panels * part / p.parts), end = (int)((int64_t)panels * (part + 1) / p.parts);
    const int steps = min(p.steps, end * kPanelSteps) - first * kPanelSteps;

    const uint8_t* wp[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)  // past the last strip: that strip again, not stored
        wp[t] = wkv7::uniform_ptr(p.weight + ((int64_t)min(strip0 + t, p.strips - 1) * p.steps + first * kPanelSteps) * kBlockBytes);
    // A's pieces of a thread: eight lanes take a row's 128 bytes.  Within a tile and step lane l's operand lies at 16 l, but for its
    // row's bits 2 and 3, changed by the piece's number, so that neither writes nor reads meet a bank twice.
    const int piece = tid & 7;
    const char* ap[kPieces];
    uint32_t at_a[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {  // past the last row: it again, not stored
        const int base = min(row0 + kThreads / 8 * i, p.M - 1);
        ap[i] = wkv7::uniform_ptr(reinterpret_cast<const char*>(p.a + base * p.a_row_stride) + first * (kPanelSteps * 64));
        at_a[i] = (uint32_t)min(tid >> 3, p.M - 1 - base) * (uint32_t)(p.a_row_stride * 2);  // at most 63 rows: below 2^31
    }
    const int row = tid >> 3;  // kThreads / 8 is a multiple of 16
    char* const to = lds + ((row >> 4) * kPanelSteps + (piece >> 2)) * 1024 + (((piece & 3) * 16 + (row & 15)) ^ (piece & 3) << 2) * 16;
    const char* const from = lds + wm * (MT * kPanelSteps * 1024) + (lane ^ quad << 2) * 16;

    u4 next[kPieces];
    const auto load_a = [&](int panel) {  // past the last step: the last one again, its products are not taken
        const uint32_t at = (uint32_t)min(panel * kPanelSteps + (piece >> 2), steps - 1) * 64 + (piece & 3) * 16;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) next[i] = *reinterpret_cast<const u4*>(ap[i] + (at_a[i] + at));
    };
    const auto store_a = [&](int slot) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            *reinterpret_cast<u4*>(to + slot * kPanel + i * (kThreads / 128 * kPanelSteps * 1024)) = next[i];
    };
    const auto load_w = [&](int step, u4* w) {
        const int64_t at = (int64_t)min(step, steps - 1) * kBlockBytes;
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = *reinterpret_cast<const u4*>(wp[t] + at + (uint32_t)lane * 16);
    };
    u4 a[kAhead], w[3][NT];
    const auto read = [&](int slot, int step, int i) {
        a[i % kAhead] = *reinterpret_cast<const u4*>(from + slot * kPanel + (i * kPanelSteps + step) * 1024);
    };
    f4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};

    load_a(0);
    load_w(0, w[0]);
    load_w(1, w[1]);
    store_a(0);
    load_a(1);
    store_a(1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(0, 0, i);
    // The panel in slot `now`, whose first step has number s and its weights in w[J]; the next panel is in LDS already.
    const auto panel = [&](int s, auto now_, auto J_, bool both) {
        constexpr int now = decltype(now_)::value, J = decltype(J_)::value;
        load_a(s / kPanelSteps + 2);
        wkv7::unroll<kPanelSteps>([&](auto q_) {
            constexpr int q = decltype(q_)::value, mine = (J + q) % 3, later = (J + q + 2) % 3;
            if (q == 0 || both) {
                load_w(s + q + 2, w[later]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[i][t] = mfma<AT>(w[mine][t], a[i % kAhead], acc[i][t]);
                    const int ahead = (i + kAhead) % MT;
                    if (i + kAhead < MT) read(now, q, ahead); else if (q == 0) read(now, 1, ahead); else read((now + 1) % 3, 0, ahead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        });
        store_a((now + 2) % 3);
        __syncthreads();
    };
    using std::integral_constant;
    int s = 0;
    for (; s + 6 <= steps; s += 6) {
        panel(s, integral_constant<int, 0>{}, integral_constant<int, 0>{}, true);
        panel(s + 2, integral_constant<int, 1>{}, integral_constant<int, 2>{}, true);
        panel(s + 4, integral_constant<int, 2>{}, integral_constant<int, 1>{}, true);
    }
    if (s < steps) panel(s, integral_constant<int, 0>{}, integral_constant<int, 0>{}, s + 1 < steps);
    if (s + 2 < steps) panel(s + 2, integral_constant<int, 1>{}, integral_constant<int, 2>{}, s + 3 < steps);
    if (s + 4 < steps) panel(s + 4, integral_constant<int, 2>{}, integral_constant<int, 1>{}, false);

    // Through LDS, kAtOnce row tiles of a wavefront at a time: rows are then stored 16 NT columns in a piece.
    constexpr int kAtOnce = 2, kPitch = 16 * NT + 4;  // floats: a tile's writes meet no bank twice
    static_assert(kAtOnce * 16 * kPitch * 4 * WM * WN <= (int)sizeof(lds) && MT % kAtOnce == 0, "");
    float* const mine = reinterpret_cast<float*>(lds) + wave * (kAtOnce * 16 * kPitch);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int g = 0; g < MT / kAtOnce; ++g) {
        wkv7::wave_lds_sync();
#pragma unroll
        for (int i = 0; i < MT; ++i)
            if (i / kAtOnce == g)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    *reinterpret_cast<f4*>(mine + (i % kAtOnce * 16 + col) * kPitch + 16 * t + 4 * quad) = acc[i][t];
        wkv7::wave_lds_sync();
#pragma unroll 1
        for (int e = lane; e < kAtOnce * 64 * NT; e += 64) {
            const int r = e / (4 * NT), c = e % (4 * NT) * 4;
            const int64_t m = row0 + 16 * (wm * MT + g * kAtOnce) + r, n = (int64_t)strip0 * kStrip + c;
            const f4 x = *reinterpret_cast<const f4*>(mine + r * kPitch + c);
            if (m < p.M) {
                if (p.parts == 1)
                    finish4(p, m, n, x);
                else if (n < p.N)
                    *reinterpret_cast<f4*>(p.sums + (part * (int64_t)p.M + m) * sums_row(p.N) + n) = x;
            }
        }
    }
}

// The parts of a split product, added in their order, four columns a thread.
__global__ __launch_bounds__(256) void dense_join_kernel(const Params p) {
    const int64_t pitch = sums_row(p.N), fours = pitch / 4, all = p.M * fours;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (int64_t)gridDim.x * 256) {
        const float* const at = p.sums + e * 4;
        f4 x = *reinterpret_cast<const f4*>(at);
        for (int i = 1; i < p.parts; ++i) x += *reinterpret_cast<const f4*>(at + (int64_t)i * p.M * pitch);
        finish4(p, e / fours, e % fours * 4, x);
    }
}

template <int AT, int MT, int NT, int WM, int WN>
void launch(const Params& p, int64_t grid, hipStream_t s) {
    hipLaunchKernelGGL((dense_tile_kernel<AT, MT, NT, WM, WN>), dim3((unsigned)grid), dim3(64 * WM * WN), 0, s, p);
}
template <int AT>
void launch_shape(const Params& p, const Plan& pl, hipStream_t s) {
    if (pl.shape == kTile256)
        launch<AT, 8, 4, 2, 4>(p, pl.grid, s);
    else if (pl.shape == kTile128x256)
        launch<AT, 8, 4, 1, 4>(p, pl.grid, s);
    else
        launch<AT, 4, 4, 2, 2>(p, pl.grid, s);
}

}  // namespace

hipError_t launch_tiles(const Params& p, const Plan& pl, int32_t dtype, hipStream_t stream) {
    if (dtype == DENSE_BF16)
        launch_shape<DENSE_BF16>(p, pl, stream);
    else
        launch_shape<DENSE_F16>(p, pl, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    const int64_t blocks = (p.M * (sums_row(p.N) / 4) + 255) / 256;
    hipLaunchKernelGGL(dense_join_kernel, dim3((unsigned)std::min<int64_t>(blocks, 4096)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace dense
