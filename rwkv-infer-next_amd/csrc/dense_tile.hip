// dense_tile.hip -- the products of include/dense.h: a workgroup's tile of the result in registers, on the matrix cores.
//
// A wavefront has 16 MT rows by 16 NT columns of sums; WN wavefronts side by side share A, and WK groups of them share K.  A comes
// through LDS, a panel of 64 columns at a time, three panels in turn; the weight, packed in operand order, goes from memory to
// registers, D - 1 steps ahead.  The operands of a row tile are read while those before it multiply, over the barrier between
// panels, so that neither LDS nor the barrier is waited for.  Products are taken as out^T = w^T a^T: a lane then has four columns
// of a row.  Measured: 4096 rows, 4096 x 16384, 443 to 476 us by 128 x 256 (two workgroups of four wavefronts a CU; by 256 x 256, eight
// wavefronts, 600), 1.16 to 1.24 PFLOP/s where a large library product reaches 1.22; the matrix cores work 58 % of the time.  64 rows
// 31 us, 4.4 TB/s of weight: bound by memory, and by the first and last of 16 panels that nothing covers; a deeper D changed nothing.
// 500 rows, 10240 x 2560, 33 to 36 us and 7 for adding the parts: one wavefront a SIMD (27 %).  A width that four does not divide stores a column a
// lane: 22 us against 16 (1175 rows, K = 64, N = 5665, 5664).  Which tile a product takes, and the measured sides of the rules: dense_plan.h.
#include "dense_device.h"

namespace dense {
namespace {

template <int AT, int MT, int NT, int WN, int WK, int D, bool STREAM>
__global__ __launch_bounds__(64 * WN * WK, 2) void dense_tile_kernel(const Params p) {
    constexpr int kThreads = 64 * WN;                  // of a group that shares K with others
    constexpr int kPanel = MT * kPanelSteps * 1024;    // bytes
    constexpr int kAhead = MT < 4 ? MT : 4;            // row tiles whose operands are read ahead
    constexpr int kPieces = kPanel / 16 / kThreads;
    constexpr int kAtOnce = MT < 2 ? MT : 2, kPitch = 16 * NT + 4;  // the epilogue's row tiles and floats between rows
    constexpr int kGroup = MT * NT * 1024 * WN;        // sums of a group
    constexpr int kEpilogue = kAtOnce * 16 * kPitch * 4 * WN, kSums = kEpilogue > (WK - 1) * kGroup ? kEpilogue : (WK - 1) * kGroup;
    static_assert(kPieces * 16 * kThreads == kPanel && MT % kAtOnce == 0 && MT % kAhead == 0 && 6 % D == 0, "");
    __shared__ __attribute__((aligned(16))) char lds_all[3 * kPanel * WK > kSums ? 3 * kPanel * WK : kSums];
    const int tid = threadIdx.x % kThreads, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
    char* const lds = lds_all + wk * (3 * kPanel);
    const int col = lane & 15, quad = lane >> 4;
    // Workgroup b runs on XCD b % 8.  Each XCD has an equal share of the tiles, in an order in which 32 that follow each other are
    // eight row groups by four column groups.
    const uint32_t tiles = (uint32_t)p.row_groups * (uint32_t)p.strip_groups, units = tiles * (uint32_t)p.parts;
    const uint32_t share = (units + 7) / 8, unit = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= share || unit >= units) return;
    const int part = (int)(unit / tiles);
    const uint32_t tile = unit % tiles, band = tile / (4 * (uint32_t)p.row_groups), in = tile % (4 * (uint32_t)p.row_groups);
    const uint32_t width = min(4u, (uint32_t)p.strip_groups - 4 * band);
    const int row0 = (int)(in / width) * (16 * MT);
    const int strip0 = (int)(((4 * band + in % width) * WN + wave) * NT);
    // This part's panels, as many as any other's but for the last ones, which have fewer or none.
    const int panels = (p.steps + kPanelSteps - 1) / kPanelSteps, share_k = (panels + p.parts * WK - 1) / (p.parts * WK);
    const int first = min((part * WK + wk) * share_k, panels);
    const int steps = min(p.steps - first * kPanelSteps, share_k * kPanelSteps), last = max(steps, 1) - 1;
    const int from_step = min(first * kPanelSteps, p.steps - 1);  // inside the weight and A also where there are none

    const uint8_t* wp[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)  // past the last strip: that strip again, not stored
        wp[t] = wkv7::uniform_ptr(p.weight + ((int64_t)min(strip0 + t, p.strips - 1) * p.steps + from_step) * kBlockBytes);
    // A's pieces of a thread: eight lanes take a row's 128 bytes.  Within a tile and step lane l's operand lies at 16 l, but for its
    // row's lower three bits, changed by the number of its piece of the 128 bytes, so that neither writes nor reads meet a bank twice.
    const int piece = tid & 7;
    const char* ap[kPieces];
    uint32_t at_a[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {  // past the last row: it again, not stored
        const int base = min(row0 + kThreads / 8 * i, p.M - 1);
        ap[i] = wkv7::uniform_ptr(reinterpret_cast<const char*>(p.a + base * p.a_row_stride) + (int64_t)from_step * 64);
        at_a[i] = (uint32_t)min(tid >> 3, p.M - 1 - base) * (uint32_t)(p.a_row_stride * 2);  // at most 63 rows: below 2^31
    }
    const int row = tid >> 3;
    char* const to = lds + ((row >> 4) * kPanelSteps + (piece >> 2)) * 1024 + (((piece & 3) * 16 + (row & 15)) ^ piece) * 16;
    const int lane_at[kPanelSteps] = {(lane ^ quad) * 16, (lane ^ quad ^ 4) * 16};

    u4 next[kPieces];
    const auto load_a = [&](int panel) {  // past the last step: the last one again, its products are not taken
        const uint32_t at = (uint32_t)min(panel * kPanelSteps + (piece >> 2), last) * 64 + (piece & 3) * 16;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) next[i] = *reinterpret_cast<const u4*>(ap[i] + (at_a[i] + at));
    };
    const auto store_a = [&](int slot) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
            *reinterpret_cast<u4*>(to + slot * kPanel + i * (kThreads / 8) / 16 * (kPanelSteps * 1024) + i * (kThreads / 8) % 16 * 16) =
                next[i];
    };
    const auto load_w = [&](int step, u4* w) {
        const int64_t at = (int64_t)min(step, last) * kBlockBytes;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const u4* const x = reinterpret_cast<const u4*>(wp[t] + at + (uint32_t)lane * 16);
            w[t] = STREAM ? __builtin_nontemporal_load(x) : *x;
        }
    };
    u4 a[kAhead], w[D][NT];
    const auto read = [&](int slot, int step, int i) {
        a[i % kAhead] = *reinterpret_cast<const u4*>(lds + slot * kPanel + (i * kPanelSteps + step) * 1024 + lane_at[step]);
    };
    f4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[i][t] = f4{0.f, 0.f, 0.f, 0.f};

    load_a(0);
#pragma unroll
    for (int d = 0; d < D - 1; ++d) load_w(d, w[d]);
    store_a(0);
    load_a(1);
    store_a(1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAhead; ++i) read(0, 0, i);
    // The panel in slot `now`, whose first step has number s and its weights in w[J]; the next panel is in LDS already.
    const auto panel = [&](int s, auto now_, auto J_, auto all) {
        constexpr int now = decltype(now_)::value, J = decltype(J_)::value;
        load_a(s / kPanelSteps + 2);
        wkv7::unroll<kPanelSteps>([&](auto q_) {
            constexpr int q = decltype(q_)::value, mine = (J + q) % D, later = (J + q + D - 1) % D;
            if (decltype(all)::value || s + q < steps) {
                load_w(s + q + D - 1, w[later]);
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
    const auto three = [&](int s, int end, auto all) {
        panel(s, integral_constant<int, 0>{}, integral_constant<int, 0>{}, all);
        if (s + 2 < end) panel(s + 2, integral_constant<int, 1>{}, integral_constant<int, 2 % D>{}, all);
        if (s + 4 < end) panel(s + 4, integral_constant<int, 2>{}, integral_constant<int, 4 % D>{}, all);
    };
    // Every wavefront comes to every barrier; steps that not all of them have are asked for one by one.
    const int most = share_k * kPanelSteps, all = min(p.steps - min((part * WK + WK - 1) * share_k, panels) * kPanelSteps, most);
    int s = 0;
    for (; s + 6 <= all; s += 6) three(s, s + 6, std::true_type{});
    for (; s < most; s += 6) three(s, most, std::false_type{});

    if constexpr (WK > 1) {  // the workgroup's parts of K, added in their order
        char* const sums = lds_all + wave * (MT * NT * 1024) + lane * 16;
        if (wk > 0)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t) *reinterpret_cast<f4*>(sums + (wk - 1) * kGroup + (i * NT + t) * 1024) = acc[i][t];
        __syncthreads();
        if (wk == 0)
            for (int g = 0; g < WK - 1; ++g)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int t = 0; t < NT; ++t) acc[i][t] += *reinterpret_cast<const f4*>(sums + g * kGroup + (i * NT + t) * 1024);
        __syncthreads();
        if (wk > 0) return;
    }
    // Through LDS, kAtOnce row tiles of a wavefront at a time: rows are then stored 16 NT columns in a piece.  (Writes of a tile, four
    // floats past a multiple of 16 from row to row, meet no bank twice.)
    float* const mine = reinterpret_cast<float*>(lds_all) + wave * (kAtOnce * 16 * kPitch);
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
        if (p.parts == 1 && !p.fours) {  // a column a lane
#pragma unroll 4
            for (int e = lane; e < kAtOnce * 256 * NT; e += 64) {
                const int r = e / (16 * NT), c = e % (16 * NT);
                const int64_t m = row0 + 16 * g * kAtOnce + r, n = (int64_t)strip0 * kStrip + c;
                if (m < p.M && n < p.N) finish(p, m, n, mine[r * kPitch + c]);
            }
            continue;
        }
#pragma unroll 2
        for (int e = lane; e < kAtOnce * 64 * NT; e += 64) {
            const int r = e / (4 * NT), c = e % (4 * NT) * 4;
            const int64_t m = row0 + 16 * g * kAtOnce + r, n = (int64_t)strip0 * kStrip + c;
            const f4 x = *reinterpret_cast<const f4*>(mine + r * kPitch + c);
            if (m < p.M && n < p.N) {
                if (p.parts == 1)
                    finish4(p, m, n, x);
                else
                    *reinterpret_cast<f4*>(p.sums + (part * (int64_t)p.M + m) * sums_row(p.N) + n) = x;
            }
        }
    }
}

// The parts of a split product, added in their order, four columns a thread, or one.
__global__ __launch_bounds__(256) void dense_join_kernel(const Params p) {
    const int64_t pitch = sums_row(p.N), fours = pitch / 4, all = p.M * fours;
    if (!p.fours) {
        for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < (int64_t)p.M * p.N; e += (int64_t)gridDim.x * 256) {
            const int64_t m = e / p.N, n = e % p.N;
            float x = 0.f;
#pragma unroll 4
            for (int i = 0; i < p.parts; ++i) x += p.sums[(i * (int64_t)p.M + m) * pitch + n];
            finish(p, m, n, x);
        }
        return;
    }
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (int64_t)gridDim.x * 256) {
        const float* const at = p.sums + e * 4;
        f4 x = *reinterpret_cast<const f4*>(at);
#pragma unroll 4
        for (int i = 1; i < p.parts; ++i) x += *reinterpret_cast<const f4*>(at + (int64_t)i * p.M * pitch);
        finish4(p, e / fours, e % fours * 4, x);
    }
}

template <int AT, Shape S, int MT, int NT, int WN, int D>
void launch(const Params& p, const Plan& pl, hipStream_t s) {
    constexpr Tile t = kTiles[S];
    static_assert(t.rows == 16 * MT && t.columns == 16 * NT * WN && t.threads == 64 * WN * t.k_groups, "");
    const dim3 grid((unsigned)pl.grid), block(t.threads);
    if constexpr (t.columns == 64)
        if (pl.stream) {
            hipLaunchKernelGGL((dense_tile_kernel<AT, MT, NT, WN, t.k_groups, D, true>), grid, block, 0, s, p);
            return;
        }
    hipLaunchKernelGGL((dense_tile_kernel<AT, MT, NT, WN, t.k_groups, D, false>), grid, block, 0, s, p);
}
template <int AT>
void launch_shape(const Params& p, const Plan& pl, hipStream_t s) {
    switch (pl.shape) {
        case k16x16: return launch<AT, k16x16, 1, 1, 1, 6>(p, pl, s);
        case k16x64: return launch<AT, k16x64, 1, 2, 2, 6>(p, pl, s);
        case k32x64: return launch<AT, k32x64, 2, 2, 2, 6>(p, pl, s);
        case k64x64: return launch<AT, k64x64, 4, 2, 2, 6>(p, pl, s);
        case k128x128: return launch<AT, k128x128, 8, 2, 4, 3>(p, pl, s);
        default: return launch<AT, k128x256, 8, 4, 4, 3>(p, pl, s);
    }
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
