// delta_capi.hip -- the C entry points of include/delta.h: checks of arguments, the choice between the kernels, the launches.
// Everything is decided from sizes and flags that the host knows.
#include "delta_device.h"
#include "wkv7_launch.h"

namespace delta {
namespace {

constexpr int kClashRows = 1024;

struct Plan {
    bool tokens, chunks;
    int32_t token_len;
    int64_t slots, rows;  // of the workspace; that can run by chunks
    size_t bytes;
};
Plan make_plan(const delta_args* a) {
    Plan pl{};
    pl.token_len = a->token_len >= 0 ? a->token_len : DELTA_TOKEN_LEN;
    const int64_t longest = a->cu_seqlens ? a->total_tokens : a->T;
    pl.chunks = !a->snapshots && longest > pl.token_len;
    pl.tokens = !pl.chunks || a->cu_seqlens;
    if (pl.chunks) {
        pl.slots = delta::chunk_slots(a->num_seqs, a->T, a->total_tokens, pl.token_len, a->cu_seqlens != nullptr).count;
        pl.rows = a->cu_seqlens ? delta::long_rows(a->num_seqs, a->total_tokens, pl.token_len) : a->num_seqs;
        pl.bytes = delta::chunk_workspace(pl.slots, a->num_seqs, a->Hk, a->Hv, a->K);
    }
    return pl;
}

// What the kernels will leave out, into the status word.
__global__ __launch_bounds__(256) void delta_status_kernel(const Params p) {
    int bits = 0;
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < p.num_seqs; n += stride) {
        if (p.cu) {
            const int64_t s = p.cu[n], e = p.cu[n + 1];
            if (s < 0 || e < s || e > p.total_tokens) bits |= DELTA_STATUS_SEQLENS;
        }
        if (p.n_keep && p.n_keep[n] < 0) bits |= DELTA_STATUS_NKEEP;
        const int64_t from = p.h0_idx ? p.h0_idx[n] : n, to = p.ht_idx ? p.ht_idx[n] : n;
        if (p.h0 && !(p.fresh && p.fresh[n]) && (from < 0 || from >= p.h0_rows)) bits |= DELTA_STATUS_SLOT;
        if (p.ht && (to < 0 || to >= p.ht_rows)) bits |= DELTA_STATUS_SLOT;
        if (p.ht && p.ht_idx && p.num_seqs <= kClashRows)
            for (int64_t m = 0; m < p.num_seqs; ++m)
                if (m != n && (p.ht_idx[m] == to || (p.h0 == p.ht && p.h0_idx && p.h0_idx[m] == to))) bits |= DELTA_STATUS_CLASH;
    }
    if (bits) atomicOr(p.status, bits);
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_sizes(const delta_args* a) {
    if (a->Hk < 1 || a->Hv < a->Hk || a->Hv % a->Hk || a->num_seqs < 0 || a->T < 0 || a->total_tokens < 0) return WKV7_ERR_SHAPE;
    if ((a->K != 64 && a->K != 128) || a->V < 16 || a->V > 256 || a->V % 16 || a->Hv > 65536) return WKV7_ERR_SHAPE;
    if (a->total_tokens > ((int64_t)1 << 30) || (!a->cu_seqlens && (int64_t)a->num_seqs * a->T > a->total_tokens))
        return WKV7_ERR_SHAPE;
    if (a->token_len < -1 || (a->snapshots && (a->cu_seqlens || a->T < 1))) return WKV7_ERR_ARG;
    if ((int64_t)a->num_seqs * a->Hv * ((a->V + 15) / 16) > (int64_t)0x7FFFFF * 4) return WKV7_ERR_SHAPE;  // work-items below 2^32
    return WKV7_OK;
}

int check(const delta_args* a) {
    const int rc = check_sizes(a);
    if (rc != WKV7_OK) return rc;
    if (a->num_seqs > 0 && a->total_tokens > 0) {
        if (!a->q || !a->k || !a->v || !a->g || !a->beta) return WKV7_ERR_NULL;
        if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->g, 4) || !aligned(a->beta, 4) ||
            !aligned(a->o, 16))
            return WKV7_ERR_ALIGN;
        const int64_t qk = (int64_t)a->Hk * a->K, v = (int64_t)a->Hv * a->V;
        if (a->q_stride % 8 || a->k_stride % 8 || a->v_stride % 8 || (a->o && a->o_stride % 8)) return WKV7_ERR_ALIGN;
        if (a->q_stride < qk || a->k_stride < qk || a->v_stride < v || a->g_stride < a->Hv || a->beta_stride < a->Hv ||
            (a->o && a->o_stride < v))
            return WKV7_ERR_SHAPE;
        for (int64_t s : {a->q_stride, a->k_stride, a->v_stride, a->g_stride, a->beta_stride, a->o ? a->o_stride : 0})
            if (s > DELTA_MAX_STRIDE) return WKV7_ERR_SHAPE;
    }
    if (!aligned(a->h0, 16) || !aligned(a->ht, 16) || !aligned(a->snapshots, 16)) return WKV7_ERR_ALIGN;
    if ((a->h0_idx && !a->h0) || (a->ht_idx && !a->ht)) return WKV7_ERR_ARG;
    if ((a->h0 && a->h0_rows < 0) || (a->ht && a->ht_rows < 0)) return WKV7_ERR_SHAPE;
    return WKV7_OK;
}

}  // namespace
}  // namespace delta

extern "C" {

size_t delta_args_size(void) { return sizeof(delta_args); }

int delta_workspace_size(const delta_args* a, size_t* bytes) {
    if (!a || !bytes) return WKV7_ERR_NULL;
    *bytes = 0;
    const int rc = delta::check_sizes(a);
    if (rc == WKV7_OK && a->num_seqs > 0) *bytes = delta::make_plan(a).bytes;
    return rc;
}

int delta_run(const delta_args* a, void* stream) {
    if (!a) return WKV7_ERR_NULL;
    const int rc = delta::check(a);
    if (rc != WKV7_OK) return rc;
    if (a->num_seqs == 0) return WKV7_OK;
    const delta::Plan pl = delta::make_plan(a);
    if (pl.bytes && (!a->workspace || a->workspace_bytes < pl.bytes)) return WKV7_ERR_WORKSPACE;
    if (pl.bytes && !delta::aligned(a->workspace, 256)) return WKV7_ERR_ALIGN;
    if (pl.chunks && (pl.slots * a->Hk >= 0xFFFFFF || delta::chunk_groups(pl.rows, a->Hv, a->V) > 0x7FFFFF))
        return WKV7_ERR_SHAPE;  // work-items of a launch below 2^32
    delta::Params p;
    p.q = a->q, p.k = a->k, p.v = a->v, p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride;
    p.g = a->g, p.beta = a->beta, p.g_stride = a->g_stride, p.beta_stride = a->beta_stride;
    p.o = a->o, p.o_stride = a->o_stride;
    p.h0 = a->h0, p.h0_idx = a->h0_idx, p.h0_rows = a->h0_rows, p.ht = a->ht, p.ht_idx = a->ht_idx, p.ht_rows = a->ht_rows;
    p.fresh = a->fresh, p.cu = a->cu_seqlens, p.n_keep = a->n_keep, p.snapshots = a->snapshots, p.status = a->status;
    p.workspace = static_cast<char*>(a->workspace), p.total_tokens = a->total_tokens;
    p.num_seqs = a->num_seqs, p.T = a->T, p.Hk = a->Hk, p.Hv = a->Hv, p.K = a->K, p.V = a->V, p.share = a->Hv / a->Hk;
    p.scale = a->scale, p.qk_norm = a->qk_norm, p.token_len = pl.token_len;
    const auto s = static_cast<hipStream_t>(stream);
    if (p.status) {
        hipLaunchKernelGGL(delta::delta_status_kernel, dim3((unsigned)((p.num_seqs + 255) / 256 < 64 ? (p.num_seqs + 255) / 256 : 64)),
                           dim3(256), 0, s, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return static_cast<int>(e);
    }
    if (pl.chunks) {
        const hipError_t e = delta::launch_chunks(p, wkv7::device_cu_count(), s);
        if (e != hipSuccess) return static_cast<int>(e);
    }
    return pl.tokens ? static_cast<int>(delta::launch_tokens(p, s)) : WKV7_OK;
}

}  // extern "C"
