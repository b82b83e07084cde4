"""The gated delta rule on MI355X over the HIP library (include/delta.h): a recurrence beside wkv7, on the same kind of slot pools.

Per value head h, with query/key head h // (Hv // Hk) and the state S (K x V, fp32):

    S_t = a_t S_{t-1} + k_t d_t^T,   d_t = beta_t (v_t - a_t S_{t-1}^T k_t),   a_t = exp(g_t)
    o_t = scale S_t^T q_t

    gated_delta(q, k, v, g, beta, state=None, ...)      -> (o, final state | None)
    gated_delta_pool_(q, k, v, g, beta, pool, slots, ...) -> o, states in a pool of slots, updated in place
                                                        (op rwkv_next_amd::gated_delta_pool_)

Layouts: q, k (B, T, Hk, K) and v (B, T, Hv, V) bfloat16, parts of one projection's result or tensors of their own (the strides
between tokens are free); g (B, T, Hv) log decays <= 0 and beta (B, T, Hv), float32; states (N, Hv, K, V) float32; o like v.
K is 64 or 128, V a multiple of 16 up to 256, Hv a multiple of Hk.  A value that is not finite reaches its own token and later ones of
its column (v) or head (k, g, beta), nothing else.  Inference only: there is no backward pass.  Every call runs on
the current stream, no host sync, and can be recorded into a HIP graph.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from .. import _lib
from ._workspace import on_device, stream_handle
from .wkv7 import _index_tensor, _require


_increment_version = torch.autograd.graph.increment_version
_MOST_TOKENS = 1 << 30  # of a call: a longer token_len is no other


def _tokens(t, dtype, shape, inner, align, name):
    """`t` (B, T, ...) as it is where its tokens, `inner` contiguous elements each, follow each other at one stride, else a contiguous
    copy; with that stride in elements and its address."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)} (got {tuple(t.shape)})")
    ptr = t.data_ptr()
    if ptr % (16 if align > 1 else 4) == 0:
        if t.is_contiguous():
            return t, inner, ptr
        B, T = shape[:2]
        st = t.stride()
        token = st[1] if T > 1 else st[0] if B > 1 else inner
        ok = (B == 1 or T == 1 or st[0] == T * st[1]) and inner <= token <= _lib.DELTA_MAX_STRIDE and token % align == 0
        want = 1
        for n, s in zip(reversed(shape[2:]), reversed(st[2:])):
            ok = ok and (n == 1 or s == want)
            want *= n
        if ok:
            return t, token, ptr
    t = t.detach().clone(memory_format=torch.contiguous_format)  # its own memory, aligned
    return t, inner, t.data_ptr()


def _launch(q, k, v, g, beta, *, o, h0=None, h0_idx=None, ht=None, ht_idx=None, fresh=None, cu=None, n_keep=None,
            snapshots=None, status=None, scale, qk_norm, token_len):
    qs = q.shape
    B, T, Hk, K = qs
    Hv, V = v.shape[2:]
    if K not in (64, 128) or V % 16 or not 16 <= V <= 256:
        raise ValueError(f"head sizes must be K in (64, 128) and V a multiple of 16 up to 256 (got K={K}, V={V})")
    if Hk < 1 or Hv < Hk or Hv % Hk:
        raise ValueError(f"value heads must be a multiple of the query/key heads (got Hk={Hk}, Hv={Hv})")
    token_len = min(token_len, _MOST_TOKENS)
    dev, index = q.device, q.get_device()
    if index < 0:
        raise ValueError(f"operands must be on a GPU (got {dev})")
    for t in (k, v, g, beta, h0, h0_idx, fresh, cu, n_keep, snapshots, status):
        if t is not None and t.get_device() != index:
            raise ValueError(f"all operands must be on {dev} (got {tuple(t.shape)} {t.dtype} on {t.device})")
    q, q_s, q_p = _tokens(q, torch.bfloat16, qs, Hk * K, 8, "q")
    k, k_s, k_p = _tokens(k, torch.bfloat16, qs, Hk * K, 8, "k")
    v, v_s, v_p = _tokens(v, torch.bfloat16, (B, T, Hv, V), Hv * V, 8, "v")
    heads = (B, T, Hv)
    g, g_s, g_p = _tokens(g, torch.float32, heads, Hv, 1, "g")
    beta, b_s, b_p = _tokens(beta, torch.float32, heads, Hv, 1, "beta")
    h_p = 0 if h0 is None else h0.data_ptr()
    fields = [q_p, k_p, v_p, q_s, k_s, v_s, g_p, b_p, g_s, b_s, 0 if o is None else o.data_ptr(), Hv * V,
              h_p, 0 if h0_idx is None else h0_idx.data_ptr(), 0 if h0 is None else h0.shape[0],
              0 if ht is None else h_p if ht is h0 else ht.data_ptr(), 0 if ht_idx is None else ht_idx.data_ptr(),
              0 if ht is None else ht.shape[0], 0 if fresh is None else fresh.data_ptr(), 0 if cu is None else cu.data_ptr(),
              0 if n_keep is None else n_keep.data_ptr(), 0 if snapshots is None else snapshots.data_ptr(),
              0 if status is None else status.data_ptr(), 0, 0, B * T, B if cu is None else cu.numel() - 1,
              T if cu is None else 0, Hk, Hv, K, V, K ** -0.5 if scale is None else float(scale), int(qk_norm),
              token_len]  # in the order of the fields
    lib = _lib.load()
    args = _lib.pack_delta(*fields)
    if cu is not None or T > (_lib.DELTA_TOKEN_LEN if token_len < 0 else token_len):  # else token by token, without a workspace
        size = ctypes.c_size_t(0)
        _lib.check(lib.delta_workspace_size(args, ctypes.byref(size)))
        if size.value:  # what it holds does not matter: from the caching allocator, in the stream's order
            workspace = torch.empty(size.value, dtype=torch.uint8, device=dev)
            fields[23:25] = workspace.data_ptr(), size.value
            args = _lib.pack_delta(*fields)
    with on_device(dev):
        _lib.check(lib.delta_run(args, stream_handle(dev)))


def _state(t, N, Hv, K, V, name):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape[1:] != (Hv, K, V) or t.dim() != 4 or (N is not None and t.shape[0] != N):
        raise ValueError(f"{name} must be a float32 ({'S' if N is None else N}, {Hv}, {K}, {V}) tensor "
                         f"(got {t.dtype} {tuple(t.shape)})")
    return t


def _rows(q, cu_seqlens):
    """(cu_seqlens as int32 on the device or None, number of sequences)"""
    if q.dim() != 4:
        raise ValueError(f"q, k must be (B, T, Hk, K) (got {tuple(q.shape)})")
    if cu_seqlens is None:
        return None, q.shape[0]
    if q.shape[0] != 1:
        raise ValueError("cu_seqlens requires B == 1 (packed varlen)")
    cu = _index_tensor(cu_seqlens, q.device, torch.int32, "cu_seqlens")
    if cu.dim() != 1 or cu.numel() < 1:
        raise ValueError(f"cu_seqlens must hold N + 1 offsets (got {tuple(cu.shape)})")
    return cu, cu.numel() - 1


def _heads(q, v):
    """K, Hv, V"""
    qs, vs = q.shape, v.shape
    if len(qs) != 4 or len(vs) != 4:
        raise ValueError(f"q, k must be (B, T, Hk, K) and v (B, T, Hv, V) (got {tuple(qs)}, {tuple(vs)})")
    return qs[3], vs[2], vs[3]


@torch.no_grad()
def gated_delta(q, k, v, g, beta, state=None, *, cu_seqlens=None, scale=None, qk_norm: bool = False, final: bool = True,
                token_len: int = -1):
    """(o, final state (N, Hv, K, V) or None) from `state` (N, Hv, K, V) float32 or None (zeros); N = B rows of T tokens, or
    the rows of cu_seqlens (N + 1,) in a packed (1, sumT, ..) batch.

    scale: K ** -0.5 where None.  qk_norm: q and k are divided by sqrt(sum of squares + 1e-6) first.  token_len: rows of at most
    so many tokens run token by token instead of by chunks (-1: the library's choice)."""
    cu, N = _rows(q, cu_seqlens)
    K, Hv, V = _heads(q, v)
    h0 = _state(state, N, Hv, K, V, "state")
    h0 = None if h0 is None else h0.contiguous()
    o = torch.empty(v.shape, dtype=torch.bfloat16, device=v.device)
    ht = torch.empty(N, Hv, K, V, dtype=torch.float32, device=v.device) if final else None
    _launch(q, k, v, g, beta, o=o, h0=h0, ht=ht, cu=cu, scale=scale, qk_norm=qk_norm, token_len=token_len)
    return o, ht


def _pool(q, k, v, g, beta, pool, slots, cu_seqlens, n_keep, fresh, scale, qk_norm, final, store_o, snapshots, status, token_len):
    N = q.shape[0] if cu_seqlens is None else cu_seqlens.numel() - 1
    K, Hv, V = _heads(q, v)
    if pool.dtype is not torch.float32 or pool.shape[1:] != (Hv, K, V) or not pool.is_contiguous():
        _require(pool, "pool", torch.float32, (None, Hv, K, V))
    if slots.dtype is not torch.int64 or slots.shape != (N,) or not slots.is_contiguous():
        _require(slots, "slots", torch.int64, (N,))
    if cu_seqlens is not None:
        _require(cu_seqlens, "cu_seqlens", torch.int32, (None,))
    if n_keep is not None:
        _require(n_keep, "n_keep", torch.int64, (N,))
    if fresh is not None:
        _require(fresh, "fresh", torch.uint8, (N,))
    if snapshots is not None:
        if cu_seqlens is not None:
            raise ValueError("snapshots are kept for dense (N, T) rows")
        _require(snapshots, "snapshots", torch.float32, (N, q.shape[1], Hv, K, V))
    if status is not None:
        _require(status, "status", torch.int32, (None,))
        if status.numel() < 1:
            raise ValueError("status must hold at least one int32")
    o = torch.empty(v.shape if store_o else (0,), dtype=torch.bfloat16, device=v.device)
    _launch(q, k, v, g, beta, o=o if store_o else None, h0=pool, h0_idx=slots, ht=pool if final else None,
            ht_idx=slots if final else None, fresh=fresh, cu=cu_seqlens, n_keep=n_keep, snapshots=snapshots, status=status,
            scale=scale, qk_norm=qk_norm, token_len=token_len)
    return o


@torch.library.custom_op("rwkv_next_amd::gated_delta_pool_", mutates_args=("pool", "snapshots", "status"))
def gated_delta_pool_op(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, pool: Tensor, slots: Tensor,
                        cu_seqlens: Optional[Tensor], n_keep: Optional[Tensor], fresh: Optional[Tensor],
                        scale: Optional[float], qk_norm: bool, final: bool, store_o: bool, snapshots: Optional[Tensor],
                        status: Optional[Tensor], token_len: int) -> Tensor:
    """The slot-pool recurrence as a registered op (indices int64, cu_seqlens int32, fresh uint8).  Returns o, or an empty tensor
    when store_o is False."""
    return _pool(q, k, v, g, beta, pool, slots, cu_seqlens, n_keep, fresh, scale, qk_norm, final, store_o, snapshots, status,
                 token_len)


@gated_delta_pool_op.register_fake
def _(q, k, v, g, beta, pool, slots, cu_seqlens, n_keep, fresh, scale, qk_norm, final, store_o, snapshots, status, token_len):
    return v.new_empty(v.shape if store_o else (0,))


def gated_delta_pool_(q, k, v, g, beta, pool, slots, *, cu_seqlens=None, n_keep=None, fresh=None, scale=None,
                      qk_norm: bool = False, final: bool = True, store_o: bool = True, snapshots=None, status=None,
                      token_len: int = -1):
    """The recurrence for N sequences whose states live in `pool` (S, Hv, K, V) float32, updated in place.

    slots (N,) int64: each sequence's row of the pool, distinct within a call.  Rows, cu_seqlens, scale, qk_norm and token_len as in
    gated_delta; fresh, n_keep, final, store_o and status as in wkv7_pool_.
    snapshots: optional (N, T, Hv, K, V) float32, the state after each token of dense rows; they run token by token.  Rolling back
    to the first n tokens is SlotCaches((snapshots.flatten(0, 1), 0)).copy_slots(row * T + n - 1, slots,
    into=SlotCaches((pool, 0))), or, on the pool as it was before, a call with n_keep=n, store_o=False on the same operands: where
    token by token, the same bits.
    Returns o like v (None when store_o is False).  Under torch.compile or another tracer it is the registered op
    rwkv_next_amd::gated_delta_pool_; an eager call goes straight to the library, as dense_matmul's (the dispatch of an op took 12 of
    a single token's 27 us)."""
    cu, N = _rows(q, cu_seqlens)
    dev = q.device
    sl = slots
    if type(slots) is not Tensor or slots.dtype is not torch.int64 or slots.device != dev or not slots.is_contiguous():
        sl = _index_tensor(slots, dev, torch.int64, "slots")
    nk = None if n_keep is None else _index_tensor(n_keep, dev, torch.int64, "n_keep")
    fr = None
    if fresh is not None:
        fr = fresh if isinstance(fresh, Tensor) and fresh.device == dev else torch.as_tensor(fresh, device=dev)
        if fr.dtype == torch.bool:
            fr = fr.view(torch.uint8)
        fr = (fr if fr.dtype == torch.uint8 else fr.to(torch.uint8)).contiguous()
    traced = torch.compiler.is_compiling() or type(pool) is not Tensor or torch._C._len_torch_dispatch_stack() > 0
    o = (gated_delta_pool_op if traced else _pool)(q, k, v, g, beta, pool, sl, cu, nk, fr, scale, bool(qk_norm), final, store_o,
                                                   snapshots, status, int(token_len))
    if not traced:  # written in place, as autograd is told
        if final and not pool.is_inference():
            _increment_version(pool)
        for t in (snapshots, status):
            if t is not None and not t.is_inference():
                _increment_version(t)
    return o if store_o else None
