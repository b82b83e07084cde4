"""Products with 16-bit weights on the HIP kernels of include/dense.h, with bias, activation and residual in the epilogue: the
projections, low-rank parts and channel mix of a layer whose weights are not quantised (rwkv_next/model.py:113-175 computes
them with torch operations), beside int4_matmul and int6_matmul.

    prepack_dense(w)                                     -> DensePacked, made once when the weights are loaded
    dense_matmul(a, packed, bias=None, activation=None, residual=None, out_dtype=None)
                                                         -> act(a @ w + bias) + residual
    dense_matmul_op(a, weight, K, N, bias, activation, residual, out_dtype=None)
                                                         op rwkv_next_amd::dense_matmul, the fields of a DensePacked

Activations and weights are both bfloat16 or both float16; sums and the epilogue are fp32, the result is rounded once.  K is a
multiple of 32, N is any.  Every call runs on the current stream, no host sync, and can be recorded into a HIP graph.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from .. import _lib
from ._workspace import on_device, stream_handle

_CODES = {torch.bfloat16: _lib.DENSE_BF16, torch.float16: _lib.DENSE_F16, torch.float32: _lib.DENSE_F32}
ACTIVATIONS = {None: _lib.DENSE_NONE, "none": _lib.DENSE_NONE, "relu": _lib.DENSE_RELU, "relu2": _lib.DENSE_RELU2,
               "tanh": _lib.DENSE_TANH, "sigmoid": _lib.DENSE_SIGMOID, "silu": _lib.DENSE_SILU, "gelu": _lib.DENSE_GELU}


class DensePacked(NamedTuple):
    """A 16-bit weight in the order in which the kernels read it (include/dense.h, dense_pack), from prepack_dense."""
    weight: torch.Tensor   # of the weight's type, 16-byte aligned
    K: int
    N: int


_SIZES: dict = {}  # (K, N) -> elements of a packed weight


def _size(K, N):
    s = _SIZES.get((K, N))
    if s is None:
        n = ctypes.c_size_t(0)
        _lib.check(_lib.load().dense_packed_size(K, N, ctypes.byref(n)))
        s = _SIZES[(K, N)] = int(n.value) // 2
    return s


@torch.no_grad()
def prepack_dense(w) -> DensePacked:
    """Lays a (K, N) bfloat16 or float16 weight out for dense_matmul, on its device; any strides (a Linear's (N, K) weight is
    prepack_dense(weight.t()))."""
    if w.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"prepack_dense takes a bfloat16 or float16 weight (got {w.dtype})")
    if w.dim() != 2 or w.shape[0] < 32 or w.shape[0] % 32 or w.shape[1] < 1:
        raise ValueError(f"prepack_dense takes a (K, N) weight with K % 32 == 0 (got {tuple(w.shape)})")
    if not w.is_cuda:
        raise ValueError(f"prepack_dense takes a weight on a GPU (got {w.device})")
    K, N = w.shape
    packed = torch.empty(_size(K, N), dtype=w.dtype, device=w.device)
    with on_device(w.device):
        _lib.check(_lib.load().dense_pack(w.data_ptr(), w.stride(0), w.stride(1), K, N, packed.data_ptr(),
                                          stream_handle(w.device)))
    return DensePacked(packed, K, N)


def dense_matmul(a, packed: DensePacked, *, bias=None, activation: Optional[str] = None, residual=None, out_dtype=None):
    """act(a (..., K) @ w (K, N) + bias (N,)) + residual (..., N), in a.dtype or out_dtype (bfloat16 / float16 / float32).

    activation: None ("none"), "relu", "relu2" (the squared ReLU of RWKV's channel mix), "tanh", "sigmoid", "silu" or "gelu" (by
    erf).  bias and residual: bfloat16, float16 or float32, whatever the others are."""
    weight, K, N = packed
    adt = a.dtype
    odt = adt if out_dtype is None else out_dtype
    if (adt is not torch.bfloat16 and adt is not torch.float16) or weight.dtype is not adt:
        raise TypeError(f"dense_matmul takes bfloat16 or float16 activations of the weight's type (got {adt}, {weight.dtype})")
    if odt not in _CODES:
        raise TypeError(f"dense_matmul writes bfloat16, float16 or float32 (got {odt})")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {[x for x in ACTIVATIONS if x]} or None (got {activation!r})")
    index = a.get_device()
    if index < 0 or weight.get_device() != index:
        raise ValueError(f"dense_matmul needs a and the weight on one GPU (got {a.device}, {weight.device})")
    shape = a.shape
    if len(shape) < 1 or shape[-1] != K:
        raise ValueError(f"K mismatch: a is {tuple(shape)}, the weight has {K} rows")
    if not weight.is_contiguous() or weight.numel() != _size(K, N):
        raise ValueError("the packed weight is not prepack_dense's")
    dev = a.device
    b_p = b_t = r_p = r_t = r_row = 0
    if bias is not None:
        if bias.dtype not in _CODES or bias.shape != (N,) or bias.get_device() != index:
            raise ValueError(f"bias must be ({N},), bfloat16, float16 or float32, on {dev} (got {bias.dtype} {tuple(bias.shape)} on "
                             f"{bias.device})")
        bias = bias.contiguous()
        b_p, b_t = bias.data_ptr(), _CODES[bias.dtype]
    x = a if len(shape) == 2 else a.reshape(-1, K)
    M = x.size(0)
    if residual is not None:
        if residual.dtype not in _CODES or residual.shape != (*shape[:-1], N) or residual.get_device() != index:
            raise ValueError(f"residual must be {(*shape[:-1], N)}, bfloat16, float16 or float32, on {dev} (got {residual.dtype} "
                             f"{tuple(residual.shape)} on {residual.device})")
        res = residual if len(shape) == 2 else residual.reshape(-1, N)
        r_row = res.stride(0) if M > 1 else N
        if (N > 1 and res.stride(1) != 1) or r_row < N:
            res = res.clone(memory_format=torch.contiguous_format)
            r_row = N
        r_p, r_t = res.data_ptr(), _CODES[res.dtype]
    out = torch.empty(*shape[:-1], N, dtype=odt, device=dev)
    if M == 0:
        return out
    row, ptr = x.stride(0) if M > 1 else K, x.data_ptr()
    if x.stride(1) != 1 or row % 8 or row < K or row > _lib.DENSE_MAX_ROW_STRIDE or ptr % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        row, ptr = K, x.data_ptr()
    lib, sums, sums_p, size = _lib.load(), None, 0, 0
    with on_device(dev):
        if M > _lib.DENSE_UNSPLIT_ROWS or K >= _lib.DENSE_UNSPLIT_K:
            need = ctypes.c_size_t(0)
            _lib.check(lib.dense_workspace_size(M, N, K, ctypes.byref(need)))
            size = need.value
            if size:  # what it holds does not matter: from the caching allocator, in the stream's order
                sums = torch.empty(size, dtype=torch.uint8, device=dev)
                sums_p = sums.data_ptr()
        args = _lib.pack_dense(ptr, row, weight.data_ptr(), b_p, r_p, r_row, out.data_ptr(), N, M, N, K, _CODES[adt], _CODES[odt],
                               b_t, r_t, ACTIVATIONS[activation], sums_p, size)  # in the order of the fields
        _lib.check(lib.dense_matmul(args, stream_handle(dev)))
    return out


@torch.library.custom_op("rwkv_next_amd::dense_matmul", mutates_args=())
def dense_matmul_op(a: torch.Tensor, weight: torch.Tensor, K: int, N: int, bias: Optional[torch.Tensor], activation: str,
                    residual: Optional[torch.Tensor], out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """dense_matmul as a registered op, for torch.compile: the fields of a DensePacked."""
    return dense_matmul(a, DensePacked(weight, K, N), bias=bias, activation=activation, residual=residual, out_dtype=out_dtype)


@dense_matmul_op.register_fake
def _(a, weight, K, N, bias, activation, residual, out_dtype=None):
    return a.new_empty((*a.shape[:-1], N), dtype=a.dtype if out_dtype is None else out_dtype)
