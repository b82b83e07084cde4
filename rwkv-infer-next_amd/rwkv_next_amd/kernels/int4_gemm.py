"""Products with 4-bit weights (W4A16) on the HIP kernels of include/w4a16.h: the output head and the projections of a decode
step, at two thirds of the 6-bit weights' bytes.  No counterpart in the reference, whose weights have 6 or 8 bits.

    quantize_int4(w, group_k=128, clip_search=True) -> (codes, scales, group_k)
    dequantize_int4(codes, scales, group_k, dtype)  -> w
    prepack_int4(codes, scales, group_k)            -> Int4Packed, made once when the weights are loaded
    int4_matmul(a, packed, out_dtype=None)          -> a @ w
    int4_matmul_op(a, weight, scales, K, N, group_k)   op rwkv_next_amd::int4_matmul, the fields of an Int4Packed

Format: a (K, N) weight is quantised to q in [-8, 7] per (group of group_k rows, column) with an fp16 scale, w ~ s q; two codes
u = q + 8 to a byte, codes[j] = u(row 2j) | u(row 2j + 1) << 4.  K and group_k are multiples of 32, N is any.

Activations are bf16 or fp16, sums fp32, the result has the activations' type or out_dtype.  The kernel is made for the rows of a
decode or verification step; it takes any number, but a prompt of thousands of rows is served better by dequantize_int4 and a
library product.  Every call runs on the current stream, no host sync.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from .. import _lib
from ._workspace import on_device, stream_handle

STEP = 32                 # rows that K and group_k are multiples of
QMIN, QMAX = -8, 7
_RATIOS = (1.0, 0.97, 0.94, 0.91, 0.88, 0.85, 0.82, 0.79)
_CODES = {torch.bfloat16: _lib.W4A16_BF16, torch.float16: _lib.W4A16_F16, torch.float32: _lib.W4A16_F32}


def _check_group(K, group_k):
    g = group_k if group_k and 0 < group_k < K else K
    if K < STEP or K % STEP or g % STEP or K % g:
        raise ValueError(f"int4 needs K % 32 == 0 and group_k % 32 == 0 dividing K (K={K}, group_k={group_k})")
    return g


@torch.no_grad()
def quantize_int4(w, group_k=128, clip_search=True):
    """(K, N) float -> (codes uint8 (K/2, N), scales fp16 (K/group_k, N), group_k); a group_k outside (0, K) means one group.

    The scale of a (group, column) is fp16(absmax * r / 7.5) for the clip ratio r in (1, .97, .. .79) (only 1 without
    clip_search) whose rounded weights have the least squared error, the first such r on ties; q = clamp(round(w / s), -8, 7)
    with the stored fp16 scale.  A column of zeros has a scale of the smallest normal fp16 and codes of 0."""
    if w.dim() != 2:
        raise ValueError(f"quantize_int4 takes a (K, N) weight (got {tuple(w.shape)})")
    K, N = w.shape
    g = _check_group(K, group_k)
    G = K // g
    codes = torch.empty((K // 2, N), dtype=torch.uint8, device=w.device)
    scales = torch.empty((G, N), dtype=torch.float16, device=w.device)
    cols = max(256, (1 << 23) // K)  # column blocks keep the fp32 temporaries to ~32 MB
    for n0 in range(0, N, cols):
        n1 = min(N, n0 + cols)
        x = w[:, n0:n1].float().view(G, g, n1 - n0)
        amax = x.abs().amax(dim=1, keepdim=True)
        best_s = best_err = None
        for r in (_RATIOS if clip_search else _RATIOS[:1]):
            s = (amax * (r / 7.5)).half().clamp_min(2.0 ** -14).float()
            err = (torch.round(x / s).clamp(QMIN, QMAX) * s - x).square().sum(dim=1, keepdim=True)
            if best_s is None:
                best_s, best_err = s, err
            else:
                better = err < best_err
                best_s, best_err = torch.where(better, s, best_s), torch.where(better, err, best_err)
        u = (torch.round(x / best_s).clamp(QMIN, QMAX) + 8).to(torch.uint8).view(K // 2, 2, n1 - n0)
        codes[:, n0:n1] = u[:, 0] | (u[:, 1] << 4)
        scales[:, n0:n1] = best_s.view(G, n1 - n0).half()
    return codes, scales, g


def _weight(codes, scales, group_k):
    if codes.dtype != torch.uint8 or scales.dtype != torch.float16:
        raise TypeError(f"int4 weights are (codes uint8, scales float16) (got {codes.dtype}, {scales.dtype})")
    if codes.dim() != 2 or scales.dim() != 2 or codes.shape[1] != scales.shape[1] or codes.shape[1] < 1:
        raise ValueError(f"int4 codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not match")
    if codes.device.type != "cuda" or scales.device != codes.device:
        raise ValueError(f"int4 codes and scales must be on one GPU (got {codes.device}, {scales.device})")
    K, N = 2 * codes.shape[0], codes.shape[1]
    g = _check_group(K, group_k)
    if scales.shape[0] != K // g:
        raise ValueError(f"group_k {group_k} does not match K = {K} with {scales.shape[0]} scale rows")
    return codes.contiguous(), scales.contiguous(), K, N, g


@torch.no_grad()
def dequantize_int4(codes, scales, group_k, dtype=torch.float32):
    """w = s q, (K, N) in `dtype` (bfloat16, float16 or float32; float32 is exact), on the device."""
    codes, scales, K, N, g = _weight(codes, scales, group_k)
    if dtype not in _CODES:
        raise TypeError(f"dequantize_int4 writes bfloat16, float16 or float32 (got {dtype})")
    w = torch.empty((K, N), dtype=dtype, device=codes.device)
    with on_device(w.device):
        _lib.check(_lib.load().w4a16_dequantize(codes.data_ptr(), scales.data_ptr(), w.data_ptr(), K, N, g,
                                                _CODES[dtype], stream_handle(w.device)))
    return w


class Int4Packed(NamedTuple):
    """A 4-bit weight in the order in which the kernel reads it (include/w4a16.h, w4a16_pack), from prepack_int4."""
    weight: torch.Tensor   # uint8, 16-byte aligned
    scales: torch.Tensor   # float16, 16-byte aligned
    K: int
    N: int
    group_k: int


def _packed_size(K, N, g):
    wb, sb = ctypes.c_size_t(0), ctypes.c_size_t(0)
    _lib.check(_lib.load().w4a16_packed_size(K, N, g, ctypes.byref(wb), ctypes.byref(sb)))
    return int(wb.value), int(sb.value) // 2


@torch.no_grad()
def prepack_int4(codes, scales, group_k) -> Int4Packed:
    """Lays a quantised weight out for int4_matmul, on its device: the same codes and scales."""
    codes, scales, K, N, g = _weight(codes, scales, group_k)
    nw, ns = _packed_size(K, N, g)
    weight = torch.empty(nw, dtype=torch.uint8, device=codes.device)
    sc = torch.empty(ns, dtype=torch.float16, device=codes.device)
    with on_device(codes.device):
        _lib.check(_lib.load().w4a16_pack(codes.data_ptr(), scales.data_ptr(), K, N, g, weight.data_ptr(),
                                          sc.data_ptr(), stream_handle(codes.device)))
    return Int4Packed(weight, sc, K, N, g)


def int4_matmul(a, packed: Int4Packed, *, out_dtype=None):
    """a (..., K) bf16 or fp16 @ dequant(packed (K, N)) -> (..., N) in a.dtype, or out_dtype (bfloat16 / float16 / float32).
    An infinity or NaN in a row of `a` makes the whole row NaN."""
    weight, scales, K, N, g = packed
    adt = a.dtype
    odt = adt if out_dtype is None else out_dtype
    if adt is not torch.bfloat16 and adt is not torch.float16:
        raise TypeError(f"int4_matmul takes bfloat16 or float16 activations (got {adt})")
    if odt not in _CODES:
        raise TypeError(f"int4_matmul writes bfloat16, float16 or float32 (got {odt})")
    index = a.get_device()
    if index < 0 or weight.get_device() != index or scales.get_device() != index:
        raise ValueError(f"int4_matmul needs a and the weight on one GPU (got {a.device}, {weight.device})")
    shape = a.shape
    if len(shape) < 1 or shape[-1] != K:
        raise ValueError(f"K mismatch: a is {tuple(shape)}, int4 weight has {K} rows")
    if weight.dtype is not torch.uint8 or scales.dtype is not torch.float16 or not weight.is_contiguous() or \
            not scales.is_contiguous() or (weight.numel(), scales.numel()) != _sizes(K, N, g):
        raise ValueError("the packed weight and scales are not prepack_int4's")
    dev = a.device
    x = a if len(shape) == 2 else a.reshape(-1, K)
    M = x.size(0)
    out = torch.empty(*shape[:-1], N, dtype=odt, device=dev)
    if M == 0:
        return out
    row, ptr = x.stride(0) if M > 1 else K, x.data_ptr()
    if x.stride(1) != 1 or row % 8 or row < K or row > _lib.W4A16_MAX_ROW_STRIDE or ptr % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        row, ptr = K, x.data_ptr()
    args = _lib.pack_w4a16(ptr, row, weight.data_ptr(), scales.data_ptr(), out.data_ptr(), N, M, N, K, g, _CODES[adt],
                           _CODES[odt])  # in the order of the fields
    with on_device(dev):
        _lib.check(_lib.load().w4a16_matmul(args, stream_handle(dev)))
    return out


_SIZES: dict = {}  # (K, N, group_k) -> elements of a packed weight and of its scales


def _sizes(K, N, g):
    s = _SIZES.get((K, N, g))
    if s is None:
        s = _SIZES[(K, N, g)] = _packed_size(K, N, g)
    return s


@torch.library.custom_op("rwkv_next_amd::int4_matmul", mutates_args=())
def int4_matmul_op(a: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor, K: int, N: int,
                   group_k: int) -> torch.Tensor:
    """int4_matmul as a registered op, for torch.compile: the fields of an Int4Packed."""
    return int4_matmul(a, Int4Packed(weight, scales, K, N, group_k))


@int4_matmul_op.register_fake
def _(a, weight, scales, K, N, group_k):
    return a.new_empty((*a.shape[:-1], N))
