"""From logits to tokens on the HIP kernels of include/logits.h: what the reference's sampler and its speculative step do with
torch operations (rwkv_next/sampler.py:1-81, rwkv_next/spec.py:35-84).

    penalize_logits(logits, ...)        penalties for repeated tokens, per-request biases, grammar masks
    sample_logits(logits, noise, ...)   temperature, top-k, top-p, min-p, and a draw by given noise
    next_tokens(x, head, noise, ...)    a decode step's end: head product, penalties, draw, the drawn tokens counted

Logits are (B, V), one token for each sequence, or (B, T, V), T positions of a block of drafted tokens, in bfloat16, float16 or
float32.  A per-sequence parameter is a tensor of B entries on the logits' device, or one number for all.  Every call runs on the
current stream, no host sync, and can be recorded into a HIP graph; `status` (wkv7.new_status) reports indices that the kernels
left out (check_status names them).
"""
from __future__ import annotations

import ctypes
import threading

import numpy as np
import torch

from .. import _lib
from ._workspace import on_device, retire, stream_handle, stream_workspace
from .int4_gemm import Int4Packed, int4_matmul

_DTYPES = {torch.bfloat16: _lib.LOGITS_BF16, torch.float16: _lib.LOGITS_F16, torch.float32: _lib.LOGITS_F32}
_COUNTS = {torch.int32: _lib.LOGITS_COUNTS_I32, torch.float32: _lib.LOGITS_COUNTS_F32}


def _shape(logits):
    """(B, T, V, sequence stride, position stride, the last stride) of (B, V) or (B, T, V) logits."""
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits must be bfloat16, float16 or float32 (got {logits.dtype})")
    if not logits.is_cuda:
        raise ValueError(f"logits must be on a GPU (got {logits.device})")
    n = logits.dim()
    if n == 2:
        (B, V), (seq, last) = logits.shape, logits.stride()
        return B, 1, V, seq, 0, last
    if n != 3:
        raise ValueError(f"logits must be (B, V) or (B, T, V) (got {tuple(logits.shape)})")
    return (*logits.shape, *logits.stride())


def _on(t, dev, name):
    if t.get_device() != dev.index:
        raise ValueError(f"{name} must be on {dev} (got {t.device})")


def _per_sequence(x, dtype, B, dev, name):
    """(pointer, scalar) of a parameter: a tensor of B entries, or a number (pointer 0)."""
    if not isinstance(x, torch.Tensor):
        return 0, x
    if x.dtype is dtype and x.shape == (B,) and x.is_contiguous() and x.get_device() == dev.index:
        return x.data_ptr(), 0
    _on(x, dev, name)
    raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor of {B} entries "
                     f"(got {x.dtype} {tuple(x.shape)})")


def _rows(x, dtype, lead, least, dev, name):
    """(tensor, its row stride) of a tensor of rows of at least `least` contiguous elements whose leading sizes are `lead`; a copy
    where rows share memory, as one row broadcast to all sequences."""
    _on(x, dev, name)
    shape, stride = x.shape, x.stride()
    if x.dtype is not dtype or shape[:-1] != lead or shape[-1] < least or (stride[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"{name} must be a {dtype} {(*lead, least)} tensor with contiguous rows "
                         f"(got {x.dtype} {tuple(shape)}, strides {stride})")
    if lead[0] > 1 and stride[0] < shape[-1]:
        x = x.contiguous()
        return x, x.stride(0)
    return x, stride[0] if lead[0] > 1 else max(stride[0], shape[-1])


def _overlaps(t):
    """Whether rows of a (B, V) or (B, T, V) tensor with contiguous rows may share memory."""
    least = t.shape[-1]
    for stride, size in sorted((s, n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        if stride < least:
            return True
        least = stride * (size - 1) + least
    return False


def _share_memory(a, b):
    """Whether rows of two (B, V) or (B, T, V) tensors with contiguous rows have memory in common.  Where their address ranges
    are apart, the usual case, at the cost of a few additions; else (columns of one buffer, say) by the rows' addresses."""
    ranges = []
    for t in (a, b):
        if t.numel() == 0:
            return False
        at = t.data_ptr()
        ranges.append((at, at + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()))
    if ranges[0][1] <= ranges[1][0] or ranges[1][1] <= ranges[0][0]:
        return False
    starts = [np.sort((t.data_ptr() + t.element_size() * sum(
        np.arange(n, dtype=np.int64).reshape(-1, *(1,) * (t.dim() - 2 - i)) * s
        for i, (n, s) in enumerate(zip(t.shape[:-1], t.stride()[:-1])))).reshape(-1)) for t in (a, b)]
    rows, others = starts
    # of the rows of b that begin before a row of a ends, the last one: does it end after that row begins?
    before = np.searchsorted(others, rows + a.shape[-1] * a.element_size(), side="left")
    last = others[np.maximum(before - 1, 0)] + b.shape[-1] * b.element_size()
    return bool(((before > 0) & (last > rows)).any())


def _counts(counts, slots, B, V, dev):
    """(pointer, row stride, rows, type, slots' pointer) of a count table (S, V)."""
    if counts is None:
        if slots is not None:
            raise ValueError("slots without counts")
        return 0, 0, 0, 0, 0
    _on(counts, dev, "counts")
    code, shape, stride = _COUNTS.get(counts.dtype), counts.shape, counts.stride()
    if code is None or len(shape) != 2 or shape[1] != V or (stride[1] != 1 and V > 1) or (shape[0] > 1 and stride[0] < V):
        raise ValueError(f"counts must be an int32 or float32 (S, {V}) tensor with contiguous rows "
                         f"(got {counts.dtype} {tuple(shape)}, strides {stride})")
    if slots is None:
        if shape[0] < B:
            raise ValueError(f"counts has {shape[0]} rows for {B} sequences (or pass slots)")
        return counts.data_ptr(), max(stride[0], V), shape[0], code, 0
    if not isinstance(slots, torch.Tensor):
        raise TypeError(f"slots must be an int64 tensor of {B} entries (got {type(slots).__name__})")
    sl = _per_sequence(slots, torch.int64, B, dev, "slots")[0]
    # a table without rows has no address, and NULL would be no table: every slot lies outside it, and its memory is not read
    return counts.data_ptr() if shape[0] else sl, max(stride[0], V), shape[0], code, sl


def _status(status, dev):
    if status is None:
        return 0
    _on(status, dev, "status")
    if status.dtype != torch.int32 or status.numel() < 1:
        raise ValueError("status must be an int32 tensor (new_status)")
    return status.data_ptr()


def penalize_logits(logits, *, counts=None, slots=None, repetition=1.0, presence=0.0, frequency=0.0, drafts=None,
                    bias_ids=None, bias_values=None, mask=None, mask_rows=None, out=None, status=None):
    """Per sequence b, position t and token v, with x the logit and c = counts[slots[b], v] + the number of drafts[b, :t] that
    are v:

        c > 0:  x = (x / repetition if x > 0 else x * repetition) - (frequency * c + presence)
        x += bias_values[b, i] for every i with bias_ids[b, i] == v, in their order
        x = -inf where the mask's bit of v is 0

    in fp32, rounded once.  Returns a new tensor of the logits' type, or fills and returns `out` (any of the three types;
    `logits` itself for an update in place, else apart from the logits).

    counts (S, V) int32 or float32, row slots[b] (int64; row b without slots) of sequence b; the reference's penalty table.
    drafts (B, >= T - 1) int64: the tokens fed at positions 1 .. T - 1, not yet in `counts` (negative: none).
    bias_ids (B, P) int64 (negative: an unused place), bias_values (B, P) float32.
    mask int32, ceil(V / 32) words to a row, bit v % 32 of word v / 32 set where v is allowed: one row for each row of the logits
    ((B, words) or (B, T, words)), or a table (R, words) with mask_rows int64 in the shape of the rows (negative: no mask).
    """
    B, T, V, seq_stride, pos_stride, last = _shape(logits)
    dev, in_place = logits.device, out is logits
    if last != 1 and V > 1:
        if in_place:
            raise ValueError("logits must have contiguous rows to be changed in place")
        logits = logits.contiguous()
        _, _, _, seq_stride, pos_stride, _ = _shape(logits)
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
        out_seq, out_pos = (V, 0) if logits.dim() == 2 else (T * V, V)
    else:
        if not in_place:
            _on(out, dev, "out")
            if out.shape != logits.shape or out.dtype not in _DTYPES or (out.stride(-1) != 1 and V > 1):
                raise ValueError(f"out must be bfloat16, float16 or float32 {tuple(logits.shape)} with contiguous rows "
                                 f"(got {out.dtype} {tuple(out.shape)}, strides {out.stride()})")
            if (out.data_ptr() != logits.data_ptr() or out.dtype != logits.dtype or out.stride() != logits.stride()) and \
                    _share_memory(out, logits):
                raise ValueError("out may share memory with the logits only as the logits themselves: at their address, of their "
                                 "type and strides")
        if _overlaps(out):
            raise ValueError(f"out must not share memory between its rows (strides {out.stride()})")
        out_seq, out_pos = out.stride(0), out.stride(1) if out.dim() == 3 else 0
    if not (B and T and V):
        return out
    lead = (B,) if logits.dim() == 2 else (B, T)
    ct, ct_stride, ct_rows, ct_type, slots_p = _counts(counts, slots, B, V, dev)
    rep_p, rep = _per_sequence(repetition, torch.float32, B, dev, "repetition")
    pres_p, pres = _per_sequence(presence, torch.float32, B, dev, "presence")
    freq_p, freq = _per_sequence(frequency, torch.float32, B, dev, "frequency")
    if not rep_p and not rep > 0:
        raise ValueError(f"repetition must be positive (got {rep})")
    dr_p = dr_stride = 0
    if drafts is not None and T > 1:
        drafts, dr_stride = _rows(drafts, torch.int64, (B,), T - 1, dev, "drafts")
        dr_p = drafts.data_ptr()
    bi_p = bv_p = bias_stride = n_bias = 0
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if bias_ids is not None:
        n_bias = bias_ids.size(-1)
        bias_ids, bias_stride = _rows(bias_ids, torch.int64, (B,), 0, dev, "bias_ids")
        bias_values, value_stride = _rows(bias_values, torch.float32, (B,), 0, dev, "bias_values")
        if bias_values.size(-1) != n_bias:
            raise ValueError(f"bias_ids and bias_values must have one shape (got {n_bias} and {bias_values.size(-1)} places)")
        if value_stride != bias_stride:
            bias_ids, bias_values, bias_stride = bias_ids.contiguous(), bias_values.contiguous(), n_bias
        bi_p, bv_p = bias_ids.data_ptr(), bias_values.data_ptr()
    m_p = m_stride = m_rows = mr_p = 0
    if mask is not None:
        words = (V + 31) // 32
        if mask_rows is None:
            m_rows = B * T
            mask, m_stride = _rows(mask, torch.int32, lead, words, dev, "mask")
            if len(lead) == 2:  # rows of (b, t) one after another
                if not mask.is_contiguous():
                    mask = mask.contiguous()
                m_stride = mask.size(-1)
        else:
            _on(mask_rows, dev, "mask_rows")
            if mask_rows.dtype is not torch.int64 or mask_rows.shape != lead or not mask_rows.is_contiguous():
                raise ValueError(f"mask_rows must be a contiguous int64 {lead} tensor "
                                 f"(got {mask_rows.dtype} {tuple(mask_rows.shape)})")
            if mask.dim() != 2:
                raise ValueError(f"mask must be a table (R, words) where mask_rows is given (got {tuple(mask.shape)})")
            m_rows = mask.size(0)
            mask, m_stride = _rows(mask, torch.int32, (m_rows,), words, dev, "mask") if m_rows else (mask, words)
            mr_p = mask_rows.data_ptr()
        m_p = mask.data_ptr() if m_rows else mr_p  # as for counts: a table without rows is one that no index lies in
    elif mask_rows is not None:
        raise ValueError("mask_rows without a mask")
    args = _lib.pack_penalize(
        logits.data_ptr(), seq_stride, pos_stride, out.data_ptr(), out_seq, out_pos, ct, ct_stride, ct_rows, slots_p,
        rep_p, pres_p, freq_p, dr_p, dr_stride, bi_p, bv_p, bias_stride, m_p, m_stride, m_rows, mr_p,
        _status(status, dev), rep, pres, freq, B, T, V, n_bias, _DTYPES[logits.dtype], _DTYPES[out.dtype],
        ct_type)  # in the order of the fields
    with on_device(dev):
        _lib.check(_lib.load().logits_penalize(args, stream_handle(dev)))
    return out


_WORKSPACES: dict = {}  # (device index, stream handle) -> [buffer, zeroed in stream order, capture id]
# A call's launches pass a row's state on through the stream's workspace, and the library runs without Python's lock: of threads
# on one stream one at a time looks its workspace up and launches.
_LAUNCHES = threading.Lock()
_BYTES: list = []  # of the workspace, once it is known


def _workspace(dev):
    """The workspace of the current stream, see `_workspace.stream_workspace`: 20 MiB, which serve any number of rows (as many as a
    set of launches takes).  One of a call's own rows alone would be replaced, and kept for captured graphs, whenever they grow."""
    if not _BYTES:
        size = ctypes.c_size_t(0)
        _lib.check(_lib.load().logits_sample_workspace_size(_lib.SampleArgs(B=2 ** 31 - 1, T=1, V=1), ctypes.byref(size)))
        _BYTES.append(int(size.value))
    return stream_workspace(_WORKSPACES, dev, _BYTES[0], _lib.LOGITS_SAMPLE_STATE_BYTES)


def reset_workspaces() -> None:
    """The next call of every stream gets a new, zeroed workspace (wkv7.reset_workspaces calls this too)."""
    with _LAUNCHES:
        retire(_WORKSPACES)


def sample_logits(logits, noise=None, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, counts=None, slots=None,
                  status=None):
    """(tokens int64, log-probabilities float32), each (B,) or (B, T): one token for each row of the logits.

    With d = (max - x) / temperature and w = exp(-d), tokens are ordered by (d, index).  Kept are the first top_k (all where
    top_k <= 0), of those the smallest prefix whose weights reach top_p of their sum (all where top_p >= 1), of those the ones
    with w >= min_p; the first always.  The token is the kept one with the largest w / noise, the lowest index of equals: with
    noise of the exponential distribution (torch.empty_like(logits, dtype=torch.float32).exponential_()) a draw by the kept
    weights.  Rows with a temperature of 0, and all rows without noise, take the largest logit.  The log-probability is that of
    the row's softmax at its temperature, before the filters (at a temperature of 1 in greedy rows).

    NaN counts as -inf, and tokens of -inf are never chosen; a row of nothing else gives -1 and -inf.  A row's result depends on
    that row alone.  Calls of one stream share a workspace, from any threads; graphs captured on one stream share it too, and are
    replayed one after another, or captured on streams of their own.  noise float32 in the logits' shape; top_k int32 where it is a tensor, the other parameters float32.
    counts (S, V) int32 or float32 with slots, for (B, V) logits: counts[slots[b], token] += 1, the next step's penalties.
    """
    B, T, V, seq_stride, pos_stride, last = _shape(logits)
    dev = logits.device
    if V < 1:
        raise ValueError("logits without a token to choose")
    if last != 1 and V > 1:
        logits = logits.contiguous()
        _, _, _, seq_stride, pos_stride, _ = _shape(logits)
    three = logits.dim() == 3
    nz = nz_seq = nz_pos = 0
    if noise is not None:
        _on(noise, dev, "noise")
        if noise.dtype is not torch.float32 or noise.shape != logits.shape:
            raise ValueError(f"noise must be float32 {tuple(logits.shape)} (got {noise.dtype} {tuple(noise.shape)})")
        if noise.stride(-1) != 1 and V > 1:
            noise = noise.contiguous()
        nz, nz_seq, nz_pos = noise.data_ptr(), noise.stride(0), noise.stride(1) if three else 0
    t_p, t = _per_sequence(temperature, torch.float32, B, dev, "temperature")
    k_p, k = _per_sequence(top_k, torch.int32, B, dev, "top_k")
    p_p, p = _per_sequence(top_p, torch.float32, B, dev, "top_p")
    m_p, m = _per_sequence(min_p, torch.float32, B, dev, "min_p")
    if counts is not None and three:
        raise ValueError("counts are kept for (B, V) logits: a block's accepted tokens are known only later")
    ct, ct_stride, ct_rows, ct_type, slots_p = _counts(counts, slots, B, V, dev)
    if three:
        token = torch.empty(B, T, dtype=torch.int64, device=dev)
        logprob = torch.empty(B, T, dtype=torch.float32, device=dev)
    else:
        token = torch.empty(B, dtype=torch.int64, device=dev)
        logprob = torch.empty(B, dtype=torch.float32, device=dev)
    if not (B and T):
        return token, logprob
    with on_device(dev), _LAUNCHES:
        ws = _workspace(dev)
        args = _lib.pack_sample(
            logits.data_ptr(), seq_stride, pos_stride, nz, nz_seq, nz_pos, t_p, k_p, p_p, m_p, token.data_ptr(),
            logprob.data_ptr(), ct, ct_stride, ct_rows, slots_p, _status(status, dev), ws.data_ptr(), ws.numel(), t, p, m,
            max(-1, min(int(k), 2 ** 31 - 1)), B, T, V, _DTYPES[logits.dtype], ct_type)  # in the order of the fields
        rc = _lib.load().logits_sample(args, stream_handle(dev))
        if rc > 0:  # a launch failed, after others perhaps: what they left in the workspace serves no further call
            retire(_WORKSPACES)
        _lib.check(rc)
    return token, logprob


def next_tokens(x, head: Int4Packed, noise=None, *, counts=None, slots=None, repetition=1.0, presence=0.0,
                frequency=0.0, bias_ids=None, bias_values=None, mask=None, mask_rows=None, temperature=1.0, top_k=0,
                top_p=1.0, min_p=0.0, status=None):
    """The end of a decode step: the output head's product with the last hidden states x (B, C) in fp32, the penalties, the
    draw, and the drawn tokens counted in `counts`.  Returns (tokens, log-probabilities), each (B,).  Arguments as in
    int4_matmul, penalize_logits and sample_logits; the whole can be recorded into a HIP graph."""
    if x.dim() != 2:
        raise ValueError(f"x must be (B, C), the hidden state of one token for each sequence (got {tuple(x.shape)})")
    logits = int4_matmul(x, head, out_dtype=torch.float32)
    penalize_logits(logits, counts=counts, slots=slots, repetition=repetition, presence=presence, frequency=frequency,
                    bias_ids=bias_ids, bias_values=bias_values, mask=mask, mask_rows=mask_rows, out=logits, status=status)
    return sample_logits(logits, noise, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, counts=counts,
                         slots=slots, status=status)
