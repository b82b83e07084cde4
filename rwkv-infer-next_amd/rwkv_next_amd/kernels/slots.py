"""The slots of a served model's caches (include/slots.h): copies and forks, compaction, freeing, over all tensors at once, beside
StatePool's reset_slots and move_slots (rwkv_next/model.py:310-316), which know one tensor of fp32 states.

    caches = SlotCaches(pool.wkv, (shifts, 1), (counts, 0))   # (layers, slots, ..) tensors, or (tensor, dimension of its slots)
    caches.copy_slots(src, dst)                # one source may go to many: a shared prompt forked
    caches.copy_slots(src, dst, into=other)    # to caches of as many slots as they like: a store of prompts, and back
    caches.free_slots(idx)                     # zeroed
    where, count = caches.compact_slots(live)  # live slots to the front; where each went

Indices are int64 on the device; one launch a call, on the current stream, no host sync, can be recorded into a HIP graph.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._workspace import on_device, stream_handle


def _apart(a, slots_a, b, slots_b):
    """Whether no slot of cache `a` shares memory with one of cache `b`, each (tensor, layer, slot, row, layers) with strides in bytes:
    their extents are apart, or both lie in one grid of slots (two ranges of a tensor's slots, or two parts of its rows)."""
    (t, layer, slot, row, layers), (u, layer_u, slot_u, row_u, layers_u) = a, b
    if not (row and layers and slots_a and row_u and layers_u and slots_b):
        return True
    end = t.data_ptr() + (layers - 1) * layer + (slots_a - 1) * slot + row
    end_u = u.data_ptr() + (layers_u - 1) * layer_u + (slots_b - 1) * slot_u + row_u
    if end <= u.data_ptr() or end_u <= t.data_ptr():
        return True
    if slots_a == 1 and layers == 1 or slots_b == 1 and layers_u == 1:
        return False
    inner, outer = (slot, layer) if layers == 1 or slot <= layer else (layer, slot)
    if {slot, layer if layers > 1 else 0} != {slot_u, layer_u if layers_u > 1 else 0}:
        return False
    far = u.data_ptr() - t.data_ptr()
    if outer % inner == 0 and row <= far % inner and far % inner + row_u <= inner:
        return True  # beside each other within every row of the grid
    if far % inner or not outer or (slot, layer) != (slot_u, layer_u) or slot > layer:
        return False
    first = far % outer // slot  # a layer's slots of `b` begin so many after those of `a`
    return slots_a <= first and (first + slots_b) * slot <= outer


_increment_version = torch.autograd.graph.increment_version


class SlotCaches:
    """A model's cache tensors that share their slots.  Each argument is a tensor (layers, slots, ..) or (tensor, dim) with dim 0 for
    (slots, ..) and 1 for (layers, slots, ..); a slot's part of a layer is contiguous.  At most 16 tensors, of any types.  A tensor that
    is given other memory or another shape later (t.data = .., set_, resize_) is taken as it is at a call."""

    def __init__(self, *caches):
        if not 1 <= len(caches) <= _lib.SLOTS_MAX_CACHES:
            raise ValueError(f"SlotCaches takes 1 to {_lib.SLOTS_MAX_CACHES} tensors (got {len(caches)})")
        self._caches = [x if isinstance(x, tuple) else (x, 1) for x in caches]
        self._lay_out()

    def _places(self):
        """What the layout follows from, of every tensor."""
        return [(t.data_ptr(), t.shape, t.stride(), t.dtype, t.get_device()) for t, _ in self._caches]

    def _current(self):
        """Before every call: addresses are those that the tensors have now."""
        if self._places() != self._laid:
            self._lay_out()

    def _lay_out(self):
        """All of it, taken when it is found right."""
        places, rows, slots, device, shared = self._places(), [], None, None, False
        for t, dim in self._caches:
            if dim not in (0, 1) or t.dim() <= dim:
                raise ValueError(f"the slots are dimension 0 or 1 of a cache (got dimension {dim} of {tuple(t.shape)})")
            if not t.is_cuda:
                raise ValueError(f"caches must be on a GPU (got {t.device})")
            if device is None:
                device, slots = t.device, t.shape[dim]
            if t.device != device or t.shape[dim] != slots:
                raise ValueError(f"caches must have {slots} slots on {device} (got {t.shape[dim]} on {t.device})")
            layers, shape, strides, size = t.shape[0] if dim else 1, t.shape[dim + 1:], t.stride(), t.element_size()
            row = 1
            for n, s in zip(reversed(shape), reversed(strides[dim + 1:])):
                if n > 1 and s != row:
                    raise ValueError(f"a slot's part of a cache must be contiguous (got {tuple(t.shape)}, strides {strides})")
                row *= n
            row *= size
            slot = strides[dim] * size if slots > 1 else row
            layer = strides[0] * size if dim and layers > 1 else 0
            if row and (slot < row or (layers > 1 and layer < row)):
                raise ValueError(f"slots of a cache must not share memory (got {tuple(t.shape)}, strides {strides})")
            # layers outside slots or within them, but not interlocked
            if row and layers > 1 and slots > 1 and layer < slots * slot and slot < layers * layer:
                raise ValueError(f"slots of a cache must not share memory (got {tuple(t.shape)}, strides {strides})")
            rows.append((t, layer, slot, row, layers))
            shared |= not all(_apart(rows[-1], slots, x, slots) for x in rows[:-1])
        self._rows, self.slots, self.device, self._shared = rows, slots, device, shared
        self._own, self._laid = self._pairs(self), places

    def _pairs(self, other):
        a = (_lib.SlotsCache * len(self._rows))()
        for x, (t, layer, slot, row, layers), (u, to_layer, to_slot, to_row, to_layers) in zip(a, self._rows, other._rows):
            if (row, layers) != (to_row, to_layers) or t.dtype != u.dtype:
                raise ValueError(f"caches of one shape but for their slots are needed (got {tuple(t.shape)}, {tuple(u.shape)})")
            x.from_, x.to, x.from_layer_stride, x.from_slot_stride = t.data_ptr(), u.data_ptr(), layer, slot
            x.to_layer_stride, x.to_slot_stride, x.row_bytes, x.layers = to_layer, to_slot, row, layers
        return a

    def _index(self, x, name):
        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(x, dtype=torch.int64, device=self.device)
        if x.device != self.device:
            raise ValueError(f"{name} must be on {self.device} (got {x.device})")
        if x.dtype is not torch.int64 or x.dim() != 1:
            raise ValueError(f"{name} must be an int64 tensor of one dimension (got {x.dtype} {tuple(x.shape)})")
        return x.contiguous()

    def _written(self):
        """In place, as autograd is told."""
        for t, _ in self._caches:
            if not t.is_inference():
                _increment_version(t)

    def _require_apart(self):
        if self._shared:
            raise ValueError("caches whose slots move must not share memory with each other")

    def _status(self, status):
        if status is None:
            return None
        if status.device != self.device or status.dtype != torch.int32 or status.numel() < 1:
            raise ValueError(f"status must be an int32 tensor on {self.device} (new_status)")
        return status.data_ptr()

    def copy_slots(self, src, dst, *, into: "SlotCaches | None" = None, status=None) -> None:
        """into's slot dst[i] = this one's slot src[i] (into: these caches themselves where None, or caches apart from them), as if all sources were read
        before any destination is written: swaps and chains are exact.  A source may be named any number of times; of equal
        destinations the last one counts.  A negative index leaves its entry out, one past the slots does too and sets
        SLOTS_STATUS_SLOT in `status`.  At most 1024 entries."""
        self._current()
        src, dst = self._index(src, "src"), self._index(dst, "dst")
        n = src.numel()
        if n != dst.numel():
            raise ValueError(f"src and dst must have the same length (got {n} and {dst.numel()})")
        if n > _lib.SLOTS_MAX_PAIRS:
            raise ValueError(f"at most {_lib.SLOTS_MAX_PAIRS} copies per call (got {n})")
        a, to = self._own, self.slots
        self._require_apart()
        if into is not None and into is not self:
            into._current()
            into._require_apart()
            if into.device != self.device or len(into._rows) != len(self._rows):
                raise ValueError(f"into must be {len(self._rows)} caches on {self.device}")
            for x in self._rows:
                for y in into._rows:
                    if not _apart(x, self.slots, y, into.slots):
                        raise ValueError("into must not share memory with these caches, but for being the same")
            a, to = self._pairs(into), into.slots
        with on_device(self.device):
            _lib.check(_lib.load().slots_copy(a, len(a), src.data_ptr(), dst.data_ptr(), n, self.slots, to,
                                              self._status(status), stream_handle(self.device)))
        (self if into is None else into)._written()

    def free_slots(self, idx, *, status=None) -> None:
        """Slot idx[i] = 0 in every cache, indices as in copy_slots.  At most 65535."""
        self._current()
        idx = self._index(idx, "idx")
        if idx.numel() > 65535:
            raise ValueError(f"at most 65535 slots per call (got {idx.numel()})")
        with on_device(self.device):
            _lib.check(_lib.load().slots_free(self._own, len(self._own), idx.data_ptr(), idx.numel(), self.slots,
                                              self._status(status), stream_handle(self.device)))
        self._written()

    def compact_slots(self, live):
        """Moves the live slots to the front: with k the number of live ones (live (S,) bool), those at k and behind go, in their
        order, to the free ones before k, in theirs.  Returns (where, count): where (S,) int64 a slot's place after, -1 for a free
        one, count (1,) int32 k, both on the device.  Slots that nothing moves to keep what they hold (free_slots zeroes)."""
        self._current()
        if not isinstance(live, torch.Tensor) or live.device != self.device or live.dtype not in (torch.bool, torch.uint8) or \
                live.shape != (self.slots,):
            raise ValueError(f"live must be a bool ({self.slots},) tensor on {self.device}")
        self._require_apart()
        if self.slots > _lib.SLOTS_MAX_COMPACT:
            raise ValueError(f"at most {_lib.SLOTS_MAX_COMPACT} slots are compacted (got {self.slots})")
        live = live.contiguous()
        where = torch.empty(self.slots, dtype=torch.int64, device=self.device)
        count = torch.empty(1, dtype=torch.int32, device=self.device)
        with on_device(self.device):
            _lib.check(_lib.load().slots_compact(self._own, len(self._own), live.data_ptr(), self.slots, where.data_ptr(),
                                                 count.data_ptr(), stream_handle(self.device)))
        self._written()
        return where, count
