"""Which caches SlotCaches takes for apart, against the bytes of their slots counted one by one (no GPU: the rule looks at addresses and
strides alone)."""
import random

import pytest

pytest.importorskip("torch")

from rwkv_next_amd.kernels.slots import _apart  # noqa: E402


class _At:
    def __init__(self, at):
        self.at = at

    def data_ptr(self):
        return self.at


def _bytes(at, layer, slot, row, layers, slots):
    return {at + i * layer + j * slot + k for i in range(layers) for j in range(slots) for k in range(row)}


def test_never_apart_where_a_byte_is_shared():
    rng = random.Random(5)
    seen = [0, 0]
    for _ in range(40000):
        sides = []
        grid = (rng.choice((2, 4, 8)), rng.choice((8, 16, 24, 32)))
        for _ in range(2):
            layers, slots, row = rng.randint(1, 3), rng.randint(1, 4), rng.randint(0, 4)
            slot, layer = grid if rng.random() < 0.8 else (rng.randint(1, 9), rng.randint(1, 40))
            if rng.random() < 0.2:
                slot, layer = layer, slot
            if slots == 1:  # as SlotCaches has them: a row within its slot and layer, slots and layers not interlocked
                slot = row
            if layers == 1:
                layer = 0
            if row > slot or layers > 1 and (row > layer or slots > 1 and layer < slots * slot and slot < layers * layer):
                slots = layers = 1
                slot, layer = row, 0
            sides.append(((_At(rng.randint(0, 70)), layer, slot, row, layers), slots))
        (a, m), (b, n) = sides
        shared = _bytes(a[0].at, *a[1:4], a[4], m) & _bytes(b[0].at, *b[1:4], b[4], n)
        got = _apart(a, m, b, n)
        assert not (got and shared), (a[0].at, a[1:], m, b[0].at, b[1:], n)
        assert got == _apart(b, n, a, m) or not shared
        seen[got] += 1
    assert min(seen) > 1000


@pytest.mark.parametrize("a,m,b,n", [
    ((0, 64, 16, 16, 3), 2, (32, 64, 16, 16, 3), 2),     # two ranges of the slots of (layers, 4, 16) bytes
    ((0, 64, 16, 8, 3), 4, (8, 64, 16, 8, 3), 4),        # two parts of every row
    ((0, 16, 64, 8, 4), 3, (8, 16, 64, 8, 4), 3),        # layers within slots
    ((0, 0, 16, 16, 1), 2, (32, 0, 16, 16, 1), 5),       # one after the other
    ((0, 64, 16, 0, 3), 2, (0, 64, 16, 16, 3), 2)])      # an empty row
def test_parts_of_one_tensor_are_apart(a, m, b, n):
    assert _apart((_At(a[0]), *a[1:]), m, (_At(b[0]), *b[1:]), n) and _apart((_At(b[0]), *b[1:]), n, (_At(a[0]), *a[1:]), m)


@pytest.mark.parametrize("b,n", [((0, 64, 16, 16, 3), 4), ((16, 64, 16, 16, 3), 3), ((48, 64, 16, 16, 2), 2), ((8, 64, 16, 16, 3), 4),
                                 ((0, 0, 16, 16, 1), 4), ((64, 0, 16, 4, 1), 1)])
def test_parts_that_share_slots_are_not(b, n):
    assert not _apart((_At(0), 64, 16, 16, 3), 4, (_At(b[0]), *b[1:]), n)
