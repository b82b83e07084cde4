"""The slot operators (rwkv-infer-next_amd/csrc/slots.hip): they move bytes, so all results are compared bit for bit with plain
indexing on the host."""
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _caches(S, gen, layers=3):
    """Tensors of every alignment, some of them parts of larger ones."""
    ints = lambda *n: torch.randint(-2 ** 31, 2 ** 31 - 1, n, device=DEV, generator=gen, dtype=torch.int32)  # noqa: E731
    big = ints(layers, S + 5, 70)
    return [
        (ints(layers, S, 5, 64, 8), 1),                                       # 16-byte units
        (ints(layers, S, 3).view(torch.float32).view(layers, S, 3), 1),        # 4-byte units
        (ints(layers, S, 9).to(torch.int16), 1),                               # 2-byte units
        (ints(S, 7).to(torch.uint8), 0),                                       # bytes, and no layers
        (big[:, 2:S + 2, 3:67], 1),                                            # a part of another tensor
        (ints(S, layers, 16).transpose(0, 1), 1),                              # slots outside layers
        (ints(S, 65536 // 4), 0),
        (ints(layers, S), 1),                                                  # a number a slot
        (ints(layers, S, 0), 1),                                               # nothing
    ]


def _host(caches):
    return [t.cpu().clone() for t, _ in caches]


def _same(caches, want):
    return all(torch.equal(t.cpu().view(w.shape).view(torch.uint8) if t.is_contiguous() else t.cpu().contiguous().view(torch.uint8),
                           w.contiguous().view(torch.uint8)) for (t, _), w in zip(caches, want) if w.numel())


def _copy(host, to, caches, src, dst):
    """All sources first, then the destinations in their order."""
    for h, t, (_, dim) in zip(host, to, caches):
        was = h.clone()
        S, S2 = h.shape[dim], t.shape[dim]
        for s, d in zip(src, dst):
            if 0 <= s < S and 0 <= d < S2:
                t.select(dim, d).copy_(was.select(dim, s))


@pytest.mark.parametrize("S,src,dst", [
    (1, [0], [0]), (2, [0], [1]), (2, [0, 1], [1, 0]), (9, [3, 3, 3, 3], [0, 1, 2, 8]),
    (9, [0, 1, 2, 3, 4], [1, 2, 3, 4, 5]),          # a chain
    (9, [7, 6, 5, 7], [1, 1, 1, 2]),                # one destination three times: the last counts
    (9, [1, 1, 4], [2, 1, 4]),                      # a slot onto itself
    (9, [4, 0, 2], [0, 4, 4]),                      # a swap that a later entry overrules
    (9, [], []), (5, [-1, 2, 3], [0, -7, 4]),       # unused entries
    (5, [5, 2, 99, 1], [0, 5, 3, 2]),               # past the slots
])
def test_copy(S, src, dst):
    from rwkv_next_amd.kernels import SlotCaches, new_status
    say("copy", S, src, dst)
    caches = _caches(S, torch.Generator(device=DEV).manual_seed(S))
    want, status = _host(caches), new_status(DEV)
    _copy(want, want, caches, src, dst)
    SlotCaches(*caches).copy_slots(torch.tensor(src, device=DEV, dtype=torch.int64), torch.tensor(dst, device=DEV, dtype=torch.int64),
                                   status=status)
    assert _same(caches, want)
    assert int(status) == (1024 if any(x >= S for x in src + dst) else 0)


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 63, 64, 65, 255, 256, 257, 700, 1024])
def test_copy_many(n):
    """Every size of a range, permutations with repeated sources and destinations, within 600 slots."""
    from rwkv_next_amd.kernels import SlotCaches
    say("copy", n)
    S, gen = 600, torch.Generator(device=DEV).manual_seed(n)
    caches = _caches(S, gen, layers=2)
    src = torch.randint(0, S, (n,), device=DEV, generator=gen)
    dst = torch.randint(0, S, (n,), device=DEV, generator=gen)
    want = _host(caches)
    _copy(want, want, caches, src.tolist(), dst.tolist())
    SlotCaches(*caches).copy_slots(src, dst)
    assert _same(caches, want)


def test_copy_into_other_caches_and_back():
    from rwkv_next_amd.kernels import SlotCaches
    gen = torch.Generator(device=DEV).manual_seed(1)
    here, there = _caches(7, gen), _caches(40, gen)
    want, other = _host(here), _host(there)
    a, b = SlotCaches(*here), SlotCaches(*there)
    idx = lambda *x: torch.tensor(x, device=DEV)  # noqa: E731
    _copy(want, other, here, [6, 0, 6], [39, 2, 0])
    a.copy_slots(idx(6, 0, 6), idx(39, 2, 0), into=b)
    assert _same(here, want) and _same(there, other)
    _copy(other, want, here, [39, 39, 8], [1, 2, 6])
    b.copy_slots(idx(39, 39, 8), idx(1, 2, 6), into=a)
    assert _same(here, want) and _same(there, other)


@pytest.mark.parametrize("S,idx", [(4, [0]), (9, [8, 1, 1, -3, 4]), (9, []), (6, [6, 2, 1 << 40])])
def test_free(S, idx):
    from rwkv_next_amd.kernels import SlotCaches, new_status
    say("free", S, idx)
    caches = _caches(S, torch.Generator(device=DEV).manual_seed(S))
    want, status = _host(caches), new_status(DEV)
    for h, (_, dim) in zip(want, caches):
        for i in idx:
            if 0 <= i < S:
                h.select(dim, i).zero_()
    SlotCaches(*caches).free_slots(torch.tensor(idx, device=DEV, dtype=torch.int64), status=status)
    assert _same(caches, want)
    assert int(status) == (1024 if any(x >= S for x in idx) else 0)


def _compacted(live):
    """(where, count, moves) from the definition."""
    k = sum(live)
    holes, movers = [s for s in range(k) if not live[s]], [s for s in range(k, len(live)) if live[s]]
    where = [s if on else -1 for s, on in enumerate(live)]
    for h, m in zip(holes, movers):
        where[m] = h
    return where, k, list(zip(movers, holes))


@pytest.mark.parametrize("S", [1, 2, 3, 64, 65, 255, 256, 257, 1000, 8192])
@pytest.mark.parametrize("share", [0.0, 0.02, 0.5, 0.97, 1.0, "last", "alternating"])
def test_compact(S, share):
    from rwkv_next_amd.kernels import SlotCaches
    say("compact", S, share)
    gen = torch.Generator(device=DEV).manual_seed(S)
    caches = [(torch.randint(0, 2 ** 31 - 1, (2, S, 20), device=DEV, generator=gen, dtype=torch.int32), 1),
              (torch.randint(0, 2 ** 31 - 1, (S, 3), device=DEV, generator=gen, dtype=torch.int32).to(torch.int16), 0)]
    if share == "last":
        live = torch.arange(S, device=DEV) == S - 1
    elif share == "alternating":
        live = torch.arange(S, device=DEV) % 2 == 1
    else:
        live = torch.rand(S, device=DEV, generator=gen) < share
    where, k, moves = _compacted(live.tolist())
    want = _host(caches)
    _copy(want, want, caches, [m for m, _ in moves], [h for _, h in moves])
    got, count = SlotCaches(*caches).compact_slots(live)
    assert _same(caches, want) and got.tolist() == where and int(count) == k
    got, count = SlotCaches(*caches).compact_slots(torch.arange(S, device=DEV) < k)  # nothing left to do
    assert _same(caches, want) and got.tolist() == [s if s < k else -1 for s in range(S)] and int(count) == k


def test_compact_every_alignment():
    from rwkv_next_amd.kernels import SlotCaches
    gen = torch.Generator(device=DEV).manual_seed(2)
    caches = _caches(50, gen)
    live = torch.rand(50, device=DEV, generator=gen) < 0.6
    _, _, moves = _compacted(live.tolist())
    want = _host(caches)
    _copy(want, want, caches, [m for m, _ in moves], [h for _, h in moves])
    SlotCaches(*caches).compact_slots(live.to(torch.uint8) * 3)  # any value but 0 is live
    assert _same(caches, want)


def test_offsets_past_32_bits():
    from rwkv_next_amd.kernels import SlotCaches
    t = torch.zeros(2, 4200, 1 << 20, device=DEV, dtype=torch.uint8)
    mark = torch.arange(1 << 20, device=DEV).to(torch.uint8)
    t[:, 4199], t[:, 5] = mark, 7
    caches = SlotCaches(t)
    caches.copy_slots(torch.tensor([4199, 5], device=DEV), torch.tensor([1, 4198], device=DEV))
    assert torch.equal(t[1, 1], mark) and (t[1, 4198] == 7).all() and torch.equal(t[0, 1], mark) and not t[:, 2].any()
    live = torch.zeros(4200, dtype=torch.bool, device=DEV)
    live[4198:] = True
    where, count = caches.compact_slots(live)
    assert where[4198:].tolist() == [0, 1] and int(count) == 2 and (t[1, 0] == 7).all() and torch.equal(t[1, 1], mark)
    caches.free_slots(torch.tensor([4199, 0], device=DEV))
    assert not t[:, 4199].any() and not t[:, 0].any() and torch.equal(t[0, 1], mark)


def test_graph():
    """The indices and the plan are the device's: a captured step follows them."""
    from rwkv_next_amd.kernels import SlotCaches
    gen = torch.Generator(device=DEV).manual_seed(4)
    caches = _caches(12, gen)
    c = SlotCaches(*caches)
    src, dst = torch.tensor([0, 0], device=DEV), torch.tensor([1, 2], device=DEV)
    idx, live = torch.tensor([3], device=DEV), torch.ones(12, dtype=torch.bool, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.copy_slots(src, dst)
        c.free_slots(idx)
        where, count = c.compact_slots(live)
    for step in range(4):
        say("replay", step)
        src.copy_(torch.randint(0, 12, (2,), device=DEV, generator=gen))
        dst.copy_(torch.randperm(12, device=DEV, generator=gen)[:2])
        idx.copy_(torch.randint(0, 12, (1,), device=DEV, generator=gen))
        live.copy_(torch.rand(12, device=DEV, generator=gen) < 0.5)
        want = _host(caches)
        _copy(want, want, caches, src.tolist(), dst.tolist())
        for h, (_, dim) in zip(want, caches):
            h.select(dim, int(idx)).zero_()
        w, k, moves = _compacted(live.tolist())
        _copy(want, want, caches, [m for m, _ in moves], [h for _, h in moves])
        g.replay()
        torch.cuda.synchronize()
        assert _same(caches, want) and where.tolist() == w and int(count) == k


def test_refusals():
    from rwkv_next_amd.kernels import SlotCaches
    t = torch.zeros(2, 6, 8, device=DEV)
    i = torch.tensor([0], device=DEV)
    for bad in ((), (t,) * 17, (t.cpu(),), ((t, 2),), (torch.zeros(6, device=DEV),), (t, torch.zeros(2, 7, 8, device=DEV)),
                (t[..., ::2],), (t[:, :1].expand(2, 6, 8),), (t[:1].expand(2, 6, 8),),
                (torch.zeros(400, device=DEV).as_strided((2, 6, 8), (16, 8, 1)),)):
        with pytest.raises(ValueError):
            SlotCaches(*bad)
    c = SlotCaches(t)
    for src, dst in ((i, i.int()), (i, i.cpu()), (i, i[None]), (i, torch.tensor([0, 1], device=DEV)),
                     (torch.zeros(1025, dtype=torch.int64, device=DEV),) * 2):
        with pytest.raises(ValueError):
            c.copy_slots(src, dst)
    for other in (SlotCaches(t, t), SlotCaches(torch.zeros(2, 6, 9, device=DEV)), SlotCaches(torch.zeros(3, 6, 8, device=DEV)),
                  SlotCaches(torch.zeros(2, 6, 8, device=DEV, dtype=torch.int32))):
        with pytest.raises(ValueError):
            c.copy_slots(i, i, into=other)
    for live in (torch.ones(5, dtype=torch.bool, device=DEV), torch.ones(6, device=DEV), torch.ones(6, dtype=torch.bool)):
        with pytest.raises(ValueError):
            c.compact_slots(live)
    with pytest.raises(ValueError):
        SlotCaches((torch.zeros(8193, 1, device=DEV), 0)).compact_slots(torch.ones(8193, dtype=torch.bool, device=DEV))
    with pytest.raises(ValueError):
        c.free_slots(i.float())
    with pytest.raises(ValueError):
        c.free_slots(i, status=torch.zeros(1, device=DEV))
