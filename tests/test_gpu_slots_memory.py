"""SlotCaches whose tensors are given other memory or another shape after it was made: every call takes them as they are."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _idx(*x):
    return torch.tensor(x, device=DEV)


def _fresh(*n):
    return torch.arange(1, torch.Size(n).numel() + 1, device=DEV, dtype=torch.float32).view(n)


@pytest.mark.parametrize("how", ["data", "set_", "resize_", "storage"])
def test_other_memory_is_followed(how):
    from rwkv_next_amd.kernels import SlotCaches
    t, u = _fresh(3, 6, 8), _fresh(6, 5)
    caches = SlotCaches(t, (u, 0))
    keep = t.detach()  # the old memory stays, so that a write to it would show
    was = keep.clone()
    if how == "data":
        t.data = _fresh(3, 6, 8) * 2
    elif how == "set_":
        t.set_(_fresh(3, 6, 8) * 2)
    elif how == "resize_":
        keep, was = None, None
        t.resize_(4, 6, 8)  # more layers: memory of its own, larger
        t.copy_(_fresh(4, 6, 8))
    else:
        keep, was = None, None
        t.untyped_storage().resize_(2 * t.untyped_storage().nbytes())
        t.copy_(_fresh(3, 6, 8))
    want, other = t.clone(), u.clone()
    want[:, 1], other[1] = t[:, 4], u[4]
    caches.copy_slots(_idx(4), _idx(1))
    assert torch.equal(t, want) and torch.equal(u, other)
    want[:, 5], other[5] = 0, 0
    caches.free_slots(_idx(5))
    assert torch.equal(t, want) and torch.equal(u, other)
    live = torch.tensor([False, True, True, True, True, False], device=DEV)
    want[:, 0], other[0] = t[:, 4], u[4]
    where, count = caches.compact_slots(live)
    assert torch.equal(t, want) and torch.equal(u, other) and int(count) == 4 and where.tolist() == [-1, 1, 2, 3, 0, -1]
    assert keep is None or torch.equal(keep, was)


def test_other_memory_of_into_is_followed():
    from rwkv_next_amd.kernels import SlotCaches
    t, u = _fresh(3, 6, 8), _fresh(3, 9, 8)
    here, there = SlotCaches(t), SlotCaches(u)
    keep = u.detach()
    was = keep.clone()
    u.data = _fresh(3, 20, 8) * 2  # more slots too
    want = u.clone()
    want[:, 17] = t[:, 2]
    here.copy_slots(_idx(2), _idx(17), into=there)
    assert torch.equal(u, want) and torch.equal(keep, was) and there.slots == 20


def test_what_no_longer_fits_is_refused():
    from rwkv_next_amd.kernels import SlotCaches
    t, u = _fresh(3, 6, 8), _fresh(6, 5)
    caches = SlotCaches(t, (u, 0))
    live = torch.ones(6, dtype=torch.bool, device=DEV)
    calls = (lambda: caches.copy_slots(_idx(0), _idx(1)), lambda: caches.free_slots(_idx(0)), lambda: caches.compact_slots(live))
    for bad in (_fresh(3, 7, 8), _fresh(3, 6, 16)[..., ::2], torch.zeros(3, 6, 8), _fresh(1, 6, 8).expand(3, 6, 8)):
        t.data = bad
        was, other = t.clone(), u.clone()
        for call in calls:  # again and again, not the first time alone
            with pytest.raises(ValueError):
                call()
        assert torch.equal(t, was) and torch.equal(u, other) and caches.slots == 6 and caches.device == u.device
    t.data = u.view(1, 6, 5)  # the other cache's memory
    for call in (calls[0], calls[2]):
        with pytest.raises(ValueError, match="share memory"):
            call()
    t.data = _fresh(3, 6, 8)
    for call in calls:
        call()
    assert not t[:, 0].any() and not u[0].any() and torch.equal(t[:, 1], _fresh(3, 6, 8)[:, 0])


def test_a_captured_call_keeps_the_memory_of_its_capture():
    """A graph holds addresses, as torch's own do: later memory is taken by later calls."""
    from rwkv_next_amd.kernels import SlotCaches
    t = _fresh(2, 4, 8)
    caches = SlotCaches(t)
    src, dst = _idx(0), _idx(3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        caches.copy_slots(src, dst)
    keep = t.detach()
    t.data = _fresh(2, 4, 8) * 3
    new = t.clone()
    for _ in range(3):
        keep.copy_(_fresh(2, 4, 8))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(keep[:, 3], keep[:, 0]) and torch.equal(t, new)
    caches.copy_slots(src, dst)
    assert torch.equal(t[:, 3], new[:, 0])


def test_autograd_is_told_of_what_is_written():
    from rwkv_next_amd.kernels import SlotCaches
    t, u, v = _fresh(2, 4, 8), _fresh(4, 3), _fresh(2, 9, 8)
    caches, other = SlotCaches(t, (u, 0)), SlotCaches(v, (_fresh(9, 3), 0))
    live = torch.tensor([False, True, True, False], device=DEV)
    for call in (lambda: caches.copy_slots(_idx(0), _idx(1)), lambda: caches.free_slots(_idx(3)), lambda: caches.compact_slots(live)):
        w = torch.ones(2, 4, 8, device=DEV, requires_grad=True)
        versions = t._version, u._version
        y = (w * t).sum()
        call()
        assert t._version > versions[0] and u._version > versions[1]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    versions = t._version, u._version, v._version
    caches.copy_slots(_idx(0), _idx(8), into=other)  # read alone
    assert (t._version, u._version) == versions[:2] and v._version > versions[2]
    with torch.inference_mode():  # inference tensors have no counter
        SlotCaches(_fresh(2, 4, 8)).copy_slots(_idx(0), _idx(1))
        caches.free_slots(_idx(0))
    assert not t[:, 0].any()


def test_as_many_slots_are_freed_as_a_call_may_name():
    """65535 slots in three caches of 61 layers: more than a launch has workgroups for, were each to have one slot."""
    from rwkv_next_amd.kernels import SlotCaches, new_status
    S, n = 70000, 65535
    gen = torch.Generator(device=DEV).manual_seed(1)
    caches = [torch.randint(1, 100, (61, S, w), device=DEV, generator=gen, dtype=torch.uint8) for w in (1, 2, 16)]
    idx = torch.randperm(S + 500, device=DEV, generator=gen)[:n]
    idx[5::1000] = -1
    want, status = [t.clone() for t in caches], new_status(DEV)
    for t in want:
        t[:, idx[(idx >= 0) & (idx < S)]] = 0
    SlotCaches(*caches).free_slots(idx, status=status)
    assert int(status) == 1024 and all(torch.equal(t, w) for t, w in zip(caches, want))
