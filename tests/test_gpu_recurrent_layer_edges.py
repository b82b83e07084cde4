"""The gated delta rule, the products and the slots where calls meet each other and the ends of their operands.  Tolerances of the delta rule as
in test_gpu_gated_delta.py: a state is off by sqrt(T) (K / 8 + 12) 2^-24 of its size, an output by 2^-8 + 2^-15."""
import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
O_TOL = 2.0 ** -8 + 2.0 ** -15


def _tol(T, K):
    return max(1.0, T) ** 0.5 * (K / 8 + 12) * 2.0 ** -24


def _np(x):
    return x.detach().double().cpu().numpy()


def _rel(got, want):
    return np.linalg.norm(_np(got) - want) / max(np.linalg.norm(want), 1e-30)


def _inputs(total, Hk, Hv, K, V, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *n: torch.randn(*n, device=DEV, generator=gen)  # noqa: E731
    g = -torch.rand(1, total, Hv, device=DEV, generator=gen) * 0.2
    return [randn(1, total, Hk, K).bfloat16(), randn(1, total, Hk, K).bfloat16(), randn(1, total, Hv, V).bfloat16(), g,
            torch.sigmoid(randn(1, total, Hv))]


def _same(x, y):
    """To the bit (keys are not normalised here: some states grow until they are not numbers)."""
    size = {2: torch.int16, 4: torch.int32}[x.element_size()]
    return torch.equal(x.view(size), y.view(size))


def _check_rows(ops, lens, o, pool, was, slots, K, first=0):
    for n, T in enumerate(lens):
        want, states = oracle.delta_ref.gated_delta_ref(*(_np(x[0, first:first + T]) for x in ops), _np(was[slots[n]]), qk_norm=True)
        if T:
            assert _rel(o[0, first:first + T], want) <= O_TOL, (n, T)
        assert _rel(pool[slots[n]], states[-1]) <= _tol(T, K), (n, T)
        first += T


@pytest.mark.parametrize("lens", [
    [17000, 3, 64, 16321, 0, 200],                       # rows of more chunks than the order of rows tells apart
    [1 + 13 * i % 150 for i in range(300)],              # more rows than one pass of the ordering workgroup takes
    [0] * 270 + [40] + [0] * 30 + [1, 18, 17, 16],
])
def test_ragged_rows_of_every_kind_together(lens):
    from rwkv_next_amd.kernels import gated_delta_pool_, new_status
    say("ragged", len(lens), max(lens))
    N, total, Hk, Hv, K, V = len(lens), sum(lens), 1, 2, 64, 16
    ops = _inputs(total, Hk, Hv, K, V, N)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    was = torch.randn(N, Hv, K, V, device=DEV)
    slots = torch.randperm(N, device=DEV)
    pool, status = was.clone(), new_status(DEV)
    o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=cu, qk_norm=True, status=status)
    assert int(status) == 0
    _check_rows(ops, lens, o, pool, was, slots, K)
    for _ in range(3):  # the order of rows is free, results are not
        again = was.clone()
        assert torch.equal(gated_delta_pool_(*ops, again, slots, cu_seqlens=cu, qk_norm=True), o) and torch.equal(again, pool)


@pytest.mark.parametrize("Hk,Hv,K,V", [(4, 16, 64, 64), (8, 8, 128, 96), (2, 16, 128, 128)])
def test_many_rows_by_wide_columns(Hk, Hv, K, V):
    """Enough rows for 32 columns a workgroup."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    lens = [70 + 3 * i for i in range(40)]
    ops = _inputs(sum(lens), Hk, Hv, K, V, K + V)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    was = torch.randn(40, Hv, K, V, device=DEV)
    slots = torch.randperm(40, device=DEV)
    pool = was.clone()
    o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=cu, qk_norm=True)
    _check_rows(ops, lens[:4], o, pool, was, slots[:4], K)
    _check_rows(ops, lens[-3:], o, pool, was, slots[-3:], K, first=sum(lens[:-3]))


@pytest.mark.parametrize("token_len", [0, 1 << 30])
def test_nothing_behind_the_last_token_is_used(token_len):
    """NaN in the tokens before the first and behind the last row, and behind n_keep, reaches nothing."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    for cu, keep in (([5, 90, 171], None), ([0, 90, 180], [70, 33])):
        ops = _inputs(180, 2, 4, 128, 64, 3)
        cu = torch.tensor(cu, device=DEV, dtype=torch.int32)
        nk = None if keep is None else torch.tensor(keep, device=DEV)
        was = torch.randn(2, 4, 128, 64, device=DEV)
        slots = torch.arange(2, device=DEV)
        pool = was.clone()
        o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=cu, n_keep=nk, qk_norm=True, token_len=token_len)
        used = torch.zeros(180, dtype=torch.bool, device=DEV)
        for n in range(2):
            used[int(cu[n]):min(int(cu[n + 1]), int(cu[n]) + (1000 if keep is None else keep[n]))] = True
        for x in ops:
            x[:, ~used] = float("nan")
        again = was.clone()
        o2 = gated_delta_pool_(*ops, again, slots, cu_seqlens=cu, n_keep=nk, qk_norm=True, token_len=token_len)
        assert torch.equal(pool, again) and torch.isfinite(pool).all()
        assert torch.equal(o2[:, used], o[:, used]) and torch.isfinite(o2[:, used]).all()


@pytest.mark.parametrize("T", [1, 5, 100])
def test_an_eager_call_is_the_op(T):
    from rwkv_next_amd.kernels import gated_delta_pool_, gated_delta_pool_op
    ops = [x.reshape(2, T, *x.shape[2:]) for x in _inputs(2 * T, 2, 4, 64, 64, T)]
    was, slots = torch.randn(4, 4, 64, 64, device=DEV), torch.tensor([3, 1], device=DEV)
    one, two = was.clone(), was.clone()
    version = one._version
    o = gated_delta_pool_(*ops, one, slots)
    assert one._version == version + 1  # written in place, as autograd is told
    assert _same(gated_delta_pool_op(*ops, two, slots, None, None, None, None, False, True, True, None, None, -1), o)
    assert _same(one, two)
    with torch.inference_mode():
        three = was.clone()
        assert _same(gated_delta_pool_(*ops, three, slots), o) and _same(three, one)
    need = [x.clone().requires_grad_() for x in ops]
    four = was.clone()
    got = gated_delta_pool_(*need, four, slots)
    assert not got.requires_grad and _same(got, o) and _same(four, one)


def test_indices_of_any_kind():
    """Slots as a list, of another type, strided: taken as they are meant."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    ops = [x.reshape(2, 3, *x.shape[2:]) for x in _inputs(6, 1, 2, 64, 64, 1)]
    was = torch.randn(4, 2, 64, 64, device=DEV)
    want = was.clone()
    o = gated_delta_pool_(*ops, want, torch.tensor([3, 1], device=DEV), qk_norm=True, n_keep=torch.tensor([2, 3], device=DEV))
    for slots in ([3, 1], torch.tensor([3, 1]), torch.tensor([3, 1], device=DEV, dtype=torch.int32),
                  torch.tensor([3, 7, 1, 7], device=DEV)[::2]):
        pool = was.clone()
        assert torch.equal(gated_delta_pool_(*ops, pool, slots, qk_norm=True, n_keep=[2, 3])[1], o[1]) and torch.equal(pool, want)


def test_caches_that_share_memory():
    from rwkv_next_amd.kernels import SlotCaches
    gen = torch.Generator(device=DEV).manual_seed(3)
    both = torch.randn(3, 12, 5, device=DEV, generator=gen)
    low, high = SlotCaches(both[:, :8]), SlotCaches(both[:, 8:])
    want = both.clone()
    want[:, 8 + 2], want[:, 8] = both[:, 7], both[:, 1]
    low.copy_slots(torch.tensor([7, 1], device=DEV), torch.tensor([2, 0], device=DEV), into=high)
    assert torch.equal(both, want)
    idx = torch.tensor([0], device=DEV)
    for other in (both[:, 1:9], both[:, 7:], both.view(torch.int32)[:, :8], both[1:, :8].flatten(2)):
        with pytest.raises(ValueError, match="share memory|one shape"):
            low.copy_slots(idx, idx, into=SlotCaches(other))
    live = torch.ones(12, dtype=torch.bool, device=DEV)
    for pair in ((both, both), (both, (both[0], 0)), (both, both.view(torch.int32))):
        caches = SlotCaches(*pair)
        caches.free_slots(idx)  # the same zeros twice
        for call in (lambda: caches.copy_slots(idx, idx), lambda: caches.compact_slots(live),
                     lambda: caches.copy_slots(idx, idx, into=caches)):
            with pytest.raises(ValueError, match="share memory"):
                call()
    SlotCaches(both[..., :3].contiguous(), both).copy_slots(idx, idx)


def test_products_of_one_weight_from_two_threads():
    import threading
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    gen = torch.Generator(device=DEV).manual_seed(4)
    w = (torch.randn(4128, 2564, device=DEV, generator=gen) / 64).bfloat16()
    p = prepack_dense(w)
    a = [torch.randn(n, 4128, device=DEV, generator=gen).bfloat16() for n in (7, 130)]
    want = [dense_matmul(x, p) for x in a]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(dense_matmul(a[i], p), want[i]):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
