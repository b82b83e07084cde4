"""Ragged calls of the gated delta rule with many rows, of which few or none run by chunks.  Tolerances as in test_gpu_gated_delta.py: a state is
off by sqrt(T) (K / 8 + 12) 2^-24 of its size, an output by 2^-8 + 2^-15."""
import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
O_TOL = 2.0 ** -8 + 2.0 ** -15


def _inputs(total, Hk, Hv, K, V, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *n: torch.randn(*n, device=DEV, generator=gen)  # noqa: E731
    g = -torch.rand(1, total, Hv, device=DEV, generator=gen) * 0.2
    return [randn(1, total, Hk, K).bfloat16(), randn(1, total, Hk, K).bfloat16(), randn(1, total, Hv, V).bfloat16(), g,
            torch.sigmoid(randn(1, total, Hv))]


def _np(x):
    return x.detach().double().cpu().numpy()


def _rel(got, want):
    return np.linalg.norm(_np(got) - want) / max(np.linalg.norm(want), 1e-30)


@pytest.mark.parametrize("token_len", [-1, 0, 3, 31, 100])
@pytest.mark.parametrize("K,V", [(64, 32), (128, 16)])
def test_few_long_rows_among_many_short_ones(K, V, token_len):
    from rwkv_next_amd.kernels import gated_delta_pool_, new_status
    lens = [1] * 400
    for at, n in ((0, 17), (1, 18), (7, 33), (50, 64), (51, 65), (52, 16), (200, 2), (201, 130), (333, 0), (334, 32), (399, 200)):
        lens[at] = n
    say("ragged", K, V, token_len)
    total, Hk, Hv = sum(lens), 1, 2
    ops = _inputs(total, Hk, Hv, K, V, K)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    was = torch.randn(410, Hv, K, V, device=DEV)
    slots = torch.randperm(410, device=DEV)[:400]
    pool, status = was.clone(), new_status(DEV)
    o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=cu, qk_norm=True, status=status, token_len=token_len)
    assert int(status) == 0
    first = 0
    for n, T in enumerate(lens):
        want, states = oracle.delta_ref.gated_delta_ref(*(_np(x[0, first:first + T]) for x in ops), _np(was[slots[n]]), qk_norm=True)
        if T:
            assert _rel(o[0, first:first + T], want) <= O_TOL, (n, T)
        assert _rel(pool[slots[n]], states[-1]) <= max(1.0, T) ** 0.5 * (K / 8 + 12) * 2.0 ** -24, (n, T)
        first += T
    rest = torch.ones(410, dtype=torch.bool, device=DEV)
    rest[slots] = False
    assert torch.equal(pool[rest], was[rest])


def test_a_step_of_single_tokens_needs_little_memory():
    """1024 rows, 32 heads of 128 x 128: what the call allocates besides its output is in proportion to the tokens, and its bits are those
    of the same rows in a dense call."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    N, Hk, Hv, K, V = 1024, 16, 32, 128, 128
    ops = _inputs(N, Hk, Hv, K, V, 1)
    was = torch.randn(8, Hv, K, V, device=DEV)
    slots = torch.full((N,), -1, device=DEV)
    slots[100:108] = torch.randperm(8, device=DEV)
    pool, dense = was.clone(), was.clone()
    cu = torch.arange(N + 1, device=DEV, dtype=torch.int32)
    gated_delta_pool_(*ops, was.clone(), slots, cu_seqlens=cu, qk_norm=True)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=cu, qk_norm=True)
    # the output, and a slot for each 16 tokens and one, of K, Q, K^T and a record of each value head
    allowed = o.numel() * 2 + (N // 16 + 1) * (Hk * 3 * K * 64 * 2 + Hv * 32000) + (1 << 22)
    assert torch.cuda.max_memory_allocated() - before <= allowed
    o2 = gated_delta_pool_(*(x.transpose(0, 1) for x in ops), dense, slots, qk_norm=True)
    assert torch.equal(o[0], o2[:, 0]) and torch.equal(pool, dense)


def test_many_rows_of_many_heads():
    """8192 single tokens of 128 heads: more than a launch by chunks could hold if every row ran so."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    N, Hv, K, V = 8192, 128, 64, 256
    ops = _inputs(N, 1, Hv, K, V, 2)
    pool = torch.randn(2, Hv, K, V, device=DEV)
    was = pool.clone()
    slots = torch.full((N,), -1, device=DEV)
    slots[4321], slots[8191] = 1, 0
    o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=torch.arange(N + 1, device=DEV, dtype=torch.int32), qk_norm=True)
    for n in (0, 4321, 8191):
        state = None if slots[n] < 0 else _np(was[slots[n]])
        want, states = oracle.delta_ref.gated_delta_ref(*(_np(x[0, n:n + 1]) for x in ops), state, qk_norm=True)
        assert _rel(o[0, n:n + 1], want) <= O_TOL
        if state is not None:
            assert _rel(pool[slots[n]], states[-1]) <= (K / 8 + 12) * 2.0 ** -24


@pytest.mark.parametrize("rows,total", [(40, 300), (4, 700)])
def test_a_captured_call_follows_its_offsets(rows, total):
    """One graph, other rows at every replay: which of them run by chunks, and where these lie, is found on the device."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    Hk, Hv, K, V = 1, 2, 64, 32
    ops = _inputs(total, Hk, Hv, K, V, rows)
    rng = np.random.default_rng(rows)
    pool = torch.randn(rows, Hv, K, V, device=DEV)
    mine, slots = pool.clone(), torch.randperm(rows, device=DEV)
    cu = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
    keep = torch.full((rows,), 1000, device=DEV)
    gated_delta_pool_(*ops, mine, slots, cu_seqlens=cu, n_keep=keep, qk_norm=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = gated_delta_pool_(*ops, mine, slots, cu_seqlens=cu, n_keep=keep, qk_norm=True)
    for replay in range(6):
        ends = np.sort(rng.integers(0, total + 1, rows - 1)) if replay % 2 else np.minimum(np.arange(1, rows) + (total - rows if replay else 0), total)
        cu.copy_(torch.tensor([0, *ends, total], dtype=torch.int32))
        keep.copy_(torch.from_numpy(rng.integers(0, 200, rows)))
        mine.copy_(pool)
        graph.replay()
        torch.cuda.synchronize()
        eager = pool.clone()
        want = gated_delta_pool_(*ops, eager, slots, cu_seqlens=cu, n_keep=keep, qk_norm=True)
        assert torch.equal(mine, eager), replay
        for n, (a, b) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
            b = min(b, a + int(keep[n]))
            assert torch.equal(o[0, a:b], want[0, a:b]), (replay, n)
            ref, states = oracle.delta_ref.gated_delta_ref(*(_np(x[0, a:b]) for x in ops), _np(pool[slots[n]]), qk_norm=True)
            assert b == a or _rel(o[0, a:b], ref) <= O_TOL, (replay, n)
            assert _rel(mine[slots[n]], states[-1]) <= max(1.0, b - a) ** 0.5 * (K / 8 + 12) * 2.0 ** -24, (replay, n)
