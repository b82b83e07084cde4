"""The gated delta rule (rwkv-infer-next_amd/csrc/delta_*.hip) against the oracle in 64 bits.

u = 2^-24.  Token by token a step rounds the state K / 8 + 12 times at most along any path (the sum over K in eights, three sums over
lanes, the update), so its state is off by (K / 8 + 12) u of its size, 1.7e-6 at K = 128; a step's rule does not lengthen errors (|k| = 1,
beta <= 1, decays <= 1) and they go both ways: sqrt(T) of it over T tokens, in the 2-norm.  By chunks of 64 the sums of one chunk have
K + 2 64 terms, each product of three parts of 8 bits left to the last of 24: sqrt(K + 128) u, 1e-6, a chunk, in the same way.
An output is rounded to bf16 once: 8 significant bits, half a step is 2^-8 of the value at most; its sums keep 16 bits of both
factors: 2^-15."""
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


def _inputs(B, T, Hk, Hv, K, V, seed, norm=False, strong=False):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *n: torch.randn(*n, device=DEV, generator=gen)  # noqa: E731
    rand = lambda *n: torch.rand(*n, device=DEV, generator=gen)  # noqa: E731
    q, k, v = randn(B, T, Hk, K), randn(B, T, Hk, K), randn(B, T, Hv, V)
    if not norm:
        q, k = (x / x.square().sum(-1, keepdim=True).sqrt() for x in (q, k))
    g = -(1 + 15 * rand(Hv)) * torch.exp(rand(B, T, Hv) * 4.6 - 6.9)
    if strong:  # whole forgetting here and there
        g = torch.where(rand(B, T, Hv) < 0.2, -30 * rand(B, T, Hv), g)
    return [q.bfloat16(), k.bfloat16(), v.bfloat16(), g, torch.sigmoid(randn(B, T, Hv))]


def _np(x):
    return x.detach().double().cpu().numpy()


def _rel(got, want):
    return np.linalg.norm(_np(got) - want) / max(np.linalg.norm(want), 1e-30)


def _row(ops, n, first, len_, state, keep=None, **kw):
    return oracle.delta_ref.gated_delta_ref(*(_np(x[n, first:first + len_]) for x in ops), None if state is None else _np(state),
                                            keep=keep, **kw)


def _check(o, ht, ops, state, T, K, **kw):
    for n in range(ops[0].shape[0]):
        want, states = _row(ops, n, 0, T, None if state is None else state[n], **kw)
        if T:
            assert _rel(o[n], want) <= O_TOL, (n, _rel(o[n], want))
        assert _rel(ht[n], states[-1]) <= _tol(T, K), (n, _rel(ht[n], states[-1]), _tol(T, K))


SHAPES = [  # B, T, Hk, Hv, K, V
    (1, 1, 1, 1, 64, 64), (1, 1, 16, 32, 128, 128), (3, 1, 2, 6, 128, 64), (2, 2, 1, 4, 64, 16), (2, 5, 3, 3, 128, 48),
    (5, 8, 2, 2, 64, 256), (1, 16, 2, 2, 128, 128), (1, 17, 2, 4, 128, 128), (1, 33, 12, 12, 64, 64), (2, 63, 2, 2, 128, 128),
    (2, 64, 2, 2, 128, 128), (1, 65, 2, 4, 64, 80), (1, 127, 3, 3, 128, 16), (2, 129, 1, 2, 128, 96), (3, 200, 2, 4, 64, 64),
    (1, 500, 4, 4, 64, 64), (1, 640, 2, 4, 128, 128), (1, 1000, 1, 1, 128, 256),
]


@pytest.mark.parametrize("B,T,Hk,Hv,K,V", SHAPES)
@pytest.mark.parametrize("norm,with_state", [(False, True), (True, False), (True, True)])
def test_rows(B, T, Hk, Hv, K, V, norm, with_state):
    from rwkv_next_amd.kernels import gated_delta
    say("delta", B, T, Hk, Hv, K, V, norm, with_state)
    ops = _inputs(B, T, Hk, Hv, K, V, B + T + Hv, norm)
    state = torch.randn(B, Hv, K, V, device=DEV) * 0.2 if with_state else None
    was = None if state is None else state.clone()
    o, ht = gated_delta(*ops, state, qk_norm=norm)
    assert o.dtype == torch.bfloat16 and o.shape == (B, T, Hv, V) and ht.shape == (B, Hv, K, V)
    _check(o, ht, ops, state, T, K, qk_norm=norm)
    assert state is None or torch.equal(state, was)
    o2, none = gated_delta(*ops, state, qk_norm=norm, final=False)
    assert none is None and torch.equal(o2, o)


@pytest.mark.parametrize("token_len", [0, 1 << 30])
@pytest.mark.parametrize("T", [1, 3, 16, 64, 150])
def test_both_ways(T, token_len):
    """Token by token and by chunks, for lengths at which the library takes the other."""
    from rwkv_next_amd.kernels import gated_delta
    say("delta", T, token_len)
    ops = _inputs(2, T, 2, 4, 128, 128, T, True)
    state = torch.randn(2, 4, 128, 128, device=DEV)
    o, ht = gated_delta(*ops, state, qk_norm=True, token_len=token_len)
    _check(o, ht, ops, state, T, 128, qk_norm=True)


@pytest.mark.parametrize("T", [1, 7, 100, 300])
def test_strong_decays_and_scales(T):
    from rwkv_next_amd.kernels import gated_delta
    for kw in (dict(), dict(scale=1.0), dict(scale=0.0)):
        ops = _inputs(1, T, 1, 2, 64, 64, T, False, strong=True)
        state = torch.randn(1, 2, 64, 64, device=DEV) * 10
        o, ht = gated_delta(*ops, state, **kw)
        _check(o, ht, ops, state, T, 64, **kw)
    ops[3][:, T // 2] = float("-inf")  # a reset
    o, ht = gated_delta(*ops, state)
    _check(o, ht, ops, state, T, 64)
    ops[3][:, T // 2:] = -1000.0
    o, ht = gated_delta(*ops, state)
    _check(o, ht, ops, state, T, 64)
    ops[3].zero_()
    ops[4].fill_(1.0)  # nothing forgotten, everything replaced
    o, ht = gated_delta(*ops, state)
    _check(o, ht, ops, state, T, 64)
    ops[4].zero_()     # nothing written
    o, ht = gated_delta(*ops, state)
    assert torch.equal(ht, state)


@pytest.mark.parametrize("T", [4, 90])
def test_keys_alike(T):
    """The same key again and again, and zeros: the chunk's system is far from the identity."""
    from rwkv_next_amd.kernels import gated_delta
    ops = _inputs(1, T, 1, 1, 128, 128, 3)
    ops[1][:] = ops[1][:, :1]
    ops[3].mul_(0.01)
    ops[4].fill_(0.99)
    o, ht = gated_delta(*ops)
    _check(o, ht, ops, None, T, 128)
    ops[1].zero_()
    o, ht = gated_delta(*ops, qk_norm=True)  # 0 / sqrt(1e-6)
    assert not o.any() and not ht.any()


@pytest.mark.parametrize("lens", [[0], [1], [5, 0, 70], [1, 1, 1, 130, 1, 64, 0, 63], [300, 2, 129], [0, 0, 0], [16, 17, 200, 1]])
def test_ragged_pool(lens):
    from rwkv_next_amd.kernels import gated_delta_pool_, new_status
    say("ragged", lens)
    N, total, S = len(lens), sum(lens), len(lens) + 4
    ops = _inputs(1, total, 2, 4, 128, 64, total, True)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).int()
    pool = torch.randn(S, 4, 128, 64, device=DEV)
    slots = torch.randperm(S, device=DEV)[:N]
    fresh = torch.arange(N, device=DEV) % 3 == 2
    was, status = pool.clone(), new_status(DEV)
    o = gated_delta_pool_(*ops, pool, slots, cu_seqlens=cu, fresh=fresh, qk_norm=True, status=status)
    assert int(status) == 0
    first = 0
    for n, T in enumerate(lens):
        state = torch.zeros_like(was[0]) if fresh[n] else was[slots[n]]
        want, states = _row(ops, 0, first, T, state, qk_norm=True)
        if T:
            assert _rel(o[0, first:first + T], want) <= O_TOL
        assert _rel(pool[slots[n]], states[-1]) <= _tol(T, 128) or not states[-1].any() and not pool[slots[n]].any()
        first += T
    rest = torch.ones(S, dtype=torch.bool, device=DEV)
    rest[slots] = False
    assert torch.equal(pool[rest], was[rest])


def test_rows_behind_the_last_are_left():
    """Tokens past the last sequence, and past n_keep, are not written."""
    from rwkv_next_amd.kernels import gated_delta_pool_
    from rwkv_next_amd.kernels.gated_delta import _launch
    ops = _inputs(1, 200, 1, 2, 64, 64, 9)
    for token_len in (0, 1 << 30):
        o = torch.full((1, 200, 2, 64), 7.0, device=DEV, dtype=torch.bfloat16)
        cu = torch.tensor([3, 100, 150], device=DEV, dtype=torch.int32)
        _launch(*ops, o=o, cu=cu, scale=None, qk_norm=False, token_len=token_len)
        assert (o[0, :3] == 7).all() and (o[0, 150:] == 7).all() and not (o[0, 3:150] == 7).all(dim=(1, 2)).any()
    ops = _inputs(4, 90, 1, 2, 64, 64, 9)
    for token_len in (0, 1 << 30):
        pool = torch.randn(4, 2, 64, 64, device=DEV)
        was = pool.clone()
        keep = torch.tensor([0, 90, 70, 1000], device=DEV)
        gated_delta_pool_(*ops, pool, torch.arange(4, device=DEV), n_keep=keep, store_o=False, token_len=token_len)
        for n, T in enumerate((0, 90, 70, 90)):
            assert _rel(pool[n], _row(ops, n, 0, 90, was[n], keep=T)[1][-1]) <= _tol(T, 64)


def test_decode_verify_and_replay_give_the_same_bits():
    from rwkv_next_amd.kernels import SlotCaches, gated_delta_pool_
    B, T, S = 6, 5, 9
    ops = _inputs(B, T, 2, 4, 128, 128, 21, True)
    pool = torch.randn(S, 4, 128, 128, device=DEV)
    slots = torch.randperm(S, device=DEV)[:B]
    was = pool.clone()
    snaps = torch.empty(B, T, 4, 128, 128, device=DEV)
    o = gated_delta_pool_(*ops, pool, slots, qk_norm=True, final=False, snapshots=snaps)
    assert torch.equal(pool, was)
    steps = was.clone()
    for t in range(T):
        ot = gated_delta_pool_(*(x[:, t:t + 1] for x in ops), steps, slots, qk_norm=True)
        assert torch.equal(ot, o[:, t:t + 1]) and torch.equal(steps[slots], snaps[:, t])
    n = torch.tensor([0, 1, 2, 3, 4, 5], device=DEV)
    replayed, restored = was.clone(), was.clone()
    assert gated_delta_pool_(*ops, replayed, slots, qk_norm=True, n_keep=n, store_o=False) is None
    at = torch.where(n > 0, torch.arange(B, device=DEV) * T + n - 1, -1)
    SlotCaches((snaps.flatten(0, 1), 0)).copy_slots(at, slots, into=SlotCaches((restored, 0)))
    assert torch.equal(replayed, restored)
    assert torch.equal(restored[slots[0]], was[slots[0]]) and torch.equal(restored[slots[5]], steps[slots[5]])


@pytest.mark.parametrize("T", [1, 200])
def test_strides(T):
    """q, k, v as parts of one projection's result, g and beta of another; batches apart."""
    from rwkv_next_amd.kernels import gated_delta
    ops = _inputs(2, T, 2, 4, 128, 64, 5)
    state = torch.randn(2, 4, 128, 64, device=DEV)
    want = gated_delta(*ops, state)
    fused = torch.cat([x.flatten(2) for x in ops[:3]] + [ops[0].flatten(2)[..., :8]], dim=2)
    q, k, v = fused[..., :256].unflatten(2, (2, 128)), fused[..., 256:512].unflatten(2, (2, 128)), fused[..., 512:768].unflatten(2, (4, 64))
    gb = torch.cat([ops[3], ops[4]], dim=2)
    got = gated_delta(q, k, v, gb[..., :4], gb[..., 4:], state)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.cat([fused[..., :3], fused], dim=2)[..., 3:]  # not aligned
    got = gated_delta(odd[..., :256].unflatten(2, (2, 128)), ops[1].transpose(1, 2).contiguous().transpose(1, 2),
                      ops[2].repeat(1, 2, 1, 1)[:, :T], ops[3].transpose(0, 1).contiguous().transpose(0, 1), ops[4], state.transpose(2, 3).contiguous().transpose(2, 3))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_bad_indices_are_reported():
    from rwkv_next_amd.kernels import check_status, gated_delta_pool_, new_status
    ops = _inputs(1, 150, 1, 1, 64, 64, 2)
    pool = torch.randn(3, 1, 64, 64, device=DEV)

    def bits(ops=ops, **kw):
        status, p = new_status(DEV), pool.clone()
        slots = torch.tensor(kw.pop("slots"), device=DEV)
        for name in ("cu_seqlens", "n_keep"):
            if name in kw:
                kw[name] = torch.tensor(kw[name], device=DEV)
        o = gated_delta_pool_(*ops, p, slots, status=status, **kw)
        return int(status), o, p

    assert bits(slots=[1])[0] == 0
    got, o, p = bits(slots=[3])
    assert got == 2048 and torch.equal(p, pool)
    assert _rel(o[0], _row(ops, 0, 0, 150, None)[0]) <= O_TOL  # from zeros
    assert bits(slots=[-1])[0] == 2048
    assert bits(slots=[0, 1], cu_seqlens=[0, 100, 151])[0] == 4096
    assert bits(slots=[0, 1], cu_seqlens=[0, 100, 90])[0] == 4096
    assert bits(slots=[0, 1], cu_seqlens=[-5, 100, 150])[0] == 4096
    assert bits(slots=[0, 1], cu_seqlens=[120, 2 ** 30, 20])[0] == 4096
    assert bits(slots=[0], n_keep=[-1])[0] == 8192
    assert bits(slots=[1, 1], cu_seqlens=[0, 100, 150])[0] == 16384
    status = new_status(DEV)
    gated_delta_pool_(*ops, pool.clone(), torch.tensor([7], device=DEV), status=status)
    with pytest.raises(ValueError, match="gated_delta: a slot outside the pool"):
        check_status(status)


@pytest.mark.parametrize("T", [1, 5, 140])
def test_graph_and_streams(T):
    from rwkv_next_amd.kernels import gated_delta_pool_
    ops = _inputs(3, T, 2, 4, 128, 128, T)
    pool = torch.randn(5, 4, 128, 128, device=DEV)
    slots = torch.tensor([4, 0, 2], device=DEV)
    p = pool.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = gated_delta_pool_(*ops, p, slots)
    eager = pool.clone()
    p.copy_(pool)
    for step in range(4):
        want = gated_delta_pool_(*ops, eager, slots)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(p, eager), step
        slots.copy_(slots.roll(1) if step else torch.tensor([1, 3, 0], device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    was, mine = eager.clone(), eager.clone()
    with torch.cuda.stream(side):
        got = gated_delta_pool_(*ops, mine, slots)
    other = gated_delta_pool_(*ops, was, slots)  # at the same time
    torch.cuda.synchronize()
    assert torch.equal(got, other) and torch.equal(mine, was)


def test_values_that_are_not_finite_stay_in_their_head_and_row():
    from rwkv_next_amd.kernels import gated_delta
    for T in (4, 130):
        ops = _inputs(2, T, 2, 4, 64, 64, T)
        want = gated_delta(*ops)
        ops[2][1, T // 2, 2, 5] = float("nan")
        o, ht = gated_delta(*ops)
        assert torch.equal(o[0], want[0][0]) and torch.equal(ht[0], want[1][0])
        for h in (0, 1, 3):
            assert torch.equal(o[1, :, h], want[0][1, :, h]) and torch.equal(ht[1, h], want[1][1, h])
        assert torch.isnan(o[1, T // 2, 2, 5]) and torch.isnan(ht[1, 2, :, 5]).any()


def test_op_and_refusals():
    from rwkv_next_amd.kernels import gated_delta, gated_delta_pool_, gated_delta_pool_op
    ops = _inputs(2, 3, 2, 4, 64, 64, 1)
    pool, slots = torch.randn(4, 4, 64, 64, device=DEV), torch.tensor([2, 0], device=DEV)
    torch.library.opcheck(gated_delta_pool_op, (*ops, pool, slots, None, None, None, None, True, True, True, None, None, -1))
    q, k, v, g, b = ops
    cu = torch.tensor([0, 3], device=DEV)
    for bad in ((q.float(), k, v, g, b), (q, k, v, g.bfloat16(), b), (q, k, v, g, b.bfloat16()), (q.half(), k, v, g, b)):
        with pytest.raises(TypeError):
            gated_delta(*bad)
    for bad in ((q[..., :32], k[..., :32], v, g, b), (q, k[:, :2], v, g, b), (q, k, v[..., :8], g, b), (q, k, v[:, :, :3], g[:, :, :3], b[:, :, :3]),
                (q, k, v, g[..., :3], b), (q, k, v, g, b[:1]), (q.flatten(2), k, v, g, b), (q.cpu(), k.cpu(), v.cpu(), g.cpu(), b.cpu()),
                (q, k.cpu(), v, g, b)):
        with pytest.raises(ValueError):
            gated_delta(*bad)
    for kw in (dict(cu_seqlens=cu), dict(state=pool), dict(state=pool[:2].double()), dict(state=pool[:2, :3])):
        with pytest.raises(ValueError):
            gated_delta(*ops, **kw)
    snaps = torch.empty(2, 3, 4, 64, 64, device=DEV)
    for kw in (dict(pool=pool.half()), dict(pool=pool[:, :3]), dict(pool=pool.transpose(2, 3)), dict(slots=slots[:1]),
               dict(n_keep=slots[:1]), dict(fresh=slots[:1]), dict(snapshots=snaps[:1]), dict(snapshots=snaps.double()),
               dict(status=torch.zeros(1, device=DEV))):
        with pytest.raises(ValueError):
            gated_delta_pool_(*ops, kw.pop("pool", pool), kw.pop("slots", slots), **kw)
    one = [x.reshape(1, 6, *x.shape[2:]) for x in ops]
    with pytest.raises(ValueError):
        gated_delta_pool_(*one, pool, slots, cu_seqlens=torch.tensor([0, 3, 6], device=DEV), snapshots=snaps)
