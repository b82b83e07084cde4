"""The delta rule and the slot operators where there is nothing: no rows, no tokens, no slots, no entries; and limits past every size."""
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _ops(B, T, Hk=1, Hv=2, K=64, V=32):
    r = lambda *n: torch.randn(*n, device=DEV)  # noqa: E731
    return [r(B, T, Hk, K).bfloat16(), r(B, T, Hk, K).bfloat16(), r(B, T, Hv, V).bfloat16(), -torch.rand(B, T, Hv, device=DEV),
            torch.rand(B, T, Hv, device=DEV)]


@pytest.mark.parametrize("B,T", [(0, 0), (0, 5), (0, 100), (3, 0)])
def test_no_rows_or_no_tokens(B, T):
    from rwkv_next_amd.kernels import gated_delta, gated_delta_pool_
    state = torch.randn(B, 2, 64, 32, device=DEV)
    o, ht = gated_delta(*_ops(B, T), state)
    assert o.shape == (B, T, 2, 32) and torch.equal(ht, state)
    assert not gated_delta(*_ops(B, T))[1].any()
    pool = torch.randn(4, 2, 64, 32, device=DEV)
    was = pool.clone()
    assert gated_delta_pool_(*_ops(B, T), pool, torch.arange(B, device=DEV)).shape == (B, T, 2, 32) and torch.equal(pool, was)
    fresh = torch.ones(B, dtype=torch.bool, device=DEV)
    gated_delta_pool_(*_ops(B, T), pool, torch.arange(B, device=DEV), fresh=fresh)
    assert not pool[:B].any() and torch.equal(pool[B:], was[B:])


def test_no_ragged_rows():
    from rwkv_next_amd.kernels import gated_delta_pool_, new_status
    pool = torch.randn(4, 2, 64, 32, device=DEV)
    was, status = pool.clone(), new_status(DEV)
    for total in (0, 50):
        gated_delta_pool_(*_ops(1, total), pool, torch.arange(0, device=DEV), cu_seqlens=torch.tensor([0], device=DEV), status=status)
        gated_delta_pool_(*_ops(1, total), pool, torch.arange(3, device=DEV), cu_seqlens=torch.tensor([0] * 4, device=DEV), status=status)
    assert torch.equal(pool, was) and int(status) == 0


@pytest.mark.parametrize("token_len", [1 << 31, sys.maxsize])
@pytest.mark.parametrize("T", [1, 40])
def test_a_token_len_past_every_length(T, token_len):
    from rwkv_next_amd.kernels import gated_delta
    ops = _ops(2, T)
    want, got = gated_delta(*ops, token_len=1 << 30), gated_delta(*ops, token_len=token_len)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_no_slots():
    from rwkv_next_amd.kernels import SlotCaches, new_status
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    empty = SlotCaches(torch.zeros(2, 0, 8, device=DEV), (torch.zeros(0, 3, device=DEV), 0))
    empty.copy_slots(none, none)
    empty.free_slots(none)
    where, count = empty.compact_slots(torch.zeros(0, dtype=torch.bool, device=DEV))
    assert where.shape == (0,) and int(count) == 0
    t, u = torch.randn(2, 5, 8, device=DEV), torch.randn(5, 3, device=DEV)
    was, other = t.clone(), u.clone()
    some = SlotCaches(t, (u, 0))
    one = torch.tensor([0], device=DEV)
    for call in (lambda s: empty.copy_slots(one, one, status=s), lambda s: empty.free_slots(one, status=s),
                 lambda s: empty.copy_slots(one, one, into=some, status=s), lambda s: some.copy_slots(one, one, into=empty, status=s),
                 lambda s: SlotCaches(torch.zeros(2, 5, 0, device=DEV)).free_slots(one + 5, status=s)):  # past the slots, of which there are none
        status = new_status(DEV)
        call(status)
        assert int(status) == 1024
    assert torch.equal(t, was) and torch.equal(u, other)
