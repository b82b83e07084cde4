"""Values that are not finite in the gated delta rule, token by token and by chunks of 64: what they may reach.  The rule makes a column of
a head's state from that column of v alone, one token after another, so a value of token t that is not finite reaches token t and those
behind it in its column (v) or its head (k, g, beta), and nothing else, to the bit: the same products of the same numbers."""
import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")
BY = {"chunks": 0, "tokens": 1 << 30}


def _inputs(B, T, Hk, Hv, K, V, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *n: torch.randn(*n, device=DEV, generator=gen)  # noqa: E731
    q, k, v = randn(B, T, Hk, K), randn(B, T, Hk, K), randn(B, T, Hv, V)
    q, k = (x / x.square().sum(-1, keepdim=True).sqrt() for x in (q, k))
    g = -torch.rand(B, T, Hv, device=DEV, generator=gen) * 0.2
    return [q.bfloat16(), k.bfloat16(), v.bfloat16(), g, torch.sigmoid(randn(B, T, Hv))], randn(B, Hv, K, V)


def _bits(x):
    return x.contiguous().view({2: torch.int16, 4: torch.int32}[x.element_size()])


def _check(got, want, clean):
    """`clean` of the outputs has the bits of `want`; the rest is not finite."""
    assert torch.equal(_bits(got)[clean], _bits(want)[clean])
    assert torch.isfinite(want).all() and not torch.isfinite(got)[~clean].any()


@pytest.mark.parametrize("by", BY)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("t", [0, 1, 20, 31, 32, 50, 63, 64, 85, 127, 129])
@pytest.mark.parametrize("what,value", [("v", NAN), ("v", -INF), ("k", NAN), ("k", INF), ("g", NAN), ("beta", NAN), ("beta", INF)])
@pytest.mark.parametrize("K,V", [(64, 48), (128, 64)])
def test_nothing_before_it_or_beside_it(K, V, what, value, t, norm, by):
    from rwkv_next_amd.kernels import gated_delta
    say("not finite", K, V, what, value, t, norm, by)
    B, T, Hk, Hv = 2, 130, 2, 4
    ops, state = _inputs(B, T, Hk, Hv, K, V, 5 * t + K)
    want = gated_delta(*ops, state, qk_norm=norm, token_len=BY[by])
    reached, column = slice(2, 3), slice(None)
    if what == "v":
        ops[2][1, t, 2, 5], column = value, slice(5, 6)
    elif what == "k":
        ops[1][1, t, 1, 9], reached = value, slice(2, 4)  # both value heads of that key head
    else:
        ops[3 if what == "g" else 4][1, t, 2] = value
    got = gated_delta(*ops, state, qk_norm=norm, token_len=BY[by])
    clean = torch.ones(B, T, Hv, V, dtype=torch.bool, device=DEV)
    clean[1, t:, reached, column] = False
    _check(got[0], want[0], clean)
    clean = torch.ones(B, Hv, K, V, dtype=torch.bool, device=DEV)
    clean[1, reached, :, column] = False
    _check(got[1], want[1], clean)


@pytest.mark.parametrize("by", BY)
@pytest.mark.parametrize("t", [0, 40, 100])
def test_a_query_reaches_its_own_output(t, by):
    from rwkv_next_amd.kernels import gated_delta
    ops, state = _inputs(1, 130, 2, 4, 64, 64, t)
    want = gated_delta(*ops, state, token_len=BY[by])
    ops[0][0, t, 0, 3] = NAN
    got = gated_delta(*ops, state, token_len=BY[by])
    clean = torch.ones_like(want[0], dtype=torch.bool)
    clean[0, t, :2] = False
    _check(got[0], want[0], clean)
    assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("by", BY)
def test_a_state_reaches_its_column(by):
    from rwkv_next_amd.kernels import gated_delta
    ops, state = _inputs(2, 130, 2, 4, 128, 64, 1)
    want = gated_delta(*ops, state, token_len=BY[by])
    for value in (NAN, INF):
        dirty = state.clone()
        dirty[0, 3, 77, 20] = value
        got = gated_delta(*ops, dirty, token_len=BY[by])
        clean = torch.ones_like(want[0], dtype=torch.bool)
        clean[0, :, 3, 20] = False
        _check(got[0], want[0], clean)
        clean = torch.ones_like(want[1], dtype=torch.bool)
        clean[0, 3, :, 20] = False
        _check(got[1], want[1], clean)


@pytest.mark.parametrize("K,V", [(128, 128), (64, 160)])
def test_many_ragged_rows(K, V):
    """By 32 columns a workgroup; several tokens of a row, of which the first counts; rows beside it."""
    from rwkv_next_amd.kernels import gated_delta
    lens = [70 + 3 * i for i in range(40)]
    at = np.cumsum([0] + lens)
    ops, _ = _inputs(1, int(at[-1]), 2, 16, K, V, 3)
    state = torch.randn(40, 16, K, V, device=DEV)
    cu = torch.tensor(at, device=DEV).int()
    want = gated_delta(*ops, state, cu_seqlens=cu, token_len=0)
    out, fin = torch.ones_like(want[0], dtype=torch.bool), torch.ones_like(want[1], dtype=torch.bool)
    for n, h, c, tokens in ((0, 0, 0, (69, 3)), (7, 15, 127, (40, 41)), (20, 5, 17, (64,)), (39, 9, 16, (186, 100, 130))):
        for t in tokens:
            ops[2][0, at[n] + t, h, c] = NAN
        out[0, at[n] + min(tokens):at[n + 1], h, c] = False
        fin[n, h, :, c] = False
    ops[4][0, at[30] + 50, 2] = NAN
    out[0, at[30] + 50:at[31], 2] = False
    fin[30, 2] = False
    got = gated_delta(*ops, state, cu_seqlens=cu, token_len=0)
    _check(got[0], want[0], out)
    _check(got[1], want[1], fin)


@pytest.mark.parametrize("by", BY)
@pytest.mark.parametrize("size", [2.0, 4.0, 40.0])
def test_states_that_leave_the_range(by, size):
    """The same long key again and again multiplies the state by 1 - size^2 a token, until it leaves fp32.  Tokens whose state in 64 bits
    is below 1e25 are finite: the products on their way, of at most 64 terms and factors of size^2, stay below 1e38."""
    from rwkv_next_amd.kernels import gated_delta
    T, K = 192, 64
    ops, _ = _inputs(1, T, 1, 1, K, 16, 1)
    ops[1][:] = ops[1][:, :1] * size
    ops[3].zero_()
    ops[4].fill_(1.0)
    o, _ = gated_delta(*ops, token_len=BY[by])
    with np.errstate(over="ignore", invalid="ignore"):
        _, states = oracle.delta_ref.gated_delta_ref(*(x[0].double().cpu().numpy() for x in ops))
    small = np.array([np.abs(s).max() < 1e25 for s in states[1:]])
    assert 3 < small.sum() < T and not small[small.argmin():].any()
    assert torch.isfinite(o[0, torch.from_numpy(small).to(DEV)]).all()
