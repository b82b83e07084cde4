"""Values of the sampling kernels (rwkv-infer-next_amd/csrc/logits_sample.hip) that looser comparisons let through."""
import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def test_greedy_rows_have_a_temperature_of_one():
    """Rows without noise are greedy: whatever their temperature, the log-probability is that of the plain softmax."""
    from rwkv_next_amd import kernels
    say("sample greedy log-probabilities")
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((5, 1, 3001)) * 3).astype(np.float32)
    logits = _dev(x[:, 0])
    want, want_lp = kernels.sample_logits(logits)
    for t in (0.6, 2.5, torch.tensor([0.3, 0.0, 1.0, 7.0, -1.0], device=DEV)):
        token, logprob = kernels.sample_logits(logits, temperature=t, top_k=4, top_p=0.7)
        assert torch.equal(token, want) and torch.equal(logprob, want_lp)
    for b in range(5):
        ok, lp = oracle.logits_ref.choices_ref(x[b, 0], None, 0.6, 0, 1.0, 0.0, 1e-6)
        assert ok == {int(want[b])} and abs(float(want_lp[b]) - lp[int(want[b])]) <= 1e-5 * (1 + abs(lp[int(want[b])]))


@pytest.mark.parametrize("kw", [dict(), dict(min_p=0.01), dict(top_p=0.9), dict(top_k=40)])
def test_a_row_has_the_same_bits_beside_others(kw):
    """80 rows of 66000 go by segments of 8192 elements, one row by segments of 2048.  In every other row only such tokens are allowed
    as one thread of a long segment has, four of a short one's."""
    from rwkv_next_amd import kernels
    say("sample rows by themselves", kw)
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((80, 66000)) * 2).astype(np.float32)
    near = np.arange(66000) % 2048 < 8
    near[8192:] = False
    x[::2, ~near] = -np.inf
    x, noise = _dev(x), _dev(rng.exponential(size=(80, 66000)).astype(np.float32))
    temperature = _dev(rng.uniform(0.5, 1.8, 80).astype(np.float32))
    temperature[7] = 0
    token, logprob = kernels.sample_logits(x, noise, temperature=temperature, **kw)
    for b in range(80):
        one, one_lp = kernels.sample_logits(x[b:b + 1], noise[b:b + 1], temperature=temperature[b:b + 1].clone(), **kw)
        assert int(one) == int(token[b]) and float(one_lp) == float(logprob[b]), b


def test_top_p_at_a_bins_end():
    """The first bin's weight is half of all, to the last bit of the sums: whether that reaches a top-p of a half or needs one token more,
    it never takes all of the next bin.  Logits are at the starts of bins, 32nds below the largest, so many tokens at each."""
    from rwkv_next_amd import kernels
    say("sample top-p at a bin's end")
    at = [0] * 7 + [55] * 3 + [56] * 35 + [59, 67, 88, 126, 150, 188, 208, 219, 255, 275, 343, 364, 381, 385, 395, 505, 682, 878, 1009]
    x = torch.full((1, 200), -np.inf)
    x[0, :len(at)] = -torch.tensor(at) / 32
    noise = torch.ones(1, 200)
    noise[0, 9] = 1e-6  # the last of the second bin
    token, _ = kernels.sample_logits(x.to(DEV), noise.to(DEV), top_p=0.5)
    assert int(token) == 0
