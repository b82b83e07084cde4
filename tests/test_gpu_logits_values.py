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


@pytest.mark.parametrize("kw", [dict(), dict(top_k=50), dict(top_p=0.9)])
def test_sums_lean_to_no_side(kw):
    """The mean error of 256 rows' log-probabilities at a temperature of 1, logits in whole 1024ths, so that every d is exact.  What may
    lean to one side is the exponential instruction's last place, for a bin's first weight and for a weight in its bin, 2^-23 each;
    roundings go both ways and leave less than 0.6e-7 in a mean over 256: 3e-7."""
    from rwkv_next_amd import kernels
    say("sample sums", kw)
    rng = np.random.default_rng(3)
    x = np.round(rng.standard_normal((256, 4096)) * 2048) / 1024
    x[:, :40] += 4
    noise = rng.exponential(size=x.shape)
    token, logprob = kernels.sample_logits(_dev(x.astype(np.float32)), _dev(noise.astype(np.float32)), **kw)
    d = x.max(axis=1, keepdims=True) - x
    want = -d[np.arange(256), token.cpu().numpy()] - np.log(np.exp(-d).sum(axis=1))
    error = (logprob.double().cpu().numpy() - want).mean()
    assert abs(error) <= 3e-7, error


@pytest.mark.parametrize("kw", [dict(), dict(top_k=2), dict(top_k=3, min_p=0.0)])
def test_rare_tokens_have_their_weight(kw):
    """Two tokens, d apart, their noise such that one's score is 5e-7 to 1.5e-6 above the other's.  A weight is off by the exponential
    instruction's last place (2^-23) and two roundings, a score by one more: 3e-7 in all for a ratio of two."""
    from rwkv_next_amd import kernels
    say("sample rare tokens", kw)
    rng = np.random.default_rng(4)
    n = 3000
    d = np.round(rng.uniform(1, 30, n) * 1024) / 1024
    x = np.full((n, 16), -np.inf, np.float32)
    x[:, 3], x[:, 9] = 0.0, -d
    noise = np.ones((n, 16), np.float32)
    noise[:, 3] = rng.uniform(0.5, 2, n)
    noise[:, 9] = noise[:, 3] * np.exp(-d) * (1 + rng.choice([-1, 1], n) * rng.uniform(5.5e-7, 1.5e-6, n))
    first, second = 1 / noise[:, 3].astype(np.float64), np.exp(-d) / noise[:, 9].astype(np.float64)
    sure = np.abs(first / second - 1) >= 5e-7
    assert sure.sum() > n * 0.9
    token, _ = kernels.sample_logits(_dev(x), _dev(noise), **kw)
    want = np.where(first > second, 3, 9)
    got = token.cpu().numpy()
    wrong = sure & (got != want)
    assert not wrong.any(), (int(wrong.sum()), d[wrong][:8])


@pytest.mark.parametrize("kw", [dict(), dict(top_k=2), dict(top_p=0.9)])
def test_scores_of_very_large_and_small_noise(kw):
    """Scores below the normal numbers and noise whose reciprocal is none still have their order."""
    from rwkv_next_amd import kernels
    say("sample noise at its ends", kw)
    x = torch.tensor([[0.0, -1.0], [-1.0, 0.0]], device=DEV)
    big = torch.tensor([[3e38, 1e38], [1e38, 2.9e38]], device=DEV)    # 1 / 3e38 < e^-1 / 1e38, and so in the second row
    assert kernels.sample_logits(x, big, **kw)[0].tolist() == [1, 0]
    x = torch.tensor([[-1.0, 0.0]], device=DEV)
    small = torch.tensor([[5e-39, 6e-39]], device=DEV)                # e^-1 / 5e-39 < 1 / 6e-39, both finite
    assert kernels.sample_logits(x, small, **kw)[0].tolist() == [1]


@pytest.mark.parametrize("kw", [dict(), dict(top_k=4), dict(top_p=0.99)])
def test_noise_of_nothing_and_below(kw):
    """A noise of 0 wins, the lowest index of several; negative, infinite or no noise never does, and where nothing else is left the
    largest logit is taken.  Equal quotients of different tokens: the lowest index."""
    from rwkv_next_amd import kernels
    say("sample noise at and below 0", kw)
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[0.0, -1.0, -0.5, -2.0]], device=DEV)
    for noise, want in (([1.0, 0.0, 1e-30, 0.0], 1), ([1.0, -1e-3, 2.0, 0.2], 0), ([-1.0, nan, inf, -0.5], 0), ([inf, nan, -1.0, 5.0], 3)):
        assert kernels.sample_logits(x, torch.tensor([noise], device=DEV), **kw)[0].tolist() == [want], noise
    x = torch.zeros(1, 50, device=DEV)
    noise = torch.full((1, 50), 3.0, device=DEV)
    noise[0, 30:] = 0.1
    assert kernels.sample_logits(x, noise, **dict(kw, **({"top_k": 45} if "top_k" in kw else {})))[0].tolist() == [30]


@pytest.mark.parametrize("V", [131072, 131074, 600000, 2097152])
def test_one_bin_of_a_whole_vocabulary(V):
    """Equal logits: a bin's word holds V tokens at its first weight.  A top-p of a half keeps the first half, a top-k of k the first k;
    the logarithm of V is off by its function's last place and a rounding: 2e-6."""
    from rwkv_next_amd import kernels
    say("sample one bin", V)
    x, noise = torch.zeros(1, V, device=DEV), torch.ones(1, V, device=DEV)
    for last, kw in ((V // 2 - 1, dict(top_p=0.5)), (V - 8, dict(top_k=V - 7)), (99, dict(top_k=100)), (V - 1, dict())):
        noise[0, last:last + 2] = torch.tensor([1e-3, 1e-6], device=DEV)[:V - last]  # the token after the last one would win
        token, logprob = kernels.sample_logits(x, noise, **kw)
        assert int(token) == last and abs(float(logprob) + np.log(V)) <= 2e-6, kw
        noise.fill_(1)


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
