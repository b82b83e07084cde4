"""The choice of a token (rwkv-infer-next_amd/csrc/logits_sample.hip) against the oracle in 64 bits, at the sizes, filters and
values where it can go wrong.

The kernel's weights are off by a few ulp of fp32: d = (max - x) / T is rounded three times, w = exp2(c d) adds the rounding of
c d, of at most 1.44 * 30 * 2^-24 in the exponent for weights that matter, and the instruction's ulp; a bin's weights are whole
numbers of 2^-20 of their bin's first.  Together below 8e-6: SLACK.  A token is right when it is one that some weights within
SLACK of the exact ones give; tokens of the same logit are ordered by their index, exactly.  The log-probability is off by the
roundings of d and of the sum: 1e-5 (1 + its size)."""
import math

import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SLACK = 8e-6
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _draws(rng, shape):
    return rng.exponential(size=shape).astype(np.float32)


def _peaked(rng, B, T, V, dtype="f32"):
    """Logits of a language model: a bulk and some tokens that stand out."""
    x = rng.standard_normal((B, T, V)) * 2
    for b in range(B):
        for t in range(T):
            at = rng.integers(0, V, min(V, 40))
            x[b, t, at] = 14 - 1.5 * rng.exponential(size=at.size)
    return torch.from_numpy(x.astype(np.float32)).to(DTYPES[dtype])


def _check(x, noise, token, logprob, temperature, top_k, top_p, min_p):
    B, T, V = x.shape
    xs = x.double().cpu().numpy()
    per = lambda v: np.broadcast_to(np.asarray(v, np.float64), (B,))  # noqa: E731
    temperature, top_k, top_p, min_p = per(temperature), per(top_k), per(top_p), per(min_p)
    token, logprob = token.cpu().numpy().reshape(B, T), logprob.double().cpu().numpy().reshape(B, T)
    for b in range(B):
        for t in range(T):
            ok, lp = oracle.logits_ref.choices_ref(xs[b, t], None if noise is None else noise[b, t], temperature[b],
                                                   int(top_k[b]), top_p[b], min_p[b], SLACK)
            got = int(token[b, t])
            if not ok:
                assert got == -1 and logprob[b, t] == -math.inf, (b, t, got)
                continue
            assert got in ok, (b, t, got, sorted(ok)[:8], temperature[b], top_k[b], top_p[b], min_p[b])
            assert abs(logprob[b, t] - lp[got]) <= 1e-5 * (1 + abs(lp[got])), (b, t, logprob[b, t], lp[got])


def _run(x, noise, three=True, **kw):
    from rwkv_next_amd import kernels
    dev = torch.device(DEV)
    logits = x.to(dev)
    nz = None if noise is None else torch.from_numpy(noise).to(dev)
    if not three:
        logits, nz = logits[:, 0], None if nz is None else nz[:, 0]
    return kernels.sample_logits(logits, nz, **{k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in kw.items()})


FILTERS = [
    dict(),
    dict(top_k=1), dict(top_k=2), dict(top_k=50), dict(top_k=500), dict(top_k=3000),
    dict(top_p=0.0), dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.999),
    dict(min_p=0.05), dict(min_p=1.0), dict(min_p=2.0),
    dict(top_k=50, top_p=0.9), dict(top_k=400, top_p=0.99, min_p=0.01), dict(top_p=0.95, min_p=0.02),
    dict(top_k=5000, top_p=0.97),
]


@pytest.mark.parametrize("f", range(len(FILTERS)))
@pytest.mark.parametrize("V,dtype", [(1, "f32"), (7, "f16"), (1000, "bf16"), (2049, "f32"), (8191, "f16"), (30001, "bf16")])
def test_filters(f, V, dtype):
    kw = FILTERS[f]
    say("sample", V, dtype, kw)
    rng = np.random.default_rng(100 * f + V)
    B, T = 3, 2
    x = _peaked(rng, B, T, V, dtype)
    noise = _draws(rng, (B, T, V))
    for temperature in (0.7, 1.6, torch.tensor([0.0, 1.0, 3.0])):
        token, logprob = _run(x, noise, temperature=temperature, **kw)
        assert token.dtype == torch.int64 and token.shape == (B, T) and logprob.dtype == torch.float32
        _check(x, noise, token, logprob, temperature, kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_requests_differ(dtype):
    """Every request its own filters, one of them greedy; long segments (many rows) and short ones give the same."""
    say("sample requests differ", dtype)
    rng = np.random.default_rng(7)
    B, V = 80, 66000
    x = _peaked(rng, B, 1, V, dtype)
    noise = _draws(rng, (B, 1, V))
    temperature = torch.from_numpy(rng.uniform(0.5, 1.8, B).astype(np.float32))
    temperature[3] = 0
    top_k = torch.from_numpy(rng.choice([0, 1, 40, 700], B).astype(np.int32))
    top_p = torch.from_numpy(rng.choice([0.5, 0.9, 0.95, 1.0], B).astype(np.float32))
    min_p = torch.from_numpy(rng.choice([0.0, 0.02, 0.2], B).astype(np.float32))
    kw = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    token, logprob = _run(x, noise, three=False, **kw)
    assert token.shape == (B,)
    _check(x, noise, token, logprob, temperature, top_k, top_p, min_p)
    for b in (0, 3, 41, 79):  # alone: short segments
        one = {k: v[b:b + 1].clone() for k, v in kw.items()}
        t1, l1 = _run(x[b:b + 1], noise[b:b + 1], three=False, **one)
        assert int(t1) == int(token[b]) and abs(float(l1) - float(logprob[b])) <= 1e-5 * (1 + abs(float(l1)))


@pytest.mark.parametrize("kw", [dict(), dict(top_k=10), dict(top_k=5000), dict(top_p=0.5), dict(top_k=6000, top_p=0.4),
                                dict(top_p=0.9999)])
def test_equal_logits(kw):
    """Rows of few different values: bins of more tokens than the list holds, thresholds inside a run of equals."""
    say("sample equal logits", kw)
    rng = np.random.default_rng(11)
    V = 20000
    x = torch.zeros(4, 1, V)
    x[1] = torch.from_numpy(rng.choice([-1.0, 0.0, 0.5], V).astype(np.float32))
    x[2, 0, ::2] = -0.0
    x[3, 0, 5000:] = -math.inf
    noise = _draws(rng, (4, 1, V))
    token, logprob = _run(x, noise, **kw)
    _check(x, noise, token, logprob, 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.8), dict(top_k=4, top_p=0.8, min_p=0.1), dict(temperature=0.0)])
def test_strange_values(kw):
    """Rows without an allowed token, of one allowed token, with infinities, NaN, the type's lowest value and far outliers."""
    say("sample strange values", kw)
    rng = np.random.default_rng(12)
    V = 5003
    x = torch.from_numpy(rng.standard_normal((9, 1, V)).astype(np.float32))
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 0, 4999] = -3.0
    x[2, 0, 17] = math.inf
    x[3, 0, 100:200] = math.nan
    x[4] = torch.finfo(torch.float32).min
    x[5, 0, 1:] -= 1e30
    x[6] = math.nan
    x[7, 0, 50] = 1e6
    x[8, 0, 3:] = torch.finfo(torch.float32).min
    noise = _draws(rng, (9, 1, V))
    token, logprob = _run(x, noise, **kw)
    _check(x, noise, token, logprob, kw.get("temperature", 1.0), kw.get("top_k", 0), kw.get("top_p", 1.0),
           kw.get("min_p", 0.0))
    assert token[0, 0] == -1 and token[6, 0] == -1 and token[1, 0] == 4999


def test_temperatures_at_their_ends():
    say("sample temperatures")
    rng = np.random.default_rng(13)
    x = _peaked(rng, 6, 1, 3001)
    noise = _draws(rng, (6, 1, 3001))
    temperature = torch.tensor([1e-6, 1e-3, 50.0, -1.0, math.nan, 1e4])
    for kw in (dict(), dict(top_p=0.9), dict(top_k=7)):
        token, logprob = _run(x, noise, temperature=temperature, **kw)
        _check(x, noise, token, logprob, temperature, kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0)


def test_noise():
    """No noise is greedy; noise that is no number draws nothing; equal scores give the lowest index."""
    from rwkv_next_amd import kernels
    say("sample noise")
    rng = np.random.default_rng(14)
    x = _peaked(rng, 3, 1, 9001)
    token, logprob = _run(x, None, top_k=5, top_p=0.5)
    _check(x, None, token, logprob, 1.0, 5, 0.5, 0.0)
    noise = _draws(rng, (3, 1, 9001))
    noise[0] = math.nan
    noise[1, 0, ::3] = math.nan
    for kw in (dict(), dict(top_p=0.97), dict(top_k=30)):
        token, logprob = _run(x, noise, **kw)
        _check(x, noise, token, logprob, 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0)
    flat = torch.zeros(1, 70000, device=DEV)
    for kw in (dict(), dict(top_k=60000), dict(top_p=0.9), dict(top_k=4000)):
        assert int(kernels.sample_logits(flat, torch.ones_like(flat), **kw)[0]) == 0, kw


def test_strides_and_orders():
    """Views: rows apart, positions before sequences, offset starts, columns that are not contiguous."""
    from rwkv_next_amd import kernels
    say("sample strides")
    rng = np.random.default_rng(15)
    B, T, V = 3, 4, 1501
    x, noise = _peaked(rng, B, T, V, "bf16"), _draws(rng, (B, T, V))
    want, want_lp = _run(x, noise, top_p=0.9)
    nz = torch.from_numpy(noise).to(DEV)
    wide = torch.zeros(T, B, V + 13, dtype=torch.bfloat16, device=DEV)
    wide[..., 5:5 + V] = x.to(DEV).transpose(0, 1)
    view = wide[..., 5:5 + V].transpose(0, 1)
    nw = torch.zeros(B, T, V + 3, device=DEV)
    nw[..., 1:1 + V] = nz
    columns = x.to(DEV).permute(2, 0, 1).contiguous().permute(1, 2, 0)
    for logits, noise_t in ((view, nw[..., 1:1 + V]), (columns, nz.permute(2, 0, 1).contiguous().permute(1, 2, 0))):
        token, logprob = kernels.sample_logits(logits, noise_t, top_p=0.9)
        assert torch.equal(token, want) and torch.equal(logprob, want_lp)


def test_counts_and_status():
    from rwkv_next_amd import kernels
    say("sample counts")
    rng = np.random.default_rng(16)
    x = _peaked(rng, 4, 1, 2000)
    x[2] = -math.inf
    slots = torch.tensor([5, 1, 0, 9], device=DEV)
    for dt in (torch.int32, torch.float32):
        table = torch.zeros(8, 2010, dtype=dt, device=DEV)
        counts = table[:, 4:2004]
        status = kernels.new_status(torch.device(DEV))
        for n in (1, 2):
            token, _ = kernels.sample_logits(x[:, 0].to(DEV), None, counts=counts, slots=slots, status=status)
            want = torch.zeros_like(table)
            for b, s in ((0, 5), (1, 1)):  # row 2 has no token, slot 9 is outside
                want[s, 4 + int(token[b])] += n
            assert torch.equal(table, want)
        with pytest.raises(ValueError, match="count table"):
            kernels.check_status(status)
    counts = torch.zeros(4, 2000, dtype=torch.int32, device=DEV)
    token, _ = kernels.sample_logits(x[:2, 0].to(DEV), None, counts=counts)
    assert counts.sum() == 2 and counts[0, token[0]] == 1 and counts[1, token[1]] == 1


def test_streams_repeats_and_graphs():
    """The same bits again, on another stream, beside calls of other shapes, and from a graph replayed after eager work."""
    from rwkv_next_amd import kernels
    say("sample streams and graphs")
    rng = np.random.default_rng(17)
    x, noise = _peaked(rng, 5, 2, 40000).to(DEV), torch.from_numpy(_draws(rng, (5, 2, 40000))).to(DEV)
    small = _peaked(rng, 2, 1, 700).to(DEV)
    kw = dict(temperature=1.3, top_k=60, top_p=0.95)
    want = kernels.sample_logits(x, noise, **kw)
    other = kernels.sample_logits(small, noise[:2, :1, :700].contiguous(), top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = kernels.sample_logits(x, noise, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    logits = x.clone()
    with torch.cuda.stream(side):
        kernels.sample_logits(logits, noise, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kernels.sample_logits(logits, noise, **kw)
        got_small = kernels.sample_logits(small, noise[:2, :1, :700].contiguous(), top_p=0.9)
    for i in range(4):
        logits.copy_(x.roll(i, 0))
        g.replay()
        torch.cuda.synchronize()
        eager = kernels.sample_logits(logits, noise, **kw)
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), i
        assert all(torch.equal(a, b) for a, b in zip(got_small, other)), i


def test_many_rows():
    """More rows than one set of launches holds, and none."""
    from rwkv_next_amd import kernels
    say("sample many rows")
    rng = np.random.default_rng(18)
    x, noise = _peaked(rng, 260, 4, 300), _draws(rng, (260, 4, 300))
    token, logprob = _run(x, noise, top_k=20, top_p=0.9)
    _check(x, noise, token, logprob, 1.0, 20, 0.9, 0.0)
    for shape in ((0, 50), (0, 2, 50), (3, 0, 50)):
        token, logprob = kernels.sample_logits(torch.empty(shape, device=DEV))
        assert token.shape == shape[:-1] and logprob.shape == shape[:-1]


def test_draws_follow_the_weights():
    """4000 draws of one row of 8 kept tokens: each token's share within 5 standard deviations of its probability."""
    from rwkv_next_amd import kernels
    say("sample shares")
    p = torch.tensor([0.35, 0.25, 0.15, 0.1, 0.06, 0.04, 0.03, 0.02])
    n = 4000
    row = torch.full((64,), -20.0)
    row[8:16] = p.log()
    logits = row.to(DEV).expand(n, 64)
    gen = torch.Generator(device=DEV).manual_seed(3)
    for kw in (dict(), dict(top_k=8), dict(top_p=0.99999)):
        noise = torch.empty(n, 64, device=DEV).exponential_(generator=gen)
        token, _ = kernels.sample_logits(logits, noise, **kw)
        share = torch.bincount(token.cpu(), minlength=64)[8:16].double() / n
        assert ((share - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all(), (kw, share)
