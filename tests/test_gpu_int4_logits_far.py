"""Offsets past 32 bits: rows of logits, counts, noise and masks far apart, and a 4-bit weight of more than 4 GiB."""
import numpy as np
import pytest

from gpu_util import say
from test_gpu_int4 import _check as check_int4
from test_gpu_logits_penalize import _check as check_penalties
from test_gpu_logits_sample import _check as check_tokens

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
FAR = 2 ** 31 + 5  # elements


def _far(t, dtype=None):
    """t (2, n) on the device with rows FAR elements apart."""
    base = torch.empty(FAR + t.shape[1], dtype=dtype or t.dtype, device=DEV)
    view = base.as_strided((2, t.shape[1]), (FAR, 1))
    view.copy_(t.to(DEV))
    return view


def test_logits_far_apart():
    from rwkv_next_amd import kernels
    say("logits far apart")
    rng = np.random.default_rng(1)
    V = 5001
    x = torch.from_numpy(rng.standard_normal((2, V)).astype(np.float32))
    counts = (rng.integers(0, 3, (2, V))).astype(np.int32)
    mask = rng.integers(0, 2 ** 32, (2, (V + 31) // 32), dtype=np.uint32)
    c = dict(counts=counts, repetition=np.float32(1.25), presence=np.float32(0.5), frequency=np.float32(0.25), mask=mask[:, None])
    logits = _far(x)
    out = kernels.penalize_logits(logits, counts=_far(torch.from_numpy(counts)), repetition=1.25, presence=0.5, frequency=0.25,
                                  mask=_far(torch.from_numpy(mask.view(np.int32))), out=logits)
    assert out is logits
    check_penalties(out.contiguous()[:, None], x[:, None], c)
    noise = rng.exponential(size=(2, 1, V)).astype(np.float32)
    table = torch.zeros(2, V, dtype=torch.int32)
    far_table = _far(table)
    for kw in (dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.8)):
        token, logprob = kernels.sample_logits(out, _far(torch.from_numpy(noise[:, 0])), counts=far_table, **kw)
        check_tokens(out.cpu()[:, None], noise, token, logprob, 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), 0.0)
        for b in range(2):
            table[b, int(token[b])] += 1
    assert torch.equal(far_table.cpu(), table)


def test_slots_far_down_a_table():
    from rwkv_next_amd import kernels
    say("slots far down a table")
    V, S = 65536, 33000
    counts = torch.zeros(S, V, dtype=torch.int32, device=DEV)  # 8.7 GB
    counts[S - 1, 7] = 3
    x = torch.ones(1, V, device=DEV)
    slots = torch.tensor([S - 1], device=DEV)
    y = kernels.penalize_logits(x, counts=counts, slots=slots, presence=0.5)
    assert float(y[0, 7]) == 0.5 and float((y == 1).sum()) == V - 1
    token, _ = kernels.sample_logits(y, None, counts=counts, slots=slots)
    assert int(token) == 0 and int(counts[S - 1, 0]) == 1 and int(counts.sum()) == 4


def test_weight_past_4_gib():
    from rwkv_next_amd import kernels
    say("int4 weight past 4 GiB")
    K, N, g = 16384, 540017, 128
    gen = torch.Generator(device=DEV).manual_seed(2)
    codes = torch.randint(0, 256, (K // 2, N), dtype=torch.uint8, device=DEV, generator=gen)
    scales = ((torch.rand(K // g, N, device=DEV, generator=gen) + 0.5) / 128).half()
    pk = kernels.prepack_int4(codes, scales, g)
    assert pk.weight.numel() > 2 ** 32
    columns = torch.tensor([0, 1, 262143, 262144, 524287, 524288, 530000, N - 2, N - 1], device=DEV)
    part, part_scales = codes[:, columns].cpu().numpy(), scales[:, columns].cpu().numpy()
    del codes, scales
    for M in (1, 40):
        a = torch.randn(M, K, device=DEV, generator=gen).to(torch.bfloat16)
        y = kernels.int4_matmul(a, pk, out_dtype=torch.float32)
        check_int4(y[:, columns], a.cpu(), part, part_scales, g)
