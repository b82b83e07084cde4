"""Penalties, biases and grammar masks on logits (rwkv-infer-next_amd/csrc/logits_penalize.hip) against the oracle in 64 bits.

The kernel works in fp32 and rounds once: with u = 2^-24, at most u for the quotient or product by the repetition penalty, 2 u of
frequency c + presence, one u for each difference, sum and bias added, all below 8 u times the sum of the terms' sizes (with P biases
on one token, P u more of theirs).  Results of 16 bits are that fp32 result rounded once: compared bit for bit."""
import math

import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _case(rng, B, T, V, P=0, S=None, table="i32", masked=False):
    S = S or B + 2
    c = dict(counts=rng.integers(0, 4, (S, V)) * (rng.random((S, V)) < 0.1), slots=rng.permutation(S)[:B],
             repetition=rng.uniform(0.8, 1.5, B).astype(np.float32), presence=rng.uniform(-0.5, 1, B).astype(np.float32),
             frequency=rng.uniform(0, 1, B).astype(np.float32), drafts=rng.integers(0, V, (B, max(T - 1, 0))))
    c["counts"] = c["counts"].astype(np.int32) if table == "i32" else (c["counts"] * 0.75).astype(np.float32)
    if P:
        c["bias_ids"] = rng.integers(-1, V, (B, P))
        c["bias_values"] = (rng.standard_normal((B, P)) * 3).astype(np.float32)
    if masked:
        c["mask"] = rng.integers(0, 2 ** 32, (B, T, (V + 31) // 32), dtype=np.uint32)
    return c


def _dev(c, T, two):
    d = {}
    for n, v in c.items():
        if isinstance(v, np.ndarray):
            v = torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to(DEV)
            if two and n in ("mask", "mask_rows") and v.dim() == (3 if n == "mask" and "mask_rows" not in c else 2) and \
                    not (n == "mask" and "mask_rows" in c):
                v = v[:, 0]
        d[n] = v
    if two:
        d.pop("drafts", None)
    return d


def _check(got, x, c):
    assert got.dtype == torch.float32
    xs = x.double().cpu().numpy()
    want = oracle.logits_ref.penalize_ref(xs, **c)
    got = got.double().cpu().numpy().reshape(want.shape)
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    B, T, V = xs.shape
    per = lambda n: np.abs(np.broadcast_to(np.asarray(c.get(n, {"repetition": 1.0}.get(n, 0.0)), np.float64), (B,)))[:, None, None]  # noqa: E731
    most = 0.0 if c.get("counts") is None else float(np.max(c["counts"], initial=0))
    size = np.abs(np.where(np.isinf(xs), 0, xs)) * np.maximum(per("repetition"), 1 / per("repetition")) + \
        per("frequency") * (most + T) + per("presence")
    terms = 8.0
    if c.get("bias_ids") is not None:
        size = size + np.abs(c["bias_values"]).sum(axis=1)[:, None, None]
        terms += c["bias_ids"].shape[1]
    bound = terms * 2.0 ** -24 * size + 2.0 ** -24 * np.abs(want)
    assert (np.abs(got - want)[~inf] <= bound[~inf]).all(), np.max((np.abs(got - want) / bound)[~inf])


@pytest.mark.parametrize("B,T,V,P,masked", [
    (1, 1, 1, 1, True), (2, 1, 7, 0, True), (3, 1, 33, 5, False), (1, 1, 2048, 3, True), (2, 3, 2049, 40, True),
    (3, 5, 4097, 257, False), (5, 2, 1000, 700, True), (4, 1, 50001, 12, True),
])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_against_the_oracle(B, T, V, P, masked, dtype):
    from rwkv_next_amd import kernels
    say("penalize", B, T, V, P, masked, dtype)
    rng = np.random.default_rng(B + 10 * T + V)
    x = torch.from_numpy((rng.standard_normal((B, T, V)) * 5).astype(np.float32)).to(DTYPES[dtype])
    for table in ("i32", "f32"):
        c = _case(rng, B, T, V, P, table=table, masked=masked)
        f32 = torch.empty(x.shape, device=DEV)
        assert kernels.penalize_logits(x.to(DEV), out=f32, **_dev(c, T, False)) is f32
        _check(f32, x, c)
        got = kernels.penalize_logits(x.to(DEV), **_dev(c, T, False))
        assert got.dtype == x.dtype and torch.equal(got, f32.to(x.dtype))
        if T == 1:
            assert torch.equal(kernels.penalize_logits(x[:, 0].to(DEV), **_dev(c, T, True)), got[:, 0])
        for out_dtype in (torch.bfloat16, torch.float16):
            out = torch.empty(x.shape, dtype=out_dtype, device=DEV)
            assert torch.equal(kernels.penalize_logits(x.to(DEV), out=out, **_dev(c, T, False)), f32.to(out_dtype))
        same = x.to(DEV)
        assert kernels.penalize_logits(same, out=same, **_dev(c, T, False)) is same and torch.equal(same, got)


def test_parts_alone():
    """Each part without the others, and none at all: the logits as they were."""
    from rwkv_next_amd import kernels
    say("penalize parts alone")
    rng = np.random.default_rng(2)
    B, T, V = 3, 4, 2500
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32))
    x[0, 0, 5] = math.nan
    logits = x.to(DEV)
    for kw in (dict(), dict(repetition=1.3, presence=0.5, frequency=0.2)):  # nothing is counted
        assert torch.equal(kernels.penalize_logits(logits, **kw).view(torch.int32), logits.view(torch.int32))
    x[0, 0, 5] = 1.0
    logits = x.to(DEV)
    c = _case(rng, B, T, V, 6, S=B, masked=True)
    for part in (("counts", "repetition"), ("counts", "presence"), ("counts", "frequency", "slots"), ("mask",),
                 ("bias_ids", "bias_values"), ("drafts", "repetition", "frequency"), ("drafts", "presence")):
        some = {n: c[n] for n in part}
        _check(kernels.penalize_logits(logits, **_dev(some, T, False)), x, some)
    for kw in (dict(repetition=1.25), dict(presence=0.5, frequency=0.25)):  # one number for all
        some = dict(counts=c["counts"], slots=c["slots"], **kw)
        _check(kernels.penalize_logits(logits, **_dev(some, T, False)), x, some)


def test_equal_biases_add_up_in_order():
    from rwkv_next_amd import kernels
    say("penalize equal biases")
    rng = np.random.default_rng(3)
    V, P = 5000, 1000
    ids = rng.integers(2040, 2060, (1, P))  # over the edge of two workgroups' columns
    values = rng.standard_normal((1, P)).astype(np.float32)
    x = torch.zeros(1, V, device=DEV)
    got = kernels.penalize_logits(x, bias_ids=torch.from_numpy(ids).to(DEV), bias_values=torch.from_numpy(values).to(DEV))
    want = np.zeros(V, np.float32)
    for i, v in zip(ids[0], values[0]):
        want[i] = want[i] + v
    assert np.array_equal(got[0].cpu().numpy(), want)


def test_masks():
    """A mask that leaves nothing, one that leaves the last token, a table of masks, rows without one and past its end."""
    from rwkv_next_amd import kernels
    say("penalize masks")
    rng = np.random.default_rng(4)
    B, T, V, words = 2, 3, 1003, 32
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32))
    x[0, 0, 3], x[0, 1, 4], x[1, 0, :] = math.inf, -math.inf, math.nan
    table = np.zeros((4, words + 2), np.uint32)
    table[1, (V - 1) // 32] = 1 << ((V - 1) % 32)
    table[2:, :] = rng.integers(0, 2 ** 32, (2, words + 2), dtype=np.uint32)
    rows = np.array([[0, 1, 2], [0, -1, 4]])
    status = kernels.new_status(torch.device(DEV))
    dev_table = torch.from_numpy(table.view(np.int32)).to(DEV)[:, :words]
    got = kernels.penalize_logits(x.to(DEV), mask=dev_table, mask_rows=torch.from_numpy(rows).to(DEV), status=status).cpu()
    for b in range(B):
        for t in range(T):
            r = rows[b, t]
            bits = np.ones(V, bool)
            if 0 <= r < 4:
                bits = np.unpackbits(np.ascontiguousarray(table[r]).view(np.uint8), bitorder="little")[:V] != 0
            want = torch.where(torch.from_numpy(bits), x[b, t], torch.tensor(-math.inf))
            assert torch.equal(got[b, t].nan_to_num(nan=7.5), want.nan_to_num(nan=7.5)), (b, t)
    with pytest.raises(ValueError, match="mask row"):
        kernels.check_status(status)


def test_bad_indices_are_left_out():
    from rwkv_next_amd import kernels
    say("penalize bad indices")
    rng = np.random.default_rng(5)
    B, T, V = 3, 3, 3000
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32))
    c = _case(rng, B, T, V, 4)
    c["slots"] = np.array([1, 77, -1])
    status = kernels.new_status(torch.device(DEV))
    _check(kernels.penalize_logits(x.to(DEV), status=status, **_dev(c, T, False)), x, c)
    assert int(status) == 256
    c["slots"], c["drafts"] = np.array([1, 0, 2]), np.array([[V, 3], [5, 2 ** 40], [-1, -7]])
    c["bias_ids"][0, 0], c["bias_ids"][1, 1] = V, -2 ** 50
    status.zero_()
    _check(kernels.penalize_logits(x.to(DEV), status=status, **_dev(c, T, False)), x, c)
    assert int(status) == 512
    with pytest.raises(ValueError, match="vocabulary"):
        kernels.check_status(status)


def test_strides():
    """Rows apart, positions before sequences, offset starts, parameters out of larger tensors."""
    from rwkv_next_amd import kernels
    say("penalize strides")
    rng = np.random.default_rng(6)
    B, T, V = 3, 2, 2051
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32)).to(torch.bfloat16)
    c = _case(rng, B, T, V, 5, masked=True)
    d = _dev(c, T, False)
    want = kernels.penalize_logits(x.to(DEV), **d)
    wide = torch.zeros(T, B, V + 9, dtype=torch.bfloat16, device=DEV)
    wide[..., 3:3 + V] = x.to(DEV).transpose(0, 1)
    view = wide[..., 3:3 + V].transpose(0, 1)
    counts = torch.zeros(d["counts"].shape[0], V + 5, dtype=torch.int32, device=DEV)
    counts[:, 2:2 + V] = d["counts"]
    more = lambda t, n: torch.cat([t, t.new_zeros(*t.shape[:-1], n)], -1)[..., :t.shape[-1]]  # noqa: E731
    d2 = dict(d, counts=counts[:, 2:2 + V], drafts=more(d["drafts"], 3), bias_ids=more(d["bias_ids"], 2),
              bias_values=more(d["bias_values"], 7), mask=more(d["mask"], 4))
    assert torch.equal(kernels.penalize_logits(view, **d2), want)
    columns = x.to(DEV).permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(kernels.penalize_logits(columns, **d), want)
    before = wide.clone()
    kernels.penalize_logits(view, out=view, **d2)  # in place, and nothing beside it
    assert torch.equal(view, want)
    before[..., 3:3 + V] = view.transpose(0, 1)
    assert torch.equal(wide, before)
    one = torch.randn(1, 1, V, device=DEV).expand(B, T, V)
    assert torch.equal(kernels.penalize_logits(one, **d), kernels.penalize_logits(one.contiguous(), **d))


def test_streams_and_graphs():
    from rwkv_next_amd import kernels
    say("penalize streams and graphs")
    rng = np.random.default_rng(7)
    B, T, V = 4, 2, 9000
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32)).to(DEV)
    d = _dev(_case(rng, B, T, V, 20, masked=True), T, False)
    want = kernels.penalize_logits(x, **d)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = kernels.penalize_logits(x, **d)
    torch.cuda.synchronize()
    assert torch.equal(again, want)
    logits = x.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kernels.penalize_logits(logits, **d)
    for i in range(3):
        logits.copy_(x.roll(i, 2))
        d["counts"].add_(i)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, kernels.penalize_logits(logits, **d)), i


def test_empty():
    from rwkv_next_amd import kernels
    say("penalize empty")
    for shape in ((0, 50), (2, 0, 50), (0, 3, 50), (4, 0)):
        assert kernels.penalize_logits(torch.empty(shape, device=DEV)).shape == shape
    x = torch.ones(2, 40, device=DEV)
    ids, values = torch.empty(2, 0, dtype=torch.int64, device=DEV), torch.empty(2, 0, device=DEV)
    assert torch.equal(kernels.penalize_logits(x, bias_ids=ids, bias_values=values), x)
