"""The products with 16-bit weights and an epilogue (rwkv-infer-next_amd/csrc/dense.hip) against the oracle in 64 bits.

With u = 2^-24, a sum of K exact products in fp32, whatever their order, is off by at most (K + 8) u times the sum of their sizes,
element by element; roundings go both ways, so over a whole result they come to much less: 4e-6 of its 2-norm.  An activation is off
by its slope (at most 1.13, relu2 2 |x|) times that, and by a few units in the last place of its own: 16 u of its value, tanh and the
others of the device library being good to 2 to 6; the residual's addition by u of the result.  Results of 16 bits are the fp32 ones rounded once: compared bit
for bit."""
import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NORM_TOL = 4e-6
U = 2.0 ** -24
ref = oracle.delta_ref


def _np(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _check(got, a, w, bias, act, residual):
    assert got.dtype == torch.float32
    K = a.shape[-1]
    want, x = ref.dense_ref(_np(a), _np(w), _np(bias), act, _np(residual))
    size = np.abs(_np(a)) @ np.abs(_np(w)) + (0 if bias is None else np.abs(_np(bias)))
    off = (K + 8) * U * size
    slope = 2 * (np.abs(x) + off) if act == "relu2" else 1.13
    bound = slope * off + 16 * U * np.abs(ref.ACTIVATIONS[act](x)) + 2 * U * np.abs(want) + 1e-37
    err = np.abs(_np(got) - want)
    assert (err <= bound).all(), np.max(err / bound)
    if act in (None, "none"):
        assert np.linalg.norm(err) <= NORM_TOL * max(np.linalg.norm(want), 1e-30)


def _case(M, K, N, dtype, seed, bias=None, residual=None):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    a = torch.randn(M, K, device=DEV, generator=gen).to(dtype)
    w = (torch.randn(K, N, device=DEV, generator=gen) / K ** 0.5).to(dtype)
    b = None if bias is None else torch.randn(N, device=DEV, generator=gen).to(bias)
    r = None if residual is None else torch.randn(M, N, device=DEV, generator=gen).to(residual)
    return a, w, b, r


SHAPES = [
    (1, 32, 1), (1, 32, 16), (2, 64, 17), (3, 96, 40), (1, 4096, 512), (5, 1088, 1000), (16, 2560, 300), (17, 640, 272),
    (23, 2560, 96), (31, 768, 2049), (33, 4096, 100), (64, 384, 8208), (65, 1024, 31), (130, 2560, 777), (203, 256, 8191),
    (256, 128, 256), (257, 160, 513), (300, 416, 65), (500, 2560, 640), (1000, 96, 2000), (1025, 1056, 1031), (1, 256, 66000),
    (20, 128, 40000), (4, 16384, 64), (2048, 512, 256), (700, 10240, 300),
]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_product(M, K, N, dtype):
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    say("dense", M, K, N, dtype)
    a, w, b, r = _case(M, K, N, dtype, M + K + N, torch.float32, dtype)
    p = prepack_dense(w)
    y = dense_matmul(a, p, out_dtype=torch.float32)
    _check(y, a, w, None, None, None)
    assert torch.equal(dense_matmul(a, p), y.to(dtype))
    z = dense_matmul(a, p, bias=b, activation="silu", residual=r, out_dtype=torch.float32)
    _check(z, a, w, b, "silu", r)
    assert torch.equal(dense_matmul(a, p, bias=b, activation="silu", residual=r), z.to(dtype))
    assert torch.equal(dense_matmul(a, p), y.to(dtype))  # nothing of a call is kept


@pytest.mark.parametrize("act", [None, "none", "relu", "relu2", "tanh", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("M,N", [(3, 50), (40, 300), (300, 520)])
@pytest.mark.parametrize("bias,residual", [(None, None), (torch.float16, torch.float32), (torch.bfloat16, None), (None, torch.bfloat16)])
def test_epilogue(act, M, N, bias, residual):
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    a, w, b, r = _case(M, 320, N, torch.bfloat16, 7, bias, residual)
    a = a * 3  # into the flat parts too
    p = prepack_dense(w)
    y = dense_matmul(a, p, bias=b, activation=act, residual=r, out_dtype=torch.float32)
    _check(y, a, w, b, act, r)
    for t in (torch.bfloat16, torch.float16):
        assert torch.equal(dense_matmul(a, p, bias=b, activation=act, residual=r, out_dtype=t), y.to(t))


@pytest.mark.parametrize("M", [1, 7, 70, 600])
def test_strides_and_shapes(M):
    from rwkv_next_amd.kernels import dense_matmul, dense_matmul_op, prepack_dense
    a, w, b, r = _case(M, 160, 100, torch.bfloat16, 3, torch.float32, torch.bfloat16)
    p = prepack_dense(w)
    want = dense_matmul(a, p, bias=b, residual=r)
    assert torch.equal(prepack_dense(w.t().contiguous().t()).weight, p.weight)  # the other order of a matrix
    wide = torch.zeros(M, 400, device=DEV, dtype=torch.bfloat16)
    for first in (8, 3):  # rows apart; rows apart and not aligned
        view = wide[:, first:first + 160]
        view.copy_(a)
        assert torch.equal(dense_matmul(view, p, bias=b, residual=r), want)
    assert torch.equal(dense_matmul(a.t().contiguous().t(), p, bias=b, residual=r), want)
    res = torch.zeros(M, 333, device=DEV, dtype=torch.bfloat16)[:, 5:105]
    res.copy_(r)
    assert torch.equal(dense_matmul(a, p, bias=b, residual=res), want)
    row = r[:1].expand(M, 100)
    assert torch.equal(dense_matmul(a, p, residual=row), dense_matmul(a, p, residual=row.contiguous()))
    assert torch.equal(dense_matmul(a.view(M, 1, 160), p, bias=b, residual=r.view(M, 1, 100)), want.view(M, 1, 100))
    assert torch.equal(dense_matmul(a[0], p, bias=b, residual=r[0]).float(), dense_matmul(a[:1], p, bias=b, residual=r[:1])[0].float())
    assert dense_matmul(a[:0], p, bias=b, residual=r[:0]).shape == (0, 100)
    assert torch.equal(dense_matmul_op(a, p.weight, 160, 100, b, "none", r), want)


@pytest.mark.parametrize("M", [2, 40, 300])
def test_values_that_are_not_finite(M):
    """An infinity or NaN stays in its row of the activations, and in its column of the weight."""
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    a, w, _, _ = _case(M, 256, 64, torch.bfloat16, 5)
    clean = dense_matmul(a, prepack_dense(w))
    a2 = a.clone()
    a2[1, 77] = float("inf")
    y = dense_matmul(a2, prepack_dense(w))
    keep = torch.arange(M, device=DEV) != 1
    assert torch.equal(y[keep], clean[keep]) and not torch.isfinite(y[1]).any()
    w2 = w.clone()
    w2[9, 63] = float("nan")
    y = dense_matmul(a, prepack_dense(w2))
    assert torch.equal(y[:, :63], clean[:, :63]) and torch.isnan(y[:, 63]).all()
    assert torch.isnan(dense_matmul(a, prepack_dense(w2), activation="relu2")[:, 63]).all()
    big = torch.full((M, 256), 3e38, device=DEV, dtype=torch.bfloat16)
    ones = torch.ones(256, 16, device=DEV, dtype=torch.bfloat16)
    p = prepack_dense(ones)
    assert (dense_matmul(big, p, activation="sigmoid") == 1).all() and (dense_matmul(-big, p, activation="sigmoid") == 0).all()
    assert (dense_matmul(-big, p, activation="relu") == 0).all() and (dense_matmul(big, p, activation="tanh") == 1).all()


@pytest.mark.parametrize("M", [1, 64, 400])
def test_graph_and_streams(M):
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    a, w, b, r = _case(M, 512, 320, torch.bfloat16, 11, torch.float32, torch.bfloat16)
    p = prepack_dense(w)
    want = dense_matmul(a, p, bias=b, activation="gelu", residual=r)
    other = dense_matmul(-a, p, bias=b, activation="gelu", residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dense_matmul(a, p, bias=b, activation="gelu", residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    x, g = a.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = dense_matmul(x, p, bias=b, activation="gelu", residual=r)
    for _ in range(3):
        x.copy_(a)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        x.copy_(-a)
        g.replay()
        assert torch.equal(y, other)


def test_rows_far_apart():
    """Rows of activations, residual and result at offsets past 32 bits."""
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    far = 1 << 24
    a, w, _, _ = _case(260, 64, 48, torch.bfloat16, 13)
    store = torch.empty(259 * far + 64, device=DEV, dtype=torch.bfloat16)
    x = store.as_strided((260, 64), (far, 1))
    x.copy_(a)
    p = prepack_dense(w)
    assert torch.equal(dense_matmul(x, p), dense_matmul(a, p))
    res = store.as_strided((260, 48), (far, 1))
    assert torch.equal(dense_matmul(a, p, residual=res), dense_matmul(a, p, residual=res.contiguous()))


def test_refusals():
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    a, w, b, r = _case(4, 64, 32, torch.bfloat16, 1, torch.float32, torch.bfloat16)
    p = prepack_dense(w)
    for bad in (w.float(), w.to(torch.float8_e4m3fn)):
        with pytest.raises(TypeError):
            prepack_dense(bad)
    for bad in (w[:33], w[:0], w[None], w.cpu(), w[:, :0]):
        with pytest.raises(ValueError):
            prepack_dense(bad)
    for kw in (dict(a=a.half()), dict(a=a.float()), dict(out_dtype=torch.int32)):
        with pytest.raises(TypeError):
            dense_matmul(kw.pop("a", a), p, **kw)
    for kw in (dict(a=a[:, :32]), dict(a=a.cpu()), dict(bias=b[:31]), dict(bias=b.cpu()), dict(bias=b.int()),
               dict(bias=b[None]), dict(residual=r[:3]), dict(residual=r.cpu()), dict(residual=r.long()),
               dict(residual=r[None]), dict(activation="swish"), dict(p=p._replace(N=33)), dict(p=p._replace(weight=p.weight[1:]))):
        with pytest.raises(ValueError):
            dense_matmul(kw.pop("a", a), kw.pop("p", p), **kw)
