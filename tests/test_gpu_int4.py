"""The 4-bit weight products (rwkv-infer-next_amd/csrc/w4a16.hip) against the oracle in 64 bits.

With u = 2^-24, a group's sum of n products a (16 + u_code) and its sum of a's are off by at most n u times the sum of their sizes,
the groups' sums by their number: below (136 + K / 32 + 8) u sum |a| |s| (31 + 24), element by element; such sums' roundings go both
ways, so over a whole result they come to much less: 4e-6 of its 2-norm, what the square root of the terms' number gives for weights
of random sign (sqrt(136) u 24 / 4.6 times a few).  Results of 16 bits are the fp32 result rounded once: compared bit for bit."""
import math

import numpy as np
import pytest

import oracle
from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
NORM_TOL = 4e-6


def _weight(rng, K, N, g):
    codes = rng.integers(0, 256, (K // 2, N)).astype(np.uint8)
    scales = (rng.uniform(0.5, 1.5, (K // g, N)) / math.sqrt(K)).astype(np.float16)
    return codes, scales


def _check(got, a, codes, scales, g):
    assert got.dtype == torch.float32
    want = oracle.int4_ref.int4_matmul_ref(a.double().cpu().numpy(), codes, scales, g)
    K = a.shape[-1]
    size = np.abs(a.double().cpu().numpy()) @ np.abs(np.asarray(scales, np.float64))[np.arange(K) // g]
    err = np.abs(got.double().cpu().numpy() - want)
    bound = (144 + K / 32) * 2.0 ** -24 * 55 * size
    assert (err <= bound).all(), np.max(err / bound)
    if want.size:
        assert np.linalg.norm(err) <= NORM_TOL * np.linalg.norm(want)


@pytest.mark.parametrize("M,N,K,g", [
    (1, 1, 32, 32),            # one step, one column
    (1, 16, 128, 128),
    (2, 17, 160, 32),          # a chunk and a step, a strip and a column
    (3, 40, 96, 96),           # a group that is no power of two
    (1, 4096, 512, 64),
    (5, 1000, 1088, 64),       # eight and a half chunks
    (16, 300, 2560, 128),
    (17, 272, 640, 320),       # a group that ends inside a chunk
    (31, 2049, 768, 256),
    (33, 100, 4096, 128),
    (64, 8208, 384, 128),
    (65, 31, 1024, 1024),
    (130, 777, 2560, 64),
    (203, 8191, 256, 32),
    (300, 65, 416, 32),
    (1, 66000, 256, 128),      # many strips
    (20, 40000, 128, 128),
    (4, 64, 16384, 128),       # deep
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_against_the_oracle(M, N, K, g, dtype):
    from rwkv_next_amd import kernels
    say("int4", M, N, K, g, dtype)
    rng = np.random.default_rng(M + N + K)
    codes, scales = _weight(rng, K, N, g)
    a = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).to(dtype)
    pk = kernels.prepack_int4(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), g)
    f32 = kernels.int4_matmul(a.to(DEV), pk, out_dtype=torch.float32)
    _check(f32, a, codes, scales, g)
    got = kernels.int4_matmul(a.to(DEV), pk)
    assert got.shape == (M, N) and got.dtype == dtype and torch.equal(got, f32.to(dtype))
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    assert torch.equal(kernels.int4_matmul(a.to(DEV), pk, out_dtype=other), f32.to(other))


@pytest.mark.parametrize("K,N,g", [(32, 1, 32), (160, 33, 32), (640, 50, 320), (1024, 128, 128), (192, 16, 64)])
def test_layouts(K, N, g):
    """The packed order and the dequantised weight, bit for bit."""
    from rwkv_next_amd import kernels
    say("int4 layouts", K, N, g)
    rng = np.random.default_rng(K + N)
    codes, scales = _weight(rng, K, N, g)
    c, s = torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV)
    pk = kernels.prepack_int4(c, s, g)
    assert np.array_equal(pk.weight.cpu().numpy().view(np.uint32), oracle.int4_ref.packed_ref(codes).reshape(-1))
    assert np.array_equal(pk.scales.cpu().numpy(), oracle.int4_ref.packed_scales_ref(scales, K, g).reshape(-1))
    want = torch.from_numpy(oracle.int4_ref.dequantize_ref(codes, scales, g))
    assert torch.equal(kernels.dequantize_int4(c, s, g).double().cpu(), want)  # exact in fp32
    for dt in (torch.bfloat16, torch.float16):
        assert torch.equal(kernels.dequantize_int4(c, s, g, dtype=dt).cpu(), want.float().to(dt))


def test_extremes():
    """Every code, scales from subnormal to the largest, activations of one sign and large ones, rows of zeros; an infinity or NaN
    in a row stays in that row."""
    from rwkv_next_amd import kernels
    say("int4 extremes")
    rng = np.random.default_rng(5)
    K, N, g = 256, 48, 64
    codes, scales = _weight(rng, K, N, g)
    codes[:16] = np.arange(256).reshape(16, 16)[:, :1] + np.arange(48) % 16
    scales[0, :4], scales[1, 4:8], scales[2, 8] = 6e-8, 65504, 0
    a = torch.from_numpy(rng.standard_normal((20, K)).astype(np.float32))
    a[0], a[1], a[2] = 0, a[1].abs(), a[2] * 1e30
    a[3] *= 1e-30
    a[5, 17], a[18, 100] = math.inf, math.nan
    a = a.to(torch.bfloat16)
    pk = kernels.prepack_int4(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), g)
    got = kernels.int4_matmul(a.to(DEV), pk, out_dtype=torch.float32)
    assert got[5].isnan().all() and got[18].isnan().all()
    fine = [r for r in range(20) if r not in (2, 5, 18)]
    ok = got[fine].isfinite()
    assert ok.all()
    for r in fine + [2]:
        _check(got[r:r + 1], a[r:r + 1], codes, scales, g)


def test_shapes_and_strides():
    """Leading sizes, none, rows apart, rows that 16-byte loads cannot read in place, and no rows."""
    from rwkv_next_amd import kernels
    say("int4 strides")
    rng = np.random.default_rng(6)
    K, N, g = 320, 90, 64
    codes, scales = _weight(rng, K, N, g)
    pk = kernels.prepack_int4(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), g)
    a = torch.from_numpy(rng.standard_normal((6, K)).astype(np.float32)).to(torch.bfloat16).to(DEV)
    want = kernels.int4_matmul(a, pk)
    assert torch.equal(kernels.int4_matmul(a.view(2, 3, K), pk), want.view(2, 3, N))
    assert torch.equal(kernels.int4_matmul(a[4], pk), kernels.int4_matmul(a[4:5], pk)[0])
    wide = torch.full((6, K + 24), math.nan, dtype=torch.bfloat16, device=DEV)
    for at in (0, 8, 3):
        wide[:, at:at + K] = a
        assert torch.equal(kernels.int4_matmul(wide[:, at:at + K], pk), want), at
        wide.fill_(math.nan)
    assert torch.equal(kernels.int4_matmul(a.t().contiguous().t(), pk), want)
    assert torch.equal(kernels.int4_matmul(a[:1].expand(6, K), pk), want[:1].expand(6, N))
    assert kernels.int4_matmul(a[:0], pk).shape == (0, N)
    odd = torch.empty(6 * K + 1, dtype=torch.bfloat16, device=DEV)[1:].view(6, K)
    odd.copy_(a)
    assert torch.equal(kernels.int4_matmul(odd, pk), want)


def test_rows_do_not_depend_on_each_other():
    """A row's result is the same beside other rows of the same call's shape."""
    from rwkv_next_amd import kernels
    say("int4 rows")
    rng = np.random.default_rng(7)
    K, N, g = 512, 200, 128
    codes, scales = _weight(rng, K, N, g)
    pk = kernels.prepack_int4(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), g)
    a = torch.from_numpy(rng.standard_normal((70, K)).astype(np.float32)).to(torch.bfloat16).to(DEV)
    got = kernels.int4_matmul(a, pk)
    b = a.clone()
    b[1:] = math.nan
    assert torch.equal(kernels.int4_matmul(b, pk)[0], got[0])
    assert torch.equal(kernels.int4_matmul(a.flip(0), pk).flip(0), got)


def test_op_streams_and_graphs():
    from rwkv_next_amd import kernels
    say("int4 op, streams and graphs")
    rng = np.random.default_rng(8)
    K, N, g = 512, 3000, 128
    codes, scales = _weight(rng, K, N, g)
    pk = kernels.prepack_int4(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), g)
    a = torch.from_numpy(rng.standard_normal((9, K)).astype(np.float32)).to(torch.float16).to(DEV)
    want = kernels.int4_matmul(a, pk)
    assert torch.equal(kernels.int4_matmul_op(a, *pk), want)
    torch.library.opcheck(kernels.int4_matmul_op, (a, *pk), test_utils=("test_schema", "test_faketensor"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = kernels.int4_matmul(a, pk)
    torch.cuda.synchronize()
    assert torch.equal(again, want)
    x = a.clone()
    g_ = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g_):
        got = kernels.int4_matmul(x, pk)
    for i in range(3):
        x.copy_(a.roll(i, 1))
        g_.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, kernels.int4_matmul(x, pk)), i


def test_quantised_on_the_device():
    """quantize_int4 -> prepack_int4 -> int4_matmul: as near the float product as the quantised weight is near the weight."""
    from rwkv_next_amd import kernels
    say("int4 quantised")
    gen = torch.Generator(device=DEV).manual_seed(9)
    w = torch.randn(1024, 513, device=DEV, generator=gen) / 32
    a = torch.randn(7, 1024, device=DEV, generator=gen).to(torch.bfloat16)
    codes, scales, g = kernels.quantize_int4(w, 64)
    wq = kernels.dequantize_int4(codes, scales, g)
    assert (wq - w).norm() <= 0.13 * w.norm()
    y = kernels.int4_matmul(a, kernels.prepack_int4(codes, scales, g), out_dtype=torch.float32)
    _check(y, a.cpu(), codes.cpu().numpy(), scales.cpu().numpy(), g)


def test_next_tokens():
    """The whole end of a decode step: as its three operators one after another, drawn tokens counted, from a graph too."""
    from rwkv_next_amd import kernels
    say("next_tokens")
    gen = torch.Generator(device=DEV).manual_seed(10)
    B, C, V = 6, 512, 5001
    w = torch.randn(C, V, device=DEV, generator=gen) / 8
    head = kernels.prepack_int4(*kernels.quantize_int4(w, 128))
    x = torch.randn(B, C, device=DEV, generator=gen).to(torch.bfloat16)
    noise = torch.empty(B, V, device=DEV).exponential_(generator=gen)
    counts = torch.zeros(9, V, dtype=torch.int32, device=DEV)
    slots = torch.tensor([8, 3, 0, 5, 1, 2], device=DEV)
    ids = torch.randint(0, V, (B, 4), device=DEV, generator=gen)
    kw = dict(slots=slots, repetition=1.2, presence=0.3, frequency=0.1, bias_ids=ids,
              bias_values=torch.randn(B, 4, device=DEV, generator=gen),
              mask=torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), device=DEV, generator=gen).to(torch.int32))
    pick = dict(temperature=torch.rand(B, device=DEV, generator=gen) + 0.5, top_k=40, top_p=0.9, min_p=0.01)
    want_counts = counts.clone()
    for _ in range(3):
        logits = kernels.penalize_logits(kernels.int4_matmul(x, head, out_dtype=torch.float32), counts=want_counts, **kw)
        want = kernels.sample_logits(logits, noise, counts=want_counts, slots=slots, **pick)
        got = kernels.next_tokens(x, head, noise, counts=counts, **kw, **pick)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(counts, want_counts)
    assert int(counts.sum()) == 3 * B
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = kernels.next_tokens(x, head, noise, counts=counts, **kw, **pick)
    for i in range(3):
        noise.exponential_(generator=gen)
        g.replay()
        torch.cuda.synchronize()
        want = kernels.next_tokens(x, head, noise, counts=want_counts, **kw, **pick)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(counts, want_counts), i
