"""dense_matmul by each of its tiles, with K whole, shared within a workgroup and in parts of two launches, against 64 bits.

Bounds as in test_gpu_dense.py: a sum of K exact products is off by at most (K + 8) u times the sum of their sizes, u = 2^-24, whatever the order,
that of K's groups and parts included."""
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24

# rows, K, columns: what the rule takes them to on 256 CUs
SHAPES = [
    (1, 32, 16), (9, 64, 33), (16, 1056, 8192), (100, 416, 500), (300, 1600, 400), (17, 32, 1), (40, 2080, 1000),  # 16 x 16
    (7, 10272, 300), (16, 10272, 2560), (33, 6176, 640),                                             # .. in parts
    (3, 96, 8209), (16, 1120, 8704), (64, 416, 2600), (30, 4096, 4200), (300, 3104, 700),           # 16 x 64
    (17, 64, 16400), (130, 800, 2600), (33, 96, 8100),                            # 32 x 64
    (32, 10272, 5000),                                                            # .. in parts
    (64, 64, 16385), (50, 2080, 16000), (190, 96, 4100),                          # 64 x 64
    (64, 10272, 4160),                                                            # .. in parts
    (5, 4128, 8300), (32, 2080, 16160), (60, 4128, 8700),                         # the three by loads past the caches
    (70, 10272, 2000), (128, 3104, 4112), (257, 2592, 2100), (129, 32, 33000),    # 128 x 128, whole and in parts
    (1024, 2624, 4096), (400, 10272, 2564), (2050, 96, 8193), (513, 2720, 4104),  # 128 x 256, whole and in parts
]


def _inputs(M, K, N, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    a = torch.randn(M, K, device=DEV, generator=gen).to(dtype)
    w = (torch.randn(K, N, device=DEV, generator=gen) / K ** 0.5).to(dtype)
    return a, w, torch.randn(N, device=DEV, generator=gen), torch.randn(M, N, device=DEV, generator=gen).to(dtype)


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tiles(M, K, N, dtype):
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    say("tiles", M, K, N, dtype)
    a, w, b, r = _inputs(M, K, N, dtype, M + K + N)
    p = prepack_dense(w)
    y = dense_matmul(a, p, out_dtype=torch.float32)
    want = a.double() @ w.double()
    bound = (K + 8) * U * (a.double().abs() @ w.double().abs()) + 1e-37
    assert (((y.double() - want).abs()) <= bound).all(), ((y.double() - want).abs() / bound).max()
    assert torch.equal(dense_matmul(a, p), y.to(dtype))
    for odd in (False, True):  # an odd stride of the residual: columns one by one
        res = torch.zeros(M, N + 1 if odd else N, device=DEV, dtype=dtype)[:, :N]
        res.copy_(r)
        z = dense_matmul(a, p, bias=b, residual=res, out_dtype=torch.float32)
        off = bound + 2 * U * (want.abs() + b.abs() + r.double().abs() + bound)
        assert ((z.double() - (want + b.double() + r.double())).abs() <= off).all()
        assert torch.equal(dense_matmul(a, p, bias=b, residual=res), z.to(dtype))


@pytest.mark.parametrize("M,K,N", [(5, 192, 100), (33, 6176, 640), (64, 10272, 4160), (64, 4128, 4160), (128, 3104, 4112),
                                   (400, 10272, 2564)])
def test_values_that_are_not_finite_behind_the_last_step(M, K, N):
    """The last step of K, an odd one, is multiplied once: an infinity there stays one."""
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    a, w, _, _ = _inputs(M, K, N, torch.bfloat16, 7)
    a[:] = a.abs() + 0.125
    clean = dense_matmul(a, prepack_dense(w))
    w2 = w.clone()
    w2[K - 1, N - 1] = float("inf")
    y = dense_matmul(a, prepack_dense(w2))
    assert torch.equal(y[:, :N - 1], clean[:, :N - 1]) and (y[:, N - 1] == float("inf")).all()


@pytest.mark.parametrize("M,K,N", [(7, 10272, 300), (32, 10272, 5000), (128, 3104, 4112), (400, 10272, 2564)])
def test_split_products_on_two_streams_and_in_a_graph(M, K, N):
    """Parts of K in a workspace of the call's own."""
    from rwkv_next_amd.kernels import dense_matmul, prepack_dense
    a, w, b, _ = _inputs(M, K, N, torch.bfloat16, 8)
    p = prepack_dense(w)
    want, other = dense_matmul(a, p, bias=b), dense_matmul(-a, p, bias=b)
    side, now = torch.cuda.Stream(), torch.cuda.current_stream()
    side.wait_stream(now)
    for _ in range(4):
        with torch.cuda.stream(side):
            x = dense_matmul(-a, p, bias=b)
        y = dense_matmul(a, p, bias=b)
        now.wait_stream(side)
        assert torch.equal(x, other) and torch.equal(y, want)
        side.wait_stream(now)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    xs = a.clone()
    with torch.cuda.graph(one):
        x = dense_matmul(xs, p, bias=b)
    with torch.cuda.graph(two):
        y = dense_matmul(xs, p, bias=b)
    for i in range(4):
        xs.copy_(-a if i % 2 else a)
        one.replay()
        two.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, other if i % 2 else want) and torch.equal(y, x)
        assert torch.equal(dense_matmul(a, p, bias=b), want)
