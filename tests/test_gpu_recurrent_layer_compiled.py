"""A layer of the gated delta rule under a tracer: its operators are the registered ops, with the types that they ask of each other."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _weights(gen, *sizes):
    from rwkv_next_amd.kernels import prepack_dense
    return [prepack_dense((torch.randn(k, n, device=DEV, generator=gen) / k ** 0.5).bfloat16()) for k, n in sizes]


@pytest.mark.parametrize("out_dtype", [None, torch.bfloat16, torch.float16, torch.float32])
def test_the_product_as_an_op_has_its_result_types(out_dtype):
    from rwkv_next_amd.kernels import dense_matmul, dense_matmul_op
    gen = torch.Generator(device=DEV).manual_seed(1)
    (p,) = _weights(gen, (96, 40))
    a, b = torch.randn(5, 96, device=DEV, generator=gen).bfloat16(), torch.randn(40, device=DEV, generator=gen)
    want = dense_matmul(a, p, bias=b, activation="sigmoid", out_dtype=out_dtype)
    got = dense_matmul_op(a, p.weight, p.K, p.N, b, "sigmoid", None, out_dtype)
    assert got.dtype == want.dtype == (out_dtype or torch.bfloat16) and torch.equal(got, want)
    torch.library.opcheck(dense_matmul_op, (a, p.weight, p.K, p.N, b, "sigmoid", None, out_dtype))
    assert torch.equal(dense_matmul_op(a, p.weight, p.K, p.N, b, "sigmoid", None), dense_matmul(a, p, bias=b, activation="sigmoid"))


@pytest.mark.parametrize("T", [1, 5, 40])
def test_a_compiled_layer(T):
    """Traced whole (fullgraph), its graph run as it is: the bits of the eager layer, its pool written in place."""
    from rwkv_next_amd.kernels import dense_matmul, dense_matmul_op, gated_delta_pool_
    gen = torch.Generator(device=DEV).manual_seed(2)
    C, HK, HV, K, V = 128, 2, 4, 64, 64
    qkv, step, write, out = _weights(gen, (C, 2 * HK * K + HV * V), (C, HV), (C, HV), (HV * V, C))
    bias = torch.randn(HV, device=DEV, generator=gen)

    def layer(product, x, pool, slots):
        f = product(x, qkv)
        q, k, v = (f[..., :HK * K].unflatten(-1, (HK, K)), f[..., HK * K:2 * HK * K].unflatten(-1, (HK, K)),
                   f[..., 2 * HK * K:].unflatten(-1, (HV, V)))
        g = -product(x, step, bias=bias, activation="sigmoid", out_dtype=torch.float32)
        beta = product(x, write, activation="sigmoid", out_dtype=torch.float32)
        o = gated_delta_pool_(q, k, v, g, beta, pool, slots, qk_norm=True)
        return product(o.flatten(2), out, residual=x)

    def as_op(x, p, bias=None, activation="none", residual=None, out_dtype=None):
        return dense_matmul_op(x, p.weight, p.K, p.N, bias, activation, residual, out_dtype)

    x = torch.randn(3, T, C, device=DEV, generator=gen).bfloat16()
    pool, slots = torch.randn(6, HV, K, V, device=DEV, generator=gen), torch.tensor([4, 0, 5], device=DEV)
    mine, eager = pool.clone(), pool.clone()
    compiled = torch.compile(lambda x, pool, slots: layer(as_op, x, pool, slots), backend="aot_eager", fullgraph=True)
    with torch.no_grad():
        for _ in range(2):
            assert torch.equal(compiled(x, mine, slots), layer(dense_matmul, x, eager, slots)) and torch.equal(mine, eager)
    assert not torch.equal(mine, pool)
