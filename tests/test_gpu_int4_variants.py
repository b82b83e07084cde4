"""Every variant of the 4-bit product's kernels (rwkv-infer-next_amd/csrc/w4a16.hip): each shape of a workgroup with one, two and four
scales a chunk, over enough panels that the blocks' three LDS buffers go round, ends inside a chunk and a strip, and past the last
row.  Against the product in 64 bits of the dequantised weight, both by torch on the device, with test_gpu_int4's bound."""
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"

# (shape, rows / 16, columns / 16) of a workgroup on 256 CUs, and an M and N that give it (test_int4_plan.py holds them to that)
SIZES = [
    (("strips", 1, 1), 9, 1001), (("strips", 1, 2), 16, 5003), (("strips", 1, 4), 7, 10009), (("strips", 1, 1), 50, 1001),
    (("strips", 1, 2), 40, 2003), (("strips", 1, 4), 90, 2003),
    (("block 256", 2, 2), 29, 65301), (("block 256", 4, 2), 61, 65301), (("block 256", 4, 2), 150, 22009),
    (("block 128", 2, 2), 17, 33001), (("block 128", 4, 2), 64, 33001), (("block 128", 4, 2), 203, 8191),
    (("block 64", 2, 1), 32, 16401), (("block 64", 4, 1), 47, 16401), (("block 64", 4, 1), 250, 4097),
]
# K of nine chunks (five panels of two), the last one whole, half or a quarter, with one, two or four scales a chunk
DEPTHS = [(1152, 128), (1088, 64), (1056, 32), (1152, 1152), (1344, 192), (224, 32)]


@pytest.mark.parametrize("K,g", DEPTHS)
@pytest.mark.parametrize("shape,M,N", SIZES, ids=["%s-%d-%d-M%d" % (*s, m) for s, m, _ in SIZES])
def test_variant(shape, M, N, K, g):
    from rwkv_next_amd import kernels
    say("int4 variant", *shape, M, N, K, g)
    gen = torch.Generator(device=DEV).manual_seed(M + N + K)
    codes = torch.randint(0, 256, (K // 2, N), dtype=torch.uint8, device=DEV, generator=gen)
    scales = ((torch.rand(K // g, N, device=DEV, generator=gen) + 0.5) / K ** 0.5).half()
    pk = kernels.prepack_int4(codes, scales, g)
    s = scales.double().repeat_interleave(g, 0)
    w = (torch.stack((codes & 15, codes >> 4), 1).view(K, N).double() - 8) * s
    x = torch.randn(M, K, device=DEV, generator=gen)
    for dtype in (torch.bfloat16, torch.float16):
        a = x.to(dtype)
        got = kernels.int4_matmul(a, pk, out_dtype=torch.float32)
        want, size = a.double() @ w, a.double().abs() @ s
        error = (got.double() - want).abs()
        assert (error <= (144 + K / 32) * 2.0 ** -24 * 55 * size).all()
        assert error.norm() <= 4e-6 * want.norm()
        assert torch.equal(kernels.int4_matmul(a, pk), got.to(dtype))
