"""What the logit operators and the 4-bit products refuse before any launch, by their Python entry points."""
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device=DEV)


def test_penalize_logits_refuses():
    from rwkv_next_amd import kernels
    say("penalize refusals")
    x, y = _t(2, 64), _t(2, 3, 64)
    i64, i32 = torch.int64, torch.int32
    cpu = torch.zeros(2)
    for logits, kw in [
        (x.double(), {}), (x.long(), {}), (x[0], {}), (_t(1, 2, 3, 4), {}), (x.cpu(), {}),
        (x, dict(counts=_t(2, 63, dtype=i32))), (x, dict(counts=_t(2, 64, dtype=i64))), (x, dict(counts=_t(1, 64, dtype=i32))),
        (x, dict(counts=_t(64, 2, dtype=i32).t())), (x, dict(counts=torch.zeros(2, 64, dtype=i32))),
        (x, dict(slots=_t(2, dtype=i64))), (x, dict(counts=_t(5, 64, dtype=i32), slots=_t(3, dtype=i64))),
        (x, dict(counts=_t(5, 64, dtype=i32), slots=_t(2, dtype=i32))), (x, dict(counts=_t(5, 64, dtype=i32), slots=[0, 1])),
        (x, dict(repetition=_t(3))), (x, dict(repetition=_t(2).double())), (x, dict(presence=cpu)),
        (x, dict(frequency=_t(4)[::2])), (x, dict(repetition=0.0)), (x, dict(repetition=-1.0)),
        (y, dict(drafts=_t(2, 1, dtype=i64))), (y, dict(drafts=_t(3, 2, dtype=i64))), (y, dict(drafts=_t(2, 2, dtype=i32))),
        (x, dict(bias_ids=_t(2, 3, dtype=i64))), (x, dict(bias_values=_t(2, 3))),
        (x, dict(bias_ids=_t(2, 3, dtype=i64), bias_values=_t(2, 4))), (x, dict(bias_ids=_t(2, 3, dtype=i32), bias_values=_t(2, 3))),
        (x, dict(bias_ids=_t(1, 3, dtype=i64), bias_values=_t(1, 3))),
        (x, dict(mask=_t(2, 1, dtype=i32))), (x, dict(mask=_t(2, 2))), (y, dict(mask=_t(2, 2, dtype=i32))),
        (x, dict(mask_rows=_t(2, dtype=i64))), (x, dict(mask=_t(4, 2, dtype=i32), mask_rows=_t(3, dtype=i64))),
        (x, dict(mask=_t(4, 2, dtype=i32), mask_rows=_t(2, dtype=i32))), (y, dict(mask=_t(2, 3, 2, dtype=i32), mask_rows=_t(2, 3, dtype=i64))),
        (x, dict(out=_t(2, 63))), (x, dict(out=_t(2, 64).double())), (x, dict(out=_t(64, 2).t())), (x, dict(out=cpu)),
        (x, dict(out=_t(1, 64).expand(2, 64))), (x, dict(out=x.view(torch.int32).view(torch.bfloat16)[:, :64])),
        (x, dict(status=_t(1))), (x, dict(status=torch.zeros(1, dtype=i32))),
    ]:
        with pytest.raises((ValueError, TypeError)):
            kernels.penalize_logits(logits, **kw)
    strided = _t(64, 2).t()
    with pytest.raises(ValueError):
        kernels.penalize_logits(strided, out=strided)
    same = _t(1, 64).expand(2, 64)
    with pytest.raises(ValueError):
        kernels.penalize_logits(same, out=same)


def test_sample_logits_refuses():
    from rwkv_next_amd import kernels
    say("sample refusals")
    x, y = _t(2, 64), _t(2, 3, 64)
    i64, i32 = torch.int64, torch.int32
    for logits, kw in [
        (x.double(), {}), (x[0], {}), (x.cpu(), {}), (_t(2, 0), {}),
        (x, dict(noise=_t(2, 63))), (x, dict(noise=_t(2, 64).bfloat16())), (y, dict(noise=x)), (x, dict(noise=torch.zeros(2, 64))),
        (x, dict(temperature=_t(3))), (x, dict(top_k=_t(2, dtype=i64))), (x, dict(top_p=_t(2).double())),
        (x, dict(min_p=_t(2, 1))), (x, dict(temperature=torch.ones(2))),
        (y, dict(counts=_t(2, 64, dtype=i32))), (x, dict(counts=_t(2, 65, dtype=i32))), (x, dict(slots=_t(2, dtype=i64))),
        (x, dict(counts=_t(4, 64, dtype=i32), slots=_t(2, dtype=i32))),
    ]:
        with pytest.raises((ValueError, TypeError)):
            kernels.sample_logits(logits, **kw)
    with pytest.raises(_lib_error()):
        kernels.sample_logits(_t(1, 2 ** 21 + 1))


def _lib_error():
    from rwkv_next_amd import _lib
    return _lib.Wkv7Error


def test_int4_refuses():
    from rwkv_next_amd import kernels
    say("int4 refusals")
    codes, scales = _t(64, 40, dtype=torch.uint8), _t(2, 40, dtype=torch.float16)
    pk = kernels.prepack_int4(codes, scales, 64)
    a = _t(3, 128, dtype=torch.bfloat16)
    for bad in [(codes, scales, 32), (codes, scales, 48), (codes, scales[:1], 64), (codes[:, :39], scales, 64), (codes[0], scales, 64),
                (codes, scales.cpu(), 64), (codes.int(), scales, 64), (codes, scales.float(), 64), (codes[:60], scales, 64)]:
        with pytest.raises((ValueError, TypeError)):
            kernels.prepack_int4(*bad)
        with pytest.raises((ValueError, TypeError)):
            kernels.dequantize_int4(*bad)
    with pytest.raises(TypeError):
        kernels.dequantize_int4(codes, scales, 64, dtype=torch.float64)
    for x, w, kw in [(a[:, :64], pk, {}), (a.float(), pk, {}), (a.cpu(), pk, {}), (a, pk, dict(out_dtype=torch.int32)),
                     (a, pk._replace(N=41 + 16), {}), (a, pk._replace(K=256), {}), (a, pk._replace(weight=pk.weight[:-1]), {}),
                     (a, pk._replace(scales=pk.scales.float()), {}), (a, pk._replace(scales=pk.scales.cpu()), {}),
                     (a[0, 0], pk, {})]:
        with pytest.raises((ValueError, TypeError)):
            kernels.int4_matmul(x, w, **kw)
    with pytest.raises(ValueError):
        kernels.next_tokens(a[None], pk)
