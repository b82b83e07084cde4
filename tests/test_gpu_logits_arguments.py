"""Arguments of the logit operators at their ends."""
import numpy as np
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_out_beside_the_logits():
    """Rows of `out` between rows of the logits, in one buffer; over them at another place it is refused."""
    from rwkv_next_amd import kernels
    say("penalize out beside the logits")
    B, V = 5, 300
    buf = torch.randn(2 * B + 1, V, device=DEV)
    logits = buf[0:2 * B:2]
    ids, values = torch.full((B, 1), 7, device=DEV), torch.ones(B, 1, device=DEV)
    want = logits.clone()
    want[:, 7] += 1
    for out in (buf[1:2 * B:2], buf[1:2 * B:2].view(torch.bfloat16)[:, :V]):
        assert kernels.penalize_logits(logits, bias_ids=ids, bias_values=values, out=out) is out
        assert torch.equal(out, want.to(out.dtype))
    columns = torch.randn(B, 2 * V, device=DEV)
    want = columns[:, :V].clone()
    want[:, 7] += 1
    kernels.penalize_logits(columns[:, :V], bias_ids=ids, bias_values=values, out=columns[:, V:])
    assert torch.equal(columns[:, V:], want)
    before = buf.clone()
    for x, out in ((buf[:-1], buf[1:]), (buf[1:], buf[:-1]), (columns[:, :V], columns[:, 8:8 + V]), (columns[:, :V], columns[:, V - 1:-1]),
                   (logits, buf[1:B + 1]), (buf.view(-1)[:B * V].view(B, V), buf.view(torch.bfloat16).view(-1)[4:4 + B * V].view(B, V))):
        with pytest.raises(ValueError, match="share memory"):
            kernels.penalize_logits(x, out=out)
    assert torch.equal(buf, before)


def test_tables_without_rows():
    """Every index into a table of no rows lies outside it: left out, and reported."""
    from rwkv_next_amd import kernels
    say("logits empty tables")
    V = 70
    x = torch.randn(2, V, device=DEV)
    status = kernels.new_status(torch.device(DEV))
    slots = torch.tensor([0, 3], device=DEV)
    for dt in (torch.int32, torch.float32):
        counts = torch.zeros(0, V, dtype=dt, device=DEV)
        status.zero_()
        y = kernels.penalize_logits(x, counts=counts, slots=slots, repetition=1.5, presence=1.0, status=status)
        assert torch.equal(y, x) and int(status) == 256
        status.zero_()
        token, _ = kernels.sample_logits(x, counts=counts, slots=slots, status=status)
        assert torch.equal(token, x.argmax(dim=1)) and int(status) == 256
    mask = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    for rows, bits in (([0, -1], 256), ([-1, -2], 0)):
        status.zero_()
        y = kernels.penalize_logits(x, mask=mask, mask_rows=torch.tensor(rows, device=DEV), status=status)
        assert torch.equal(y, x) and int(status) == bits


def test_one_row_for_all_sequences():
    """Broadcast rows (a stride of 0) of biases, drafts and masks: as their copies."""
    from rwkv_next_amd import kernels
    say("logits broadcast rows")
    rng = np.random.default_rng(1)
    B, T, V, P = 4, 3, 501, 5
    x = torch.from_numpy(rng.standard_normal((B, T, V)).astype(np.float32)).to(DEV)
    ids = torch.from_numpy(rng.integers(0, V, (1, P))).to(DEV).expand(B, P)
    values = torch.from_numpy(rng.standard_normal((1, P)).astype(np.float32)).to(DEV).expand(B, P)
    drafts = torch.from_numpy(rng.integers(0, V, (1, T - 1))).to(DEV).expand(B, T - 1)
    bits = torch.from_numpy(rng.integers(0, 2 ** 32, (1, 16), dtype=np.uint32).view(np.int32)).to(DEV)
    for logits, kw in [(x, dict(bias_ids=ids, bias_values=values)), (x, dict(bias_ids=ids.contiguous(), bias_values=values)),
                       (x, dict(drafts=drafts, presence=0.5)), (x, dict(mask=bits.expand(B, T, 16))),
                       (x[:, 0], dict(mask=bits.expand(B, 16))),
                       (x[:, 0], dict(mask=bits.expand(3, 16), mask_rows=torch.tensor([0, 2, 1, -1], device=DEV)))]:
        copies = {k: v.contiguous() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
        assert torch.equal(kernels.penalize_logits(logits, **kw), kernels.penalize_logits(logits, **copies)), sorted(kw)
