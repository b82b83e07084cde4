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
