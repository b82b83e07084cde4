"""Values of the sampling kernels (rwkv-infer-next_amd/csrc/logits_sample.hip) that looser comparisons let through."""
import numpy as np
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def test_top_p_at_a_bins_end():
    """The first bin's weight is half of all, to the last bit of the sums: whether that reaches a top-p of a half or needs one token more,
    it never takes all of the next bin.  Logits are at the starts of bins, 32nds below the largest, so many tokens at each."""
    from rwkv_next_amd import kernels
    say("sample top-p at a bin's end")
    at = [0] * 7 + [55] * 3 + [56] * 35 + [59, 67, 88, 126, 150, 188, 208, 219, 255, 275, 343, 364, 381, 385, 395, 505, 682, 878, 1009]
    x = torch.full((1, 200), -np.inf)
    x[0, :len(at)] = -torch.tensor(at) / 32
    noise = torch.ones(1, 200)
    noise[0, 9] = 1e-6  # the last of the second bin
    token, _ = kernels.sample_logits(x.to(DEV), noise.to(DEV), top_p=0.5)
    assert int(token) == 0
