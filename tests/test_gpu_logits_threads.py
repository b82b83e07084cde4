"""The workspace that the launches of a sample_logits call share: threads of one stream, and a state that no call left behind."""
import ctypes
import threading

import numpy as np
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_threads_of_one_stream():
    from rwkv_next_amd import kernels
    say("sample threads")
    rng = np.random.default_rng(1)
    work = []
    for rows, V, kw in ((3, 40000, dict(top_p=0.9)), (40, 3001, dict(top_k=20, top_p=0.9)), (1, 65536, dict()), (7, 500, dict(top_k=5))):
        x = torch.from_numpy((rng.standard_normal((rows, V)) * 3).astype(np.float32)).to(DEV)
        noise = torch.from_numpy(rng.exponential(size=(rows, V)).astype(np.float32)).to(DEV)
        work.append((x, noise, kw, kernels.sample_logits(x, noise, **kw)))
    torch.cuda.synchronize()
    wrong = []

    def loop(x, noise, kw, want):
        got = [kernels.sample_logits(x, noise, **kw) for _ in range(50)]
        torch.cuda.synchronize()
        wrong.extend(kw for g in got if not all(torch.equal(a, b) for a, b in zip(g, want)))

    threads = [threading.Thread(target=loop, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("field", ["max_key", "won"])
def test_a_token_past_the_row_touches_nothing(field):
    """A workspace that was not zero, as when two calls run on it at the same time: an index past the row is no token."""
    from rwkv_next_amd import _lib
    say("sample dirty workspace", field)
    V = 100
    x, noise = torch.zeros(1, V, device=DEV), torch.ones(1, V, device=DEV)
    counts = torch.zeros(1, V, dtype=torch.int32, device=DEV)
    token, logprob = torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(1, device=DEV)
    size = ctypes.c_size_t(0)
    args = _lib.SampleArgs(B=1, T=1, V=V)
    _lib.check(_lib.load().logits_sample_workspace_size(ctypes.byref(args), ctypes.byref(size)))
    ws = torch.zeros(size.value, dtype=torch.uint8, device=DEV)
    # a score (or logit) of 2^100 at index 2^30
    bits = {"max_key": 0x80000000 | 0x71800000, "won": 0x71800000}[field]
    key = np.array([bits << 32 | (~(1 << 30) & 0xFFFFFFFF)], np.uint64)
    ws[:24].view(torch.int64)[{"max_key": 0, "won": 2}[field]] = int(key.view(np.int64)[0])
    args = _lib.SampleArgs(logits=x.data_ptr(), seq_stride=V, noise=noise.data_ptr() if field == "won" else None, noise_seq_stride=V,
                           token=token.data_ptr(), logprob=logprob.data_ptr(), counts=counts.data_ptr(), counts_stride=V, counts_rows=1,
                           workspace=ws.data_ptr(), workspace_bytes=size.value, temperature_all=1.0, top_p_all=1.0, B=1, T=1, V=V,
                           dtype=_lib.LOGITS_F32, counts_dtype=_lib.LOGITS_COUNTS_I32)
    _lib.check(_lib.load().logits_sample(ctypes.byref(args), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    torch.cuda.synchronize()
    assert int(token) == -1 and float(logprob) == -float("inf") and not counts.any()
    assert not ws[:_lib.LOGITS_SAMPLE_STATE_BYTES].any()
