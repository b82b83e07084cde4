"""sample_logits between its arguments and the library, without a GPU: tensors' sizes and strides are real, the library is a stand-in."""
import contextlib
import ctypes
import threading
import time
import types

import pytest

torch = pytest.importorskip("torch")

from rwkv_next_amd.kernels import sampler  # noqa: E402


class _Logits:
    """A CPU tensor that says that it is on a GPU."""

    def __init__(self, *shape):
        self.t = torch.zeros(shape)

    is_cuda = True

    def __getattr__(self, name):
        return getattr(self.t, name)


class _Library:
    """Stands for the shared library: notes how many calls are inside logits_sample at once."""

    def __init__(self):
        self.inside = self.most = self.calls = self.code = 0

    def logits_sample(self, args, stream):
        self.inside += 1
        self.calls += 1
        self.most = max(self.most, self.inside)
        time.sleep(0.02)  # as the real one: other threads go on meanwhile
        self.inside -= 1
        return self.code

    def wkv7_strerror(self, code):
        return b"refused"


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(sampler._lib, "load", lambda: lib)
    monkeypatch.setattr(sampler, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(sampler, "stream_handle", lambda dev: 0)
    return lib


def test_threads_launch_one_after_another(library, monkeypatch):
    """A call's launches follow each other on the stream: two threads' calls do not mix them."""
    monkeypatch.setattr(sampler, "_workspace", lambda *_: torch.zeros(8))
    threads = [threading.Thread(target=lambda: [sampler.sample_logits(_Logits(2, 8)) for _ in range(3)]) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert library.calls == 12 and library.most == 1


def _bytes(t):
    at = torch.arange(t.untyped_storage().nbytes() // t.element_size()).as_strided(t.shape, t.stride(), t.storage_offset())
    return {int(i) * t.element_size() + b for i in at.reshape(-1).unique() for b in range(t.element_size())}


def test_shared_memory_is_found():
    """Against the bytes that two views of one buffer have; out over the logits at another place is refused, before any launch."""
    buf = torch.zeros(4000, dtype=torch.bfloat16)
    views = [buf.as_strided(shape, stride, at) for shape, stride in [
        ((3, 50), (50, 1)), ((3, 50), (100, 1)), ((3, 50), (120, 1)), ((1, 50), (7, 1)), ((4, 2, 25), (100, 50, 1)), ((2, 4, 25), (25, 50, 1)),
        ((2, 3, 50), (0, 60, 1)), ((3, 1), (9, 1)), ((2, 0, 5), (9, 5, 1))] for at in (0, 8, 50, 58, 150, 500, 2)]
    views += [v.view(torch.float32) for v in views if v.shape[-1] % 2 == 0 and v.storage_offset() % 2 == 0 and
              all(s % 2 == 0 for s in v.stride()[:-1])]
    seen = set()
    for a in views:
        for b in views:
            want = bool(_bytes(a) & _bytes(b))
            seen.add(want)
            assert sampler._share_memory(a, b) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert seen == {False, True}


def test_one_workspace_serves_any_number_of_rows(monkeypatch):
    """Calls of ever more rows ask for the same bytes: nothing is replaced, and so nothing kept beside it."""
    asked = set()

    def note(cache, dev, nbytes, zero_bytes):
        asked.add((nbytes, zero_bytes))
        return torch.zeros(8)

    monkeypatch.setattr(sampler, "stream_workspace", note)
    monkeypatch.setattr(sampler, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(sampler, "stream_handle", lambda dev: 0)
    real, size = sampler._lib.load(), ctypes.c_size_t(0)
    monkeypatch.setattr(sampler._lib, "load", lambda: types.SimpleNamespace(
        logits_sample=lambda args, stream: 0, logits_sample_workspace_size=real.logits_sample_workspace_size))
    for rows in (1, 132, 133, 134, 511, 512, 513, 5000):
        sampler.sample_logits(_Logits(rows, 3))
        sampler.sample_logits(_Logits(rows, 2, 3))
    assert len(asked) == 1
    nbytes, zero = asked.pop()
    assert zero == sampler._lib.LOGITS_SAMPLE_STATE_BYTES
    for rows in (1, 512, 10 ** 6):
        args = sampler._lib.SampleArgs(B=rows, T=3, V=100)
        assert real.logits_sample_workspace_size(ctypes.byref(args), ctypes.byref(size)) == 0 and size.value <= nbytes < 32 << 20


def test_a_workspace_is_given_up_after_a_failed_launch_and_on_request(library, monkeypatch):
    from rwkv_next_amd.kernels import _workspace
    from rwkv_next_amd.kernels.wkv7 import reset_workspaces
    ws = torch.zeros(8)
    monkeypatch.setattr(sampler, "_workspace", lambda *_: ws)
    monkeypatch.setattr(sampler, "_WORKSPACES", {(0, 0): [ws, True, None]})
    monkeypatch.setattr(_workspace, "_RETIRED", [])
    for code, left in ((0, 1), (sampler._lib.WKV7_ERR_SHAPE, 1), (1, 0)):  # done, refused before any launch, an error of a launch
        library.code = code
        if code:
            with pytest.raises(sampler._lib.Wkv7Error):
                sampler.sample_logits(_Logits(2, 8))
        else:
            sampler.sample_logits(_Logits(2, 8))
        assert len(sampler._WORKSPACES) == left and len(_workspace._RETIRED) == 1 - left
    sampler._WORKSPACES[0, 0] = [ws, True, None]
    reset_workspaces()
    assert not sampler._WORKSPACES and len(_workspace._RETIRED) == 2  # captured graphs may still address them
