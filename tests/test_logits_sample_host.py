"""sample_logits between its arguments and the library, without a GPU: tensors' sizes and strides are real, the library is a stand-in."""
import contextlib
import threading
import time

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
        self.inside = self.most = self.calls = 0

    def logits_sample(self, args, stream):
        self.inside += 1
        self.calls += 1
        self.most = max(self.most, self.inside)
        time.sleep(0.02)  # as the real one: other threads go on meanwhile
        self.inside -= 1
        return 0


@pytest.fixture
def library(monkeypatch):
    lib = _Library()
    monkeypatch.setattr(sampler._lib, "load", lambda: lib)
    monkeypatch.setattr(sampler, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(sampler, "stream_handle", lambda dev: 0)
    return lib


def test_threads_launch_one_after_another(library, monkeypatch):
    """A call's launches follow each other on the stream: two threads' calls do not mix them."""
    monkeypatch.setattr(sampler, "_workspace", lambda rows, V, dev: torch.zeros(8))
    threads = [threading.Thread(target=lambda: [sampler.sample_logits(_Logits(2, 8)) for _ in range(3)]) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert library.calls == 12 and library.most == 1
