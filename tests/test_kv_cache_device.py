"""KVCache on another device than the current one, without a GPU: what the C calls get and
which device is current then."""
import contextlib

import pytest
import torch

from ttjam_gottagofast_b200 import KVCache, kv_cache


@pytest.fixture
def devices(monkeypatch):
    """Two made-up devices, 0 the current one; [current device] at the time."""
    current = [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], torch.device(d).index
        yield
        current[0] = before

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: type("Stream", (), {"cuda_stream": 0}))
    monkeypatch.setattr(kv_cache, "_current_device", lambda: current[0])
    monkeypatch.setattr(kv_cache, "_raw_stream", lambda index: 0)  # the default stream of whichever
    return current


class _Lib:
    def __init__(self, current):
        self.current, self.calls = current, []

    def tt_kv_read_status(self, cache, code, detail, stream):
        self.calls.append((self.current[0], stream))
        return 0


def test_status_is_read_on_the_caches_device(devices):
    """The default stream's handle is that of the current device: read there, the status
    would not wait for the cache's kernels."""
    cache = KVCache.__new__(KVCache)
    cache.device, cache._index, cache._structs = torch.device("cuda:1"), 1, [None]
    cache._lib = _Lib(devices)
    assert cache.read_device_status() == (0, 0)
    assert cache._lib.calls == [(1, 0)]
    assert devices[0] == 0
