"""What KVCache.advance knows of `lengths`: a bound on the host as long as it alone
changes them, else what it reads."""
import contextlib

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(max_tokens=64, batch=2):
    from ttjam_gottagofast_b200 import KVCache

    return KVCache(batch, max_tokens, 1, 16, page_size=16)


@contextlib.contextmanager
def _no_sync():
    torch.cuda.set_sync_debug_mode("error")
    try:
        yield
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_a_graph_of_the_callers_that_counts_tokens():
    """Its replays change lengths without a count that the host could see."""
    cache = _cache()
    cache.advance(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.lengths.add_(10)
    cache.advance(1)
    for _ in range(6):
        graph.replay()
    with pytest.raises(ValueError, match="full"):
        cache.advance(3)
    assert cache.lengths.tolist() == [62, 62]
    cache.advance(2)
    cache.reset()
    cache.advance(1)
    for _ in range(6):
        graph.replay()
    with pytest.raises(ValueError, match="full"):
        cache.advance(4)
    assert cache.lengths.tolist() == [61, 61]


def test_a_captured_reset_and_advance():
    cache = _cache()
    cache.advance(60)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.reset()
        cache.advance(50)
    with pytest.raises(ValueError, match="full"):
        cache.advance(5)
    graph.replay()
    cache.advance(14)
    assert cache.lengths.tolist() == [64, 64]


def test_changes_that_torch_does_not_count():
    cache = _cache()
    cache.advance(1)
    cache.lengths_changed()
    cache.advance(1)
    cache.lengths.data.fill_(60)
    with pytest.raises(ValueError, match="full"):
        cache.advance(5)
    assert cache.lengths.tolist() == [60, 60]


def test_a_cache_over_the_callers_tensors_reads_them():
    from ttjam_gottagofast_b200 import KVCache

    own = _cache()
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = KVCache.from_tensors(own.k, own.v, own.k_scale, own.v_scale, own.block_table, lengths)
    cache.advance(1)
    lengths.data.fill_(60)
    with pytest.raises(ValueError, match="full"):
        cache.advance(5)
    assert lengths.tolist() == [60, 60]


def test_a_cache_of_its_own_lengths_is_not_read():
    """Advanced and reset by itself alone, also in inference mode: no host sync."""
    for mode in (contextlib.nullcontext, torch.inference_mode):
        with mode():
            cache = _cache(max_tokens=1024)
            counts = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
            with _no_sync():
                cache.advance(200)
                cache.advance(3, new_tokens=counts)
                cache.reset()
                for _ in range(1024):
                    cache.advance(1)
            assert cache.lengths.tolist() == [1024, 1024]
            with pytest.raises(ValueError, match="full"):
                cache.advance(1)
