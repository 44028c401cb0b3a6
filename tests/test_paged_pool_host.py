"""The page accounting of PagedKVCache where calls are refused, on the CPU with the GPU calls
replaced."""

import pytest
import torch

from ascendc_kernel_b200 import paged_cache


@pytest.fixture
def cache(monkeypatch):
    """Two sequences of 9 rows in a pool of 9 pages of 8; eviction refuses what the operator
    refuses, and fails where `cache.broken` is set."""
    made = paged_cache.PagedKVCache(2, 9, 8, 40, 1, 64, track_weights=True, device="cpu")
    made.broken = False

    def evict(kp, vp, weights, table, lens, dst, *, budget, n_first, n_recent):
        assert budget >= 1 and n_first >= 0 and n_recent >= 0 and n_first + n_recent <= budget
        if made.broken:
            raise RuntimeError("the launch failed")
        return None, torch.clamp(lens, max=budget)

    monkeypatch.setattr(paged_cache, "cache_append", lambda *a: None)
    monkeypatch.setattr(paged_cache, "cache_evict", evict)
    made.append(torch.zeros(2, 9, 1, 64))
    return made


def state(c):
    return list(c.free), [list(x) for x in c.pages], list(c.host_lens), c.block_table.tolist()


@pytest.mark.parametrize("args", [(8, 5, 4), (8, -1, 0), (0, 0, 0), (-3, 0, 0), (8, 0, 9)])
def test_a_refused_eviction_keeps_the_pages(cache, args):
    before = state(cache)
    for _ in range(3):
        with pytest.raises(AssertionError):
            cache.evict(*args)
        assert state(cache) == before


def test_a_failed_eviction_keeps_the_pages(cache):
    before = state(cache)
    cache.broken = True
    with pytest.raises(RuntimeError, match="launch"):
        cache.evict(4)
    assert state(cache) == before
    cache.broken = False
    cache.evict(4)
    assert cache.host_lens == [4, 4]
    assert sorted(cache.free + cache.pages[0] + cache.pages[1]) == list(range(9))
