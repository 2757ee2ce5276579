"""What CachedStepGraph asks of a cache, on the CPU (the recording is replaced by plain calls):
a device cursor, a status, a host ``length`` and ``_check_room``; a paged cache has its own
host state."""

from __future__ import annotations

import pytest
import torch

from dexter_amd.models import KVCache, PagedKVCache
from dexter_amd.runtime import CachedStepGraph, graph


class Plain:
    """A cache of a user's own."""

    def __init__(self, capacity):
        self.capacity, self.length = capacity, 4
        self.cursor = torch.tensor([4], dtype=torch.int32)
        self.status = torch.zeros(1, dtype=torch.int32)

    def _check_room(self, n):
        if self.length + n > self.capacity:
            raise RuntimeError("KV cache full")

    def commit(self, n):
        self.length += n
        self.cursor.add_(n)


@pytest.fixture(autouse=True)
def no_graph(monkeypatch):
    def record(fn, static, warmup, after_each_warmup=None):
        for _ in range(warmup):
            fn(*static)
            after_each_warmup()
        fn(*static)  # a capture runs the host code alone
        for c in record.caches:
            c.cursor.sub_(record.rows)
        return lambda *args: args
    monkeypatch.setattr(graph, "_record", record)
    return record


def _run(cache, record, rows, length):
    record.caches, record.rows = [cache], rows
    x = torch.zeros(1)

    def fn(x):
        cache._check_room(rows)
        cache.commit(rows)
    step = CachedStepGraph(fn, (x,), [cache], rows)
    assert length(cache) == 4 and int(cache.cursor[0]) == 4
    for i in range(3):
        step(x)
        assert length(cache) == 4 + rows * (i + 1)
    return step


def test_a_cache_of_a_users_own(no_graph):
    step = _run(Plain(20), no_graph, 5, lambda c: c.length)
    with pytest.raises(RuntimeError, match="full"):
        step(torch.zeros(1))


def test_the_framework_s_caches(no_graph):
    kv = KVCache(1, 1, 64, 1, 4, "cpu", torch.float32, device_cursor=True)
    kv.commit(4)
    _run(kv, no_graph, 5, lambda c: c.length)
    paged = PagedKVCache(1, 2, 8, 16, 1, 4, "cpu", torch.float32)
    paged.reserve(4)
    paged.commit(4)
    _run(paged, no_graph, 5, lambda c: c.lengths[0])
    assert paged.lengths == [19, 19]
