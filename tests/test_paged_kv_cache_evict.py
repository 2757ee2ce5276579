"""PagedKVCache.evict's page keeping, on the CPU: its kernels are replaced by the oracle's
plain forms; every sequence's rows are compared with a plain list of what it was given."""

from __future__ import annotations

import random

import pytest
import torch

from dexter_amd import ops
from dexter_amd.models import PagedKVCache
from oracle import keep
from test_paged_kv_cache import _check, _step, plain_ops  # noqa: F401
from test_paged_kv_cache_errors import _state


@pytest.fixture(autouse=True)
def plain_keep(monkeypatch):
    def gather(pages, table, rows, dst=None, weights=None, head_dim=None):
        dst = table if dst is None else dst
        pages.copy_(keep.gather(pages, table.tolist(), rows, dst.tolist()))
        weights.copy_(keep.gather_weights(weights, rows))
    monkeypatch.setattr(ops, "kv_keep_rows", lambda w, lens, k, recent=0: keep.keep_rows(w, lens.tolist(), k, recent))
    monkeypatch.setattr(ops, "kv_page_gather", gather)


def _cache(batch=3, pages=20, **kw):
    return PagedKVCache(2, batch, pages, 16, 1, 4, "cpu", torch.float32, track_weights=True, **kw)


def _weigh(kv, seed):
    g = torch.Generator().manual_seed(seed)
    for b, n in enumerate(kv.lengths):
        kv.weights[:, b, :, :n] += torch.rand(1, 1, n, generator=g)  # the same in both layers


def _evict(kv, want, k, recent):
    """evict(), and the same to the plain lists, by the first layer's weights."""
    rows = keep.keep_rows(kv.weights[0], kv.lengths, k, recent)
    long = [b for b in range(kv.batch) if kv.lengths[b] > k]
    assert kv.evict(k, recent) == len(long)
    for b in long:
        want[b] = [want[b][r] for r in rows[b, 0].tolist()]


def test_in_place_and_shared():
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 50, 0)
    kv.free(2)
    kv.fork(0, 2)
    want[2] = list(want[0])
    _weigh(kv, 1)
    kv.weights[:, 2] = kv.weights[:, 0] + 1  # (the same order)
    _evict(kv, want, 20, 4)
    _check(kv, want)
    # 1's rows stayed on its first pages; 0 and 2, which shared theirs, each have new ones.
    assert len({p for t in kv.tables for p in t}) == 6 and kv.free_pages == 14
    _step(kv, want, 30, 500)
    _check(kv, want)
    assert bool((kv.weights[..., 20:] == 0).all())
    assert kv.evict(60) == 0


def test_a_full_pool_refuses_with_nothing_changed():
    kv, want = _cache(batch=2, pages=8), [[], []]
    _step(kv, want, 60, 0)
    kv.free(1)
    kv.fork(0, 1)
    want[1] = list(want[0])
    kv.reserve(1)  # copies the shared last page: three are shared, three free
    before, w = _state(kv), kv.weights.clone()
    with pytest.raises(RuntimeError, match="KV cache full: 4 pages needed, 3 of 8 free"):
        kv.evict(20)
    assert _state(kv) == before and torch.equal(kv.weights, w)
    _check_rows = kv.evict(0)
    assert _check_rows == 2 and kv.lengths == [0, 0] and kv.free_pages == 8


def test_refusals():
    kv = PagedKVCache(1, 1, 4, 16, 1, 4, "cpu", torch.float32)
    with pytest.raises(RuntimeError, match="track_weights"):
        kv.evict(3)
    kv = _cache()
    for args in ((-1,), (3, -1)):
        with pytest.raises(ValueError, match="cannot keep"):
            kv.evict(*args)
    for kw in (dict(dtype=torch.float32, head_dim=64), dict(dtype=torch.bfloat16, head_dim=32)):
        with pytest.raises(ValueError, match="4 bits"):
            PagedKVCache(1, 1, 4, 16, 1, device="cpu", fp4=True, **kw)


def test_many_steps():
    rng = random.Random(4)
    kv, want = _cache(batch=4, pages=80, max_rows=200), [[] for _ in range(4)]
    for i in range(80):
        what = rng.choice(["step", "step", "evict", "fork", "free", "compact"])
        if what == "step" and max(kv.lengths) < 150:
            _step(kv, want, rng.randint(1, 40), 1000 * i)
            _weigh(kv, i)
        elif what == "evict":
            _evict(kv, want, rng.randint(0, 60), rng.randint(0, 20))
        elif what == "fork":
            a, b = rng.sample(range(4), 2)
            kv.fork(a, b)
            want[b] = list(want[a])
            assert torch.equal(kv.weights[:, a], kv.weights[:, b])
        elif what == "free":
            b = rng.randrange(4)
            kv.free(b)
            want[b] = []
            assert not kv.weights[:, b].any()
        else:
            kv.compact()
        _check(kv, want)
        for b, n in enumerate(kv.lengths):
            assert not kv.weights[:, b, :, n:].any()
