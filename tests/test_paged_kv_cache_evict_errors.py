"""PagedKVCache.evict when a call fails half-way, on the CPU (the kernels it launches are replaced
by the oracle's plain forms)."""

from __future__ import annotations

import pytest
import torch

from dexter_amd import ops
from oracle import keep
from test_paged_kv_cache import _check, _step, plain_ops  # noqa: F401
from test_paged_kv_cache_errors import _state
from test_paged_kv_cache_evict import _cache, _evict, _weigh, plain_keep  # noqa: F401


@pytest.mark.parametrize("shared", [False, True])
def test_a_choice_that_fails_changes_nothing(monkeypatch, shared):
    """Rows are chosen for every layer before any layer's move: where a later layer's choice
    raises (out of memory), no layer's rows have moved, and a later evict does it all."""
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 50, 0)
    _weigh(kv, 1)
    if shared:
        kv.fork(0, 2)
        want[2] = list(want[0])
    before, pools, w = _state(kv), [p.clone() for p in kv.pools], kv.weights.clone()
    choose, calls = ops.kv_keep_rows, []

    def fail(*args):
        calls.append(args)
        if len(calls) == 2:
            raise torch.OutOfMemoryError("no memory for the second layer's rows")
        return choose(*args)
    monkeypatch.setattr(ops, "kv_keep_rows", fail)
    with pytest.raises(torch.OutOfMemoryError):
        kv.evict(20, 4)
    assert _state(kv) == before and torch.equal(kv.weights, w)
    assert all(torch.equal(a, b) for a, b in zip(kv.pools, pools))
    monkeypatch.setattr(ops, "kv_keep_rows", choose)
    _evict(kv, want, 20, 4)
    _check(kv, want)


def _full():
    """Two sequences of 60 rows on a pool of 8 pages: three pages shared, three free."""
    kv, want = _cache(batch=2, pages=8), [[], []]
    _step(kv, want, 60, 0)
    kv.free(1)
    kv.fork(0, 1)
    want[1] = list(want[0])
    kv.reserve(1)
    _weigh(kv, 1)
    kv.weights[:, 1] = kv.weights[:, 0].flip(-1).roll(60, -1)  # other rows are its heaviest
    return kv, want


@pytest.mark.parametrize("first", [0, 1, -1])
def test_one_sequence_at_a_time_on_a_full_pool(first):
    """Together they need four new pages of the three that are free. One after the other the first
    takes two and gives back its own last one, and the second stays where it is."""
    kv, want = _full()
    before, w = _state(kv), kv.weights.clone()
    with pytest.raises(RuntimeError, match="4 pages needed, 3 of 8 free"):
        kv.evict(20, 3)
    assert _state(kv) == before and torch.equal(kv.weights, w)
    for seq in (first, 1 - first % 2):
        b, other = seq % 2, 1 - seq % 2
        rows = keep.keep_rows(kv.weights[0], kv.lengths, 20, 3)[b, 0].tolist()
        beside = kv.weights[:, other].clone()
        assert kv.evict(20, 3, seq=seq) == 1
        want[b] = [want[b][r] for r in rows]
        assert torch.equal(kv.weights[:, other], beside)
        _check(kv, want)
        assert not kv.weights[:, b, :, 20:].any() and kv.weights[:, b, :, :20].any()
    assert len({p for t in kv.tables for p in t}) == 4 and kv.free_pages == 4
    assert kv.evict(20, 3, seq=first) == kv.evict(30, seq=1 - first % 2) == 0
    _step(kv, want, 40, 900)
    _check(kv, want)


def test_a_sequence_that_does_not_exist():
    kv, want = _full()
    before, w = _state(kv), kv.weights.clone()
    for seq in (2, -3):
        with pytest.raises(IndexError):
            kv.evict(20, 3, seq=seq)
    assert _state(kv) == before and torch.equal(kv.weights, w)
    _check(kv, want)
