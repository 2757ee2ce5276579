"""PagedKVCache.evict when a call fails half-way, on the CPU (the kernels it launches are replaced
by the oracle's plain forms)."""

from __future__ import annotations

import pytest
import torch

from dexter_amd import ops
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
