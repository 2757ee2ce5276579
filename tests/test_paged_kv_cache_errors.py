"""PagedKVCache when a call fails half-way or is given a sequence that does not exist, on the
CPU (the kernels it launches are replaced by torch indexing)."""

from __future__ import annotations

import pytest
import torch

from dexter_amd import ops
from test_paged_kv_cache import _cache, _check, _step, plain_ops  # noqa: F401


def _state(kv):
    return ([list(t) for t in kv.tables], list(kv.lengths), dict(kv._users), sorted(kv._free),
            kv.block_table.tolist(), kv.cache_lens.tolist(), list(kv.prefix), kv.prefix_rows)


def test_a_failed_copy_changes_nothing(monkeypatch):
    """reserve() copies shared pages before any page changes hands: when the copy raises,
    a later reserve() finds the pages still shared and copies them."""
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 20, 0)
    kv.fork(0, 2)
    kv.fork(0, 1)
    want = [list(want[0]) for _ in range(3)]
    before = _state(kv)
    copy = ops.kv_page_copy

    def fail(*args):
        raise RuntimeError("no launch")
    monkeypatch.setattr(ops, "kv_page_copy", fail)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no launch"):
            _step(kv, want, 3, 1000)
        assert _state(kv) == before
    monkeypatch.setattr(ops, "kv_page_copy", copy)
    _step(kv, want, 3, 2000)
    _check(kv, want)
    assert len({t[1] for t in kv.tables}) == 3


@pytest.mark.parametrize("name,args", [("fork", (0, 3)), ("fork", (3, 0)), ("fork", (0, -4)),
                                       ("free", (3,)), ("hold_prefix", (3,))])
def test_a_sequence_that_does_not_exist(name, args):
    """IndexError with nothing changed: no page is counted for a sequence that is not there."""
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 20, 0)
    before = _state(kv)
    with pytest.raises(IndexError):
        getattr(kv, name)(*args)
    assert _state(kv) == before
    _check(kv, want)
