"""PagedKVCache when a call fails half-way or is given a sequence that does not exist, on the
CPU (the kernels it launches are replaced by torch indexing)."""

from __future__ import annotations

import pytest
import torch

from dexter_amd import ops
from dexter_amd.models import PagedKVCache
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


def test_a_step_takes_pages_in_every_sequence():
    """The sizes of the integration notes: 16 rollouts, 400 pages of 64 rows hold an episode of
    1,600 rows until it is held as a prefix, which frees the other 15 copies."""
    kv = PagedKVCache(1, 16, 400, 64, 1, 4, "cpu", torch.float32, max_rows=2048)
    with pytest.raises(RuntimeError, match="KV cache full: 416 pages needed, 400 of 400 free"):
        kv.reserve(1601)
    kv.reserve(1600)
    kv.commit(1600)
    assert kv.free_pages == 0
    kv.hold_prefix(0)
    assert kv.free_pages == 375 and kv.prefix_rows == 1600 and kv.lengths == [0] * 16
    kv.reserve(83)
    kv.commit(83)
    kv.fork(3, 5)
    kv.free(7)
    kv.compact()
    assert kv.lengths == [83] * 7 + [0] + [83] * 8
