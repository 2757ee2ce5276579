"""PagedKVCache's page keeping, on the CPU: the two kernels it launches are replaced by
torch indexing; every sequence's rows are compared with a plain list of what it was given."""

from __future__ import annotations

import random

import pytest
import torch

from dexter_amd import ops
from dexter_amd.models import PagedKVCache


@pytest.fixture(autouse=True)
def plain_ops(monkeypatch):
    def append(pages, k, v, table, starts, status=None):
        rows = pages.shape[2]
        for b in range(k.shape[0]):
            for t in range(k.shape[1]):
                r = int(starts[b]) + t
                page = int(table[b, r // rows]) if r // rows < table.shape[1] else -1
                if not 0 <= page < pages.shape[1]:
                    status.fill_(1)
                    continue
                pages[0, page, r % rows], pages[1, page, r % rows] = k[b, t], v[b, t]

    def copy(pools, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for p in pools:
            p[:, dst] = p[:, src]
    monkeypatch.setattr(ops, "kv_page_append", append)
    monkeypatch.setattr(ops, "kv_page_copy", copy)


def _cache(batch=3, pages=20, layers=2, **kw):
    return PagedKVCache(layers, batch, pages, 16, 1, 4, "cpu", torch.float32, **kw)


def _chunk(batch, n, value):
    return torch.arange(batch * n * 4, dtype=torch.float32).view(batch, n, 1, 4) + value


def _step(kv, want, n, value):
    """Append and commit a chunk, and the same to the plain lists."""
    k = _chunk(kv.batch, n, value)
    for layer in range(len(kv.pools)):
        kv.append(layer, k + layer, -k - layer)
    kv.commit(n)
    for b in range(kv.batch):
        want[b] = want[b] + list(k[b])


def _check(kv, want):
    assert kv.cache_lens.tolist() == kv.lengths == [len(w) for w in want]
    users = {}
    for b, rows in enumerate(want):
        table = kv.block_table[b].tolist()
        assert table[:len(kv.tables[b])] == kv.tables[b]
        assert all(p == -1 for p in table[len(kv.tables[b]):])
        for r, row in enumerate(rows):
            page = table[r // 16]
            for layer, pool in enumerate(kv.pools):
                assert torch.equal(pool[0, page, r % 16], row + layer)
                assert torch.equal(pool[1, page, r % 16], -row - layer)
        for p in kv.tables[b]:
            users[p] = users.get(p, 0) + 1
    for p in kv.prefix:
        users[p] = users.get(p, 0) + 1
    assert users == dict(kv._users)
    assert sorted(kv._free) == sorted(set(range(kv.pages)) - set(users))
    assert int(kv.status) == 0


def test_append_commit_and_reset():
    kv, want = _cache(), [[], [], []]
    for i, n in enumerate((1, 5, 16, 10, 0)):
        _step(kv, want, n, 100 * i)
        _check(kv, want)
    kv.reset()
    _check(kv, [[], [], []])
    assert kv.free_pages == kv.pages


def test_append_alone_moves_nothing():
    kv = _cache()
    kv.append(0, _chunk(3, 5, 0), _chunk(3, 5, 0))
    kv.append(0, _chunk(3, 5, 9), _chunk(3, 5, 9))  # again, over the first
    assert kv.lengths == [0, 0, 0] and kv.cache_lens.tolist() == [0, 0, 0]
    assert torch.equal(kv.pools[0][0, kv.tables[1][0], :5], _chunk(3, 5, 9)[1])


def test_fork_shares_pages_until_one_writes():
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 20, 0)
    before = kv.free_pages
    kv.fork(0, 2)
    want[2] = list(want[0])
    _check(kv, want)
    assert kv.tables[2] == kv.tables[0] and kv.free_pages == before + 2
    _step(kv, want, 3, 1000)  # the shared last page is copied once; the full one stays shared
    _check(kv, want)
    assert kv.tables[2][0] == kv.tables[0][0] and kv.tables[2][1] != kv.tables[0][1]


def test_fork_at_a_page_boundary_copies_nothing(monkeypatch):
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 32, 0)
    kv.fork(1, 0)
    want[0] = list(want[1])
    monkeypatch.setattr(ops, "kv_page_copy", lambda *a: pytest.fail("nothing to copy"))
    _step(kv, want, 1, 500)
    _check(kv, want)


def test_fork_leaves_reserved_pages_with_their_owner():
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 4, 0)
    kv.reserve(40)
    kv.fork(0, 1)
    want[1] = list(want[0])
    assert len(kv.tables[0]) == 3 and len(kv.tables[1]) == 1
    kv.fork(1, 1)
    _step(kv, want, 40, 700)
    _check(kv, want)


def test_prefix_is_held_once():
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 37, 0)
    pages = kv.tables[1][:3]
    kv.hold_prefix(1)
    assert kv.prefix == pages and kv.prefix_rows == 37 and int(kv.prefix_len) == 37
    assert kv.prefix_table.tolist()[:3] == pages and kv.free_pages == kv.pages - 3
    want = [[], [], []]
    _check(kv, want)
    _step(kv, want, 5, 2000)
    _check(kv, want)
    with pytest.raises(RuntimeError, match="ends inside a page"):
        kv.hold_prefix(0)


def test_prefix_grows_by_whole_pages():
    kv, want = _cache(), [[], [], []]
    _step(kv, want, 32, 0)
    kv.hold_prefix(0)
    _step(kv, [[], [], []], 8, 50)
    kv.hold_prefix(2)
    assert kv.prefix_rows == 40 and len(kv.prefix) == 3


def test_full_cache_changes_nothing():
    kv, want = _cache(batch=2, pages=5), [[], []]
    _step(kv, want, 32, 0)
    kv.fork(0, 1)
    want[1] = list(want[0])
    _step(kv, want, 10, 300)
    state = (list(kv.tables[0]), list(kv.tables[1]), kv.free_pages, kv.block_table.clone())
    with pytest.raises(RuntimeError, match="KV cache full: 4 pages needed, 1 of 5 free"):
        kv.append(0, _chunk(2, 30, 0), _chunk(2, 30, 0))
    assert (list(kv.tables[0]), list(kv.tables[1]), kv.free_pages) == state[:3]
    assert torch.equal(kv.block_table, state[3])
    _check(kv, want)
    small = _cache(max_rows=40)
    assert small.width == 3
    with pytest.raises(RuntimeError, match="KV cache full: 0 \\+ 49 > 48"):
        small.reserve(49)


def test_page_rows_are_checked():
    for rows in (0, 8, 24, 2048):
        with pytest.raises(ValueError, match="multiple of 16"):
            PagedKVCache(1, 1, 4, rows, 1, 4, "cpu", torch.float32)


def test_commit_takes_only_what_is_reserved():
    kv = _cache()
    with pytest.raises(RuntimeError, match="commit of 1 rows behind 0, but only 0"):
        kv.commit(1)
    kv.reserve(10)
    with pytest.raises(RuntimeError, match="commit of 17 rows"):
        kv.commit(17)
    kv.commit(16)  # the page's rows are there
    assert kv.lengths == [16, 16, 16]
    for call in (kv.commit, kv.reserve):
        with pytest.raises(ValueError, match="-1 rows"):
            call(-1)
    assert kv.lengths == kv.cache_lens.tolist() == [16, 16, 16]


@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_operations(seed):
    """Random appends, forks, frees, prefixes and compactions against plain lists."""
    rng = random.Random(seed)
    kv, want = _cache(batch=4, pages=40), [[] for _ in range(4)]
    for i in range(60):
        op = rng.choice(["step", "step", "step", "fork", "free", "compact", "prefix"])
        if op == "step":
            n = rng.choice([1, 1, 7, 16, 20])
            try:
                _step(kv, want, n, 1000 * i)
            except RuntimeError as e:
                assert "KV cache full" in str(e)
                for b in rng.sample(range(4), 2):
                    kv.free(b)
                    want[b] = []
        elif op == "fork":
            a, b = rng.randrange(4), rng.randrange(4)
            kv.fork(a, b)
            want[b] = list(want[a])
        elif op == "free":
            b = rng.randrange(4)
            kv.free(b)
            want[b] = []
        elif op == "compact":
            kv.compact()
            live = set(kv._users)
            assert live == set(range(len(live)))
        elif rng.random() < 0.2 and kv.prefix_rows % 16 == 0 and kv.prefix_rows < 200:
            held = list(want[rng.randrange(4)])
            b = next(i for i, w in enumerate(want) if len(w) == len(held))
            kv.hold_prefix(b)
            want = [[] for _ in range(4)]
        _check(kv, want)
