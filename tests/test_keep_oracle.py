"""The oracle of row weights and eviction against closed forms and numpy (no GPU)."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import keep, paged


def test_weights_and_log_sum_exps_agree_with_attention():
    """Values that are one row's unit vector read out the probabilities that the weights sum."""
    g = torch.Generator().manual_seed(5)
    rows, kv, heads, dim, lq, lens = 4, 2, 4, 16, 3, [7, 0, 10]
    pages = torch.randn(2, 9, rows, kv, dim, generator=g)
    tables = [[4, 1, -1], [-1, -1, -1], [0, 7, 3]]
    pages[1] = 0
    for b, n in enumerate(lens):
        for r in range(n):
            pages[1, tables[b][r // rows], r % rows, :, r] = 1  # dim r reads row r
    q = torch.randn(3, lq, heads, dim, generator=g)
    k = torch.randn(3, lq, kv, dim, generator=g)
    v = torch.zeros(3, lq, kv, dim)
    out = paged.paged_attention(q, k, v, pages, tables, lens, causal=True)[0]
    lse, scores = keep.log_sum_exp(q, k, pages, tables, lens, causal=True)
    w, _ = keep.key_weights(q, lse, pages, tables, lens)
    for b, n in enumerate(lens):
        want = out[b].view(lq, kv, heads // kv, dim).sum((0, 2))[:, :n]
        assert float((w[b, :, :n] - want).abs().max() if n else 0) < 1e-12
        assert bool((w[b, :, n:] == 0).all())
    assert bool((scores >= 0).all())
    none = keep.log_sum_exp(q, k[:, :0], pages, [[-1]] * 3, [4] * 3)[0]
    assert bool((none == -math.inf).all())


def test_kept_rows():
    w = torch.tensor([[[3.0, 1.0, 3.0, math.nan, -1.0, 2.0, 9.0, 9.0]]])
    got = lambda n, k, r: keep.keep_rows(w, [n], k, r)[0, 0].tolist()  # noqa: E731
    assert got(6, 3, 0) == [0, 2, 5]
    assert got(6, 1, 0) == [0]          # of equal ones the lowest
    assert got(6, 3, 2) == [0, 4, 5]
    assert got(6, 2, 9) == [4, 5]
    assert got(6, 6, 0) == [0, 1, 2, 3, 4, 5]
    assert got(2, 4, 1) == [0, 1, -1, -1]
    assert got(0, 2, 1) == [-1, -1]
    assert got(6, 5, 0) == [0, 1, 2, 4, 5]  # NaN is the lowest
    g = np.random.default_rng(6)
    x = g.integers(0, 5, (2, 3, 40)).astype(np.float32)
    rows = keep.keep_rows(torch.from_numpy(x), [40, 17], 9, 0).numpy()
    for b, n in enumerate([40, 17]):
        for h in range(3):
            order = np.lexsort((np.arange(n), -x[b, h, :n]))[:9]
            assert sorted(order.tolist()) == rows[b, h].tolist()


def test_a_move_in_place_reads_what_was_there():
    g = torch.Generator().manual_seed(7)
    pages = torch.randn(2, 4, 4, 2, 8, generator=g)
    rows = torch.tensor([[[1, 2, 6, -1], [0, 5, 7, 99]]], dtype=torch.int32)
    table = [[3, 1]]
    after = keep.gather(pages, table, rows, table)
    at = lambda p, r, h: p[:, table[0][r // 4], r % 4, h]  # noqa: E731
    for h, moved in enumerate([[1, 2, 6], [0, 5, 7]]):
        for i, r in enumerate(moved):
            assert torch.equal(at(after, i, h), at(pages, r, h))
        assert torch.equal(at(after, 3, h), at(pages, 3, h))
    w = torch.arange(16.0).view(1, 2, 8)
    assert keep.gather_weights(w, rows).tolist() == [[[1, 2, 6, 0, 0, 0, 0, 0], [8, 13, 15, 0, 0, 0, 0, 0]]]
