"""The paged-attention oracle against the explicit loops of ``oracle.brute`` over the same rows
laid out in one piece (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import brute, paged


def _close(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # Both in 64 bits, over at most 60 keys of values below 10.
    assert np.nanmax(np.abs(got - want), initial=0.0) < 1e-12


@pytest.mark.parametrize("kv", [1, 2, 4])
@pytest.mark.parametrize("mask", ["all", "causal", "blocks", "late", "past"])
@pytest.mark.parametrize("prefix_len", [0, 5, 8])
def test_pages_equal_one_piece(kv, mask, prefix_len):
    g = torch.Generator().manual_seed(1)
    rows, heads, dim, lq, lens = 4, 4, 8, 7, [0, 6, 9]
    pages = torch.randn(2, 12, rows, kv, dim, generator=g)
    order = torch.randperm(12, generator=g).tolist()
    prefix = [order.pop() for _ in range(2)]
    tables = [[order.pop() for _ in range(3)] for _ in lens]
    q = torch.randn(3, lq, heads, dim, generator=g)
    k, v = (torch.randn(3, lq, kv, dim, generator=g) for _ in range(2))
    starts = {"blocks": [0, 3, 5], "late": [2, 5], "past": [0, 4, 50]}.get(mask)
    out, weight, scores = paged.paged_attention(
        q, k, v, pages, tables, lens, prefix, prefix_len,
        None if starts is None else torch.tensor(starts), 0.3, mask == "causal")
    for b, n in enumerate(lens):
        at = [(prefix[r // rows], r % rows) for r in range(prefix_len)]
        at += [(tables[b][r // rows], r % rows) for r in range(n)]
        old = torch.stack([pages[:, p, r] for p, r in at], 1) if at else pages[:, 0, :0]
        want = brute.attention(q[b:b + 1], k[b:b + 1], v[b:b + 1], old[0][None], old[1][None], len(at),
                               starts, mask == "causal", 0.3)
        _close(out[b:b + 1].numpy(), want)
    live = ~torch.isnan(out)
    assert bool((weight[live] >= out[live].abs() - 1e-12).all()) and bool((scores >= 0).all())


def test_rows_without_a_page_are_left_out():
    g = torch.Generator().manual_seed(2)
    pages = torch.randn(2, 4, 4, 1, 8, generator=g)
    q, k, v = (torch.randn(1, 2, 1, 8, generator=g) for _ in range(3))
    table, kept = [[1, -1, 3, 4]], [[1, 3]]
    got = paged.paged_attention(q, k, v, pages, table, [99])[0]
    assert torch.equal(got, paged.paged_attention(q, k, v, pages, kept, [8])[0])
    none = paged.paged_attention(q, k[:, :0], v[:, :0], pages, [[-1]], [4])[0]
    assert bool(torch.isnan(none).all())
