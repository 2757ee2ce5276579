"""Choosing and moving rows of sequences that have dropped pages of their history (MI355X), as the
operators' documents say: the caller gives such rows a weight of -inf, and keeps no more than the
others are."""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
from oracle import fp4, keep
from test_gpu_keep import _i32, _rand, _tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in4", [False, True])
def test_rows_without_a_page_are_not_kept(device, built_lib, in4):
    rows, heads, dim, lens, k, recent = 16, 2, 128, [300, 200, 90], 70, 10
    count, tables, order = _tables(lens, rows, 3, extra=3 * 5)
    gone = [[0, 3, 4], [1, 2, 10], []]  # (none of the last `recent` rows among them)
    for b, entries in enumerate(gone):
        for e in entries:
            tables[b][e] = -1
    to = [[order.pop() for _ in range(5)] for _ in lens]
    pages = _rand((2, count, rows, heads, dim), torch.bfloat16, 4)
    pool = fp4.pack(*fp4.quantise(pages)) if in4 else pages
    dev, table, length = pool.to(device), _i32(tables, device), _i32(lens, device)
    q = _rand((3, 9, heads, dim), torch.bfloat16, 5).to(device)
    attend = ops.paged_attention_fp4 if in4 else ops.paged_attention
    kw = dict(pages=dev, block_table=table, cache_lens=length)
    _, lse = attend(q, q, q, return_lse=True, **kw)
    w = ops.paged_key_weights(q, lse, **kw)
    missing = (table < 0).repeat_interleave(rows, 1)[:, None, :w.shape[2]]
    assert bool((w.masked_select(missing.expand_as(w)) == 0).all())
    w.masked_fill_(missing, -math.inf)
    picked = ops.kv_keep_rows(w, length, k, recent)
    assert torch.equal(picked.cpu(), keep.keep_rows(w.cpu(), lens, k, recent))
    for b in range(3):
        kept = picked[b].cpu()
        assert int((kept >= 0).sum()) == heads * min(lens[b], k)
        assert not any(int(r) // rows in gone[b] for r in kept.flatten() if r >= 0)
    before = w.cpu()
    ops.kv_page_gather(dev, table, picked, _i32(to, device), w, dim if in4 else None)
    # Every kept row arrived, with its weight.
    if in4:
        want = fp4.pack(*(keep.gather(t, tables, picked.cpu(), to) for t in fp4.unpack(pool, rows, dim)))
    else:
        want = keep.gather(pool, tables, picked.cpu(), to)
    assert torch.equal(dev.cpu(), want)
    assert torch.equal(w.cpu(), keep.gather_weights(before, picked.cpu()))
    assert bool(torch.isfinite(w).all())
