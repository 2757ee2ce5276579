"""Copies of 4-bit pages, which go as rows of 16-bit elements (MI355X): every byte, at the largest pages."""

from __future__ import annotations

import pytest
import torch

from dexter_amd.models import PagedKVCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,heads,dim", [(1024, 24, 256), (1024, 3, 64), (48, 40, 128), (16, 1, 64)])
def test_forks_and_compaction(device, built_lib, rows, heads, dim):
    kv = PagedKVCache(2, 3, 9, rows, heads, dim, device, torch.bfloat16, fp4=True)
    g = torch.Generator(device=device).manual_seed(rows)
    for pool in kv.pools:
        pool.copy_(torch.randint(0, 256, pool.shape, generator=g, device=device, dtype=torch.uint8))
    kv.reserve(rows + 5)
    kv.commit(rows + 5)
    kv.free(1)
    kv.free(2)
    kv.fork(0, 1)
    kv.fork(0, 2)
    before = [pool.clone() for pool in kv.pools]
    shared = list(kv.tables[0])
    kv.reserve(3)  # two of the three sharers get a copy of the last page
    copies = {t[1] for t in kv.tables} - {shared[1]}
    assert len(copies) == 2 and all(t[0] == shared[0] for t in kv.tables)
    for pool, was in zip(kv.pools, before):
        want = was.clone()
        for page in copies:
            want[:, page] = was[:, shared[1]]
        assert torch.equal(pool, want)
    kv.free(0)
    held = [[pool[:, page].clone() for page in kv.tables[2]] for pool in kv.pools]
    before = [pool.clone() for pool in kv.pools]
    moved = kv.compact()
    for pool, was, pages in zip(kv.pools, before, held):
        for page, want in zip(kv.tables[2], pages):
            assert torch.equal(pool[:, page], want)
        assert int((pool != was).flatten(2).any(-1).any(0).sum()) <= moved
    assert sorted({p for t in kv.tables for p in t}) == list(range(3))
