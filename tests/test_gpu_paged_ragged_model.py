"""SelfAttention over sequences that stand at different rows of their episodes (MI355X): each is
rotated by its own positions. Contiguous caches, one for each sequence's history, are the
reference (both are given the whole batch, so the projections are the same calls): cached
rows are equal bit for bit, outputs within the bound of ``test_gpu_paged_model``."""

from __future__ import annotations

import pytest
import torch

from dexter_amd.bench.workloads import rope_table
from dexter_amd.models import KVCache, PagedKVCache
from test_gpu_paged_model import DIM, DT, HEADS, LAYERS, _layers, _same, _step, _x

pytestmark = pytest.mark.gpu


def _tables(device, firsts, n):
    """cos, sin [B, n, D / 2] of positions from each of `firsts` on."""
    pairs = [rope_table(torch.arange(f, f + n), DIM // HEADS) for f in firsts]
    return tuple(torch.stack(t).to(device) for t in zip(*pairs))


def _ragged_step(layers, kv, x, firsts):
    cos, sin = _tables(x.device, firsts, x.shape[1])
    outs = [m(x, cos, sin, kv, i, write=True) for i, m in enumerate(layers)]
    kv.commit(x.shape[1])
    return outs


@pytest.mark.parametrize("chunk", [1, 50, 83])
@pytest.mark.parametrize("prefix", [False, True])
def test_each_sequence_at_its_own_positions(device, built_lib, chunk, prefix):
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 2, 60, 16, HEADS, DIM // HEADS, device, DT)
    refs = [KVCache(LAYERS, 2, 600, HEADS, DIM // HEADS, device, DT) for _ in range(2)]
    at = [0, 0]
    if prefix:  # one history for both
        x = _x(device, 1, 37, 1).expand(2, -1, -1)
        for c in (kv, *refs):
            _step(layers, c, x, 0)
        kv.hold_prefix(0)
        at = [37, 37]
    x = _x(device, 2, 21, 2)
    _step(layers, kv, x, at[0])
    _step(layers, refs[0], x, at[0])
    kv.free(1)  # it starts again, behind the prefix
    at[0] += 21
    assert kv.lengths == [21, 0]
    for i in range(3):
        x = _x(device, 2, chunk, 10 + i)
        new = _ragged_step(layers, kv, x, at)
        old = [_step(layers, ref, x, first) for ref, first in zip(refs, at)]
        at = [n + chunk for n in at]
        for seq in range(2):
            _same(new, old[seq], kv, refs[seq], seq, at[seq])
    # One table for all is a table of equal positions for each.
    x = _x(device, 2, chunk, 20)
    cos, sin = _tables(device, [500, 500], chunk)
    for m, layer in zip(layers, range(LAYERS)):
        assert torch.equal(m(x, cos, sin, kv, layer), m(x, cos[0], sin[0], kv, layer))


def test_tables_of_another_batch_are_refused(device, built_lib):
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 2, 4, 16, HEADS, DIM // HEADS, device, DT)
    x = _x(device, 2, 5, 0)
    cos, sin = _tables(device, [0, 0], 5)
    for c, s in ((cos[:1], sin[:1]), (cos[:, :4], sin[:, :4]), (cos, sin[0]), (cos[0], sin)):
        with pytest.raises(ValueError, match="cos/sin must"):
            layers[0](x, c, s, kv, 0, write=True)
    assert kv.free_pages == 4 and kv.lengths == [0, 0]
