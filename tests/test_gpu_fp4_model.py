"""SelfAttention over a PagedKVCache in 4 bits, and one that evicts (MI355X): the operators
together, as a user runs them.

The projections and the prologue are the same kernels over either cache, so what a 4-bit
pool stands for has to be ``oracle.fp4.stored`` of the contiguous cache's rows, bit for bit.
Outputs are then compared with a step over a contiguous cache that holds those values: each
run is off from the exact value by its own roundings (see ``test_gpu_paged_model.py``), so the
two differ by at most ``6 u max |v|``.
"""

from __future__ import annotations

import pytest
import torch

from dexter_amd.models import KVCache, PagedKVCache
from dexter_amd.runtime import CachedStepGraph
from oracle import fp4, keep
from test_gpu_paged_model import DIM, DT, HEADS, LAYERS, _layers, _step, _x

pytestmark = pytest.mark.gpu
D = DIM // HEADS


def _rows(kv, layer, seq):
    """What a sequence's own rows stand for: [2, n, H, D]."""
    pool = kv.pools[layer].cpu()
    pool = fp4.values(pool, kv.page_rows, D) if kv.fp4 else pool.double()
    return torch.cat([pool[:, p] for p in kv.tables[seq]] or [pool[:, 0, :0]], 1)[:, :kv.lengths[seq]]


def _close(a, b, vmax):
    assert torch.isfinite(a.float()).all()
    assert (a.float() - b.float()).abs().max().item() <= 6 * torch.finfo(DT).eps / 2 * vmax * 1.01


@pytest.mark.parametrize("chunk", [1, 50, 83])
def test_steps_over_4_bits(device, built_lib, chunk):
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 2, 40, 32, HEADS, D, device, DT, fp4=True)
    ref = KVCache(LAYERS, 2, 600, HEADS, D, device, DT)
    at = 0
    for i in range(4):
        x = _x(device, 2, chunk, i)
        new, old = (_step(layers, c, x, at) for c in (kv, ref))
        for layer in range(LAYERS):
            # Rows of earlier steps are stored values in ref already: storing those is exact.
            ref.cache[layer][:, :, at:at + chunk] = fp4.stored(
                ref.cache[layer][:, :, at:at + chunk].cpu()).to(DT).to(device)
        at += chunk
        vmax = float(max(ref.cache[n][1].abs().max() for n in range(LAYERS))) * 1.2 + 1
        for layer in range(LAYERS):
            for seq in range(2):
                assert torch.equal(_rows(kv, layer, seq), ref.cache[layer][:, seq, :at].double().cpu())
            _close(new[layer], old[layer], vmax)
    assert kv.lengths == [at, at] and not kv.overflowed()


def test_forks_prefix_and_compaction_in_4_bits(device, built_lib):
    layers = _layers(device)
    kv, ref = (PagedKVCache(LAYERS, 3, 60, 16, HEADS, D, device, DT, fp4=f) for f in (True, False))
    prime = _x(device, 3, 90, 0)
    for c in (kv, ref):
        _step(layers, c, prime, 0)
        c.hold_prefix(0)
        _step(layers, c, _x(device, 3, 21, 1), 90)
        c.fork(0, 2)
        c.free(1)
        c.reserve(5)
        assert len({t[-1] for t in c.tables}) == 3  # the shared last page was copied
        c.compact()
    assert kv.tables == ref.tables and kv.prefix == ref.prefix
    for layer in range(LAYERS):
        for seq in range(3):
            assert torch.equal(_rows(kv, layer, seq), fp4.stored(_rows(ref, layer, seq).to(DT)))
        # The same values in 16 bits.
        ref.pools[layer].copy_(fp4.values(kv.pools[layer].cpu(), 16, D).to(DT))
    x = _x(device, 3, 40, 2)
    new, old = (_step(layers, c, x, 111, write=False) for c in (kv, ref))
    for layer in range(LAYERS):
        _close(new[layer], old[layer], float(ref.pools[layer][1].abs().max()) + 4)


@pytest.mark.parametrize("in4", [False, True])
def test_eviction(device, built_lib, in4):
    """Weights accumulate over the steps; a shared page is left alone; steps go on behind."""
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 3, 60, 16, HEADS, D, device, DT, fp4=in4, track_weights=True)
    for i in range(4):
        _step(layers, kv, _x(device, 3, 25, i), 25 * i)
    kv.free(1)
    kv.fork(0, 1)
    _step(layers, kv, _x(device, 3, 7, 9), 100, write=False)
    kv.fork(2, 0)  # 1 keeps the first episode's pages alone; 0 and 2 share the second's
    assert kv.lengths == [100, 100, 100]
    # Each query's weights over the rows and its new keys add up to 1: less than 7 per head here.
    total = kv.weights.double().sum(-1)
    assert bool((total > 0).all()) and bool((kv.weights[..., 100:] == 0).all())
    before = [[_rows(kv, layer, s) for s in range(3)] for layer in range(LAYERS)]
    w = kv.weights.cpu()
    free = kv.free_pages
    assert kv.evict(100) == 0
    assert kv.evict(40, 10) == 3
    assert kv.lengths == [40] * 3 and kv.cache_lens.tolist() == [40] * 3
    assert len({p for t in kv.tables for p in t}) == 9 and kv.free_pages == 60 - 9 > free
    for layer in range(LAYERS):
        rows = keep.keep_rows(w[layer], [100] * 3, 40, 10)
        assert torch.equal(kv.weights[layer].cpu(), keep.gather_weights(w[layer], rows))
        for s in range(3):
            want = torch.stack([before[layer][s][:, rows[s, h].long(), h] for h in range(HEADS)], 2)
            assert torch.equal(_rows(kv, layer, s), want)
    outs = _step(layers, kv, _x(device, 3, 30, 20), 107)
    assert all(torch.isfinite(o.float()).all() for o in outs) and kv.lengths == [70] * 3
    assert not kv.overflowed()


@pytest.mark.parametrize("in4", [False, True])
def test_a_captured_step_with_weights(device, built_lib, in4):
    """Warming up and capturing leave weights as they were; replays with an eviction between
    them equal eager steps bit for bit."""
    layers = _layers(device)
    n = 10
    caches = [PagedKVCache(LAYERS, 2, 40, 16, HEADS, D, device, DT, max_rows=200, fp4=in4, track_weights=True)
              for _ in range(2)]
    from dexter_amd.bench.workloads import rope_table

    def run(kv, x, cos, sin):
        outs = [m(x, cos, sin, kv, i, write=True) for i, m in enumerate(layers)]
        kv.commit(n)
        return outs
    for kv in caches:
        _step(layers, kv, _x(device, 2, 45, 0), 0)
        _step(layers, kv, _x(device, 2, 3, 1), 45, write=False)
    x = _x(device, 2, n, 2)
    table = lambda first: [t.to(device) for t in rope_table(torch.arange(first, first + n), D)]  # noqa: E731
    was = caches[0].weights.clone()
    step = CachedStepGraph(lambda x, c, s: run(caches[0], x, c, s), (x, *table(45)), [caches[0]], n)
    assert torch.equal(caches[0].weights, was) and caches[0].lengths == [45, 45]
    for i in range(7):
        x, (cos, sin) = _x(device, 2, n, 30 + i), table(45 + n * i)
        got = [t.clone() for t in step(x, cos, sin)]
        torch.cuda.synchronize()
        want = run(caches[1], x, cos, sin)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(caches[0].weights, caches[1].weights)
        assert caches[0].lengths == caches[1].lengths
        if i % 3 == 2:
            assert [c.evict(30, 12) for c in caches] == [2, 2]
    assert caches[0].cache_lens.tolist() == caches[0].lengths


def test_a_prefix_is_not_evicted(device, built_lib):
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 2, 40, 16, HEADS, D, device, DT, track_weights=True)
    _step(layers, kv, _x(device, 2, 50, 0), 0)
    kv.hold_prefix(0)
    assert bool((kv.weights == 0).all())
    for i in range(2):
        _step(layers, kv, _x(device, 2, 30, 1 + i), 50 + 30 * i)
    held = [kv.pools[0][:, p].clone() for p in kv.prefix]
    assert kv.evict(20, 5) == 2 and kv.prefix_rows == 50 and kv.lengths == [20, 20]
    assert all(torch.equal(kv.pools[0][:, p], h) for p, h in zip(kv.prefix, held))
    assert all(torch.isfinite(o.float()).all() for o in _step(layers, kv, _x(device, 2, 9, 7), 110))
