"""SelfAttention over a PagedKVCache (MI355X): the operators together, as a user runs them.

An episode is primed, forked and continued; the same steps over a contiguous
``KVCache`` are the reference. The projections and the prologue are the same kernels,
so the cached rows have to be equal bit for bit. The output projection is the
identity here, so outputs are the attention's: each run is off from the exact value by
its own roundings, ``u |out| + 2 u sum p |v|`` with ``u = eps / 2`` (see
``oracle.paged.error_bound``; fp32 terms are below a hundredth of that), so the two
differ by at most ``6 u max |v|``.
"""

from __future__ import annotations

import pytest
import torch

from dexter_amd.bench.workloads import rope_table
from dexter_amd.models import KVCache, PagedKVCache, SelfAttention
from dexter_amd.runtime import CachedStepGraph

pytestmark = pytest.mark.gpu

DIM, HEADS, LAYERS = 512, 4, 2
DT = torch.bfloat16


def _layers(device):
    g = torch.Generator().manual_seed(1)
    out = []
    for _ in range(LAYERS):
        m = SelfAttention(DIM, HEADS, dtype=DT, device=device)
        with torch.no_grad():
            for lin in (m.q, m.k, m.v):
                lin.weight.copy_(torch.randn(DIM, DIM, generator=g) * DIM ** -0.5)
                lin.bias.copy_(torch.randn(DIM, generator=g) * 0.02)
            m.o.weight.copy_(torch.eye(DIM))
            m.o.bias.zero_()
        out.append(m)
    return out


def _x(device, batch, n, seed):
    return torch.randn(batch, n, DIM, generator=torch.Generator().manual_seed(seed)).to(DT).to(device)


def _step(layers, kv, x, first, write=True, blocks=None):
    cos, sin = (t.to(x.device) for t in rope_table(torch.arange(first, first + x.shape[1]), DIM // HEADS))
    outs = [m(x, cos, sin, kv, i, block_boundaries=blocks, write=write) for i, m in enumerate(layers)]
    if write:
        kv.commit(x.shape[1])
    return outs


def _rows(kv, layer, seq, n):
    """Cached rows [0, n) of a sequence, prefix first: [2, n, H, D]."""
    if isinstance(kv, KVCache):
        return kv.cache[layer][:, seq, :n]
    rows = [kv.pools[layer][:, p] for p in kv.prefix]
    flat = torch.cat(rows, 1)[:, :kv.prefix_rows] if rows else None
    own = [kv.pools[layer][:, p] for p in kv.tables[seq]]
    own = torch.cat(own, 1)[:, :kv.lengths[seq]]
    return (own if flat is None else torch.cat((flat, own), 1))[:, :n]


def _same(paged, plain, kv, ref, seq, n):
    """Sequence `seq` of both runs: equal rows, outputs within the bound."""
    for layer, (a, b) in enumerate(zip(paged, plain)):
        rows = _rows(kv, layer, seq, n)
        assert torch.equal(rows, _rows(ref, layer, seq, n))
        bound = 6 * torch.finfo(DT).eps / 2 * float(rows[1].float().abs().max()) * 1.01
        assert torch.isfinite(a[seq].float()).all()
        assert (a[seq].float() - b[seq].float()).abs().max().item() <= bound


@pytest.mark.parametrize("chunk", [1, 50, 83])
def test_steps_equal_the_contiguous_cache(device, built_lib, chunk):
    """Chunks written and committed, and a read-only step, over both caches."""
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 2, 40, 32, HEADS, DIM // HEADS, device, DT)
    ref = KVCache(LAYERS, 2, 600, HEADS, DIM // HEADS, device, DT)
    at = 0
    for i in range(5):
        x = _x(device, 2, chunk, i)
        new = _step(layers, kv, x, at)
        old = _step(layers, ref, x, at)
        at += chunk
        for seq in range(2):
            _same(new, old, kv, ref, seq, at)
    x = _x(device, 2, chunk, 99)
    blocks = torch.arange(0, chunk, 20, device=device)
    new, old = (_step(layers, c, x, at, write=False, blocks=blocks) for c in (kv, ref))
    for seq in range(2):
        _same(new, old, kv, ref, seq, at)
    assert kv.lengths == [at, at] and not kv.overflowed()


def test_prefill_sized_chunk(device, built_lib):
    """More than 128 tokens: the projections and the prologue are separate calls."""
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 1, 12, 64, HEADS, DIM // HEADS, device, DT)
    ref = KVCache(LAYERS, 1, 700, HEADS, DIM // HEADS, device, DT)
    blocks = torch.arange(0, 300, 100, device=device)
    for i in range(2):
        x = _x(device, 1, 300, i)
        new, old = (_step(layers, c, x, 300 * i, blocks=blocks) for c in (kv, ref))
        _same(new, old, kv, ref, 0, 300 * (i + 1))


def test_fork_prefix_and_compaction_run(device, built_lib):
    """One episode is primed on sequence 0 and held as the prefix of three rollouts, which
    take different chunks; one forks into another, one is freed, pages are compacted."""
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 3, 60, 16, HEADS, DIM // HEADS, device, DT)
    ref = KVCache(LAYERS, 3, 400, HEADS, DIM // HEADS, device, DT)
    prime = _x(device, 1, 90, 0).expand(3, -1, -1)
    _step(layers, kv, prime, 0)
    _step(layers, ref, prime, 0)
    kv.hold_prefix(0)
    assert len(kv.prefix) == 6 and kv.free_pages == 54
    at = 90
    for i in range(3):
        x = _x(device, 3, 21, 10 + i)
        new, old = _step(layers, kv, x, at), _step(layers, ref, x, at)
        at += 21
        for seq in range(3):
            _same(new, old, kv, ref, seq, at)
    kv.fork(0, 2)
    for c in ref.cache:
        c[:, 2] = c[:, 0]
    kv.free(1)
    kv.fork(2, 1)
    for c in ref.cache:
        c[:, 1] = c[:, 0]
    assert kv.compact() > 0
    for i in range(2):
        x = _x(device, 3, 13, 20 + i)
        new, old = _step(layers, kv, x, at), _step(layers, ref, x, at)
        at += 13
        for seq in range(3):
            _same(new, old, kv, ref, seq, at)


def test_captured_step_reserves_between_replays(device, built_lib):
    """A captured cache-writing step over pages: pages are reserved before each replay, and
    each replay equals the eager step bit for bit; a fork between replays is followed."""
    layers = _layers(device)

    def make():
        kv = PagedKVCache(LAYERS, 2, 30, 16, HEADS, DIM // HEADS, device, DT, max_rows=240)
        _step(layers, kv, _x(device, 2, 37, 0), 0)
        return kv
    kv, eager = make(), make()
    cos, sin = (t.to(device) for t in rope_table(torch.arange(37, 37 + 11), DIM // HEADS))

    def last(x, cache):
        outs = [m(x, cos, sin, cache, i, write=True) for i, m in enumerate(layers)]
        cache.commit(11)
        return tuple(outs)
    step = CachedStepGraph(lambda x: last(x, kv), (_x(device, 2, 11, 1),), [kv], 11)
    assert kv.lengths == [37, 37] and kv.cache_lens.tolist() == [37, 37]
    for i in range(5):
        if i == 2:
            for c in (kv, eager):
                c.fork(1, 0)
        x = _x(device, 2, 11, 30 + i)
        got = step(x)
        want = last(x, eager)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), f"replay {i}"
        assert kv.lengths == eager.lengths == kv.cache_lens.tolist()
        for layer in range(LAYERS):
            for seq in range(2):
                n = kv.lengths[seq]
                assert torch.equal(_rows(kv, layer, seq, n), _rows(eager, layer, seq, n))
    while True:
        try:
            step(_x(device, 2, 11, 50))
        except RuntimeError as e:
            assert "KV cache full" in str(e)
            break
    assert kv.lengths == kv.cache_lens.tolist() and not kv.overflowed()


def test_captured_step_refuses_another_prefix(device, built_lib):
    """Which attention a step calls is captured with it: a prefix that comes or goes after
    the capture is refused, with nothing moved."""
    layers = _layers(device)
    kv = PagedKVCache(LAYERS, 2, 30, 16, HEADS, DIM // HEADS, device, DT)
    _step(layers, kv, _x(device, 2, 20, 0), 0)
    cos, sin = (t.to(device) for t in rope_table(torch.arange(20, 25), DIM // HEADS))

    def last(x):
        outs = [m(x, cos, sin, kv, i, write=True) for i, m in enumerate(layers)]
        kv.commit(5)
        return tuple(outs)
    x = _x(device, 2, 5, 1)
    step = CachedStepGraph(last, (x,), [kv], 5)
    step(x)
    kv.hold_prefix(0)
    with pytest.raises(RuntimeError, match="capture it again"):
        step(x)
    assert kv.lengths == [0, 0] and kv.prefix_rows == 25
    again = CachedStepGraph(last, (x,), [kv], 5)
    again(x)
    kv.reset()
    with pytest.raises(RuntimeError, match="capture it again"):
        again(x)
    step(x)
    assert kv.lengths == kv.cache_lens.tolist() == [5, 5]


@pytest.mark.parametrize("name,args", [("fork", (0, 1)), ("free", (0,)), ("hold_prefix", (0,)),
                                       ("compact", ()), ("reset", ())])
def test_page_keeping_inside_a_capture_is_refused(device, built_lib, name, args):
    kv = PagedKVCache(1, 2, 8, 16, HEADS, DIM // HEADS, device, DT)
    k = _x(device, 2, 3, 0).view(2, 3, HEADS, DIM // HEADS)
    kv.append(0, k, k)
    kv.commit(3)
    tables = [list(t) for t in kv.tables]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            k2 = k + 1  # noqa: F841 (something to capture)
            with pytest.raises(RuntimeError, match="before a capture"):
                getattr(kv, name)(*args)
    assert kv.tables == tables and kv.lengths == [3, 3] and kv.free_pages == 6


def test_reserve_inside_a_capture_is_refused(device, built_lib):
    kv = PagedKVCache(1, 1, 4, 16, HEADS, DIM // HEADS, device, DT)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    k = _x(device, 1, 3, 0).view(1, 3, HEADS, DIM // HEADS)
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            k2 = k + 1
            with pytest.raises(RuntimeError, match="before a capture"):
                kv.append(0, k2, k2)
    assert kv.free_pages == 4
