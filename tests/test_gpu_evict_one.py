"""PagedKVCache.evict of one sequence at a time (MI355X): the rows and weights of all at once, bit
for bit, on a pool that has room for that and on one that does not."""

from __future__ import annotations

import pytest
import torch

from dexter_amd.models import PagedKVCache
from test_gpu_fp4_model import _rows
from test_gpu_paged_model import DIM, DT, HEADS, LAYERS, _layers, _step, _x

pytestmark = pytest.mark.gpu
D = DIM // HEADS


def _cache(device, layers, pages, in4):
    kv = PagedKVCache(LAYERS, 3, pages, 16, HEADS, D, device, DT, max_rows=320, fp4=in4, track_weights=True)
    for i in range(3):
        _step(layers, kv, _x(device, 3, 30, i), 30 * i)
    kv.fork(0, 2)
    _step(layers, kv, _x(device, 3, 5, 9), 90, write=False)  # the sharers' weights part
    return kv


@pytest.mark.parametrize("in4", [False, True])
def test_one_sequence_at_a_time(device, built_lib, in4):
    layers = _layers(device)
    # 12 pages are taken: six by 0 and 2 together, six by 1.
    roomy, full = (_cache(device, layers, pages, in4) for pages in (40, 18))
    assert full.free_pages == 6
    with pytest.raises(RuntimeError, match="8 pages needed, 6 of 18 free"):
        full.evict(50, 10)
    assert roomy.evict(50, 10) == 3
    assert [full.evict(50, 10, seq=s) for s in (0, 1, 2)] == [1, 1, 1]
    assert full.lengths == roomy.lengths == [50] * 3
    assert full.cache_lens.tolist() == [50] * 3
    assert torch.equal(full.weights, roomy.weights)
    for layer in range(LAYERS):
        for s in range(3):
            assert torch.equal(_rows(full, layer, s), _rows(roomy, layer, s))
    assert not torch.equal(_rows(full, 0, 0), _rows(full, 0, 2))  # sharers chose by their own weights
    a, b = (_step(layers, kv, _x(device, 3, 20, 20), 95) for kv in (full, roomy))
    for x, y in zip(a, b):
        assert torch.isfinite(x.float()).all() and torch.equal(x, y)
    assert not full.overflowed()
