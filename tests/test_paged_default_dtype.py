"""torch's default dtype is the caller's (a model built in bf16 may set it): log-sum-exps and row
weights are fp32 whatever it is. The kernels write 4 bytes for each of their elements. No GPU: the
library's entry points are replaced."""

from __future__ import annotations

import pytest
import torch

from dexter_amd.models import PagedKVCache
from dexter_amd.ops.gfx950 import _lib, keep, paged


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64], ids=lambda t: str(t)[6:])
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


@pytest.fixture
def no_launch(monkeypatch):
    class Library:
        def __getattr__(self, name):
            return lambda *args: 0
    for module in (paged, keep):
        monkeypatch.setattr(module, "_elsewhere", lambda device: False)
    monkeypatch.setattr(paged, "_workspace_bytes", lambda *args: 0)
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 0)


def test_a_cache_that_tracks_weights(default_dtype):
    kv = PagedKVCache(2, 3, 4, 16, 2, 64, "cpu", torch.bfloat16, track_weights=True)
    assert kv.weights.dtype == torch.float32 and kv.weights.shape == (2, 3, 2, 64)
    assert kv.pools[0].dtype == torch.bfloat16 and kv.cache_lens.dtype == torch.int32


@pytest.mark.parametrize("fp4", [False, True])
@pytest.mark.parametrize("prefix", [False, True])
def test_a_log_sum_exp(default_dtype, no_launch, fp4, prefix):
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(2, 3, 2, 64, dtype=torch.bfloat16)
    pool = (torch.zeros(2, 5, 2, 16 * 34, dtype=torch.uint8) if fp4 else
            torch.zeros(2, 5, 16, 2, 64, dtype=torch.bfloat16))
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for n in (3, 0):
        out, lse = paged._attend("attention", q[:, :n], k[:, :n], k[:, :n], pool,
                                 (table[0], lens[:1]) if prefix else None, table, lens, None, None, False,
                                 True, fp4)
        assert lse.dtype == torch.float32 and lse.shape == (2, n, 4) and out.dtype == torch.bfloat16


def test_row_weights(default_dtype, no_launch):
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 5, 16, 2, 64, dtype=torch.bfloat16)
    lse = torch.zeros(2, 3, 4, dtype=torch.float32)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    got = keep.paged_key_weights(q, lse, None, pool, table, lens, None)
    assert got.dtype == torch.float32 and got.shape == (2, 2, 64)
