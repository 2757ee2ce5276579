"""The rotary tables that SelfAttention takes over a paged cache, on the CPU: refusals come
before a page is reserved, and a table per sequence reaches the prologue row by row."""

from __future__ import annotations

import pytest
import torch

from dexter_amd import ops
from dexter_amd.models import PagedKVCache, SelfAttention

B, L, DIM, HEADS = 3, 5, 16, 4


def _setup():
    g = torch.Generator().manual_seed(0)
    m = SelfAttention(DIM, HEADS, dtype=torch.float32)
    kv = PagedKVCache(1, B, 6, 16, HEADS, DIM // HEADS, "cpu", torch.float32)
    x = torch.randn(B, L, DIM, generator=g)
    cos, sin = (torch.randn(B, L, DIM // HEADS // 2, generator=g) for _ in range(2))
    return m, kv, x, cos, sin


@pytest.mark.parametrize("change", [lambda c, s: (c[:2], s[:2]), lambda c, s: (c[:, :4], s[:, :4]),
                                    lambda c, s: (c, s[0]), lambda c, s: (c[0], s),
                                    lambda c, s: (c[None], s[None])])
def test_refusals_change_nothing(change):
    m, kv, x, cos, sin = _setup()
    with pytest.raises(ValueError, match="cos/sin must be"):
        m(x, *change(cos, sin), kv, 0, write=True)
    assert kv.free_pages == 6 and kv.lengths == [0] * B


def test_each_row_gets_its_sequences_table(monkeypatch):
    m, kv, x, cos, sin = _setup()
    seen = []

    def prologue(q, k, q_weight, k_weight, cos, sin, eps):
        # Rows are told apart by their tables: returned in place of q and k.
        b, n, heads, dim = q.shape
        assert cos.shape == sin.shape == (n, dim // 2)
        t = torch.cat((cos, sin), -1)[None, :, None].expand(b, n, heads, dim)
        return t.contiguous(), t.contiguous()

    def attend(layer, q, k, v, block_boundaries=None):
        seen.append((q, k, v))
        return q
    monkeypatch.setattr(ops, "qk_norm_rope", prologue)
    monkeypatch.setattr(kv, "attend", attend)
    m(x, cos, sin, kv, 0)
    want = torch.cat((cos, sin), -1)[:, :, None].expand(B, L, HEADS, DIM // HEADS)
    q, k, v = seen[0]
    assert torch.equal(q, want) and torch.equal(k, want)
    assert torch.equal(v, torch.nn.functional.linear(x, m.v.weight, m.v.bias).view(B, L, HEADS, -1))
    m(x, cos[1], sin[1], kv, 0)
    assert torch.equal(seen[1][0], want[1:2].expand(B, -1, -1, -1))
