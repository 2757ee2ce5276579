"""Lines of attention items that the device cuts into pieces (MI355X): pieces that begin
behind an item's tiles, in calls whose shapes take the paths under test (computed here from
the line's arithmetic, so that a case cannot drift off its path without failing)."""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
from oracle import paged as opaged
from test_gpu_paged import _check, _i32, _rand, _tables

pytestmark = pytest.mark.gpu


def _tiles(rows):
    return -(-rows // 32)


def _pieces(weights, cost, most):
    """(start, stop) of the pieces that a line of items of these tiles is cut into."""
    total = sum(weights) + cost * len(weights)
    n = min(-(-total // cost), most)
    q, longer = divmod(total, n)
    at = [w * q + min(w, longer) for w in range(n + 1)]
    return list(zip(at, at[1:]))


def _behind(weights, cost, most):
    """How many pieces begin behind an item's tiles and go on into the next item."""
    ends, at = [], 0
    for w in weights:
        ends.append((at + w, at + w + cost))  # the item's tiles end here, the item there
        at += w + cost
    return sum(tiles <= start < item < stop for start, stop in _pieces(weights, cost, most)
               for tiles, item in ends)


@pytest.mark.parametrize("dtype,dim,cost", [(torch.bfloat16, 128, 8), (torch.float16, 64, 8),
                                            (torch.bfloat16, 256, 8), (torch.float32, 64, 8),
                                            (torch.float32, 128, 4)])
@pytest.mark.parametrize("lq", [9, 31])
def test_pieces_that_begin_behind_an_item(device, built_lib, dtype, dim, cost, lq):
    """Every item's last new key has infinite values that only its last query sees, so every
    item's workgroup goes through it twice, those of pieces that begin behind an item's
    tiles among them: the other queries' bits are what they were."""
    rows, heads, lens = 16, 2, [0, 1, 40, 95, 130, 7, 64]
    weights = [_tiles(n) + 1 for n in lens for _ in range(heads)]
    assert _behind(weights, cost, 256) >= 2
    # Wide enough that 16-bit calls are planned as a line to cut.
    count, tables, _ = _tables(lens, rows, 1, width=160)
    pages = _rand((2, count, rows, heads, dim), dtype, 2)
    q, k, v = (_rand((len(lens), lq, heads, dim), dtype, s) for s in (3, 4, 5))
    args = dict(pages=pages.to(device), block_table=_i32(tables, device),
                cache_lens=_i32(lens, device), causal=True)
    want = ops.paged_attention(q.to(device), k.to(device), v.to(device), **args)
    ref = opaged.paged_attention(q, k, v, pages, tables, lens, causal=True)
    vmax = max(float(t.double().abs().max()) for t in (pages[1], v))
    _check(want, ref, dtype, dim, max(lens) + lq, vmax, f"behind D{dim} {dtype}")
    v[:, -1, :, 3] = math.inf
    v[:, -1, :, 40] = math.nan
    for _ in range(3):
        got = ops.paged_attention(q.to(device), k.to(device), v.to(device), **args)
        assert torch.equal(got[:, :-1], want[:, :-1])
        assert bool((got[:, -1, :, 3] == math.inf).all() and got[:, -1, :, 40].isnan().all())
        clean = [c for c in range(dim) if c not in (3, 40)]
        assert torch.equal(got[:, -1][..., clean], want[:, -1][..., clean])
