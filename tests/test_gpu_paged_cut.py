"""Lines of attention items that the device cuts into pieces (MI355X): pieces that begin
behind an item's tiles, more items than workgroups, more sequences than lanes, prefix and own
keys on one full grid. That the shapes here take those paths is computed from the lines'
arithmetic, so that a case cannot drift off its path without failing."""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
from oracle import paged as opaged
from test_gpu_paged import _case, _check, _i32, _rand, _tables

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


# ---------------------------------------------------------------------------
# Full grids (that these shapes fill them is pinned without a GPU by test_paged_plan.py). The
# scale makes a few keys carry each result, so that a part of the keys left out shows.
# ---------------------------------------------------------------------------
def _lens(batch, top, step=37):
    """Ragged: every ninth sequence empty, one of a single row, the others up to `top`."""
    lens = [0 if b % 9 == 4 else (step * b) % top for b in range(batch)]
    lens[1] = 1
    return lens


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LINES = {
    # More items than workgroups: a record per workgroup, whatever items those leave broken.
    # Lists of sequences longer than a wave (two and three steps of the scan).
    "70 x 3 fp32": dict(dtype=F32, dim=64, lens=_lens(70, 90), lq=3, heads=8, kv=8),
    "70 x 1 long fp32": dict(dtype=F32, dim=128, lens=_lens(70, 600, 211), lq=1, heads=8, kv=8),
    "150 x 1 fp32": dict(dtype=F32, dim=64, lens=_lens(150, 50), lq=1, heads=8, kv=8),
    "70 x 2 bf16": dict(dtype=BF16, dim=128, lens=_lens(70, 90), lq=2, heads=16, kv=8, wide=True),
    "130 x 1 f16": dict(dtype=F16, dim=64, lens=_lens(130, 200, 53), lq=1, heads=8, kv=8, wide=True),
    "70 x 3 D256": dict(dtype=BF16, dim=256, lens=_lens(70, 90), lq=3, heads=8, kv=8, wide=True),
    # Four row waves to an item.
    "70 x 20 bf16": dict(dtype=BF16, dim=64, lens=_lens(70, 90), lq=20, heads=16, kv=8, wide=True),
}
SHARED = {
    # Prefix and own keys both cut, and together more work than the grid has workgroups for:
    # it is dealt in proportion. Row waves of prefix and own items: 4 and 1, 1 and 1, 4 and 4.
    "64 x 1": dict(dtype=BF16, dim=128, lens=_lens(64, 500, 97), lq=1, heads=8, kv=8, prefix_len=4001),
    "70 x 1 fp32": dict(dtype=F32, dim=64, lens=_lens(70, 300, 97), lq=1, heads=8, kv=8,
                        prefix_len=3000),
    "20 x 1": dict(dtype=F16, dim=64, lens=_lens(20, 900, 331), lq=1, heads=8, kv=8, prefix_len=12000),
    "2 x 60": dict(dtype=BF16, dim=64, lens=[4000, 3500], lq=60, heads=8, kv=8, prefix_len=4001),
    "2 x 40 D256": dict(dtype=BF16, dim=256, lens=[1500, 1200], lq=40, heads=8, kv=8, prefix_len=2100),
}


@pytest.mark.parametrize("mask", ["none", "causal", "blocks"])
@pytest.mark.parametrize("name", list(LINES))
def test_more_items_than_workgroups(device, built_lib, name, mask):
    call = dict(LINES[name])
    kw = {"none": {}, "causal": {"causal": True},
          "blocks": {"bb": list(range(0, call["lq"], 2))}}[mask]
    _case(device, call.pop("dtype"), call.pop("dim"), scale=0.5, what=f"{name} {mask}", **call, **kw)


@pytest.mark.parametrize("mask", ["none", "causal", "blocks"])
@pytest.mark.parametrize("name", list(SHARED))
def test_prefix_and_own_keys_share_the_grid(device, built_lib, name, mask):
    call = dict(SHARED[name])
    kw = {"none": {}, "causal": {"causal": True},
          "blocks": {"bb": list(range(0, call["lq"], 7))}}[mask]
    _case(device, call.pop("dtype"), call.pop("dim"), scale=0.5, what=f"{name} {mask}", **call, **kw)
