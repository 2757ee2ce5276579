"""Cut lines and full grids (the shapes of ``test_gpu_paged_cut.py``) over pages in 4 bits and with
log-sum-exps (MI355X). Launches are planned by sizes alone, so that these take the paths that are
pinned for those shapes; fp32 ones are taken in bf16 over wide tables, which are cut as theirs."""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
import test_gpu_fp4
from oracle import keep
from test_gpu_paged import _i32, _rand, _tables
from test_gpu_paged_cut import LINES, SHARED, _behind, _tiles

pytestmark = pytest.mark.gpu
WIDE = 132  # table entries of 16 rows behind the longest sequence: 66 32-key tiles


def _kw(mask, lq, step):
    return {"none": {}, "causal": {"causal": True}, "blocks": {"bb": list(range(0, lq, step))}}[mask]


@pytest.mark.parametrize("mask", ["none", "causal", "blocks"])
@pytest.mark.parametrize("name", list(LINES))
def test_more_items_than_workgroups_in_4_bits(device, built_lib, name, mask):
    c = LINES[name]
    dtype = torch.bfloat16 if c["dtype"] == torch.float32 else c["dtype"]
    test_gpu_fp4._case(device, dtype, c["dim"], lens=c["lens"], lq=c["lq"], heads=c["heads"], kv=c["kv"],
                       scale=0.5, wide=WIDE, what=f"{name} {mask}", **_kw(mask, c["lq"], 2))


@pytest.mark.parametrize("mask", ["none", "causal", "blocks"])
@pytest.mark.parametrize("name", list(SHARED))
def test_prefix_and_own_keys_share_the_grid_in_4_bits(device, built_lib, name, mask):
    c = SHARED[name]
    dtype = torch.bfloat16 if c["dtype"] == torch.float32 else c["dtype"]
    test_gpu_fp4._case(device, dtype, c["dim"], lens=c["lens"], lq=c["lq"], heads=c["heads"], kv=c["kv"],
                       scale=0.5, prefix_len=c["prefix_len"], what=f"{name} {mask}", **_kw(mask, c["lq"], 7))


@pytest.mark.parametrize("name", list(LINES) + list(SHARED))
def test_log_sum_exps(device, built_lib, name):
    """The plain call's result, bit for bit (which those tests compare with the oracle), and
    log-sum-exps within their bound."""
    c = (LINES | SHARED)[name]
    dtype, dim, lens, lq, kv, pre = c["dtype"], c["dim"], c["lens"], c["lq"], c["kv"], c.get("prefix_len", 0)
    count, tables, prefix = _tables(lens, 16, 1, prefix_rows=pre)
    if c.get("wide"):
        tables = [t + [-1] * WIDE for t in tables]
    q = _rand((len(lens), lq, c["heads"], dim), dtype, 2)
    k, v = (_rand((len(lens), lq, kv, dim), dtype, s) for s in (3, 4))
    pages = _rand((2, count, 16, kv, dim), dtype, 5)
    kw = dict(pages=pages.to(device), block_table=_i32(tables, device), cache_lens=_i32(lens, device),
              softmax_scale=0.5, causal=True)
    call = ops.paged_attention
    if pre:
        call = ops.shared_prefix_attention
        kw.update(prefix_table=_i32(prefix, device), prefix_len=_i32([pre], device))
    d = [t.to(device) for t in (q, k, v)]
    out, lse = call(*d, return_lse=True, **kw)
    assert torch.equal(out, call(*d, **kw)) and bool(torch.isfinite(out.float()).all())
    want, size = keep.log_sum_exp(q, k, pages, tables, lens, prefix, pre, None, 0.5, True)
    off = (lse.double().cpu() - want).abs() / keep.lse_bound(want, dim, pre + max(lens) + lq, size)
    print(f"[cut] {name}: lse {float(off.max()):.3f} of the bound")
    assert float(off.max()) <= 1.0


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 256)])
@pytest.mark.parametrize("lq", [9, 31])
def test_pieces_that_begin_behind_an_item_in_4_bits(device, built_lib, dtype, dim, lq):
    """Infinite new values that only each item's last query sees: the others' bits are what they
    were, and so are all log-sum-exps."""
    rows, heads, lens = 16, 2, [0, 1, 40, 95, 130, 7, 64]
    assert _behind([_tiles(n) + 1 for n in lens for _ in range(heads)], 8, 256) >= 2
    count, tables, _ = _tables(lens, rows, 1, width=160)
    g = torch.Generator().manual_seed(2)
    pool = torch.randint(0, 256, (2, count, heads, rows * (dim // 2 + dim // 32)), generator=g, dtype=torch.uint8)
    pool[..., rows * dim // 2:] = 124 + pool[..., rows * dim // 2:] % 3  # scales of 2^-3 to 2^-1
    q, k, v = (_rand((len(lens), lq, heads, dim), dtype, s) for s in (3, 4, 5))
    args = dict(pages=pool.to(device), block_table=_i32(tables, device), cache_lens=_i32(lens, device),
                causal=True, return_lse=True)
    want, sums = ops.paged_attention_fp4(q.to(device), k.to(device), v.to(device), **args)
    assert bool(torch.isfinite(want.float()).all())
    v[:, -1, :, 3] = math.inf
    v[:, -1, :, 40] = math.nan
    clean = [c for c in range(dim) if c not in (3, 40)]
    for _ in range(3):
        got, again = ops.paged_attention_fp4(q.to(device), k.to(device), v.to(device), **args)
        assert torch.equal(got[:, :-1], want[:, :-1]) and torch.equal(again, sums)
        assert bool((got[:, -1, :, 3] == math.inf).all() and got[:, -1, :, 40].isnan().all())
        assert torch.equal(got[:, -1][..., clean], want[:, -1][..., clean])
