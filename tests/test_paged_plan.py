"""Which plan the shapes of test_gpu_paged_cut.py take, told by the workspace that the library
asks for (no GPU: it then plans for 256 compute units)."""

from __future__ import annotations

import pytest

from dexter_amd.ops.gfx950 import _lib
from test_gpu_paged_cut import LINES, SHARED, _pieces, _tiles

ROWS = 16  # of a page


def _shape(call):
    """(sequences, rows of a sequence and K/V head, table width, workgroups that run at once)"""
    batch, rows = len(call["lens"]), call["lq"] * call["heads"] // call["kv"]
    width = max(1, max(-(-n // ROWS) for n in call["lens"]))
    if call.get("wide"):
        width += -(-66 * 32 // ROWS)
    return batch, rows, width, 256 if call["dim"] == 256 else 512


def _workspace(call, width, prefix_width=0):
    n = _lib.load().dx_paged_attention_workspace_bytes(
        _lib.dtype_code(call["dtype"]), len(call["lens"]), call["lq"], call["lq"], call["heads"],
        call["kv"], call["dim"], ROWS, width, int(prefix_width > 0), prefix_width)
    assert n >= 0
    return n


def _cost(call, rows):
    """What an item adds to its tiles: two rounds of a workgroup's streams."""
    line = call["dim"] * (4 if call["dtype"].itemsize == 4 else 2)
    if rows > 32:
        return 4 if line < 512 else 2
    return 2 * (2 if line * (1 if call["dim"] == 256 else 2) >= 1024 else 4)


def _slot(call, rows):
    return (32 if rows <= 32 else 128) * (call["dim"] * 4 + 8)


@pytest.mark.parametrize("name", list(LINES))
def test_records_are_kept_by_workgroup(built_lib, name):
    call = LINES[name]
    batch, rows, width, slots = _shape(call)
    items = batch * call["kv"]
    assert batch > 64 and rows <= 128 and items > slots
    # Cut (two partials per workgroup), with fewer records than items.
    assert _workspace(call, width) == 2 * slots * _slot(call, rows) + 16 * slots
    # All workgroups get a piece, and some cover several items.
    tiles = [_tiles(n) + _tiles(call["lq"]) for n in call["lens"] for _ in range(call["kv"])]
    pieces = _pieces(tiles, _cost(call, rows), slots)
    assert len(pieces) == slots
    ends, at = [], 0
    for t in tiles:
        at += t + _cost(call, rows)
        ends.append(at)
    assert max(sum(a < e <= b for e in ends) for a, b in pieces) >= 2


@pytest.mark.parametrize("name", list(SHARED))
def test_prefix_and_own_keys_fill_the_grid(built_lib, name):
    call = SHARED[name]
    batch, rows, width, slots = _shape(call)
    pre_rows, pre_width = batch * rows, -(-call["prefix_len"] // ROWS)
    assert rows <= 128 and pre_rows <= 128
    items = batch * call["kv"]
    # Both are cut: partials for every item and one more per workgroup, a record per item.
    assert _workspace(call, width, pre_width) == (
        (items + slots) * _slot(call, rows) + (call["kv"] + slots) * _slot(call, pre_rows)
        + 16 * (items + call["kv"]))
    cost, pre_cost = _cost(call, rows), _cost(call, pre_rows)
    own = sum(_tiles(n) + _tiles(call["lq"]) + cost for n in call["lens"]) * call["kv"]
    pre = (_tiles(call["prefix_len"]) + pre_cost) * call["kv"]
    assert min(-(-own // cost), slots) + min(-(-pre // pre_cost), slots) > slots
