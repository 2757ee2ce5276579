"""A KV cache in pages (MI355X): append, page copies, attention over pages, shared prefixes.

Appends and copies move bits: results are equal to torch indexing, every other
row of the pool included. Attention is compared with ``oracle/paged.py`` (64 bits,
one query at a time) within ``oracle.paged.error_bound``, which counts the
roundings of the formula; nothing is tuned to what the kernels give.
"""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
from oracle import paged as opaged

pytestmark = pytest.mark.gpu

TYPES = [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float16, 64),
         (torch.float16, 128), (torch.float16, 256), (torch.float32, 64), (torch.float32, 128)]
IDS = [f"{str(dt)[6:]}-D{d}" for dt, d in TYPES]


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _tables(lens, rows, seed, spare=2, prefix_rows=0, width=None):
    """Page tables of sequences of `lens` rows over one shuffled pool: (pages, tables, prefix)."""
    held = [-(-n // rows) for n in lens]
    pre = -(-prefix_rows // rows)
    total = sum(held) + pre + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max([1] + held) if width is None else width
    tables = [[order.pop() if j < n else -1 for j in range(width)] for n in held]
    return total, tables, [order.pop() for _ in range(pre)]


def _poisoned(pages, tables, lens, prefix, prefix_len):
    """The pool with NaN and inf in every row that no sequence holds."""
    _, count, rows = pages.shape[:3]
    live = torch.zeros(count, rows, dtype=torch.bool)
    for table, n in list(zip(tables, lens)) + [(prefix, prefix_len)]:
        for r in range(n):
            if 0 <= table[r // rows] < count:
                live[table[r // rows], r % rows] = True
    out = pages.clone()
    out[0][~live] = math.nan
    out[1][~live] = math.inf
    return out


def _check(got, want, dtype, dim, keys, vmax, what):
    ref, weight, scores = want
    assert got.dtype == dtype and got.shape == ref.shape
    got = got.double().cpu()
    none = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), none), f"{what}: NaN elements differ"
    bound = opaged.error_bound(ref, weight, dtype, dim, keys, scores, vmax)
    err = (got - ref).abs()
    worst = float((err / bound)[~none].max()) if (~none).any() else 0.0
    print(f"[paged] {what}: {worst:.3f} of the bound, max-abs {float(err[~none].max()) if (~none).any() else 0:.2e}")
    assert worst <= 1.0, f"{what}: error {worst:.3f} times its bound"


def _case(device, dtype, dim, *, lens, lq, heads=2, kv=2, rows=16, prefix_len=0, lk=None, bb=None,
          causal=False, scale=None, seed=0, tables=None, prefix=None, poison=True, what="",
          device_lens=None, strided=False, own=True, wide=False):
    """One attention call against the oracle."""
    b = len(lens)
    lk = lq if lk is None else lk
    count, t0, p0 = _tables(lens, rows, seed, prefix_rows=prefix_len)
    tables = t0 if tables is None else tables
    prefix = p0 if prefix is None else prefix
    if wide:  # room for 66 more 32-key tiles: the launch is planned for long sequences
        tables = [t + [-1] * (-(-66 * 32 // rows)) for t in tables]
    q = _rand((b, lq, heads, dim), dtype, seed + 1)
    k = _rand((b, lk, kv, dim), dtype, seed + 2)
    v = _rand((b, lk, kv, dim), dtype, seed + 3)
    pages = _rand((2, count, rows, kv, dim), dtype, seed + 4)
    dev_pages = _poisoned(pages, tables, lens, prefix, prefix_len) if poison else pages
    dev = lambda t: t.to(device)  # noqa: E731
    if strided:  # rows of a wider tensor, and a head-major pool
        qd = dev(torch.cat((q, q), -1))[..., :dim]
        kd = dev(torch.cat((k, k), 1))[:, :lk]
        pd = dev(dev_pages.transpose(2, 3).contiguous()).transpose(2, 3)
    else:
        qd, kd, pd = dev(q), dev(k), dev(dev_pages)
    kw = dict(pages=pd, block_boundaries=None if bb is None else torch.tensor(bb).to(device),
              softmax_scale=scale, causal=causal)
    if own:
        kw.update(block_table=_i32(tables, device),
                  cache_lens=_i32(lens if device_lens is None else device_lens, device))
    if prefix_len or prefix:
        got = ops.shared_prefix_attention(qd, kd, dev(v), prefix_table=_i32(prefix, device),
                                          prefix_len=_i32([prefix_len], device), **kw)
    else:
        got = ops.paged_attention(qd, kd, dev(v), **kw)
    want = opaged.paged_attention(
        q, k, v, pages, tables if own else None, lens if own else None, prefix, prefix_len,
        None if bb is None else torch.tensor(bb), scale, causal)
    keys = prefix_len + max(lens) + lk
    vmax = max(float(t.double().abs().max()) if t.numel() else 0.0 for t in (pages[1], v))
    _check(got, want, dtype, dim, keys, vmax, what)
    return got


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,starts,rows", [(1, [0, 7, 15], 16), (1, [5, 100, 31], 5),
                                           (83, [0, 13, 200], 64), (50, [16, 47, 3], 48),
                                           (333, [1, 0, 64], 32)])
def test_append(device, built_lib, dtype, n, starts, rows):
    heads, dim = 3, 72
    count, tables, _ = _tables([s + n for s in starts], rows, 1)
    pages = _rand((2, count, rows, heads, dim), dtype, 2)
    k, v = (_rand((3, n, heads, dim), dtype, s) for s in (3, 4))
    want = pages.clone()
    for b, s in enumerate(starts):
        for t in range(n):
            page, r = tables[b][(s + t) // rows], (s + t) % rows
            want[0, page, r], want[1, page, r] = k[b, t], v[b, t]
    got = pages.to(device)
    status = _i32([0], device)
    ops.kv_page_append(got, k.to(device), v.to(device), _i32(tables, device), _i32(starts, device),
                       status)
    assert torch.equal(got.cpu(), want) and int(status) == 0
    # A head-major pool, and k and v that are views of a fused projection's rows.
    major = pages.transpose(2, 3).contiguous().to(device).transpose(2, 3)
    kv = torch.cat((k, v), 2).to(device)
    ops.kv_page_append(major, kv[:, :, :heads], kv[:, :, heads:], _i32(tables, device),
                       _i32(starts, device))
    assert torch.equal(major.cpu(), want)


def test_append_rows_without_a_page(device, built_lib):
    """Rows before 0, past the table, or in an entry that names no page: not written, the
    others are, and the status word says so."""
    rows, heads, dim, n = 16, 2, 64, 40
    pages = _rand((2, 4, rows, heads, dim), torch.bfloat16, 1)
    k, v = (_rand((3, n, heads, dim), torch.bfloat16, s) for s in (2, 3))
    tables = [[0, 1], [4, 2], [3, -1]]  # 4 is outside the pool
    starts = [-3, 0, 10]
    want, holes = pages.clone(), [0, 0, 0]
    for b, s in enumerate(starts):
        for t in range(n):
            r = s + t
            page = tables[b][r // rows] if 0 <= r < 2 * rows else -1
            if 0 <= page < 4:
                want[0, page, r % rows], want[1, page, r % rows] = k[b, t], v[b, t]
            else:
                holes[b] += 1
    assert all(holes)
    for b in range(3):  # each sequence alone sets the status, and together
        status = _i32([0], device)
        scratch = pages.to(device)
        ops.kv_page_append(scratch, k[b:b + 1].to(device), v[b:b + 1].to(device),
                           _i32(tables[b:b + 1], device), _i32(starts[b:b + 1], device), status)
        assert int(status) == 1
    got = pages.to(device)
    ops.kv_page_append(got, k.to(device), v.to(device), _i32(tables, device), _i32(starts, device))
    assert torch.equal(got.cpu(), want)
    # Nothing to write.
    empty = torch.empty(0, n, heads, dim, dtype=torch.bfloat16, device=device)
    ops.kv_page_append(got, empty, empty, torch.empty(0, 2, dtype=torch.int32, device=device),
                       torch.empty(0, dtype=torch.int32, device=device))
    assert torch.equal(got.cpu(), want)


# ---------------------------------------------------------------------------
# Copy
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layers,rows,src,dst,dtype", [
    (1, 16, [3], [0], torch.bfloat16),
    (5, 7, [0, 0, 6], [1, 5, 2], torch.float32),
    (70, 16, [2, 4], [1, 3], torch.float16),  # more pools than one launch takes
])
def test_copy(device, built_lib, layers, rows, src, dst, dtype):
    pools = [_rand((2, 8, rows, 3, 40), dtype, i) for i in range(layers)]
    want = [p.clone() for p in pools]
    for w, p in zip(want, pools):
        w[:, dst] = p[:, src]
    got = [p.to(device) for p in pools]
    ops.kv_page_copy(got, src, dst)
    assert all(torch.equal(g.cpu(), w) for g, w in zip(got, want))
    major = pools[0].transpose(2, 3).contiguous().to(device).transpose(2, 3)
    ops.kv_page_copy(major, src, dst)
    assert torch.equal(major.cpu(), want[0])
    ops.kv_page_copy(major, [], [])
    assert torch.equal(major.cpu(), want[0])


def test_copy_of_many_pages(device, built_lib):
    """More pairs than one launch takes, pages of more than one workgroup's piece."""
    pages = _rand((2, 620, 48, 1, 512), torch.bfloat16, 1)
    order = torch.randperm(620, generator=torch.Generator().manual_seed(2)).tolist()
    src, dst = order[:300], order[300:600]
    got = pages.to(device)
    ops.kv_page_copy(got, src, dst)
    pages[:, dst] = pages[:, src]
    assert torch.equal(got.cpu(), pages)


# ---------------------------------------------------------------------------
# Attention over pages
# ---------------------------------------------------------------------------
MASKS = {"none": {}, "causal": {"causal": True}, "blocks": {"bb": [0, 10, 20, 30, 40]},
         "late": {"bb": [20, 33]}, "any": {"bb": [30, -25, 7, 40]}}


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("mask", list(MASKS))
def test_masks_and_lengths(device, built_lib, dtype, dim, mask):
    """Rows 0..: lengths of zero, one and odd ones; "late" leaves the rows before the first
    block start without a key where nothing is cached (NaN)."""
    _case(device, dtype, dim, lens=[0, 1, 77, 160], lq=45, what=f"{mask} D{dim} {dtype}",
          **MASKS[mask])


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lq,heads,kv", [(1, 8, 1), (1, 3, 3), (7, 6, 2), (40, 4, 2), (130, 2, 1),
                                         (90, 1, 1)])
def test_rows_per_kv_head(device, built_lib, dtype, dim, lq, heads, kv):
    """One token to several row tiles, one query head per K/V head to eight."""
    _case(device, dtype, dim, lens=[300, 33], lq=lq, heads=heads, kv=kv, causal=lq > 1,
          what=f"lq {lq} {heads}/{kv} D{dim} {dtype}")


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("lq", [9, 45])
def test_short_rows_in_wide_tables(device, built_lib, dtype, dim, mask, lq):
    """What is planned for long sequences holds short ones: pieces of several items, items of
    several pieces, and more workgroups than there is work."""
    kw = dict(MASKS[mask])
    if "bb" in kw:
        kw["bb"] = [min(x, lq) for x in kw["bb"]]
    _case(device, dtype, dim, lens=[0, 1, 77, 160, 700], lq=lq, wide=True,
          what=f"wide {mask} {lq} D{dim} {dtype}", **kw)


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lq,heads,kv,n,wide", [
    (1, 8, 2, 3000, False), (20, 2, 2, 2049, False), (83, 3, 3, 5000, False), (1, 2, 1, 40, True),
    (83, 1, 1, 0, True), (40, 2, 1, 33, True)])
def test_one_sequence_in_ranges(device, built_lib, dtype, dim, lq, heads, kv, n, wide):
    """A single sequence's keys are split evenly: more ranges than tiles, or many of each."""
    _case(device, dtype, dim, lens=[n], lq=lq, heads=heads, kv=kv, causal=lq == 83, wide=wide,
          what=f"one sequence {n} + {lq} D{dim} {dtype}")


@pytest.mark.parametrize("rows", [16, 32, 48, 80, 112, 256, 1024])
def test_page_sizes(device, built_lib, rows):
    """Pages that end inside a tile, are whole tiles, or hold several."""
    _case(device, torch.bfloat16, 128, lens=[517, 2 * rows, rows - 1, rows + 1], lq=5, rows=rows,
          what=f"pages of {rows}")


@pytest.mark.parametrize("lq,lk", [(1, 0), (40, 0), (40, 1), (3, 130), (1, 33)])
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_new_keys_of_another_length(device, built_lib, lq, lk, dtype, dim):
    _case(device, dtype, dim, lens=[100, 7], lq=lq, lk=lk, what=f"lk {lk} for {lq}")


def test_no_keys_is_nan(device, built_lib):
    out = _case(device, torch.bfloat16, 64, lens=[0, 5], lq=2, lk=0, what="no keys")
    assert torch.isnan(out[0].float()).all() and torch.isfinite(out[1].float()).all()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 256),
                                       (torch.float32, 64)])
def test_long_caches_split(device, built_lib, dtype, dim):
    """A few rows over a long cache: key splits and their merge; one sequence is empty."""
    _case(device, dtype, dim, lens=[5003, 0, 1500], lq=3, rows=64, what=f"long D{dim} {dtype}")


@pytest.mark.parametrize("scale", [0.0, -0.11, 0.7])
def test_scales(device, built_lib, scale):
    _case(device, torch.float32, 64, lens=[70], lq=9, scale=scale, what=f"scale {scale}")
    _case(device, torch.bfloat16, 128, lens=[70], lq=9, scale=scale, what=f"scale {scale}")


def test_strided_inputs(device, built_lib):
    for dtype, dim in ((torch.bfloat16, 128), (torch.float32, 64)):
        _case(device, dtype, dim, lens=[40, 90], lq=20, causal=True, strided=True, what="strided")
        _case(device, dtype, dim, lens=[40, 90], lq=20, prefix_len=50, strided=True, what="strided")


def test_misaligned_inputs_are_copied(device, built_lib):
    """Contiguous q, k, v that begin off a 16-byte boundary."""
    lens, lq, heads, dim, rows = [20], 5, 2, 64, 16
    count, tables, _ = _tables(lens, rows, 1)
    pages = _rand((2, count, rows, heads, dim), torch.bfloat16, 2).to(device)
    q, k, v = (_rand((1, lq, heads, dim), torch.bfloat16, s).to(device) for s in (3, 4, 5))
    odd = [torch.cat((torch.zeros_like(t.flatten()[:1]), t.flatten()))[1:].view(t.shape)
           for t in (q, k, v)]
    assert all(t.data_ptr() % 16 and t.is_contiguous() for t in odd)
    args = dict(pages=pages, block_table=_i32(tables, device), cache_lens=_i32(lens, device))
    assert torch.equal(ops.paged_attention(*odd, **args), ops.paged_attention(q, k, v, **args))
    other = pages.clone()
    ops.kv_page_append(pages, k, v, args["block_table"], _i32([3], device))
    ops.kv_page_append(other, *odd[1:], args["block_table"], _i32([3], device))
    assert torch.equal(pages, other)


def test_entries_without_a_page_hide_their_keys(device, built_lib):
    """Dropped pages (-1), numbers past the pool: their keys are not seen, whichever half of a
    tile they fall in; lengths past the table, and negative ones, are clamped."""
    count, tables, _ = _tables([200, 130], 16, 3)
    tables[0][0] = tables[0][5] = -1
    tables[0][7] = count
    tables[1][1] = 2 ** 31 - 1
    tables[1][2] = -(2 ** 31)
    for dtype, dim in ((torch.bfloat16, 128), (torch.float32, 128)):
        _case(device, dtype, dim, lens=[200, 130], lq=20, tables=tables, seed=3, what="holes")
    _, tables, _ = _tables([96, 96], 16, 4)
    _case(device, torch.bfloat16, 64, lens=[96, 0], lq=4, tables=tables, seed=4,
          device_lens=[2 ** 31 - 1, -5], poison=False, what="clamped")


def test_all_pages_dropped(device, built_lib):
    """A cache without any page left: the new keys alone, or no key at all (NaN)."""
    tables = [[-1] * 4, [-1] * 4]
    _case(device, torch.bfloat16, 128, lens=[64, 50], lq=6, tables=tables, what="all dropped")
    out = _case(device, torch.bfloat16, 128, lens=[64, 50], lq=6, lk=0, tables=tables,
                what="all dropped, no new keys")
    assert torch.isnan(out.float()).all()


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lq,prefix_len", [(9, 0), (45, 0), (200, 0), (45, 70)])
@pytest.mark.parametrize("mask", ["causal", "blocks"])
@pytest.mark.parametrize("width", [None, 160])
def test_nothing_unseen_is_taken(device, built_lib, dtype, dim, lq, prefix_len, mask, width):
    """Infinities and NaN in keys and values that a query does not see, in the same tile as
    some that it does: its result is bit for bit what it was. Queries that see them get a
    result that is not finite in the columns that are not, and the others' bits elsewhere."""
    b, heads, rows, lens = 2, 2, 16, [21, 40]
    count, tables, prefix = _tables(lens, rows, 1, prefix_rows=prefix_len, width=width)
    pages = _rand((2, count, rows, heads, dim), dtype, 2).to(device)
    q, k, v = (_rand((b, lq, heads, dim), dtype, s).to(device) for s in (3, 4, 5))
    args = dict(pages=pages, block_table=_i32(tables, device), cache_lens=_i32(lens, device))
    if mask == "causal":
        args["causal"] = True
        end = torch.arange(lq)
    else:
        args["block_boundaries"] = torch.arange(0, lq, 7).to(device)
        end = (torch.arange(lq) // 7 + 1) * 7 - 1

    def run():
        if prefix_len:
            return ops.shared_prefix_attention(q, k, v, prefix_table=_i32(prefix, device),
                                               prefix_len=_i32([prefix_len], device), **args)
        return ops.paged_attention(q, k, v, **args)
    want = run()
    for at, col, bad in ((5, 3, math.inf), (5, 30, math.nan), (lq - 2, 50, -math.inf), (7, 63, math.nan)):
        v[1, at, 1, col] = bad
    got = run()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1, :, 0], want[1, :, 0])
    for at, cols in ((5, [3, 30]), (lq - 2, [50]), (7, [63])):
        sees = (end >= at).to(device)
        hit = got[1, :, 1][:, cols]
        assert torch.equal(hit[~sees], want[1, :, 1][:, cols][~sees])
        assert not torch.isfinite(hit[sees].float()).any()
    clean = [c for c in range(dim) if c not in (3, 30, 50, 63)]
    assert torch.equal(got[1, :, 1][:, clean], want[1, :, 1][:, clean])
    assert torch.equal(got[1, end >= 5, 1, 3].float().isinf().cpu(), torch.ones(int((end >= 5).sum()), dtype=torch.bool))
    # A key that is not finite: whole rows, of those that see it.
    k[0, 6, 0, 1] = math.nan
    got = run()
    sees = (end >= 6).to(device)
    assert torch.equal(got[0, ~sees, 0], want[0, ~sees, 0])
    assert torch.isnan(got[0, sees, 0].float()).all()
    assert torch.equal(got[0, :, 1], want[0, :, 1])


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lq,lens,prefix_len", [(3, [2080], 0), (130, [2080], 0), (70, [2000], 0),
                                                (50, [16, 21, 40], 2080), (2, [16, 21, 40], 2080)])
def test_infinities_that_every_query_sees(device, built_lib, dtype, dim, lq, lens, prefix_len):
    """Key j of the long run of keys has an infinite value in column j % dim, and all keys
    weigh the same: every result is that infinity, wherever the work is split."""
    heads, rows = 2, 16
    count, tables, prefix = _tables(lens, rows, 1, prefix_rows=prefix_len)
    pages = _rand((2, count, rows, heads, dim), dtype, 2)
    pages[0] = 0
    n = prefix_len or lens[0]
    j = torch.arange(n)
    held = torch.tensor(prefix or tables[0])
    pages[1, held[j // rows], j % rows, :, j % dim] = math.inf
    q, k, v = (_rand((len(lens), lq, heads, dim), dtype, s).to(device) for s in (3, 4, 5))
    k.zero_()
    args = dict(pages=pages.to(device), block_table=_i32(tables, device), cache_lens=_i32(lens, device))
    if prefix_len:
        got = ops.shared_prefix_attention(q, k, v, prefix_table=_i32(prefix, device),
                                          prefix_len=_i32([prefix_len], device), **args)
    else:
        got = ops.paged_attention(q, k, v, causal=True, **args)
    assert bool((got == math.inf).all())


def test_one_query_does_not_spoil_another(device, built_lib):
    """NaN in a query: its own row alone."""
    for dtype, dim in ((torch.bfloat16, 128), (torch.float32, 64)):
        lens, rows, heads, lq = [40, 9], 16, 2, 40
        count, tables, _ = _tables(lens, rows, 1)
        pages = _rand((2, count, rows, heads, dim), dtype, 2).to(device)
        q, k, v = (_rand((2, lq, heads, dim), dtype, s).to(device) for s in (3, 4, 5))
        args = dict(pages=pages, block_table=_i32(tables, device), cache_lens=_i32(lens, device))
        want = ops.paged_attention(q, k, v, **args)
        q[1, 7, 1, 5] = math.nan
        got = ops.paged_attention(q, k, v, **args)
        assert torch.isnan(got[1, 7, 1].float()).all()
        got[1, 7, 1] = want[1, 7, 1]
        assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# Shared prefix
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("mask", list(MASKS))
def test_shared_prefix_masks(device, built_lib, dtype, dim, mask):
    _case(device, dtype, dim, lens=[0, 1, 40], lq=45, prefix_len=203, what=f"{mask} D{dim} {dtype}",
          **MASKS[mask])


@pytest.mark.parametrize("b,lq,heads,kv,prefix_len,rows", [
    (1, 1, 1, 1, 1, 16),       # one query, one row of prefix
    (3, 1, 4, 4, 1000, 16),    # rows of several sequences in one tile
    (20, 1, 8, 2, 333, 32),
    (5, 13, 3, 3, 700, 48),    # sequences begin inside a 32-row block
    (2, 83, 4, 2, 129, 64),
    (33, 2, 2, 1, 2500, 16),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shared_prefix_batches(device, built_lib, b, lq, heads, kv, prefix_len, rows, dtype):
    lens = [(37 * i) % 90 for i in range(b)]
    _case(device, dtype, 128, lens=lens, lq=lq, heads=heads, kv=kv, prefix_len=prefix_len, rows=rows,
          causal=True, what=f"{b} x {lq}, prefix {prefix_len}")


def test_shared_prefix_without_own_rows(device, built_lib):
    _case(device, torch.bfloat16, 128, lens=[0, 0, 0], lq=9, prefix_len=100, own=False,
          what="no own cache")
    _case(device, torch.bfloat16, 128, lens=[0, 0], lq=9, lk=0, prefix_len=100, own=False,
          what="prefix alone")


def test_shared_prefix_of_no_rows(device, built_lib):
    """An empty prefix, dropped pages in it, all of it dropped: the other keys alone."""
    _case(device, torch.bfloat16, 128, lens=[30, 0], lq=9, prefix_len=0, prefix=[0], causal=True,
          what="empty prefix")
    _case(device, torch.bfloat16, 128, lens=[30, 0], lq=9, prefix_len=60, prefix=[-1, 1, 99, 0],
          seed=9, what="holes in the prefix")
    _case(device, torch.bfloat16, 128, lens=[30, 0], lq=9, prefix_len=60, prefix=[-1] * 4,
          what="prefix dropped")


def test_shared_prefix_equals_paged_attention_over_it(device, built_lib):
    """A prefix that fills its pages, put in front of every table: the same keys, so the same
    result up to how fp32 sums are split (2 u of the result and fp32 terms: see the bound)."""
    b, lq, heads, dim, rows, pre = 6, 10, 4, 128, 32, 256
    lens = [0, 5, 64, 33, 90, 1]
    count, tables, prefix = _tables(lens, rows, 1, prefix_rows=pre)
    pages = _rand((2, count, rows, heads, dim), torch.float32, 2).to(device)
    q, k, v = (_rand((b, lq, heads, dim), torch.float32, s).to(device) for s in (3, 4, 5))
    shared = ops.shared_prefix_attention(
        q, k, v, pages=pages, prefix_table=_i32(prefix, device), prefix_len=_i32([pre], device),
        block_table=_i32(tables, device), cache_lens=_i32(lens, device), causal=True)
    joined = ops.paged_attention(
        q, k, v, pages=pages, block_table=_i32([prefix + t for t in tables], device),
        cache_lens=_i32([pre + n for n in lens], device), causal=True)
    # Both are within fp32 sums of the exact value: 2 (keys + 64 + ...) 2^-24 sum p |v| each.
    assert (shared - joined).abs().max().item() <= 2e-4
    contiguous = torch.zeros(2, b, pre + max(lens), heads, dim, device=device)
    for i, n in enumerate(lens):
        flat = pages[:, prefix + tables[i]].flatten(1, 2) if n else pages[:, prefix].flatten(1, 2)
        contiguous[:, i, :pre + n] = flat[:, :pre + n]
    varlen = ops.blockwise_causal_attention_varlen(
        q, k, v, kv_cache=contiguous, cache_lens=[pre + n for n in lens], causal=True)
    assert (joined - varlen).abs().max().item() <= 2e-4


# ---------------------------------------------------------------------------
# Large offsets, streams, graphs, repeated calls
# ---------------------------------------------------------------------------
def test_offsets_past_32_bits(device, built_lib):
    """Pages and rows whose byte offsets pass 2^31 and 2^32, in one plane."""
    rows, heads, dim = 1024, 16, 128
    count = 1100  # 4.6 GB a plane
    pages = torch.zeros(2, count, rows, heads, dim, dtype=torch.bfloat16, device=device)
    ids = [1099, 3, 600, 1024]
    live = _rand((2, len(ids), rows, heads, dim), torch.bfloat16, 1)
    pages[:, ids] = live.to(device)
    q, k, v = (_rand((1, 3, heads, dim), torch.bfloat16, s) for s in (2, 3, 4))
    n = 3 * rows + 100
    got = ops.paged_attention(q.to(device), k.to(device), v.to(device), pages=pages,
                              block_table=_i32([ids], device), cache_lens=_i32([n], device))
    want = opaged.paged_attention(q, k, v, live, [[0, 1, 2, 3]], [n])
    _check(got, want, torch.bfloat16, dim, n + 3, float(live.abs().max()), "4.6 GB planes")
    new = _rand((1, 50, heads, dim), torch.bfloat16, 5).to(device)
    ops.kv_page_append(pages, new, new, _i32([ids], device), _i32([n], device))
    ops.kv_page_copy(pages, [1024], [1098])
    for page in (1024, 1098):
        assert torch.equal(pages[:, page, 100:150], torch.stack((new[0], new[0])))
        assert torch.equal(pages[:, page, :100].cpu(), live[:, 3, :100])


def _decode_state(device, b=4, lq=3, heads=4, kv=2, dim=128, rows=16, width=40):
    pool = b * width + width
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(5)).tolist()
    tables = [[order.pop() for _ in range(width)] for _ in range(b)]
    return dict(
        pages=_rand((2, pool, rows, kv, dim), torch.bfloat16, 6).to(device),
        table=_i32(tables, device), lens=_i32([5, 100, 0, 300], device),
        prefix=_i32(order[:width], device), plen=_i32([500], device),
        q=_rand((b, lq, heads, dim), torch.bfloat16, 7).to(device),
        k=_rand((b, lq, kv, dim), torch.bfloat16, 8).to(device),
        v=_rand((b, lq, kv, dim), torch.bfloat16, 9).to(device))


def _step(s):
    """A decode step: write the chunk, attend to everything before it and to itself."""
    ops.kv_page_append(s["pages"], s["k"], s["v"], s["table"], s["lens"])
    own = ops.paged_attention(s["q"], s["k"], s["v"], pages=s["pages"], block_table=s["table"],
                              cache_lens=s["lens"], causal=True)
    both = ops.shared_prefix_attention(
        s["q"], s["k"], s["v"], pages=s["pages"], prefix_table=s["prefix"], prefix_len=s["plen"],
        block_table=s["table"], cache_lens=s["lens"], causal=True)
    s["lens"].add_(s["q"].shape[1])
    return own, both


def test_captured_steps_follow_tables_and_lengths(device, built_lib):
    """A decode step captured once: replays append at, and attend up to, lengths and tables
    that changed since; each replay equals the eager step bit for bit, with eager calls and
    a second graph's replays between them."""
    s, e = _decode_state(device), _decode_state(device)
    warm = _decode_state(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(warm)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = _step(s)
    with torch.cuda.graph(other, stream=side):
        _step(warm)
    for turn in range(5):
        if turn == 3:  # a sequence moves to other pages, another loses one
            for x in (s, e):
                x["table"][1] = x["table"][1].flip(0)
                x["table"][3, 2] = -1
                x["plen"].fill_(77)
        other.replay()
        graph.replay()
        other.replay()
        want = _step(e)
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref), f"replay {turn}"
        assert torch.equal(s["pages"], e["pages"]) and torch.equal(s["lens"], e["lens"])


def test_two_streams_at_once(device, built_lib):
    """The same calls on two streams, issued together, give what one stream gives."""
    s = _decode_state(device, b=4, lq=1)
    args = dict(pages=s["pages"], prefix_table=s["prefix"], prefix_len=s["plen"],
                block_table=s["table"], cache_lens=s["lens"])
    want = ops.shared_prefix_attention(s["q"], s["k"], s["v"], **args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(ops.shared_prefix_attention(s["q"], s["k"], s["v"], **args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_repeated_calls_agree_bit_for_bit(device, built_lib):
    s = _decode_state(device)
    first = ops.paged_attention(s["q"], s["k"], s["v"], pages=s["pages"], block_table=s["table"],
                                cache_lens=s["lens"])
    for _ in range(5):
        again = ops.paged_attention(s["q"], s["k"], s["v"], pages=s["pages"],
                                    block_table=s["table"], cache_lens=s["lens"])
        assert torch.equal(again, first)


def test_empty_batches(device, built_lib):
    pages = torch.zeros(2, 3, 16, 2, 64, dtype=torch.bfloat16, device=device)
    for b, lq in ((0, 4), (2, 0)):
        q = torch.empty(b, lq, 2, 64, dtype=torch.bfloat16, device=device)
        out = ops.paged_attention(q, q, q, pages=pages,
                                  block_table=torch.zeros(b, 1, dtype=torch.int32, device=device),
                                  cache_lens=torch.zeros(b, dtype=torch.int32, device=device))
        assert out.shape == q.shape
