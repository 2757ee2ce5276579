"""A KV cache's pages in 4 bits (MI355X): writing, reading back, attention over them.

Codes, scales and the values read back are compared bit for bit with ``oracle/fp4.py``; the
rest of a pool stays as it was. Attention is compared with ``oracle/paged.py`` (64 bits) over
the values that the pool stands for, within ``oracle.paged.error_bound``: reading 4 bits adds
no rounding to those of attention over 16. Log-sum-exps are compared within
``oracle.keep.lse_bound``.
"""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
from oracle import fp4, keep
from oracle import paged as opaged

pytestmark = pytest.mark.gpu

TYPES = [(dt, d) for dt in (torch.bfloat16, torch.float16) for d in (64, 128, 256)]
IDS = [f"{str(dt)[6:]}-D{d}" for dt, d in TYPES]
MASKS = {"none": {}, "causal": {"causal": True}, "blocks": {"bb": [0, 10, 20, 30, 40]},
         "late": {"bb": [20, 33]}, "any": {"bb": [30, -25, 7, 40]}}


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _tables(lens, rows, seed, spare=2, prefix_rows=0):
    held = [-(-n // rows) for n in lens]
    pre = -(-prefix_rows // rows)
    total = sum(held) + pre + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max([1] + held)
    return (total, [[order.pop() if j < n else -1 for j in range(width)] for n in held],
            [order.pop() for _ in range(pre)])


def _bytes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)


# ---------------------------------------------------------------------------
# Writing and reading back
# ---------------------------------------------------------------------------
def _write_case(device, k, v, starts, rows, seed, tables=None, count=None, views=False):
    """Append and read back against the oracle, byte for byte."""
    b, n, heads, dim = k.shape
    if tables is None:
        count, tables, _ = _tables([max(s, 0) + n for s in starts], rows, seed)
    pool = _bytes((2, count, heads, rows * (dim // 2 + dim // 32)), seed)
    codes, scales = (t.clone() for t in fp4.unpack(pool, rows, dim))
    back = torch.zeros(2, b, n, heads, dim, dtype=torch.float64)
    holes = 0
    for plane, x in enumerate((k, v)):
        c, e = fp4.quantise(x)
        for i, s in enumerate(starts):
            for t in range(n):
                r = s + t
                page = tables[i][r // rows] if 0 <= r < len(tables[i]) * rows else -1
                if not 0 <= page < count:
                    holes += 1
                    continue
                codes[plane, page, r % rows], scales[plane, page, r % rows] = c[i, t], e[i, t]
                back[plane, i, t] = fp4.dequantise(c[i, t], e[i, t])
    got, status = pool.to(device), _i32([0], device)
    if views:  # k and v of one projection's rows; a pool that is part of a larger one
        kv = torch.cat((k, v), 2).to(device)
        kd, vd = kv[:, :, :heads], kv[:, :, heads:]
        got = torch.cat((got, got), 2)[:, :, :heads]
    else:
        kd, vd = k.to(device), v.to(device)
    args = _i32(tables, device), _i32(starts, device)
    ops.kv_page_append_fp4(got, kd, vd, *args, status)
    assert torch.equal(got.cpu(), fp4.pack(codes, scales))
    assert int(status) == (1 if holes else 0)
    status.zero_()
    read = ops.kv_page_read_fp4(got, *args, n, dim, k.dtype, status)
    assert int(status) == (1 if holes else 0)
    for x, want in zip(read, back):
        assert x.dtype == k.dtype and x.shape == k.shape and x.is_contiguous()
        assert torch.equal(torch.isnan(x.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(x.double().cpu(), nan=0.5), torch.nan_to_num(want, nan=0.5))


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("n,starts,rows,heads", [(1, [0, 7, 15], 16, 3), (83, [0, 13, 200], 64, 2),
                                                 (50, [16, 47], 48, 1), (17, [1023, 0], 1024, 5)])
def test_write_and_read(device, built_lib, dtype, dim, n, starts, rows, heads):
    k, v = (_rand((len(starts), n, heads, dim), dtype, s) for s in (3, 4))
    _write_case(device, k, v, starts, rows, 1)
    _write_case(device, k, v, starts, rows, 1, views=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_blocks_at_the_edges(device, built_lib, dtype):
    """Ties, 7 and just above it, zeros of both signs, the smallest and the largest numbers,
    every exponent, infinities and NaN."""
    x = _rand((1, 64, 2, 64), dtype, 5)
    g = torch.Generator().manual_seed(6)
    e = torch.arange(64).float() * (4 if dtype == torch.bfloat16 else 0.6) - (126 if dtype == torch.bfloat16 else 24)
    x[0, :, 0] = (x[0, :, 0].double() * torch.exp2(e.double())[:, None]).to(dtype)
    x[0, :40, 1] = (torch.randint(-28, 29, (40, 64), generator=g) / 4).to(dtype)
    x[0, 0, 1, :32] = 0
    x[0, 1, 1, :32] = -0.0
    x[0, 2, 1] = torch.finfo(dtype).max
    x[0, 3, 1] = torch.finfo(dtype).tiny
    x[0, 4, 1] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the smallest of all
    x[0, 5, 1, 7], x[0, 6, 1, 40], x[0, 7, 1, 0] = math.inf, math.nan, -math.inf
    x[0, 8, 1, 0] = 7.0
    x[0, 9, 1, 0] = 7.0 * (1 + torch.finfo(dtype).eps)
    _write_case(device, x, x.flip(1).contiguous(), [3], 16, 7)


def test_rows_without_a_page(device, built_lib):
    k, v = (_rand((3, 40, 2, 64), torch.bfloat16, s) for s in (2, 3))
    tables, starts = [[0, 1, 5], [4, 2, -1], [3, -1, 2 ** 31 - 1]], [-3, 0, 10]
    _write_case(device, k, v, starts, 16, 8, tables, 4)
    # Nothing to write or to read.
    pool = _bytes((2, 4, 2, 16 * 34), 9).to(device)
    want = pool.clone()
    empty = torch.empty(0, 4, 2, 64, dtype=torch.bfloat16, device=device)
    t0, s0 = (torch.empty(*s, dtype=torch.int32, device=device) for s in ((0, 2), (0,)))
    ops.kv_page_append_fp4(pool, empty, empty, t0, s0)
    a = ops.kv_page_read_fp4(pool, t0, s0, 3, 64)[0]
    c = ops.kv_page_read_fp4(pool, _i32([[1]], device), _i32([0], device), 0, 64)[1]
    assert a.shape == (0, 3, 2, 64) and c.shape == (1, 0, 2, 64) and torch.equal(pool, want)


def test_a_read_in_the_other_type(device, built_lib):
    """f16 rows are exact in bf16 too; bf16 rows past f16's largest number read as infinity."""
    for dtype, other, scale in ((torch.float16, torch.bfloat16, 1.0), (torch.bfloat16, torch.float16, 2.0 ** 40)):
        k, v = (_rand((1, 16, 1, 128), dtype, s, scale) for s in (1, 2))
        pool = torch.zeros(2, 1, 1, 16 * 68, dtype=torch.uint8, device=device)
        args = _i32([[0]], device), _i32([0], device)
        ops.kv_page_append_fp4(pool, k.to(device), v.to(device), *args)
        got = ops.kv_page_read_fp4(pool, *args, 16, 128, other)
        for x, want in zip(got, (k, v)):
            assert torch.equal(x.cpu(), fp4.stored(want).to(other))


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _check(got, lse, want, want_lse, dtype, dim, keys, vmax, what):
    ref, weight, scores = want
    got = got.double().cpu()
    none = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), none), f"{what}: NaN elements differ"
    bound = opaged.error_bound(ref, weight, dtype, dim, keys, scores, vmax)
    # (A stored value may be 0, and what is made of it alone exact, with a bound of 0.)
    worst = torch.where(got == ref, 0.0, (got - ref).abs() / bound)[~none]
    worst = float(worst.max()) if worst.numel() else 0.0
    ref, size = want_lse
    assert lse.dtype == torch.float32 and lse.shape == ref.shape
    lse = lse.double().cpu()
    none = ref == -math.inf
    assert torch.equal(lse == -math.inf, none), f"{what}: lse of rows without a key"
    off = (lse - ref).abs() / keep.lse_bound(ref, dim, keys, size)
    off = float(off[~none].max()) if (~none).any() else 0.0
    print(f"[fp4] {what}: {worst:.3f} of the bound, lse {off:.3f}")
    assert worst <= 1.0 and off <= 1.0, f"{what}: error {worst:.3f}, lse {off:.3f} times the bound"


def _case(device, dtype, dim, *, lens, lq, heads=2, kv=2, rows=16, prefix_len=0, lk=None, bb=None,
          causal=False, scale=None, seed=0, tables=None, own=True, wide=0, device_lens=None,
          strided=False, what=""):
    """One call against the oracle. Rows and pages that no sequence holds are bytes of 255: NaN."""
    b, lk = len(lens), lq if lk is None else lk
    count, t0, prefix = _tables(lens, rows, seed, prefix_rows=prefix_len)
    tables = t0 if tables is None else tables
    tables = [t + [-1] * wide for t in tables]
    q = _rand((b, lq, heads, dim), dtype, seed + 1)
    k = _rand((b, lk, kv, dim), dtype, seed + 2)
    v = _rand((b, lk, kv, dim), dtype, seed + 3)
    pages = _rand((2, count, rows, kv, dim), dtype, seed + 4)
    codes, scales = fp4.quantise(pages)
    values = fp4.dequantise(codes, scales)
    live = torch.zeros(count, rows, dtype=torch.bool)
    for table, n in list(zip(tables, lens)) + [(prefix, prefix_len)]:
        for r in range(n):
            if 0 <= table[r // rows] < count:
                live[table[r // rows], r % rows] = True
    scales[:, ~live] = 255
    pool = fp4.pack(codes, scales).to(device)
    qd = q.to(device)
    if strided:
        qd = torch.cat((qd, qd), -1)[..., :dim]
        pool = torch.cat((pool, pool), 1)[:, :count]
    kw = dict(pages=pool, block_boundaries=None if bb is None else torch.tensor(bb).to(device),
              softmax_scale=scale, causal=causal)
    if own:
        kw.update(block_table=_i32(tables, device),
                  cache_lens=_i32(lens if device_lens is None else device_lens, device))
    call = ops.paged_attention_fp4
    if prefix_len:
        call = ops.shared_prefix_attention_fp4
        kw.update(prefix_table=_i32(prefix, device), prefix_len=_i32([prefix_len], device))
    kd, vd = k.to(device), v.to(device)
    out, lse = call(qd, kd, vd, return_lse=True, **kw)
    assert out.dtype == dtype
    alone = call(qd, kd, vd, **kw)
    assert torch.equal(torch.nan_to_num(alone, nan=3.0), torch.nan_to_num(out, nan=3.0))
    args = (values, tables if own else None, lens if own else None, prefix, prefix_len,
            None if bb is None else torch.tensor(bb), scale, causal)
    want = opaged.paged_attention(q, k, v, *args)
    vmax = max(float(t.double().abs().max()) if t.numel() else 0.0 for t in (values[1], v))
    _check(out, lse, want, keep.log_sum_exp(q, k, *args), dtype, dim, prefix_len + max(lens) + lk, vmax, what)
    return out


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("mask", list(MASKS))
def test_masks_and_lengths(device, built_lib, dtype, dim, mask):
    _case(device, dtype, dim, lens=[0, 1, 77, 160], lq=45, what=f"{mask} D{dim}", **MASKS[mask])


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lq,heads,kv", [(1, 8, 1), (1, 3, 3), (7, 6, 2), (40, 4, 2), (130, 2, 1)])
def test_rows_per_kv_head(device, built_lib, dtype, dim, lq, heads, kv):
    _case(device, dtype, dim, lens=[300, 33], lq=lq, heads=heads, kv=kv, causal=lq > 1,
          what=f"lq {lq} {heads}/{kv} D{dim}")


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("mask", ["none", "late", "any"])
@pytest.mark.parametrize("lq", [9, 45])
def test_short_rows_in_wide_tables(device, built_lib, dtype, dim, mask, lq):
    kw = dict(MASKS[mask])
    if "bb" in kw:
        kw["bb"] = [min(x, lq) for x in kw["bb"]]
    _case(device, dtype, dim, lens=[0, 1, 77, 160, 700], lq=lq, wide=132, what=f"wide {mask} {lq} D{dim}", **kw)


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lq,heads,kv,n", [(1, 8, 2, 3000), (20, 2, 2, 2049), (83, 1, 1, 4000), (83, 1, 1, 0)])
def test_one_sequence(device, built_lib, dtype, dim, lq, heads, kv, n):
    _case(device, dtype, dim, lens=[n], lq=lq, heads=heads, kv=kv, causal=lq == 83,
          what=f"one sequence {n} + {lq} D{dim}")


@pytest.mark.parametrize("rows", [16, 32, 48, 80, 112, 256, 1024])
@pytest.mark.parametrize("lq", [5, 40])
def test_page_sizes(device, built_lib, rows, lq):
    _case(device, torch.bfloat16, 128, lens=[517, 2 * rows, rows - 1, rows + 1], lq=lq, rows=rows,
          what=f"pages of {rows}")


@pytest.mark.parametrize("lq,lk", [(1, 0), (40, 0), (40, 1), (3, 130), (1, 33)])
def test_new_keys_of_another_length(device, built_lib, lq, lk):
    _case(device, torch.bfloat16, 128, lens=[100, 7], lq=lq, lk=lk, what=f"lk {lk} for {lq}")


def test_no_keys(device, built_lib):
    out = _case(device, torch.bfloat16, 64, lens=[0, 5], lq=2, lk=0, what="no keys")
    assert torch.isnan(out[0].float()).all() and torch.isfinite(out[1].float()).all()


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lens,lq,prefix_len,kw", [
    ([0, 33, 200], 45, 100, {"causal": True}), ([5, 0, 77, 130, 16], 1, 333, {}),
    ([40, 90], 20, 17, {"bb": [0, 7, 14]}), ([0, 0, 0, 0], 50, 500, {})])
def test_prefixes(device, built_lib, dtype, dim, lens, lq, prefix_len, kw):
    heads, kv = (8, 2) if lq == 1 else (2, 2)
    _case(device, dtype, dim, lens=lens, lq=lq, heads=heads, kv=kv, prefix_len=prefix_len,
          what=f"prefix {prefix_len} lq {lq} D{dim}", **kw)


def test_a_prefix_alone(device, built_lib):
    _case(device, torch.bfloat16, 128, lens=[0, 0], lq=3, prefix_len=60, own=False, what="prefix alone")


@pytest.mark.parametrize("scale", [0.0, -0.11, 0.7])
def test_scales(device, built_lib, scale):
    for lq in (9, 50):
        _case(device, torch.bfloat16, 128, lens=[70], lq=lq, scale=scale, what=f"scale {scale}")


def test_strided_inputs(device, built_lib):
    _case(device, torch.bfloat16, 128, lens=[40, 90], lq=20, causal=True, strided=True, what="strided")
    _case(device, torch.float16, 64, lens=[40, 90], lq=50, prefix_len=50, strided=True, what="strided")


@pytest.mark.parametrize("lq", [3, 40])
def test_entries_without_a_page(device, built_lib, lq):
    """Their keys are not seen, whichever half of a tile they fall in; lengths are clamped."""
    count, tables, _ = _tables([200, 130], 16, 3)
    tables[0][0] = tables[0][5] = -1
    tables[0][7] = count
    tables[1][1] = 2 ** 31 - 1
    tables[1][2] = -(2 ** 31)
    for dim in (64, 128, 256):
        _case(device, torch.bfloat16, dim, lens=[200, 130], lq=lq, tables=tables, seed=3, what="holes")
    _, tables, _ = _tables([96, 96], 16, 4)
    _case(device, torch.bfloat16, 64, lens=[96, 0], lq=lq, tables=tables, seed=4,
          device_lens=[2 ** 31 - 1, -5], what="clamped")
    _, tables, _ = _tables([64, 64], 16, 5)
    _case(device, torch.bfloat16, 128, lens=[64, 64], lq=lq, lk=0, seed=5,
          tables=[[-1] * 4, tables[1]], what="all dropped")


@pytest.mark.parametrize("lq", [2, 50])
def test_a_block_that_is_no_number(device, built_lib, lq):
    """In a seen row's V it makes its 32 dims NaN, for the queries of its head alone; in K the
    query's result."""
    rows, dim, n = 16, 128, 100
    count, tables, _ = _tables([n], rows, 1)
    pool = fp4.pack(*fp4.quantise(_rand((2, count, rows, 2, dim), torch.bfloat16, 2)))
    q, k, v = (_rand((1, lq, 2, dim), torch.bfloat16, s).to(device) for s in (3, 4, 5))
    for plane in (0, 1):
        bad = pool.clone()
        bad[plane, tables[0][2], 1, rows * 64 + 4 * 5 + 3] = 255  # row 37, the last block, head 1
        out = ops.paged_attention_fp4(q, k, v, pages=bad.to(device), block_table=_i32(tables, device),
                                      cache_lens=_i32([n], device))
        nan = torch.isnan(out[0].float().cpu())
        assert not nan[:, 0].any()
        assert nan[:, 1, 96:].all() and (nan[:, 1].all() if plane == 0 else not nan[:, 1, :96].any())


@pytest.mark.parametrize("lq", [20, 70])
def test_what_a_query_does_not_see_of_the_new_keys(device, built_lib, lq):
    """Infinities and NaN in new values that a causal mask hides leave the others' bits alone."""
    lens, rows, dim = [50], 16, 128
    count, tables, _ = _tables(lens, rows, 1)
    pool = fp4.pack(*fp4.quantise(_rand((2, count, rows, 2, dim), torch.bfloat16, 2))).to(device)
    q, k, v = (_rand((1, lq, 2, dim), torch.bfloat16, s).to(device) for s in (3, 4, 5))
    kw = dict(pages=pool, block_table=_i32(tables, device), cache_lens=_i32(lens, device), causal=True)
    clean = ops.paged_attention_fp4(q, k, v, **kw)
    wild = v.clone()
    wild[0, lq // 2:] = math.inf
    wild[0, lq // 2 + 3] = math.nan
    out = ops.paged_attention_fp4(q, k, wild, **kw)
    assert torch.equal(out[:, :lq // 2], clean[:, :lq // 2])
    assert not torch.isfinite(out[:, lq // 2:].float()).any()


def test_a_pool_past_4_gb(device, built_lib):
    """Pages whose bytes lie past 2^32."""
    dim, rows, heads = 128, 1024, 8
    size = rows * 68 * heads
    count = (1 << 32) // size + 3
    pool = torch.empty(2, count, heads, rows * 68, dtype=torch.uint8, device=device)
    lens, table = [1500], [[count - 1, 0]]
    k, v = (_rand((1, 1500, heads, dim), torch.bfloat16, s).to(device) for s in (1, 2))
    at = _i32(table, device)
    ops.kv_page_append_fp4(pool, k, v, at, _i32([0], device))
    small = torch.zeros(2, 2, heads, rows * 68, dtype=torch.uint8, device=device)
    there = _i32([[1, 0]], device)
    ops.kv_page_append_fp4(small, k, v, there, _i32([0], device))
    assert torch.equal(small[:, 1], pool[:, count - 1])
    for x, y in zip(ops.kv_page_read_fp4(pool, at, _i32([0], device), 1500, dim),
                    ops.kv_page_read_fp4(small, there, _i32([0], device), 1500, dim)):
        assert torch.equal(x, y)
    for lq in (1, 50):
        q, kn, vn = (_rand((1, lq, heads, dim), torch.bfloat16, s).to(device) for s in (3, 4, 5))
        got = [ops.paged_attention_fp4(q, kn, vn, pages=p, block_table=t, cache_lens=_i32(lens, device),
                                       return_lse=True) for p, t in ((pool, at), (small, there))]
        assert torch.equal(got[0][0], got[1][0])
        w = [ops.paged_key_weights(q, g[1], pages=p, block_table=t, cache_lens=_i32(lens, device))
             for g, p, t in zip(got, (pool, small), (at, there))]
        assert torch.equal(*w)


def test_replays_follow_lengths_and_tables(device, built_lib):
    """A captured append and attention, replayed as the cache grows, against eager calls."""
    rows, heads, dim, b, n = 16, 2, 128, 3, 5
    pool = torch.zeros(2, 40, heads, rows * 68, dtype=torch.uint8, device=device)
    other = pool.clone()
    tables = torch.full((b, 8), -1, dtype=torch.int32)
    lens = [0, 30, 77]
    order = torch.randperm(40, generator=torch.Generator().manual_seed(1)).tolist()
    for i, x in enumerate(lens):
        for j in range(-(-x // rows)):
            tables[i, j] = order.pop()
    table, length = tables.to(device), _i32(lens, device)
    x = [torch.zeros(b, n, heads, dim, dtype=torch.bfloat16, device=device) for _ in range(3)]

    def step(p):
        ops.kv_page_append_fp4(p, x[1], x[2], table, length)
        return ops.paged_attention_fp4(*x, pages=p, block_table=table, cache_lens=length, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(other)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = step(pool)
    pool.zero_()
    other.zero_()
    for i in range(6):
        for j in range(b):  # pages for the next rows
            while (tables[j] >= 0).sum() * rows < lens[j] + n:
                tables[j, int((tables[j] >= 0).sum())] = order.pop()
        table.copy_(tables)
        length.copy_(torch.tensor(lens, dtype=torch.int32))
        for t, s in zip(x, (1, 2, 3)):
            t.copy_(_rand((b, n, heads, dim), torch.bfloat16, 10 * i + s))
        graph.replay()
        torch.cuda.synchronize()
        want, want_lse = step(other)
        assert torch.equal(pool, other)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        lens = [y + n for y in lens]
