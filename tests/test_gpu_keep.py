"""Log-sum-exps, row weights, which rows to keep, and their move (MI355X).

Row numbers, moved rows and moved weights are equal to ``oracle/keep.py``; weights lie within
``oracle.keep.weights_bound`` and log-sum-exps within ``lse_bound`` of 64 bits.
"""

from __future__ import annotations

import math

import pytest
import torch

import dexter_amd.ops as ops
from oracle import fp4, keep
from oracle import paged as opaged

pytestmark = pytest.mark.gpu

TYPES = [(dt, d, False) for dt in (torch.bfloat16, torch.float16) for d in (64, 128, 256)]
TYPES += [(torch.float32, 64, False), (torch.float32, 128, False)]
TYPES += [(dt, d, True) for dt in (torch.bfloat16, torch.float16) for d in (64, 128, 256)]
IDS = [f"{str(dt)[6:]}-D{d}{'-fp4' if f else ''}" for dt, d, f in TYPES]


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _tables(lens, rows, seed, spare=2, extra=0):
    held = [-(-n // rows) for n in lens]
    total = sum(held) + spare + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max([1] + held)
    return total, [[order.pop() if j < n else -1 for j in range(width)] for n in held], order


# ---------------------------------------------------------------------------
# Log-sum-exps of attention over 16- and 32-bit pages
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,dim", [t[:2] for t in TYPES[:8]], ids=IDS[:8])
@pytest.mark.parametrize("lens,lq,heads,kv,prefix_len,kw", [
    ([0, 1, 77, 700], 45, 2, 2, 0, {"causal": True}), ([300, 33, 0], 1, 8, 2, 0, {}),
    ([3000], 83, 1, 1, 0, {}), ([5, 0, 77], 1, 8, 2, 333, {}), ([0, 33], 45, 2, 2, 100, {"bb": [20, 33]}),
    ([0, 0], 45, 2, 2, 0, {"bb": [20, 33]})])
def test_log_sum_exps(device, built_lib, dtype, dim, lens, lq, heads, kv, prefix_len, kw):
    rows = 16
    pre = -(-prefix_len // rows)
    count, tables, order = _tables(lens, rows, 1, extra=pre)
    prefix = [order.pop() for _ in range(pre)]
    q = _rand((len(lens), lq, heads, dim), dtype, 2)
    k, v = (_rand((len(lens), lq, kv, dim), dtype, s) for s in (3, 4))
    pages = _rand((2, count, rows, kv, dim), dtype, 5)
    bb = torch.tensor(kw["bb"]) if "bb" in kw else None
    args = dict(pages=pages.to(device), block_table=_i32(tables, device), cache_lens=_i32(lens, device),
                causal=kw.get("causal", False), block_boundaries=None if bb is None else bb.to(device))
    call = ops.paged_attention
    if prefix_len:
        call = ops.shared_prefix_attention
        args.update(prefix_table=_i32(prefix, device), prefix_len=_i32([prefix_len], device))
    d = [t.to(device) for t in (q, k, v)]
    out, lse = call(*d, return_lse=True, **args)
    ref = (pages, tables, lens, prefix, prefix_len, bb, None, kw.get("causal", False))
    want, weight, scores = opaged.paged_attention(q, k, v, *ref)
    keys = prefix_len + max(lens) + lq
    none = torch.isnan(want)
    got = out.double().cpu()
    assert torch.equal(torch.isnan(got), none)
    vmax = float(max(pages[1].double().abs().max(), v.double().abs().max()))
    bound = opaged.error_bound(want, weight, dtype, dim, keys, scores, vmax)
    assert float(((got - want).abs() / bound)[~none].max()) <= 1.0
    want, size = keep.log_sum_exp(q, k, *ref)
    lse, none = lse.double().cpu(), want == -math.inf
    assert torch.equal(lse == -math.inf, none)
    worst = float(((lse - want).abs() / keep.lse_bound(want, dim, keys, size))[~none].max())
    print(f"[lse] {dtype} D{dim} {lens} lq {lq}: {worst:.3f} of the bound")
    assert worst <= 1.0
    plain = call(*d, **args)  # and without it: the same within both's bounds
    assert float(((plain.double().cpu() - got).abs() / (2 * bound))[~torch.isnan(got)].max()) <= 1.0


# ---------------------------------------------------------------------------
# Weights
# ---------------------------------------------------------------------------
def _weights_case(device, dtype, dim, in4, *, lens, lq, heads, kv, rows=16, seed=0, scale=None,
                  device_lens=None, tables=None, lse=None, strided=False):
    count, t0, _ = _tables(lens, rows, seed)
    tables = t0 if tables is None else tables
    b = len(lens)
    q = _rand((b, lq, heads, dim), dtype, seed + 1)
    pages = _rand((2, count, rows, kv, dim), dtype, seed + 2)
    if lse is None:
        none = q[:, :0, :kv]
        lse = keep.log_sum_exp(q, none, fp4.stored(pages) if in4 else pages, tables, lens,
                               softmax_scale=scale)[0]
        lse = torch.where(lse == -math.inf, 0.0, lse).float() + 0.1
    # Rows that no sequence holds: NaN.
    live = torch.zeros(count, rows, dtype=torch.bool)
    for table, n in zip(tables, lens):
        for r in range(n):
            if 0 <= table[r // rows] < count:
                live[table[r // rows], r % rows] = True
    if in4:
        codes, scales = fp4.quantise(pages)
        values = fp4.dequantise(codes, scales)
        scales[:, ~live] = 255
        pool = fp4.pack(codes, scales)
    else:
        values, pool = pages, pages.clone()
        pool[:, ~live] = math.nan
    pool, qd, ld = pool.to(device), q.to(device), lse.to(device)
    if strided:
        qd = torch.cat((qd, qd), -1)[..., :dim]
        ld = ld.transpose(1, 2).contiguous().transpose(1, 2)
        pool = torch.cat((pool, pool), 1)[:, :count]
    kw = dict(pages=pool, block_table=_i32(tables, device), softmax_scale=scale,
              cache_lens=_i32(lens if device_lens is None else device_lens, device))
    got = ops.paged_key_weights(qd, ld, **kw)
    want, size = keep.key_weights(q, lse, values, tables, lens, scale)
    assert got.dtype == torch.float32 and got.shape == want.shape
    bound = keep.weights_bound(want, size, dim, lq * heads // kv)
    x = got.double().cpu()
    worst = float(((x - want).abs() / bound)[size > 0].max()) if (size > 0).any() else 0.0
    print(f"[weights] {dtype} D{dim} {'fp4 ' if in4 else ''}{lens} lq {lq}: {worst:.3f} of the bound")
    assert worst <= 1.0 and bool((x[size == 0] == 0).all())
    # Added to what is there, rows without a page or past a length left alone; the same bits again.
    start = _rand(got.shape, torch.float32, seed + 9).to(device)
    into = start.clone()
    assert ops.paged_key_weights(qd, ld, into, **kw) is into
    assert torch.equal(into, torch.where((size > 0).to(device), start + got, start))
    assert torch.equal(ops.paged_key_weights(qd, ld, **kw), got)


@pytest.mark.parametrize("dtype,dim,in4", TYPES, ids=IDS)
@pytest.mark.parametrize("lens,lq,heads,kv,rows", [([0, 1, 77, 160], 45, 2, 2, 16), ([700, 33], 1, 8, 2, 48),
                                                   ([300], 83, 3, 1, 1024), ([130, 5], 200, 2, 2, 32)])
def test_weights(device, built_lib, dtype, dim, in4, lens, lq, heads, kv, rows):
    _weights_case(device, dtype, dim, in4, lens=lens, lq=lq, heads=heads, kv=kv, rows=rows)


@pytest.mark.parametrize("in4", [False, True])
def test_weights_of_strided_inputs_and_scales(device, built_lib, in4):
    for scale in (None, -0.1, 0.0):
        _weights_case(device, torch.bfloat16, 128, in4, lens=[90, 300], lq=7, heads=4, kv=2, scale=scale,
                      strided=True)


@pytest.mark.parametrize("in4", [False, True])
def test_weights_without_pages(device, built_lib, in4):
    count, tables, _ = _tables([200, 130], 16, 3)
    tables[0][0] = tables[0][5] = -1
    tables[0][7] = count
    tables[1][1], tables[1][2] = 2 ** 31 - 1, -(2 ** 31)
    _weights_case(device, torch.bfloat16, 128, in4, lens=[200, 130], lq=9, heads=2, kv=2, seed=3, tables=tables)
    _, tables, _ = _tables([96, 96], 16, 4)
    _weights_case(device, torch.bfloat16, 64, in4, lens=[96, 0], lq=3, heads=2, kv=2, seed=4, tables=tables,
                  device_lens=[2 ** 31 - 1, -5])


def test_queries_that_saw_no_key_give_nothing(device, built_lib):
    lse = torch.zeros(1, 40, 2)
    lse[0, 3], lse[0, 30:] = -math.inf, -math.inf
    _weights_case(device, torch.bfloat16, 128, False, lens=[50], lq=40, heads=2, kv=2, lse=lse)
    q = _rand((1, 0, 2, 64), torch.bfloat16, 1).to(device)
    pages = _rand((2, 3, 16, 2, 64), torch.bfloat16, 2).to(device)
    kw = dict(pages=pages, block_table=_i32([[0, 1]], device), cache_lens=_i32([20], device))
    none = torch.empty(1, 0, 2, device=device)
    assert bool((ops.paged_key_weights(q, none, **kw) == 0).all())
    kept = torch.ones(1, 2, 32, device=device)
    assert bool((ops.paged_key_weights(q, none, kept, **kw) == 1).all())
    # No page in the pool, a table without entries, no sequences.
    q = _rand((2, 3, 2, 64), torch.bfloat16, 1).to(device)
    lse = torch.zeros(2, 3, 2, device=device)
    got = ops.paged_key_weights(q, lse, pages=pages[:, :0], block_table=_i32([[0], [1]], device),
                                cache_lens=_i32([16, 16], device))
    assert got.shape == (2, 2, 16) and bool((got == 0).all())
    got = ops.paged_key_weights(q, lse, pages=pages, cache_lens=_i32([1, 2], device),
                                block_table=torch.empty(2, 0, dtype=torch.int32, device=device))
    assert got.shape == (2, 2, 0)
    got = ops.paged_key_weights(q[:0], lse[:0], pages=pages, cache_lens=_i32([], device),
                                block_table=torch.empty(0, 2, dtype=torch.int32, device=device))
    assert got.shape == (0, 2, 32)


@pytest.mark.parametrize("in4", [False, True])
@pytest.mark.parametrize("lq", [7, 40, 100])
def test_what_gives_nothing_may_be_no_number(device, built_lib, in4, lq):
    """Queries that saw no key hold NaN and infinities: the weights are those without them."""
    lens, rows, heads, dim = [300, 64], 16, 2, 128
    count, tables, _ = _tables(lens, rows, 5)
    pages = _rand((2, count, rows, heads, dim), torch.bfloat16, 6)
    pool = (fp4.pack(*fp4.quantise(pages)) if in4 else pages).to(device)
    q = _rand((2, lq, heads, dim), torch.bfloat16, 7).to(device)
    lse = torch.full((2, lq, heads), 9.0, device=device)
    for t in {lq - 1, lq // 2, 1}:
        lse[0, t] = -math.inf
    kw = dict(pages=pool, block_table=_i32(tables, device), cache_lens=_i32(lens, device))
    want = ops.paged_key_weights(q, lse, **kw)
    bad = q.clone()
    bad[0, lq - 1], bad[0, lq // 2, 0], bad[0, 1, 1] = math.nan, math.inf, -math.inf
    assert bool(torch.isfinite(want).all()) and float(want[0, :, :300].min()) > 0
    assert torch.equal(ops.paged_key_weights(bad, lse, **kw), want)
    # An infinite key: its weight is what the queries that count give it, the last ones of a
    # tile's rows no more than others.
    if not in4:
        pool[0, tables[1][0], 0] = math.inf
        q[1] = q[1].abs()
        got = ops.paged_key_weights(q, lse, **kw)
        assert bool((got[1, :, 0] == math.inf).all())


def test_weights_sum_to_the_queries(device, built_lib):
    """With no new keys, each query's probabilities over the cached rows add up to 1."""
    lens, rows, lq, heads, kv, dim = [1000, 37], 64, 83, 4, 2, 128
    count, tables, _ = _tables(lens, rows, 1)
    pages = _rand((2, count, rows, kv, dim), torch.bfloat16, 2).to(device)
    q = _rand((2, lq, heads, dim), torch.bfloat16, 3).to(device)
    none = q[:, :0, :kv]
    kw = dict(pages=pages, block_table=_i32(tables, device), cache_lens=_i32(lens, device))
    _, lse = ops.paged_attention(q, none, none, return_lse=True, **kw)
    w = ops.paged_key_weights(q, lse, **kw).double().sum(-1)
    # Each of the 166 rows' sums is off by at most lse_bound and the weights' own (below 1e-4).
    assert float((w / (lq * heads / kv) - 1).abs().max()) < 1e-4


# ---------------------------------------------------------------------------
# Which rows to keep
# ---------------------------------------------------------------------------
def _keep_case(device, w, lens, k, recent):
    got = ops.kv_keep_rows(w.to(device), _i32(lens, device), k, recent)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), keep.keep_rows(w, lens, k, recent))


@pytest.mark.parametrize("lens,k,recent", [([0, 1, 77, 300], 1, 0), ([0, 1, 77, 300], 77, 5),
                                           ([300, 299, 50, 64], 64, 64), ([300, 2, 65, 100], 100, 500),
                                           ([300, 300, 128, 33], 299, 0), ([300, 10, 0, 7], 300, 3),
                                           ([40, 10, 0, 7], 500, 3)])
def test_kept_rows(device, built_lib, lens, k, recent):
    for seed, make in enumerate([lambda x: x.exp(), lambda x: x, lambda x: (2 * x).round(),
                                 lambda x: x * 0, lambda x: -x.abs(), lambda x: x * 1e-42]):
        _keep_case(device, make(_rand((4, 3, 300), torch.float32, seed)), lens, k, recent)


def test_kept_rows_of_special_weights(device, built_lib):
    """Infinities, NaN (the lowest, as -inf), zeros of both signs (equal)."""
    w = _rand((2, 2, 200), torch.float32, 1)
    w[:, :, ::7] = math.nan
    w[:, :, 1::11] = math.inf
    w[:, :, 2::13] = -math.inf
    w[:, 1, 3::5] = 0.0
    w[:, 1, 5::15] = -0.0
    w[0, 0, ::14] = -math.nan
    for k in (1, 10, 60, 120, 150, 170, 199):
        _keep_case(device, w, [200, 151], k, 0)
        _keep_case(device, w, [200, 151], k, 4)
    _keep_case(device, torch.full((1, 2, 100), math.nan), [100], 40, 3)


@pytest.mark.parametrize("n,k,recent", [(1024, 512, 0), (1025, 64, 1), (5000, 4999, 0), (40001, 9000, 700),
                                        (33000, 1, 0)])
def test_kept_rows_of_long_sequences(device, built_lib, n, k, recent):
    w = _rand((2, 1, n), torch.float32, n).mul(2).exp()
    _keep_case(device, w, [n, n - 1], k, recent)
    _keep_case(device, (w * 3).floor(), [n, n // 2], k, recent)  # many ties
    # Keys that share all but their lowest bits.
    _keep_case(device, 1 + torch.randint(0, 900, (2, 1, n)).float() * 2.0 ** -23, [n, n - 3], k, recent)


def test_kept_rows_of_views_and_lengths_past_the_weights(device, built_lib):
    w = _rand((3, 4, 90), torch.float32, 1)
    lens = [90, 50, 3]
    want = keep.keep_rows(w[:, 1:3, 10:80], [70, 50, 3], 20, 2)
    got = ops.kv_keep_rows(w.to(device)[:, 1:3, 10:80], _i32([2 ** 31 - 1, 50, 3], device), 20, 2)
    assert torch.equal(got.cpu(), want)
    got = ops.kv_keep_rows(w.to(device), _i32([-4, 50, 3], device), 5)
    assert torch.equal(got.cpu(), keep.keep_rows(w, [0, 50, 3], 5, 0))
    assert ops.kv_keep_rows(w.to(device), _i32(lens, device), 0).shape == (3, 4, 0)
    assert ops.kv_keep_rows(w.to(device)[:0], _i32([], device), 3).shape == (0, 4, 3)
    one = w[:1, :1].to(device).expand(2, 3, 90)  # read only, so it may be expanded
    assert torch.equal(ops.kv_keep_rows(one, _i32([90, 60], device), 7).cpu(),
                       keep.keep_rows(one.cpu(), [90, 60], 7, 0))


# ---------------------------------------------------------------------------
# Moving them
# ---------------------------------------------------------------------------
def _gather_case(device, dtype, dim, in4, *, lens, k, recent=0, heads=3, rows=16, seed=0, new=False,
                 views=False, picked=None, extra_w=0):
    pages_each = -(-k // rows)
    count, tables, order = _tables(lens, rows, seed, extra=len(lens) * pages_each if new else 0)
    to = [[order.pop() for _ in range(pages_each)] for _ in lens] if new else tables
    width = len(tables[0]) * rows + extra_w
    weights = _rand((len(lens), heads, width), torch.float32, seed + 1)
    picked = keep.keep_rows(weights, lens, k, recent) if picked is None else picked
    if in4:
        g = torch.Generator().manual_seed(seed + 2)
        pool = torch.randint(0, 256, (2, count, heads, rows * (dim // 2 + dim // 32)), generator=g,
                             dtype=torch.uint8)
        want = fp4.pack(*(keep.gather(t, tables, picked, to) for t in fp4.unpack(pool, rows, dim)))
    else:
        pool = _rand((2, count, rows, heads, dim), dtype, seed + 2)
        want = keep.gather(pool, tables, picked, to)
    got, w = pool.to(device), weights.to(device)
    if views:
        if in4:
            got = torch.cat((got, got), 2)[:, :, :heads]
        else:
            got = got.transpose(2, 3).contiguous().transpose(2, 3)
        w = torch.cat((w, w), 1)[:, :heads]
    ops.kv_page_gather(got, _i32(tables, device), picked.to(device), _i32(to, device) if new else None, w,
                       head_dim=dim if in4 else None)
    assert torch.equal(got.cpu(), want)
    assert torch.equal(w.cpu(), keep.gather_weights(weights, picked))


GATHER = [(torch.bfloat16, 128, False), (torch.float16, 64, False), (torch.float32, 72, False),
          (torch.bfloat16, 256, False), (torch.bfloat16, 8, False), (torch.uint8, 64, True),
          (torch.uint8, 128, True), (torch.uint8, 256, True)]


@pytest.mark.parametrize("dtype,dim,in4", GATHER, ids=[f"{str(t)[6:]}-{d}" for t, d, _ in GATHER])
@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("lens,k,recent", [([0, 1, 77, 300], 50, 5), ([1300, 900], 700, 0), ([40, 40], 1, 0),
                                           ([64, 48], 64, 0)])
def test_moved_rows(device, built_lib, dtype, dim, in4, new, lens, k, recent):
    _gather_case(device, dtype, dim, in4, lens=lens, k=k, recent=recent, new=new)


@pytest.mark.parametrize("in4", [False, True])
@pytest.mark.parametrize("new", [False, True])
def test_moved_rows_of_long_sequences_and_views(device, built_lib, in4, new):
    """Many steps of a workgroup, each reading what lies just behind what the last one wrote."""
    _gather_case(device, torch.uint8 if in4 else torch.bfloat16, 128, in4, lens=[5000, 4100], k=4000, new=new,
                 rows=48, heads=2, views=True, extra_w=100)
    shift = torch.arange(1, 3001, dtype=torch.int32).expand(1, 2, 3000).contiguous()
    _gather_case(device, torch.uint8 if in4 else torch.bfloat16, 64, in4, lens=[3001], k=3000, new=new, heads=2,
                 rows=64, picked=shift)


@pytest.mark.parametrize("in4", [False, True])
def test_rows_that_cannot_move(device, built_lib, in4):
    """Numbers past the table, negative ones in the middle, entries without a page."""
    picked = torch.tensor([[[3, -1, 7, 2 ** 31 - 1, 9, -7]] * 2], dtype=torch.int32)
    _gather_case(device, torch.uint8 if in4 else torch.float32, 64, in4, lens=[20], k=6, heads=2, picked=picked)
    rows, dim = 16, 64
    pool = torch.arange(2 * 4 * 1 * rows * 34 // 2, dtype=torch.int16).view(torch.uint8).view(2, 4, 1, rows * 34)
    dev = pool.to(device)
    keepers = torch.arange(32, dtype=torch.int32).view(1, 1, 32).to(device)
    ops.kv_page_gather(dev, _i32([[4, -1]], device), keepers, _i32([[0, 1]], device), head_dim=dim)
    ops.kv_page_gather(dev, _i32([[0, 1]], device), keepers, _i32([[-1, 9]], device), head_dim=dim)
    ops.kv_page_gather(dev, _i32([[0, 1]], device), keepers, head_dim=dim)  # rows where they are
    ops.kv_page_gather(dev, _i32([[0, 1]], device), keepers[..., :0], head_dim=dim)
    assert torch.equal(dev.cpu(), pool)
    w = torch.ones(1, 1, 40, device=device)
    ops.kv_page_gather(dev, _i32([[0, 1]], device), keepers[..., :0], weights=w, head_dim=dim)
    assert torch.equal(dev.cpu(), pool) and bool((w == 0).all())


def test_a_captured_eviction(device, built_lib):
    """Weights, choice and move, replayed with other contents, against eager calls."""
    rows, heads, dim, lens, k = 16, 2, 128, [200, 90], 64
    count, tables, _ = _tables(lens, rows, 1)
    table, length = _i32(tables, device), _i32(lens, device)
    pools = [torch.zeros(2, count, rows, heads, dim, dtype=torch.bfloat16, device=device) for _ in range(2)]
    ws = [torch.zeros(2, heads, len(tables[0]) * rows, device=device) for _ in range(2)]
    q = torch.zeros(2, 5, heads, dim, dtype=torch.bfloat16, device=device)
    kw = dict(block_table=table, cache_lens=length)

    def step(pool, w):
        _, lse = ops.paged_attention(q, q, q, pages=pool, return_lse=True, **kw)
        ops.paged_key_weights(q, lse, w, pages=pool, **kw)
        at = ops.kv_keep_rows(w, length, k, 8)
        ops.kv_page_gather(pool, table, at, None, w)
        return at
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pools[1], ws[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        at = step(pools[0], ws[0])
    for i in range(5):
        x = _rand(pools[0].shape, torch.bfloat16, i).to(device)
        q.copy_(_rand(q.shape, torch.bfloat16, 50 + i))
        length.copy_(torch.tensor([200 - 13 * i, 90 - 11 * i], dtype=torch.int32))
        for pool, w in zip(pools, ws):
            pool.copy_(x)
            w.fill_(0.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(step(pools[1], ws[1]), at)
        assert torch.equal(pools[0], pools[1]) and torch.equal(ws[0], ws[1])


@pytest.mark.parametrize("in4", [False, True])
def test_pools_past_4_gb(device, built_lib, in4):
    """Pages whose offsets pass 32 bits, against the same pages in a small pool."""
    rows, heads, dim, k = 128, 8, 128, 150
    row = 68 if in4 else 256
    count = (1 << 32) // (rows * heads * row) + 40
    shape = (heads, rows * row) if in4 else (rows, heads, dim)
    small = _rand((2, 3, rows, heads, dim), torch.bfloat16, 1)
    small = (fp4.pack(*fp4.quantise(small)) if in4 else small).to(device)
    large = torch.empty(2, count, *shape, dtype=small.dtype, device=device)
    at = [count - 1, 2, count - 9]
    large[:, at] = small
    q = _rand((1, 5, heads, dim), torch.bfloat16, 2).to(device)
    lse = torch.full((1, 5, heads), 4.0, device=device)
    got = []
    for pool, table in ((small, [[0, 1, 2]]), (large, [at])):
        kw = dict(block_table=_i32(table, device), cache_lens=_i32([330], device))
        w = ops.paged_key_weights(q, lse, pages=pool, **kw)
        rows_kept = ops.kv_keep_rows(w, kw["cache_lens"], k, 20)
        ops.kv_page_gather(pool, kw["block_table"], rows_kept, None, w, dim)
        got.append((w, rows_kept, pool[:, table[0]]))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert bool((got[0][0] > 0).any()) and int(got[0][1].max()) == 329


@pytest.mark.parametrize("in4", [False, True])
def test_two_streams_at_once(device, built_lib, in4):
    """Attention, weights, choice and move of two caches on streams of their own: each as alone."""
    lens, rows, heads, dim, lq = [900, 40, 600], 16, 4, 128, 50
    count, tables, _ = _tables(lens, rows, 4)
    kw = dict(block_table=_i32(tables, device), cache_lens=_i32(lens, device))
    attend = ops.paged_attention_fp4 if in4 else ops.paged_attention

    def run(q, pool):
        out, lse = attend(q, q, q, pages=pool, return_lse=True, **kw)
        w = ops.paged_key_weights(q, lse, pages=pool, **kw)
        kept = ops.kv_keep_rows(w, kw["cache_lens"], 100, 10)
        ops.kv_page_gather(pool, kw["block_table"], kept, None, w, dim)
        return out, lse, kept, w, pool
    inputs = []
    for i in range(2):
        pages = _rand((2, count, rows, heads, dim), torch.bfloat16, 10 + i)
        pool = (fp4.pack(*fp4.quantise(pages)) if in4 else pages).to(device)
        inputs.append((_rand((3, lq, heads, dim), torch.bfloat16, 20 + i).to(device), pool))
    want = [run(q, pool.clone()) for q, pool in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        pools = [pool.clone() for _, pool in inputs]
        torch.cuda.synchronize()
        got = []
        for s, (q, _), pool in zip(streams, inputs, pools):
            with torch.cuda.stream(s):
                got.append(run(q, pool))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b):
                assert torch.equal(x, y)
