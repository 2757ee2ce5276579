"""What a row's weights are divided by (MI355X): the sum of the probabilities as they enter the
product, with a log-sum-exp or without, over pages of 16 bits and of 4.

A product over rounded probabilities that is divided by the sum of unrounded ones gives weights
that do not add up to 1: where one key carries a row, its result is off by that key's rounding.
"""

from __future__ import annotations

import pytest
import torch

import dexter_amd.ops as ops
from oracle import fp4, keep
from test_gpu_paged import IDS, TYPES, _i32, _rand, _tables

pytestmark = pytest.mark.gpu
HALVES = [(t, i) for t, i in zip(TYPES, IDS) if t[0] != torch.float32]


@pytest.mark.parametrize("dtype,dim", TYPES, ids=IDS)
@pytest.mark.parametrize("lens,lq,heads,kv,prefix_len,kw", [
    ([0, 1, 77, 700], 45, 2, 2, 0, {"causal": True}), ([300, 33, 0], 1, 8, 2, 0, {}),
    ([3000], 83, 1, 1, 0, {}), ([5, 0, 77], 1, 8, 2, 333, {}), ([0, 33], 45, 2, 2, 100, {"bb": [20, 33]}),
    ([40, 90], 9, 2, 2, 700, {"causal": True})])
def test_a_log_sum_exp_leaves_the_result_alone(device, built_lib, dtype, dim, lens, lq, heads, kv,
                                               prefix_len, kw):
    rows = 16
    count, tables, prefix = _tables(lens, rows, 1, prefix_rows=prefix_len)
    q = _rand((len(lens), lq, heads, dim), dtype, 2).to(device)
    k, v = (_rand((len(lens), lq, kv, dim), dtype, s).to(device) for s in (3, 4))
    args = dict(pages=_rand((2, count, rows, kv, dim), dtype, 5).to(device), block_table=_i32(tables, device),
                cache_lens=_i32(lens, device), causal=kw.get("causal", False),
                block_boundaries=torch.tensor(kw["bb"]).to(device) if "bb" in kw else None)
    call = ops.paged_attention
    if prefix_len:
        call = ops.shared_prefix_attention
        args.update(prefix_table=_i32(prefix, device), prefix_len=_i32([prefix_len], device))
    for scale in (None, 0.9):
        plain = call(q, k, v, softmax_scale=scale, **args)
        out, _ = call(q, k, v, softmax_scale=scale, return_lse=True, **args)
        assert torch.equal(torch.nan_to_num(out, nan=3.0), torch.nan_to_num(plain, nan=3.0))


def _half_ulp(x, dtype):
    return 2.0 ** torch.floor(torch.log2(x.abs())) * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype,dim", [t for t, _ in HALVES], ids=[i for _, i in HALVES])
@pytest.mark.parametrize("in4", [False, True])
@pytest.mark.parametrize("lq,prefix", [(9, False), (45, False), (45, True)])
def test_one_key_that_carries_a_row(device, built_lib, dtype, dim, in4, lq, prefix):
    """Of 256 rows one, in the last tile, carries 0.85 to 0.97 of the weight; one in every 32 shares
    the rest, and the others have next to none. Only the heavy row has values: the result is
    w v, with w = p / (p + 8 + ...) and p = e^q0. An early tile's maximum is the reference, so that
    p, and p alone, is a number that its rounding to 16 bits (u at most, half of the type's
    eps, relative) changes: w is off by u (1 - w) <= 0.15 u where the weights add up to 1, and by
    u where they do not. Besides this the result's own rounding (half a step of it) and fp32's
    roundings, 2^-18 with room."""
    b, heads, n, rows = 4, 2, 256, 16
    g = torch.Generator().manual_seed(dim + lq)
    q0 = (3.85 + 1.6 * torch.rand(b, lq, heads, generator=g)).to(dtype)
    q = torch.zeros(b, lq, heads, dim, dtype=dtype)
    q[..., 0] = q0
    count = n // rows if prefix else b * n // rows
    pages = torch.zeros(2, count, rows, heads, dim, dtype=dtype)
    order = torch.randperm(count, generator=g).tolist()
    tables = [order] if prefix else [order[i * n // rows:(i + 1) * n // rows] for i in range(b)]
    # Values that 4 bits hold: of a block at most 6 times its scale, among 3, 4 and 6.
    heavy = torch.tensor([3.0, 4.0, 6.0])[torch.randint(0, 3, (len(tables), heads, dim), generator=g)]
    heavy = heavy * torch.where(torch.rand(heavy.shape, generator=g) < 0.5, -1.0, 1.0)
    heavy[..., ::32] = 6.0
    for i, table in enumerate(tables):
        for r in range(n):
            pages[0, table[r // rows], r % rows, :, 0] = 2.0 if r == 250 else 1.0 if r % 32 == 5 else -6.0
        pages[1, table[250 // rows], 250 % rows] = heavy[i].to(dtype)
    assert torch.equal(fp4.stored(pages), pages.double())
    pool = (fp4.pack(*fp4.quantise(pages)) if in4 else pages).to(device)
    kw = dict(pages=pool, softmax_scale=1.0)
    none = q[:, :0].to(device)
    if prefix:
        call = ops.shared_prefix_attention_fp4 if in4 else ops.shared_prefix_attention
        kw.update(prefix_table=_i32(order, device), prefix_len=_i32([n], device))
    else:
        call = ops.paged_attention_fp4 if in4 else ops.paged_attention
        kw.update(block_table=_i32(tables, device), cache_lens=_i32([n] * b, device))
    out, lse = call(q.to(device), none, none, return_lse=True, **kw)
    plain = call(q.to(device), none, none, **kw)
    x = q0.double()
    total = torch.exp(2 * x) + 8 * torch.exp(x) + 247 * torch.exp(-6 * x)
    w = torch.exp(2 * x) / total
    assert 0.84 < float(w.min()) and float(w.max()) < 0.97
    want = w[..., None] * (heavy if prefix else heavy[:, None]).double()
    u = torch.finfo(dtype).eps / 2
    allowed = _half_ulp(want, dtype) + want.abs() * (0.16 * u + 2.0 ** -18)
    for name, got in (("with a log-sum-exp", out), ("without", plain)):
        worst = float(((got.double().cpu() - want).abs() / allowed).max())
        print(f"[sums] {dtype} D{dim} lq {lq} {'4 bits ' if in4 else ''}{name}: {worst:.3f} of what is allowed")
        assert worst <= 1.0, name
    ref = torch.log(total)
    off = (lse.double().cpu() - ref).abs() / keep.lse_bound(ref, dim, n, 6 * x)
    assert float(off.max()) <= 1.0
