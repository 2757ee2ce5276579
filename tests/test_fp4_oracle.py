"""The 4-bit oracle against brute force over every code and every scale (no GPU)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import fp4


def _nearest(x, lo, hi):
    """One block by trying every scale and every code, in Python floats."""
    sizes = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    top = max(abs(v) for v in x)
    e = next((e for e in range(lo, hi + 1) if 7 * 2.0 ** e >= top), hi)
    out = []
    for v in x:
        d = [abs(abs(v) - s * 2.0 ** e) for s in sizes]
        best = [i for i in range(8) if d[i] == min(d)]
        i = best[0] if len(best) == 1 else next(i for i in best if i % 2 == 0)
        out.append(math.copysign(sizes[i] * 2.0 ** e, v))
    return e, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_blocks_against_every_code(dtype):
    g = torch.Generator().manual_seed(3)
    lo, hi = fp4.RANGE[dtype]
    x = torch.randn(40, 32, generator=g)
    x[:20] *= torch.exp2(torch.randint(-30, 20, (20, 1), generator=g).float())
    x[20:30] = torch.randint(-28, 29, (10, 32), generator=g) / 4  # ties, and 7 itself
    x[30] = 0
    x[31] = torch.finfo(dtype).max
    x[32] = torch.finfo(dtype).tiny / 8
    x[33, 1:] = 0
    x = x.to(dtype)
    codes, scales = fp4.quantise(x)
    got = fp4.dequantise(codes, scales)
    for row, e, back in zip(x.double().tolist(), scales[:, 0].tolist(), got.tolist()):
        want_e, want = _nearest(row, lo, hi)
        assert e == want_e + 127 and back == want
        assert np.array_equal(np.signbit(back), np.signbit(row))
    assert torch.equal(got.to(dtype).double(), got)  # the type holds every stored value


def test_a_block_that_holds_no_number_reads_as_nan():
    x = torch.ones(3, 64, dtype=torch.float16)
    x[0, 5], x[1, 40], x[2, 63] = math.inf, math.nan, -math.inf
    got = fp4.stored(x)
    assert torch.equal(torch.isnan(got).view(3, 2, 32).all(-1),
                       torch.tensor([[True, False], [False, True], [False, True]]))
    assert bool((got[~torch.isnan(got)] == 1).all())


def test_the_bytes_of_a_pool():
    g = torch.Generator().manual_seed(4)
    codes = torch.randint(0, 16, (2, 3, 16, 2, 64), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 140, (2, 3, 16, 2, 2), generator=g, dtype=torch.uint8)
    pool = fp4.pack(codes, scales)
    assert pool.shape == (2, 3, 2, 16 * 34)
    # Element 2 i in the low half of byte i; scales behind all codes.
    assert int(pool[1, 2, 0, 5 * 32 + 7]) == int(codes[1, 2, 5, 0, 14]) + 16 * int(codes[1, 2, 5, 0, 15])
    assert int(pool[0, 1, 1, 16 * 32 + 9 * 2 + 1]) == int(scales[0, 1, 9, 1, 1])
    back = fp4.unpack(pool, 16, 64)
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)
    x = torch.tensor([0x7, 0xf, 0x1, 0x9], dtype=torch.uint8).repeat(8)
    assert fp4.dequantise(x, torch.tensor([128], dtype=torch.uint8))[:4].tolist() == [12, -12, 1, -1]
