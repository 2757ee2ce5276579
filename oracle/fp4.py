"""A cache's pages in 4 bits, from their definition, in 64 bits on the CPU.

A block of 32 elements is stored with the least scale ``2**e`` for which ``7 * 2**e`` is
at least its largest magnitude (``e`` within the type's range), each element as the code
whose value times the scale is nearest, the even code of two. A block with an infinity or
NaN has the scale byte 255 and reads as NaN.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).
"""

from __future__ import annotations

import math

import torch

SIZES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
RANGE = {torch.bfloat16: (-127, 125), torch.float16: (-23, 13)}


def quantise(x):
    """Codes (0..15, one per element) and scale bytes ``[..., D / 32]`` of ``x``, bf16 or f16."""
    lo, hi = RANGE[x.dtype]
    b = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], 0.0, b)
    top = b.abs().amax(-1)
    # The exponent by search: 2^e is exact in 64 bits over the whole range.
    powers = 2.0 ** torch.arange(lo, hi + 1, dtype=torch.float64)
    e = lo + torch.searchsorted(7 * powers, top.contiguous()).clamp(max=hi - lo)
    y = b.abs() / (2.0 ** e.double())[..., None]
    off = (y[..., None] - SIZES).abs()
    nearest = off.amin(-1, keepdim=True)
    # Of two nearest codes the even one.
    order = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7])  # even codes first
    code = torch.where(off == nearest, order, 99).argmin(-1)
    code = code + 8 * torch.signbit(b)
    code = torch.where(bad[..., None], 0, code)
    return code.flatten(-2).to(torch.uint8), torch.where(bad, 255, e + 127).to(torch.uint8)


def dequantise(codes, scales):
    """fp64 values of codes (one per element) and scale bytes."""
    x = SIZES[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0).double()
    s = torch.where(scales == 255, math.nan, 2.0 ** (scales.double() - 127))
    return (x.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def stored(x):
    """What ``x`` reads as once it was written, fp64."""
    return dequantise(*quantise(x))


def pack(codes, scales):
    """The bytes ``[2, P, H, R * (D / 2 + D / 32)]`` of codes and scales ``[2, P, R, H, .]``."""
    c = codes.transpose(2, 3)
    c = (c[..., 0::2] | c[..., 1::2] << 4).flatten(-2)
    return torch.cat((c, scales.transpose(2, 3).flatten(-2)), -1).contiguous()


def unpack(pool, rows, dim):
    """Codes and scales ``[2, P, R, H, .]`` of a pool's bytes."""
    at = rows * dim // 2
    c = pool[..., :at].unflatten(-1, (rows, dim // 2))
    c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    return c.transpose(2, 3), pool[..., at:].unflatten(-1, (rows, dim // 32)).transpose(2, 3)


def values(pool, rows, dim):
    """fp64 rows ``[2, P, R, H, D]`` of a pool's bytes."""
    return dequantise(*unpack(pool, rows, dim))
