"""Attention over a cache in pages, from its definition, in 64 bits on the CPU.

Keys of sequence ``b`` are the prefix's rows, its own cached rows and its new
keys, in that order; cached row ``r`` lies at row ``r % R`` of page
``table[r // R]``, lengths are clamped to ``[0, W * R]``, and rows of a table entry
outside ``[0, P)`` are left out. The mask over the new keys is that of
``oracle.attention.visible_end``, with all cached rows (left out or not) as the
cache length. Each query is a softmax over the keys it sees; none gives NaN.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).
"""

from __future__ import annotations

import math

import torch

from .attention import visible_end


def _rows(pages, table, length):
    """Page and row numbers of the cached rows that exist, and the clamped length."""
    count, rows = pages.shape[1], pages.shape[2]
    length = min(max(int(length), 0), len(table) * rows)
    at = [(table[r // rows], r % rows) for r in range(length) if 0 <= table[r // rows] < count]
    return ([p for p, _ in at], [r for _, r in at]), length


def paged_attention(q, k, v, pages, block_table=None, cache_lens=None, prefix_table=None,
                    prefix_len=0, block_boundaries=None, softmax_scale=None, causal=False):
    """Returns (out, weight, scores): the result in fp64, per element the sum of softmax
    weight times ``|v|``, and per query the largest ``scale * sum |q| |k|``, which scale
    the error of any other evaluation."""
    b, lq, heads, dim = q.shape
    lk, kv = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else softmax_scale
    out = torch.full((b, lq, heads, dim), math.nan, dtype=torch.float64)
    weight = torch.zeros_like(out)
    scores = torch.zeros(b, lq, heads, 1, dtype=torch.float64)
    p_at, p_len = _rows(pages, prefix_table or [], prefix_len)
    for i in range(b):
        o_at, o_len = _rows(pages, block_table[i] if block_table else [],
                            cache_lens[i] if cache_lens else 0)
        history = p_len + o_len
        ends = visible_end(lq, history, block_boundaries, causal, lk) - history
        at = (p_at[0] + o_at[0], p_at[1] + o_at[1])
        for h in range(kv):
            old = pages[:, at[0], at[1], h].double()
            keys = torch.cat((old[0], k[i, :, h].double()))
            vals = torch.cat((old[1], v[i, :, h].double()))
            for e in range(h * (heads // kv), (h + 1) * (heads // kv)):
                for t in range(lq):
                    n = len(at[0]) + int(ends[t])
                    if n == 0:
                        continue
                    x = q[i, t, e].double()
                    p = torch.softmax(keys[:n] @ x * scale, 0)
                    scores[i, t, e] = (keys[:n].abs() @ x.abs()).max() * abs(scale)
                    out[i, t, e] = p @ vals[:n]
                    weight[i, t, e] = p @ vals[:n].abs()
    return out, weight, scores


def error_bound(ref, weight, dtype, dim, keys, scores, vmax):
    """Largest difference between ``ref`` and an evaluation with fp32 sums, per element.

    To first order, with u the relative rounding of ``dtype`` (eps / 2):

    * the result's rounding: ``u |ref|``;
    * 16-bit inputs: probabilities rounded to ``dtype`` before the second product, their
      sum taken of the rounded ones: ``2 u weight``;
    * each score, a sum of ``dim`` products in fp32 that is scaled and has its maximum
      taken off (``scores``: the largest ``sum |q| |k|`` times the scale, an upper bound
      of every term): ``(dim + 8) 2^-24 scores``, which a weight takes over as a
      relative error, in the numerator and in the sum;
    * the exponential (2^-22 relative) and sums over ``keys`` terms and joined parts:
      ``(keys + 64) 2^-24`` in the numerator and in the sum;
    * f16: a probability below 2^-14 is off by up to 2^-25 of the largest one, which is
      at least 2^-8 of the sum's unit: ``keys 2^-25 * 2 max |v|``.
    """
    u = torch.finfo(dtype).eps / 2
    fp32 = 2 * ((dim + 8) * scores + (keys + 64) + 4) * 2.0 ** -24
    bound = u * ref.abs() + fp32 * weight
    if dtype != torch.float32:
        bound = bound + 2 * u * weight
    if dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * 2 * vmax
    return bound * (1 + 4 * u)
