"""What attention gives each cached row, and which rows a cache keeps, from their definitions:
64 bits and plain loops on the CPU.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).
"""

from __future__ import annotations

import math

import torch

from .attention import visible_end
from .paged import _rows


def log_sum_exp(q, k, pages, block_table=None, cache_lens=None, prefix_table=None, prefix_len=0,
                block_boundaries=None, softmax_scale=None, causal=False):
    """(lse ``[B, L, H]``, and per query the largest ``scale * sum |q| |k|``) of attention over
    the prefix, the cached rows and the new keys, as ``oracle.paged.paged_attention`` has them."""
    b, lq, heads, dim = q.shape
    lk, kv = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else softmax_scale
    lse = torch.full((b, lq, heads), -math.inf, dtype=torch.float64)
    scores = torch.zeros_like(lse)
    p_at, p_len = _rows(pages, prefix_table or [], prefix_len)
    for i in range(b):
        o_at, o_len = _rows(pages, block_table[i] if block_table else [],
                            cache_lens[i] if cache_lens else 0)
        history = p_len + o_len
        ends = visible_end(lq, history, block_boundaries, causal, lk) - history
        at = (p_at[0] + o_at[0], p_at[1] + o_at[1])
        for e in range(heads):
            h = e // (heads // kv)
            keys = torch.cat((pages[0, at[0], at[1], h].double(), k[i, :, h].double()))
            for t in range(lq):
                n = len(at[0]) + int(ends[t])
                if n == 0:
                    continue
                x = q[i, t, e].double()
                lse[i, t, e] = torch.logsumexp(keys[:n] @ x * scale, 0)
                scores[i, t, e] = (keys[:n].abs() @ x.abs()).max() * abs(scale)
    return lse, scores


def lse_bound(ref, dim, keys, scores):
    """Largest difference of a log-sum-exp in fp32 from ``ref``: every score off by ``(dim + 8)
    2^-24 scores`` (a sum of ``dim`` products, scaled, its maximum taken off), the
    exponentials by 2^-22 and the sum of ``keys`` of them and of the parts by ``(keys + 64)
    2^-24``, all relative to the sum; then a logarithm, a product with ln 2 and a sum of numbers
    below ``scores + ln keys``, 2^-22 of those."""
    return ((dim + 8) * scores + keys + 64) * 2.0 ** -24 + (2 + scores + math.log(keys + 1)) * 2.0 ** -22


def key_weights(q, lse, pages, block_table, cache_lens, softmax_scale=None):
    """(weights ``[B, Hkv, W * R]``, and what scales the error of another evaluation: per row
    the sum over its queries of the term times ``1 + its |q| |k|, |score| and |lse|``)."""
    b, lq, heads, dim = q.shape
    count, rows, kv = pages.shape[1:4]
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else softmax_scale
    out = torch.zeros(b, kv, len(block_table[0]) * rows if block_table else 0, dtype=torch.float64)
    size = torch.zeros_like(out)
    for i in range(b):
        for r in range(min(max(int(cache_lens[i]), 0), out.shape[2])):
            page = block_table[i][r // rows]
            if not 0 <= page < count:
                continue
            for h in range(kv):
                group = slice(h * (heads // kv), (h + 1) * (heads // kv))
                x, key = q[i, :, group].double(), pages[0, page, r % rows, h].double()
                s, l = x @ key * scale, lse[i, :, group].double()
                term = torch.where(l == -math.inf, 0.0, torch.exp(s - l))
                out[i, h, r] = term.sum()
                term = torch.where(term == 0, 0.0, term * (1 + x.abs() @ key.abs() * abs(scale) + l.abs()))
                size[i, h, r] = term.sum()
    return out, size


def weights_bound(ref, size, dim, queries):
    """Largest difference of weights in fp32 from ``ref``: a score of ``dim`` products, scaled by
    a rounded constant, less a rounded lse, ``(dim + 8) 2^-24`` of their sizes; the exponential
    2^-22 of the term; a sum of ``queries`` terms, each of at most ``log2 32 + queries / 32 + 3``
    roundings (a tree of 32, then one by one)."""
    return (dim + 8 + 4 + queries / 32 + 8) * 2.0 ** -24 * size + 2.0 ** -126


def keep_rows(weights, lens, keep, recent):
    """Row numbers ``[B, H, keep]``: ``sorted`` of Python, a row at a time."""
    b, heads, width = weights.shape
    out = torch.full((b, heads, keep), -1, dtype=torch.int32)
    for i in range(b):
        n = min(max(int(lens[i]), 0), width)
        c = min(n, keep)
        last = min(recent, c)
        for h in range(heads):
            w = [(-math.inf if x != x else x) for x in weights[i, h, :n - last].tolist()]
            best = sorted(range(n - last), key=lambda r: (-w[r], r))[:c - last]
            got = sorted(best) + list(range(n - last, n))
            out[i, h, :c] = torch.tensor(got, dtype=torch.int32)
    return out


def gather(pages, tables, rows, to):
    """A pool ``[2, P, R, H, .]`` after row ``rows[b][h][i]`` became row ``i`` of the pages ``to``."""
    after = pages.clone()
    count, per = pages.shape[1:3]

    def find(table, r):
        page = table[r // per] if 0 <= r < len(table) * per else -1
        return page if 0 <= page < count else -1
    for b in range(rows.shape[0]):
        for h in range(rows.shape[1]):
            for i, r in enumerate(rows[b, h].tolist()):
                src, dst = find(tables[b], r), find(to[b], i)
                if src >= 0 and dst >= 0:
                    after[:, dst, i % per, h] = pages[:, src, r % per, h]
    return after


def gather_weights(weights, rows):
    out = torch.zeros_like(weights)
    for b in range(rows.shape[0]):
        for h in range(rows.shape[1]):
            for i, r in enumerate(rows[b, h].tolist()[:weights.shape[2]]):
                if 0 <= r < weights.shape[2]:
                    out[b, h, i] = weights[b, h, r]
    return out
