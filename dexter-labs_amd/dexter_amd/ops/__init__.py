"""Public op surface for the blockwise-causal attention path.

Each function asks the registry for the best implementation on this platform
and calls it, exactly as dexter's dispatchers do (``python/dexter/ops/__init__.py``):

* ``qk_norm_rope``               -> ``select("rope", "qk_norm_rope", q, k)``
  (reference ``ops/__init__.py:66-86``; same arguments and defaults)
* ``blockwise_causal_attention`` -> ``select("attention", "blockwise_causal", q, k, v)``
  (reference ``ops/__init__.py:127-147``; same keyword-only arguments)
* ``kv_cache_append``            -> ``select("cache", "append", cache, k, v)``
  (no dispatcher in the reference: ``KVCache.append`` does two torch slice
  copies, ``models/dreamzero/model.py:53-58``; here it is a kernel too)
* ``qkv_norm_rope``              -> ``select("rope", "qkv_norm_rope", x, wq, ...)``
  (no dispatcher in the reference: ``SelfAttention.forward`` runs three
  ``nn.Linear`` and ``ops.qk_norm_rope``, ``models/dreamzero/model.py:162-175``;
  here one call for decode chunks)
* ``linear_chunk``               -> ``select("gemm", "linear_chunk", x, weight, bias)``
  (no dispatcher in the reference: ``SelfAttention.forward``'s output projection
  is an ``nn.Linear``, ``models/dreamzero/model.py:183``; here one kernel for
  decode chunks)
* ``qk_norm_rope_attention``     -> ``select("attention", "qk_norm_rope_blockwise_causal", q, k, v)``
  (no dispatcher in the reference: ``SelfAttention.forward`` calls
  ``ops.qk_norm_rope``, ``KVCache.append`` and ``ops.blockwise_causal_attention``,
  ``models/dreamzero/model.py:166-182``; here one call)
* ``adaln_modulate``             -> ``select("norm", "adaln", x, scale, shift)``
  (reference ``ops/__init__.py:39-49``; same arguments and default eps)
* ``gated_residual``             -> ``select("norm", "gated_residual", x, y, gate)``
  (reference ``ops/__init__.py:52-54``)
* ``kv_page_append``             -> ``select("cache", "page_append", pages, k, v)``,
  ``kv_page_copy``               -> ``select("cache", "page_copy", pools)``,
  ``paged_attention``            -> ``select("attention", "paged", q, k, v)``,
  ``shared_prefix_attention``    -> ``select("attention", "shared_prefix", q, k, v)``
  (no counterpart in the reference, whose cache is one contiguous history per
  sequence, ``models/dreamzero/model.py:35-65``: a cache in pages that
  sequences can share, and attention over it)
* ``kv_page_append_fp4``         -> ``select("cache", "page_append_fp4", pages, k, v)``,
  ``kv_page_read_fp4``           -> ``select("cache", "page_read_fp4", pages, ...)``,
  ``paged_attention_fp4``        -> ``select("attention", "paged_fp4", q, k, v)``,
  ``shared_prefix_attention_fp4`` -> ``select("attention", "shared_prefix_fp4", q, k, v)``
  (no counterpart: the same cache with its rows in 4 bits)
* ``paged_key_weights``          -> ``select("cache", "key_weights", q, lse, weights, pages)``,
  ``kv_keep_rows``               -> ``select("cache", "keep_rows", weights)``,
  ``kv_page_gather``             -> ``select("cache", "page_gather", pages, rows)``
  (no counterpart: a cache that keeps the rows which attention weighs most)

Importing this module registers the gfx950 HIP kernels. Nothing else is
registered, so on a machine without an MI355X every call raises
``LookupError`` rather than running a slower stand-in.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from ..registry import select

__all__ = ["qk_norm_rope", "blockwise_causal_attention", "kv_cache_append",
           "qk_norm_rope_append", "blockwise_causal_attention_varlen",
           "adaln_modulate", "gated_residual", "qkv_norm_rope", "qk_norm_rope_attention",
           "linear_chunk", "kv_page_append", "kv_page_copy", "paged_attention",
           "shared_prefix_attention", "kv_page_append_fp4", "kv_page_read_fp4",
           "paged_attention_fp4", "shared_prefix_attention_fp4", "paged_key_weights",
           "kv_keep_rows", "kv_page_gather"]


def qkv_norm_rope(
    x: torch.Tensor,
    wq: torch.Tensor, bq: torch.Tensor | None,
    wk: torch.Tensor, bk: torch.Tensor | None,
    wv: torch.Tensor, bv: torch.Tensor | None,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    heads: int,
    eps: float = 1e-6,
    interleaved: bool = True,
    cache: torch.Tensor | None = None,
    start: int | torch.Tensor = 0,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The q/k/v projections of a ``[B, L, C]`` chunk, QK-norm + rotary, and the cache write.

    Equals ``q, k, v = F.linear(x, wq, bq), F.linear(x, wk, bk), F.linear(x, wv, bv)``
    viewed as ``[B, L, heads, D]``, then ``qk_norm_rope(q, k, ...)``, and, with a
    ``cache``, ``kv_cache_append(cache, k_rotated, v, start, status)``. Returns the
    rotated ``q``, ``k`` and the projected ``v``.
    """
    return select("rope", "qkv_norm_rope", x, wq, bq, wk, bk, wv, bv, q_weight, k_weight, cos,
                  sin, heads)(x, wq, bq, wk, bk, wv, bv, q_weight, k_weight, cos, sin, heads,
                              eps, interleaved, cache, start, status)


def linear_chunk(x: torch.Tensor, weight: torch.Tensor,
                 bias: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` of a ``[B, L, C]`` decode chunk (at most 128 tokens,
    ``C`` a multiple of 512, out features of 16), bf16 or f16, rounded once."""
    return select("gemm", "linear_chunk", x, weight, bias)(x, weight, bias)


def adaln_modulate(
    x: torch.Tensor,
    scale: torch.Tensor,
    shift: torch.Tensor,
    eps: float = 1e-6,
) -> torch.Tensor:
    """Modulated LayerNorm of the DiT block: normalise each ``C``-row of ``x`` (no
    affine), multiply by ``1 + scale`` and add ``shift``; one kernel, one read of ``x``.

    ``x`` is ``[B, L, C]``. ``scale`` and ``shift`` broadcast against it: per row
    (``[B, L, C]``), per batch (``[B, 1, C]``, the Wan block's modulation) or one
    row for all (``[C]``). The result has torch's promoted dtype.
    """
    return select("norm", "adaln", x, scale, shift)(x, scale, shift, eps)


def gated_residual(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor) -> torch.Tensor:
    """Residual add with a gate, ``x + y * gate``: the attention or FFN branch ``y``
    scaled by its per-channel gate and added to the stream ``x`` in one pass
    (``gate`` broadcasts like ``adaln_modulate``'s modulation)."""
    return select("norm", "gated_residual", x, y, gate)(x, y, gate)


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    eps: float = 1e-6,
    interleaved: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm over the whole ``H*D`` plane of each token, then rotary, for q and k.

    ``q``/``k`` are ``[B, L, H, D]``; the weights are ``[H*D]``; ``cos``/``sin``
    are ``[L, D//2]``. ``interleaved`` pairs ``(2j, 2j+1)`` (Wan); otherwise
    ``(j, j + D/2)``. Returns new ``(q, k)`` tensors of the input dtype.
    """
    return select("rope", "qk_norm_rope", q, k)(
        q, k, q_weight, k_weight, cos, sin, eps, interleaved)


def blockwise_causal_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    kv_cache: torch.Tensor | None = None,
    cache_len: int | torch.Tensor = 0,
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
) -> torch.Tensor:
    """Softmax attention of ``q`` over ``[cache[:cache_len] | k]`` with block causality.

    A query in the block starting at ``block_boundaries[i]`` sees the whole
    cached history and every current key before the end of its own block.
    ``None`` is one block (all current keys visible); ``causal=True`` is
    token-causal on the current keys. ``kv_cache`` is ``[2, B, S, H, D]``;
    rows ``[0, cache_len)`` are read in place, never copied. ``cache_len`` may
    be a device cursor (a one-element int32 tensor) that the kernels read when
    they run, so a captured graph follows a growing cache. ``k``/``v`` of
    another length than ``q`` (no mask) is cross-attention; ``k``/``v`` with
    fewer heads is grouped-query attention.
    """
    return select("attention", "blockwise_causal", q, k, v)(
        q, k, v, kv_cache, cache_len, block_boundaries, softmax_scale, causal)


def qk_norm_rope_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    kv_cache: torch.Tensor | None = None,
    cache_len: int = 0,
    append: bool = False,
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
    eps: float = 1e-6,
    interleaved: bool = True,
    return_qk: bool = False,
):
    """``qk_norm_rope``, the cache write of the rotated k and v (``append``), and
    ``blockwise_causal_attention``, as ``SelfAttention.forward`` chains them.

    Same results as ``qr, kr = qk_norm_rope(q, k, q_weight, k_weight, cos, sin, eps,
    interleaved)``, then (with ``append``) ``kv_cache_append(kv_cache, kr, v, cache_len)``,
    then ``blockwise_causal_attention(qr, kr, v, kv_cache=kv_cache, cache_len=cache_len,
    ...)``. Returns the attention output, and with ``return_qk`` also ``qr`` and ``kr``.
    ``cache_len`` is the row count before the append (the model reads it first).
    """
    out, qr, kr = select("attention", "qk_norm_rope_blockwise_causal", q, k, v)(
        q, k, v, q_weight, k_weight, cos, sin, kv_cache, cache_len, append, block_boundaries,
        softmax_scale, causal, eps, interleaved)
    return (out, qr, kr) if return_qk else out


def blockwise_causal_attention_varlen(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    kv_cache: torch.Tensor,
    cache_lens: list[int],
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
) -> torch.Tensor:
    """``blockwise_causal_attention`` over a ragged batch in one launch.

    Sequence ``b`` attends to ``kv_cache[:, b, :cache_lens[b]]`` followed by
    its own ``k``/``v`` rows; results equal one ``blockwise_causal_attention``
    call per sequence with ``cache_len=cache_lens[b]``. (The reference takes a
    scalar ``cache_len`` only, so a ragged batch there is a loop of calls.)
    """
    return select("attention", "blockwise_causal_varlen", q, k, v)(
        q, k, v, kv_cache, cache_lens, block_boundaries, softmax_scale, causal)


def kv_cache_append(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    start: int | torch.Tensor, status: torch.Tensor | None = None) -> None:
    """Write ``k``/``v`` ``[B, n, H, D]`` into rows ``[start, start+n)`` of both planes
    of ``cache`` ``[2, B, S, H, D]``. Raises ``RuntimeError("KV cache full ...")``
    when ``start + n > S``, before anything is launched.

    ``start`` may be a device cursor (a one-element int32 tensor), read by the
    kernel when it runs; a block that would not fit is then skipped and
    ``status`` (an int32 tensor, optional) set to 1.
    """
    return select("cache", "append", cache, k, v)(cache, k, v, start, status)


def qk_norm_rope_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    cache: torch.Tensor,
    start: int | torch.Tensor,
    eps: float = 1e-6,
    interleaved: bool = True,
    status: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``qk_norm_rope`` and ``kv_cache_append`` of the rotated k and raw v, in one pass.

    Same results as ``q, k = qk_norm_rope(...)`` followed by
    ``kv_cache_append(cache, k, v, start, status)``; ``start`` may be a device cursor.
    """
    return select("rope", "qk_norm_rope_append", q, k, v, cache)(
        q, k, v, q_weight, k_weight, cos, sin, cache, start, eps, interleaved, status)


def kv_page_append(pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   block_table: torch.Tensor, starts: torch.Tensor,
                   status: torch.Tensor | None = None) -> None:
    """Write ``k``/``v`` ``[B, n, H, D]`` into the batch's pages: row ``starts[b] + t``
    of sequence ``b`` is row ``r % R`` of page ``block_table[b, r // R]`` of ``pages``
    ``[2, P, R, H, D]``.

    ``block_table`` ``[B, W]`` and ``starts`` ``[B]`` are int32 on the device, read by
    the kernel when it runs. A row without a page (past the table, a start below 0, an
    entry outside ``[0, P)``) is not written, and ``status`` (one int32, optional) set
    to 1. Sequences that write the same row of a page in one call leave a mix of theirs.
    """
    return select("cache", "page_append", pages, k, v)(pages, k, v, block_table, starts, status)


def kv_page_copy(pages: torch.Tensor | Sequence[torch.Tensor], src: Sequence[int],
                 dst: Sequence[int]) -> None:
    """``pages[:, dst[i]] = pages[:, src[i]]`` for every ``i``: what a fork (the partly
    filled last page) and compaction need. ``pages`` is a pool ``[2, P, R, H, D]`` or one
    per layer, all of one shape, copied in one launch (of up to 64 pools and 256 pages).

    ``src`` and ``dst`` are host page numbers. A page may be a source several times;
    ``ValueError`` when one is written twice, or both read and written.
    """
    pools = [pages] if isinstance(pages, torch.Tensor) else list(pages)
    return select("cache", "page_copy", pools)(pools, src, dst)


def paged_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    pages: torch.Tensor,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``blockwise_causal_attention`` with each sequence's cached rows in pages.

    Sequence ``b`` attends to rows ``[0, cache_lens[b])`` of its pages (``block_table``
    ``[B, W]``, ``pages`` ``[2, P, R, Hkv, D]``), then to its own ``k``/``v``, under the
    same masks. ``k``/``v`` may be empty (keys all cached) or of another length than
    ``q`` (no mask), and have fewer heads (grouped-query). ``block_table`` and
    ``cache_lens`` ``[B]`` are int32 on the device, read by the kernels when they run:
    lengths are clamped to ``[0, W * R]``, keys of an entry outside ``[0, P)`` are not
    seen (a sequence may drop pages of its history), and a graph captured once follows
    both. A narrower ``block_table[:, :w]`` plans the launch for fewer rows. A query
    that sees no key gives NaN, as in ``blockwise_causal_attention``.

    With ``return_lse`` also each query's log-sum-exp, fp32 ``[B, L, H]``: ``ln`` of the
    sum of ``exp(softmax_scale * q.k)`` over the keys it sees, ``-inf`` where it sees none
    (``paged_key_weights`` takes it). The result is the same, bit for bit.
    """
    impl = select("attention", "paged", q, k, v)
    more = {"return_lse": True} if return_lse else {}
    return impl(q, k, v, pages, block_table, cache_lens, block_boundaries, softmax_scale, causal,
                **more)


def shared_prefix_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    pages: torch.Tensor,
    prefix_table: torch.Tensor,
    prefix_len: torch.Tensor,
    block_table: torch.Tensor | None = None,
    cache_lens: torch.Tensor | None = None,
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``paged_attention`` for a batch that shares a prefix, computed once for all.

    Every sequence attends to rows ``[0, prefix_len)`` of the pages ``prefix_table``
    ``[Wp]`` (both int32 on the device; ``prefix_len`` one element), then to its own
    cached rows (``block_table`` and ``cache_lens``, optional) and its ``k``/``v``. The
    result is that of ``paged_attention`` with the prefix's pages in front of each
    sequence's own (when the prefix fills its pages), but its keys and values are read
    once for all queries of the batch instead of once per sequence.
    """
    impl = select("attention", "shared_prefix", q, k, v)
    more = {"return_lse": True} if return_lse else {}
    return impl(q, k, v, pages, prefix_table, prefix_len, block_table, cache_lens, block_boundaries,
                softmax_scale, causal, **more)


def kv_page_append_fp4(pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                       block_table: torch.Tensor, starts: torch.Tensor,
                       status: torch.Tensor | None = None) -> None:
    """``kv_page_append`` into pages in 4 bits, ``pages`` uint8 ``[2, P, H, R * (D/2 + D/32)]``.

    Of each page and head first ``R`` rows of ``D/2`` code bytes (element ``2 i`` in the low
    half of byte ``i``), then ``R`` rows of ``D/32`` scale bytes. A code is a sign and one of
    0, 0.5, 1, 1.5, 2, 3, 4, 6; 32 elements share a scale ``2**(byte - 127)``, ``2**e`` for the
    least ``e`` with all of them within ``7 * 2**e`` (``-127 <= e <= 125`` for bf16, ``-23 <=
    e <= 13`` for f16), and are rounded to the nearest code, ties to even. A block that holds
    an infinity or NaN reads as NaN (scale byte 255). ``k`` and ``v`` are bf16 or f16 with a
    head dim of 64, 128 or 256; ``R`` is a multiple of 16 up to 1024. Rows without a page and
    ``status`` as in ``kv_page_append``.
    """
    return select("cache", "page_append_fp4", pages, k, v)(pages, k, v, block_table, starts, status)


def kv_page_read_fp4(pages: torch.Tensor, block_table: torch.Tensor, starts: torch.Tensor, n: int,
                     head_dim: int, dtype: torch.dtype = torch.bfloat16,
                     status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows ``[starts[b], starts[b] + n)`` of pages in 4 bits as new ``k``, ``v`` ``[B, n, H, D]``
    of ``dtype`` (bf16 or f16; exact where it is the type that the rows were written from).

    A row without a page becomes zeros, and ``status`` (one int32, optional) 1.
    """
    return select("cache", "page_read_fp4", pages, block_table, starts, n, head_dim, dtype)(
        pages, block_table, starts, n, head_dim, dtype, status)


def paged_attention_fp4(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    pages: torch.Tensor,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``paged_attention`` with the cached rows in 4 bits (``pages`` as ``kv_page_append_fp4``
    has them); ``q`` and the chunk's own ``k``/``v`` are bf16 or f16. The cached values are
    exact in that type: what they lost they lost when they were written."""
    return select("attention", "paged_fp4", q, k, v)(
        q, k, v, pages, block_table, cache_lens, block_boundaries, softmax_scale, causal, return_lse)


def shared_prefix_attention_fp4(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    pages: torch.Tensor,
    prefix_table: torch.Tensor,
    prefix_len: torch.Tensor,
    block_table: torch.Tensor | None = None,
    cache_lens: torch.Tensor | None = None,
    block_boundaries: torch.Tensor | None = None,
    softmax_scale: float | None = None,
    causal: bool = False,
    return_lse: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``shared_prefix_attention`` with the prefix and the cached rows in 4 bits."""
    return select("attention", "shared_prefix_fp4", q, k, v)(
        q, k, v, pages, prefix_table, prefix_len, block_table, cache_lens, block_boundaries,
        softmax_scale, causal, return_lse)


def paged_key_weights(
    q: torch.Tensor,
    lse: torch.Tensor,
    weights: torch.Tensor | None = None,
    *,
    pages: torch.Tensor,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """The softmax weight that each cached row received from ``q`` ``[B, L, H, D]``, with the
    ``lse`` ``[B, L, H]`` that attention returned for it: ``[B, Hkv, W * R]``, fp32, summed over
    the queries and the query heads of a K/V head.

    Row ``r`` of sequence ``b`` gets the sum of ``exp(softmax_scale * q.k_r - lse)``. Rows past
    ``cache_lens[b]`` and rows without a page get 0. ``weights``, when given, is added to in
    place and returned (such rows keep what they have): over the steps of an episode it
    accumulates. A query whose ``lse`` is ``-inf`` gives nothing. ``pages`` are a pool of q's
    type (16 bits, or fp32) or one in 4 bits. Every bit is the same from call to call.
    """
    return select("cache", "key_weights", q, lse, weights, pages)(
        q, lse, weights, pages, block_table, cache_lens, softmax_scale)


def kv_keep_rows(weights: torch.Tensor, cache_lens: torch.Tensor, keep: int,
                 recent: int = 0) -> torch.Tensor:
    """Which rows to keep, by the ``weights`` ``[B, H, N]`` that they received: int32 row numbers
    ``[B, H, keep]``, ascending, then -1.

    Of the ``n = min(cache_lens[b], N)`` rows of sequence ``b``, ``c = min(n, keep)``: the last
    ``min(recent, c)`` and those with the largest weights before them; of equal ones the
    lowest, and NaN counts as ``-inf``. It knows no table: where a sequence has dropped pages,
    give their rows a weight of ``-inf``, and keep no more rows than the others are and no
    ``recent`` ones among them. A row that is kept without a page cannot move.
    """
    return select("cache", "keep_rows", weights)(weights, cache_lens, keep, recent)


def kv_page_gather(pages: torch.Tensor, block_table: torch.Tensor, rows: torch.Tensor,
                   dst_table: torch.Tensor | None = None, weights: torch.Tensor | None = None,
                   head_dim: int | None = None) -> None:
    """Row ``rows[b, h, i]`` of head ``h`` of sequence ``b``'s pages becomes row ``i`` of the pages
    ``dst_table`` names (default: ``block_table``'s own, in place), in both planes; ``weights``
    ``[B, H, N]`` move with their rows and are 0 behind them.

    ``rows`` is what ``kv_keep_rows`` returned. For a move in place, and wherever ``weights`` are
    given (theirs is always in place), it has to be ascending with ``rows[b, h, i] >= i``. Entries
    below 0, past a table or without a page move nothing (what stood in row ``i``'s place stays
    there), nor does a row that is where it belongs. A page that rows move into must not be another sequence's, nor
    one that the call reads, but for the page that both tables name at the same place of one
    sequence. ``head_dim`` is needed for pages in 4 bits.
    """
    return select("cache", "page_gather", pages, rows)(pages, block_table, rows, dst_table, weights,
                                                       head_dim)


# Importing the implementation package is what populates the registry.
from . import gfx950  # noqa: E402,F401
