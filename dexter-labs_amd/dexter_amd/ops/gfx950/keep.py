"""A cache that keeps the rows which attention weighs most, on gfx950 (``csrc/kv_weights.hip``,
``csrc/kv_keep.hip``).

A long episode's cache grows with every chunk. Attention's own probabilities say which
of its rows matter: summed over the queries they are a weight per row and K/V head, and
a cache that is to hold ``keep`` rows keeps the heaviest, and the last ones. Rows carry
their position in their rotated keys, so the kept ones may move together, and each head
may keep rows of its own.

Registered here (pools of 16 and 32 bits, and 4-bit ones; no counterpart in the reference):

* ``cache/key_weights``  ``(q, lse, weights, pages, block_table, cache_lens, softmax_scale)``
* ``cache/keep_rows``    ``(weights, cache_lens, keep, recent)``
* ``cache/page_gather``  ``(pages, block_table, rows, dst_table, weights)``

As in ``paged.py``, tables, lengths and row numbers are device tensors that the kernels
read when they run, and bound themselves. No workspaces, no atomics on results: the same
inputs give the same bits.
"""

from __future__ import annotations

import math

import torch

from ...registry import Priority, register
from . import _lib
from ._common import CDNA4, MATRIX_DTYPES
from .paged import (_APPEND_DTYPES, _HEAD_DIMS, FP4_HEAD_DIMS, PAGE_ROWS_MAX, PAGE_ROWS_MULTIPLE,
                    _check_i32, _check_pool, _elsewhere, _fp4_rows, _on, _rows, _table)


def _check_weights(w, shape: tuple, device: torch.device, what: str) -> tuple[int, int]:
    """(batch, head stride) of weights that the kernels change in place."""
    if not (isinstance(w, torch.Tensor) and w.dtype is torch.float32 and w.shape == shape
            and w.device == device and (shape[-1] <= 1 or w.stride(-1) == 1)):
        got = f"{w.dtype} {tuple(w.shape)} on {w.device}" if isinstance(w, torch.Tensor) else repr(w)
        raise ValueError(f"{what}: weights must be float32 {list(shape)} on {device} with contiguous "
                         f"rows, got {got}")
    sb, sh, _ = w.stride()
    if (sb == 0 and shape[0] > 1) or (sh == 0 and shape[1] > 1):
        raise ValueError(f"{what}: weights must not be expanded (a stride is 0)")
    return (0 if shape[0] == 1 else sb), (0 if shape[1] == 1 else sh)


# ---------------------------------------------------------------------------
# The weight that each cached row received
# ---------------------------------------------------------------------------
def _weights_accepts(q, lse, weights, pages, *args, **kwargs) -> bool:
    if not (q.is_cuda and q.dim() == 4):
        return False
    if pages.dtype == torch.uint8:
        return q.dtype in MATRIX_DTYPES and q.shape[-1] in FP4_HEAD_DIMS
    return pages.dtype == q.dtype and q.shape[-1] in _HEAD_DIMS.get(q.dtype, ())


@register("cache", "key_weights", name="hip_paged_key_weights_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_weights_accepts)
def paged_key_weights(q, lse, weights, pages, block_table, cache_lens, softmax_scale):
    what = "paged_key_weights"
    if q.dim() != 4:
        raise ValueError(f"{what}: q must be [B, L, H, D]")
    b, q_len, heads, dim = q.shape
    device, dtype, fp4 = q.device, q.dtype, pages.dtype is torch.uint8
    if fp4:
        if dtype not in MATRIX_DTYPES:
            raise ValueError(f"{what}: a 4-bit cache serves bf16 and f16, got {dtype}")
        rows = _fp4_rows(pages, dim, what)
        kv_heads, (_, s1, s3, _), s2 = pages.shape[2], pages.stride(), 0
    else:
        _, s1, s2, s3, _ = _check_pool(pages, what)
        rows, kv_heads = pages.shape[2], pages.shape[3]
        if pages.shape[4] != dim or pages.dtype is not dtype or dim not in _HEAD_DIMS.get(dtype, ()):
            raise ValueError(f"{what}: pages {tuple(pages.shape)} of {pages.dtype} for queries of "
                             f"{dim} x {dtype}")
        if rows % PAGE_ROWS_MULTIPLE or rows > PAGE_ROWS_MAX:
            raise ValueError(f"{what}: pages of a multiple of {PAGE_ROWS_MULTIPLE} rows up to "
                             f"{PAGE_ROWS_MAX} are taken, got {rows}")
    if heads % kv_heads:
        raise ValueError(f"{what}: {kv_heads} k/v heads do not divide {heads} query heads")
    if pages.device != device:
        raise ValueError(f"pages must be on {device}, got {pages.device}")
    if not (isinstance(lse, torch.Tensor) and lse.dtype is torch.float32
            and lse.shape == (b, q_len, heads) and lse.device == device):
        raise ValueError(f"{what}: lse must be float32 {[b, q_len, heads]} on {device}")
    t_sb, width = _table(block_table, b, device, "block_table")
    _check_i32(cache_lens, (b,), device, "cache_lens")
    shape = (b, kv_heads, width * rows)
    w_sb, w_sh = kv_heads * shape[2], shape[2]
    add = weights is not None
    if add:
        w_sb, w_sh = _check_weights(weights, shape, device, what)
    if _elsewhere(device):
        with _on(device):
            return paged_key_weights(q, lse, weights, pages, block_table, cache_lens, softmax_scale)
    if not add:
        weights = torch.empty(shape, device=device, dtype=torch.float32)
    if weights.numel() == 0 or (add and q.numel() == 0):
        return weights
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(dim)
    q, *q_at = _rows(q)
    lse = lse.contiguous()
    call = _lib.WEIGHTS_CALL.pack(
        q.data_ptr(), *q_at, lse.data_ptr(), pages.data_ptr(), s1, s2, s3, pages.shape[1], rows,
        block_table.data_ptr(), t_sb, width, cache_lens.data_ptr(), weights.data_ptr(), w_sb, w_sh,
        _lib.dtype_code(dtype), int(fp4), b, q_len, heads, kv_heads, dim, int(add), scale,
        _lib.stream_handle(device))
    rc = _lib.load().dx_paged_key_weights(call)
    if rc:
        _lib.check(rc, what)
    return weights


# ---------------------------------------------------------------------------
# Which rows to keep
# ---------------------------------------------------------------------------
def _keep_accepts(weights, *args, **kwargs) -> bool:
    return weights.is_cuda and weights.dtype == torch.float32 and weights.dim() == 3


@register("cache", "keep_rows", name="hip_kv_keep_rows_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_keep_accepts)
def kv_keep_rows(weights, cache_lens, keep, recent=0):
    what = "kv_keep_rows"
    device = weights.device
    if weights.dim() != 3:
        raise ValueError(f"{what}: weights must be [B, H, N], got {tuple(weights.shape)}")
    b, heads, width = weights.shape
    sb, sh, step = weights.stride()
    if weights.dtype is not torch.float32 or (step != 1 and width > 1):
        raise ValueError(f"{what}: weights must be float32 with contiguous rows, got {weights.dtype} "
                         f"of strides {weights.stride()}")
    _check_i32(cache_lens, (b,), device, "cache_lens")
    if keep < 0 or recent < 0:
        raise ValueError(f"{what}: cannot keep {keep} rows, {recent} of them the last")
    if _elsewhere(device):
        with _on(device):
            return kv_keep_rows(weights, cache_lens, keep, recent)
    rows = torch.empty((b, heads, keep), device=device, dtype=torch.int32)
    if rows.numel() == 0:
        return rows
    rc = _lib.load().dx_kv_keep_rows(weights.data_ptr(), sb, sh, width, cache_lens.data_ptr(), keep,
                                     min(recent, keep), rows.data_ptr(), b, heads, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, what)
    return rows


# ---------------------------------------------------------------------------
# Moving them
# ---------------------------------------------------------------------------
def _gather_accepts(pages, rows, *args, **kwargs) -> bool:
    return pages.is_cuda and rows.dtype == torch.int32 and (
        (pages.dtype == torch.uint8 and pages.dim() == 4)
        or (pages.dtype in _APPEND_DTYPES and pages.dim() == 5
            and (pages.shape[-1] * pages.element_size()) % 16 == 0))


@register("cache", "page_gather", name="hip_kv_page_gather_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_gather_accepts)
def kv_page_gather(pages, block_table, rows, dst_table=None, weights=None, head_dim=None) -> None:
    what = "kv_page_gather"
    device = pages.device
    if pages.dtype is torch.uint8:
        if head_dim is None:
            raise ValueError(f"{what}: head_dim is needed for pages in 4 bits")
        page_rows, heads, code = _fp4_rows(pages, head_dim, what), pages.shape[2], _lib.DX_FP4
        (s0, s1, s3, _), s2 = pages.stride(), 0
    else:
        s0, s1, s2, s3, _ = _check_pool(pages, what)
        page_rows, heads, dim = pages.shape[2:]
        if pages.dtype not in _APPEND_DTYPES or head_dim not in (None, dim):
            raise ValueError(f"{what}: pages {tuple(pages.shape)} of {pages.dtype} with head_dim {head_dim}")
        head_dim, code = dim, _lib.dtype_code(pages.dtype)
    if not isinstance(rows, torch.Tensor) or rows.dim() != 3:
        raise ValueError(f"{what}: rows must be int32 [B, H, keep]")
    b, _, keep = rows.shape
    _check_i32(rows, (b, heads, keep), device, "rows")
    s_sb, width = _table(block_table, b, device, "block_table")
    to = block_table if dst_table is None else dst_table
    d_sb, d_width = _table(to, b, device, "dst_table")
    w_ptr, w_sb, w_sh, w_width = None, 0, 0, 0
    if weights is not None:
        w_width = weights.shape[2] if isinstance(weights, torch.Tensor) and weights.dim() == 3 else -1
        w_sb, w_sh = _check_weights(weights, (b, heads, w_width), device, what)
        w_ptr = weights.data_ptr()
    if b == 0 or (keep == 0 and w_width == 0):
        return
    if _elsewhere(device):
        with _on(device):
            return kv_page_gather(pages, block_table, rows, dst_table, weights, head_dim)
    rows = rows.contiguous()  # (held until the launch)
    rc = _lib.load().dx_kv_page_gather(
        pages.data_ptr(), s0, s1, s2, s3, code, pages.shape[1], page_rows, block_table.data_ptr(),
        s_sb, width, to.data_ptr(), d_sb, d_width, rows.data_ptr(), keep, w_ptr, w_sb,
        w_sh, w_width, b, heads, head_dim, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, what)
