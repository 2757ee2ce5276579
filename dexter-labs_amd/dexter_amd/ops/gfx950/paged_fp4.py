"""A KV cache's pages in 4 bits on gfx950: writing, reading back, and attention over them.

The format (``csrc/kv_fp4.h``): E2M1 codes, 32 to a power-of-two scale, so that a row of
a head takes ``D / 2 + D / 32`` bytes (68 at D 128, where 16 bits take 256). It is the
one that this hardware converts by itself, exactly: attention reads the rows as the
values that were stored and rounds nothing more. What storing rounds is the user's
choice (of normal data 11.2% of its norm).

A pool is uint8 ``[2, P, H, R * (D / 2 + D / 32)]``; pages, tables and lengths are those
of ``paged.py``, whose checks these operators share. No counterpart in the reference.

Registered here:

* ``cache/page_append_fp4``  ``(pages, k, v, block_table, starts, status)``
* ``cache/page_read_fp4``    ``(pages, block_table, starts, n, head_dim, dtype, status)``
* ``attention/paged_fp4``, ``attention/shared_prefix_fp4``
"""

from __future__ import annotations

import torch

from ...registry import Priority, register
from . import _lib
from ._common import CDNA4, MATRIX_DTYPES
from .paged import (FP4_HEAD_DIMS, _attend, _check_i32, _elsewhere, _fp4_rows, _on, _rows, _table)


def _append_accepts(pages, k, v, *args, **kwargs) -> bool:
    return (pages.is_cuda and pages.dtype == torch.uint8 and k.dtype in MATRIX_DTYPES
            and v.dtype == k.dtype and k.dim() == 4 and k.shape == v.shape
            and k.shape[-1] in FP4_HEAD_DIMS)


@register("cache", "page_append_fp4", name="hip_kv_page_append_fp4_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_append_accepts)
def kv_page_append_fp4(pages, k, v, block_table, starts, status=None) -> None:
    what = "kv_page_append_fp4"
    if k.shape != v.shape or k.dim() != 4:
        raise ValueError("k and v must both be [B, n, H, D]")
    b, n, heads, dim = k.shape
    device = pages.device
    rows = _fp4_rows(pages, dim, what)
    if k.dtype not in MATRIX_DTYPES or v.dtype is not k.dtype:
        raise ValueError(f"{what}: k and v must both be bf16 or f16, got {k.dtype} and {v.dtype}")
    if pages.shape[2] != heads:
        raise ValueError(f"{what}: pages of {pages.shape[2]} heads for {heads}")
    if k.device != device or v.device != device:
        raise ValueError(f"k and v must be on {device}, got {k.device} and {v.device}")
    t_sb, width = _table(block_table, b, device, "block_table")
    _check_i32(starts, (b,), device, "starts")
    if status is not None:
        _check_i32(status, (1,), device, "status")
    if b == 0 or n == 0:
        return
    if _elsewhere(device):
        with _on(device):
            return kv_page_append_fp4(pages, k, v, block_table, starts, status)
    k, k_sb, k_sl, k_sh = _rows(k)
    v, v_sb, v_sl, v_sh = _rows(v)
    s0, s1, s2, _ = pages.stride()
    rc = _lib.load().dx_kv_page_append_fp4(
        k.data_ptr(), k_sb, k_sl, k_sh, v.data_ptr(), v_sb, v_sl, v_sh, pages.data_ptr(), s0, s1,
        s2, _lib.dtype_code(k.dtype), pages.shape[1], rows, block_table.data_ptr(), t_sb, width,
        starts.data_ptr(), _lib.ptr(status), b, n, heads, dim, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, what)


def _read_accepts(pages, block_table, starts, n, head_dim, dtype, *args, **kwargs) -> bool:
    return (pages.is_cuda and pages.dtype == torch.uint8 and dtype in MATRIX_DTYPES
            and head_dim in FP4_HEAD_DIMS)


@register("cache", "page_read_fp4", name="hip_kv_page_read_fp4_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_read_accepts)
def kv_page_read_fp4(pages, block_table, starts, n, head_dim, dtype, status=None):
    what = "kv_page_read_fp4"
    device = pages.device
    rows = _fp4_rows(pages, head_dim, what)
    if dtype not in MATRIX_DTYPES:
        raise ValueError(f"{what}: rows are read as bf16 or f16, not {dtype}")
    if n < 0:
        raise ValueError(f"{what}: cannot read {n} rows")
    b = starts.shape[0] if isinstance(starts, torch.Tensor) and starts.dim() == 1 else -1
    _check_i32(starts, (b,), device, "starts")
    t_sb, width = _table(block_table, b, device, "block_table")
    if status is not None:
        _check_i32(status, (1,), device, "status")
    if _elsewhere(device):
        with _on(device):
            return kv_page_read_fp4(pages, block_table, starts, n, head_dim, dtype, status)
    k, v = (torch.empty((b, n, pages.shape[2], head_dim), device=device, dtype=dtype)
            for _ in range(2))
    if b == 0 or n == 0:
        return k, v
    s0, s1, s2, _ = pages.stride()
    rc = _lib.load().dx_kv_page_read_fp4(
        pages.data_ptr(), s0, s1, s2, _lib.dtype_code(dtype), pages.shape[1], rows,
        block_table.data_ptr(), t_sb, width, starts.data_ptr(), _lib.ptr(status), k.data_ptr(),
        v.data_ptr(), b, n, pages.shape[2], head_dim, _lib.stream_handle(device))
    if rc:
        _lib.check(rc, what)
    return k, v


def _attn_accepts(q, k, v, *args, **kwargs) -> bool:
    return (q.is_cuda and q.dim() == 4 and q.dtype in MATRIX_DTYPES and q.shape[-1] in FP4_HEAD_DIMS
            and k.dtype == q.dtype and v.dtype == q.dtype and k.shape == v.shape and k.dim() == 4
            and k.shape[-1] == q.shape[-1] and k.shape[2] > 0 and q.shape[2] % k.shape[2] == 0)


@register("attention", "paged_fp4", name="hip_paged_attention_fp4_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_attn_accepts)
def paged_attention_fp4(q, k, v, pages, block_table, cache_lens, block_boundaries, softmax_scale,
                        causal=False, return_lse=False):
    return _attend("paged_attention_fp4", q, k, v, pages, None, block_table, cache_lens,
                   block_boundaries, softmax_scale, causal, return_lse, True)


@register("attention", "shared_prefix_fp4", name="hip_shared_prefix_attention_fp4_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_attn_accepts)
def shared_prefix_attention_fp4(q, k, v, pages, prefix_table, prefix_len, block_table, cache_lens,
                                block_boundaries, softmax_scale, causal=False, return_lse=False):
    return _attend("shared_prefix_attention_fp4", q, k, v, pages, (prefix_table, prefix_len),
                   block_table, cache_lens, block_boundaries, softmax_scale, causal, return_lse, True)
