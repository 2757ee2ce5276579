"""A KV cache in pages on gfx950: chunk append, page copies, and attention over pages.

The contiguous cache (``cache.py``, ``attention.py``) gives every sequence a
row range of its own, as the reference's ``KVCache`` does
(``models/dreamzero/model.py:35-65``). Here rows lie in pages of a pool
``[2, P, R, H, D]`` (plane 0 K, plane 1 V; ``P`` pages of ``R`` rows): row ``r``
of sequence ``b`` is row ``r % R`` of page ``block_table[b, r // R]``. Sequences
can then share pages, so a rollout forks by copying its table and one partly
filled page instead of its whole history, and candidate futures of one episode
attend to one copy of it. The reference has no counterpart: its cache and its
attention op take one contiguous history per sequence
(``ops/reference/attention.py:65-67``).

Registered here:

* ``cache/page_append``     ``(pages, k, v, block_table, starts, status)``: write
  ``k``/``v`` ``[B, n, H, D]`` at rows ``[starts[b], starts[b] + n)``;
* ``cache/page_copy``       ``(pools, src, dst)``: copy pages, in every pool given;
* ``attention/paged``       ``blockwise_causal_attention`` with the cached rows in pages;
* ``attention/shared_prefix``  the same, with a prefix in front that all sequences share.

Tables, lengths and start rows are int32 tensors on the device that the kernels
read when they run: nothing synchronises, and a captured graph follows them as
they change. The host cannot check what they hold, so the kernels do: lengths
are clamped to the rows that the table has entries for, an entry outside
``[0, P)`` holds no rows (attention does not see its keys, an append writes
nothing there and sets ``status``). Workspaces come from torch's allocator per
call, so calls on different streams, and graphs, never share one.
"""

from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from ...registry import Priority, register
from . import _lib
from ._common import CDNA4, as_rows, strides
from .attention import _starts

_APPEND_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# Head dims of the attention kernels, per input dtype.
_HEAD_DIMS = {torch.bfloat16: (64, 128, 256), torch.float16: (64, 128, 256),
              torch.float32: (64, 128)}
PAGE_ROWS_MULTIPLE, PAGE_ROWS_MAX = 16, 1024


def _on(device: torch.device):
    """The context that makes ``device`` the current one (nothing when it is already)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _check_pool(pages: torch.Tensor, what: str) -> None:
    if pages.dim() != 5 or pages.shape[0] != 2:
        raise ValueError(f"{what}: pages must be [2, P, R, H, D], got {tuple(pages.shape)}")
    if 0 in pages.shape[2:]:
        raise ValueError(f"{what}: pages {tuple(pages.shape)} hold no rows")
    per16 = 16 // pages.element_size()
    steps = pages.stride()
    if not (steps[-1] == 1 and pages.data_ptr() % 16 == 0 and all(x % per16 == 0 for x in steps[:-1])):
        raise ValueError(f"{what}: pages must have a contiguous, 16-byte aligned head_dim")
    if any(n > 1 and x == 0 for n, x in zip(pages.shape, steps)):
        raise ValueError(f"{what}: pages must not be expanded (a stride is 0)")


def _check_i32(t, shape: tuple, device: torch.device, what: str) -> None:
    """A device int32 tensor that the kernels read in place (never copied: they must
    read the caller's tensor, the one the caller changes)."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != device \
            or tuple(t.shape) != shape or (t.numel() > 1 and t.stride(-1) != 1):
        got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)
        raise ValueError(f"{what} must be int32 {list(shape)} on {device} with contiguous rows, "
                         f"got {got}")


def _table(t, batch: int, device: torch.device, what: str) -> tuple[int, int]:
    """(row stride, width) of a block table [B, W]."""
    width = t.shape[1] if isinstance(t, torch.Tensor) and t.dim() == 2 else -1
    _check_i32(t, (batch, width), device, what)
    return (0 if batch == 1 else t.stride(0)), width


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def _append_accepts(pages, k, v, *args, **kwargs) -> bool:
    return (pages.is_cuda and pages.dtype in _APPEND_DTYPES and k.dtype == pages.dtype
            and v.dtype == pages.dtype and pages.dim() == 5 and k.dim() == 4
            and k.shape == v.shape and (k.shape[-1] * k.element_size()) % 16 == 0)


@register("cache", "page_append", name="hip_kv_page_append_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_append_accepts)
def kv_page_append(pages, k, v, block_table, starts, status=None) -> None:
    _check_pool(pages, "kv_page_append")
    if k.shape != v.shape or k.dim() != 4:
        raise ValueError("k and v must both be [B, n, H, D]")
    b, n, heads, dim = k.shape
    device = pages.device
    if tuple(pages.shape[3:]) != (heads, dim):
        raise ValueError(f"pages must be [2, P, R, {heads}, {dim}], got {tuple(pages.shape)}")
    if k.device != device or v.device != device:
        raise ValueError(f"k and v must be on {device}, got {k.device} and {v.device}")
    t_sb, width = _table(block_table, b, device, "block_table")
    _check_i32(starts, (b,), device, "starts")
    if status is not None:
        _check_i32(status, (1,), device, "status")
    if b == 0 or n == 0:
        return
    k, v = as_rows(k), as_rows(v)
    with _on(device):
        rc = _lib.load().dx_kv_page_append(
            k.data_ptr(), *strides(k, 3), v.data_ptr(), *strides(v, 3),
            pages.data_ptr(), *pages.stride()[:4], _lib.dtype_code(pages.dtype),
            pages.shape[1], pages.shape[2], block_table.data_ptr(), t_sb, width,
            starts.data_ptr(), _lib.ptr(status), b, n, heads, dim, _lib.stream_handle(device))
    _lib.check(rc, "kv_page_append")


# ---------------------------------------------------------------------------
# Copy
# ---------------------------------------------------------------------------
def _copy_accepts(pools, *args, **kwargs) -> bool:
    return all(p.is_cuda and p.dtype in _APPEND_DTYPES and p.dim() == 5
               and (p.shape[-1] * p.element_size()) % 16 == 0 for p in pools)


@register("cache", "page_copy", name="hip_kv_page_copy_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_copy_accepts)
def kv_page_copy(pools, src, dst) -> None:
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} source pages for {len(dst)} destinations")
    if not pools:
        raise ValueError("kv_page_copy needs a pool")
    first = pools[0]
    _check_pool(first, "kv_page_copy")
    for p in pools[1:]:
        if p.shape != first.shape or p.stride() != first.stride() or p.dtype != first.dtype \
                or p.device != first.device or p.data_ptr() % 16:
            raise ValueError("kv_page_copy: pools must agree in shape, strides, dtype and device")
    n = len(src)
    if n == 0:
        return
    _, pages, rows, heads, dim = first.shape
    device = first.device
    ptrs = (ctypes.c_void_p * len(pools))(*[p.data_ptr() for p in pools])
    ids = ctypes.c_int64 * n
    with _on(device):
        rc = _lib.load().dx_kv_page_copy(
            ptrs, len(pools), *first.stride()[:4], _lib.dtype_code(first.dtype), pages, rows,
            heads, dim, ids(*src), ids(*dst), n, _lib.stream_handle(device))
    _lib.check(rc, "kv_page_copy")


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _attn_accepts(q, k, v, *args, **kwargs) -> bool:
    return (q.is_cuda and q.dim() == 4 and q.shape[-1] in _HEAD_DIMS.get(q.dtype, ())
            and k.dtype == q.dtype and v.dtype == q.dtype and k.shape == v.shape and k.dim() == 4
            and k.shape[-1] == q.shape[-1] and k.shape[2] > 0 and q.shape[2] % k.shape[2] == 0)


def _attend(what, q, k, v, pages, prefix, block_table, cache_lens, block_boundaries,
            softmax_scale, causal):
    """``prefix``: None, or (prefix_table, prefix_len)."""
    if q.dim() != 4 or k.shape != v.shape or k.dim() != 4:
        raise ValueError("q, k, v must be [B, L, H, D] with k and v of one shape")
    b, q_len, heads, dim = q.shape
    kv_len, kv_heads = k.shape[1], k.shape[2]
    device = q.device
    if k.shape[0] != b or k.shape[3] != dim or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"k/v {tuple(k.shape)} do not match q {tuple(q.shape)} (the k/v heads "
                         "must divide the query heads)")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"k/v dtypes {k.dtype}, {v.dtype} differ from q's {q.dtype}")
    if kv_len != q_len and (block_boundaries is not None or causal):
        raise ValueError(f"k/v length {kv_len} must equal q length {q_len} with block_boundaries "
                         "or causal")
    _check_pool(pages, what)
    if tuple(pages.shape[3:]) != (kv_heads, dim) or pages.dtype != q.dtype:
        raise ValueError(f"pages must be [2, P, R, {kv_heads}, {dim}] of {q.dtype}, got "
                         f"{tuple(pages.shape)} of {pages.dtype}")
    rows = pages.shape[2]
    if rows % PAGE_ROWS_MULTIPLE or rows > PAGE_ROWS_MAX:
        raise ValueError(f"attention takes pages of a multiple of {PAGE_ROWS_MULTIPLE} rows up to "
                         f"{PAGE_ROWS_MAX}, got {rows}")
    for name, t in (("k", k), ("v", v), ("pages", pages)):
        if t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")
    if (block_table is None) != (cache_lens is None):
        raise ValueError("block_table and cache_lens go together")
    t_sb = width = p_width = 0
    if block_table is not None:
        t_sb, width = _table(block_table, b, device, "block_table")
        _check_i32(cache_lens, (b,), device, "cache_lens")
    if prefix is not None:
        p_table, p_len = prefix
        p_width = p_table.shape[0] if isinstance(p_table, torch.Tensor) and p_table.dim() == 1 else -1
        _check_i32(p_table, (p_width,), device, "prefix_table")
        _check_i32(p_len, (1,), device, "prefix_len")
    if kv_len == 0 and width == 0 and p_width == 0 and q_len > 0:
        raise ValueError("attention over no keys: k/v are empty and there is no cached page")
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(dim)
    out = torch.empty((b, q_len, heads, dim), device=device, dtype=q.dtype)
    if out.numel() == 0:
        return out
    q, k, v = as_rows(q), as_rows(k), as_rows(v)
    starts, starts_dt, n_blocks = _starts(block_boundaries, q_len, device)
    lib = _lib.load()
    code = _lib.dtype_code(q.dtype)
    with _on(device):
        ws_bytes = lib.dx_paged_attention_workspace_bytes(
            code, b, q_len, kv_len, heads, kv_heads, dim, rows, width, prefix is not None, p_width)
        if ws_bytes < 0:
            _lib.check(-ws_bytes, what)
        # From torch's allocator, on the current stream: no other call holds it.
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
        args = [q.data_ptr(), *strides(q, 3), k.data_ptr(), *strides(k, 3),
                v.data_ptr(), *strides(v, 3), pages.data_ptr(), *pages.stride()[:4],
                pages.shape[1], rows]
        if prefix is not None:
            args += [p_table.data_ptr(), p_width, p_len.data_ptr()]
        args += [_lib.ptr(block_table), t_sb, width, _lib.ptr(cache_lens),
                 out.data_ptr(), *strides(out, 3), code, b, q_len, kv_len, heads, kv_heads, dim,
                 _lib.ptr(starts), starts_dt, n_blocks, int(bool(causal)), scale,
                 _lib.ptr(ws), ws_bytes, _lib.stream_handle(device)]
        fn = lib.dx_paged_attention if prefix is None else lib.dx_shared_prefix_attention
        rc = fn(*args)
    _lib.check(rc, what)
    return out


@register("attention", "paged", name="hip_paged_attention_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_attn_accepts)
def paged_attention(q, k, v, pages, block_table, cache_lens, block_boundaries, softmax_scale,
                    causal=False):
    return _attend("paged_attention", q, k, v, pages, None, block_table, cache_lens,
                   block_boundaries, softmax_scale, causal)


@register("attention", "shared_prefix", name="hip_shared_prefix_attention_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_attn_accepts)
def shared_prefix_attention(q, k, v, pages, prefix_table, prefix_len, block_table, cache_lens,
                            block_boundaries, softmax_scale, causal=False):
    return _attend("shared_prefix_attention", q, k, v, pages, (prefix_table, prefix_len),
                   block_table, cache_lens, block_boundaries, softmax_scale, causal)
