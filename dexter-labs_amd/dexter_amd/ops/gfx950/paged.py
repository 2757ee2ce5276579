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

import ctypes
import functools
import math
from array import array

import torch

from ...registry import Priority, register
from . import _lib
from ._common import CDNA4, strides
from .attention import _starts

_APPEND_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
# Head dims of the attention kernels, per input dtype.
_HEAD_DIMS = {torch.bfloat16: (64, 128, 256), torch.float16: (64, 128, 256),
              torch.float32: (64, 128)}
PAGE_ROWS_MULTIPLE, PAGE_ROWS_MAX = 16, 1024


def _on(device: torch.device):
    """The context that makes ``device`` the current one."""
    return torch.cuda.device(device)


def _elsewhere(device: torch.device) -> bool:
    """Whether ``device`` is another GPU than the current one. Raises for none at all (a
    pinned implementation is called without its predicate)."""
    if device.type != "cuda":
        raise ValueError(f"the paged cache's kernels take tensors on a GPU, got {device}")
    return device.index != torch.cuda.current_device()


def _check_pool(pages: torch.Tensor, what: str) -> tuple:
    """The strides of a pool that the kernels can read in place."""
    shape, steps = pages.shape, pages.stride()
    if len(shape) != 5 or shape[0] != 2:
        raise ValueError(f"{what}: pages must be [2, P, R, H, D], got {tuple(shape)}")
    _, p, r, h, d = shape
    if not (r and h and d):
        raise ValueError(f"{what}: pages {tuple(shape)} hold no rows")
    s0, s1, s2, s3, s4 = steps
    if s4 != 1 or pages.data_ptr() % 16 or (s0 | s1 | s2 | s3) * pages.element_size() % 16:
        raise ValueError(f"{what}: pages must have a contiguous, 16-byte aligned head_dim")
    if not (s0 and (s1 or p <= 1) and (s2 or r == 1) and (s3 or h == 1)):
        raise ValueError(f"{what}: pages must not be expanded (a stride is 0)")
    return steps


def _check_i32(t, shape: tuple, device: torch.device, what: str) -> None:
    """A device int32 tensor that the kernels read in place (never copied: they must
    read the caller's tensor, the one the caller changes)."""
    if isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.shape == shape \
            and t.device == device and (shape[-1] <= 1 or t.stride(-1) == 1):
        return
    got = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else repr(t)
    raise ValueError(f"{what} must be int32 {list(shape)} on {device} with contiguous rows, got {got}")


def _table(t, batch: int, device: torch.device, what: str) -> tuple[int, int]:
    """(row stride, width) of a block table [B, W]."""
    width = t.shape[1] if isinstance(t, torch.Tensor) and t.dim() == 2 else -1
    _check_i32(t, (batch, width), device, what)
    return (0 if batch <= 1 else t.stride(0)), width


def _rows(t: torch.Tensor) -> tuple:
    """``(tensor, batch, row, head stride)`` of a ``[B, L, H, D]`` operand: itself where the
    kernels can read it in place, else a contiguous copy; 0 for a dim that is not stepped."""
    b, n, h, d = t.shape
    s0, s1, s2, s3 = t.stride()
    s0 = 0 if b == 1 else s0
    s1 = 0 if n == 1 else s1
    s2 = 0 if h == 1 else s2
    if (s3 != 1 and d != 1) or t.data_ptr() % 16 or (s0 | s1 | s2) * t.element_size() % 16:
        t = t.clone(memory_format=torch.contiguous_format)  # (a misaligned one is contiguous too)
        return (t, *strides(t, 3))
    return t, s0, s1, s2


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
    s0, s1, s2, s3, _ = _check_pool(pages, "kv_page_append")
    if k.shape != v.shape or k.dim() != 4:
        raise ValueError("k and v must both be [B, n, H, D]")
    b, n, heads, dim = k.shape
    device = pages.device
    if pages.shape[3:] != (heads, dim) or k.dtype is not pages.dtype or v.dtype is not pages.dtype:
        raise ValueError(f"pages must be [2, P, R, {heads}, {dim}] of k's and v's dtype, got "
                         f"{tuple(pages.shape)} of {pages.dtype}")
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
            return kv_page_append(pages, k, v, block_table, starts, status)
    k, k_sb, k_sl, k_sh = _rows(k)
    v, v_sb, v_sl, v_sh = _rows(v)
    rc = _lib.load().dx_kv_page_append(
        k.data_ptr(), k_sb, k_sl, k_sh, v.data_ptr(), v_sb, v_sl, v_sh,
        pages.data_ptr(), s0, s1, s2, s3, _lib.dtype_code(pages.dtype),
        pages.shape[1], pages.shape[2], block_table.data_ptr(), t_sb, width,
        starts.data_ptr(), _lib.ptr(status), b, n, heads, dim, _lib.stream_handle(device))
    _lib.check(rc, "kv_page_append")


# ---------------------------------------------------------------------------
# Copy
# ---------------------------------------------------------------------------
def _copy_accepts(pools, *args, **kwargs) -> bool:
    # The first speaks for all: the implementation checks that they agree.
    return len(pools) == 0 or (
        pools[0].is_cuda and pools[0].dtype in _APPEND_DTYPES and pools[0].dim() == 5
        and (pools[0].shape[-1] * pools[0].element_size()) % 16 == 0)


@register("cache", "page_copy", name="hip_kv_page_copy_gfx950",
          capability=CDNA4, priority=Priority.SPECIALISED, accepts=_copy_accepts)
def kv_page_copy(pools, src, dst) -> None:
    n = len(src)
    if n != len(dst):
        raise ValueError(f"{n} source pages for {len(dst)} destinations")
    if not pools:
        raise ValueError("kv_page_copy needs a pool")
    first = pools[0]
    steps = _check_pool(first, "kv_page_copy")
    shape, dtype, device = first.shape, first.dtype, first.device
    where = first.get_device()
    ptrs = []
    for p in pools:
        if p.shape != shape or p.stride() != steps or p.dtype is not dtype or p.get_device() != where:
            raise ValueError("kv_page_copy: pools must agree in shape, strides, dtype and device")
        ptrs.append(p.data_ptr())
    if n == 0:
        return
    src, dst = array("q", src), array("q", dst)  # OverflowError, not a page modulo 2^64
    if _elsewhere(device):
        with _on(device):
            return kv_page_copy(pools, src, dst)
    ids = ctypes.c_int64 * n
    rc = _lib.load().dx_kv_page_copy(
        (ctypes.c_void_p * len(ptrs))(*ptrs), len(ptrs), *steps[:4], _lib.dtype_code(dtype),
        *shape[1:], ids.from_buffer(src), ids.from_buffer(dst), n, _lib.stream_handle(device))
    _lib.check(rc, "kv_page_copy")


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _attn_accepts(q, k, v, *args, **kwargs) -> bool:
    return (q.is_cuda and q.dim() == 4 and q.shape[-1] in _HEAD_DIMS.get(q.dtype, ())
            and k.dtype == q.dtype and v.dtype == q.dtype and k.shape == v.shape and k.dim() == 4
            and k.shape[-1] == q.shape[-1] and k.shape[2] > 0 and q.shape[2] % k.shape[2] == 0)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(device_index, code, b, q_len, kv_len, heads, kv_heads, dim, rows, width,
                     has_prefix, p_width) -> int:
    """Of a shape on the current device (``device_index``): the library's own answer."""
    n = _lib.load().dx_paged_attention_workspace_bytes(
        code, b, q_len, kv_len, heads, kv_heads, dim, rows, width, has_prefix, p_width)
    if n < 0:
        _lib.check(-n, "paged attention workspace")
    return n


def _attend(what, q, k, v, pages, prefix, block_table, cache_lens, block_boundaries,
            softmax_scale, causal):
    """``prefix``: None, or (prefix_table, prefix_len)."""
    if q.dim() != 4 or k.shape != v.shape or k.dim() != 4:
        raise ValueError("q, k, v must be [B, L, H, D] with k and v of one shape")
    b, q_len, heads, dim = q.shape
    k_b, kv_len, kv_heads, k_dim = k.shape
    device, dtype = q.device, q.dtype
    if k_b != b or k_dim != dim or kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"k/v {tuple(k.shape)} do not match q {tuple(q.shape)} (the k/v heads "
                         "must divide the query heads)")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError(f"k/v dtypes {k.dtype}, {v.dtype} differ from q's {dtype}")
    if kv_len != q_len and (block_boundaries is not None or causal):
        raise ValueError(f"k/v length {kv_len} must equal q length {q_len} with block_boundaries "
                         "or causal")
    s0, s1, s2, s3, _ = _check_pool(pages, what)
    _, n_pages, rows, p_heads, p_dim = pages.shape
    if p_heads != kv_heads or p_dim != dim or pages.dtype is not dtype:
        raise ValueError(f"pages must be [2, P, R, {kv_heads}, {dim}] of {dtype}, got "
                         f"{tuple(pages.shape)} of {pages.dtype}")
    if rows % PAGE_ROWS_MULTIPLE or rows > PAGE_ROWS_MAX:
        raise ValueError(f"attention takes pages of a multiple of {PAGE_ROWS_MULTIPLE} rows up to "
                         f"{PAGE_ROWS_MAX}, got {rows}")
    if k.device != device or v.device != device or pages.device != device:
        raise ValueError(f"k, v and pages must be on {device}, got {k.device}, {v.device} and "
                         f"{pages.device}")
    if (block_table is None) != (cache_lens is None):
        raise ValueError("block_table and cache_lens go together")
    t_sb = width = p_width = table_ptr = lens_ptr = p_table_ptr = p_len_ptr = 0
    if block_table is not None:
        t_sb, width = _table(block_table, b, device, "block_table")
        _check_i32(cache_lens, (b,), device, "cache_lens")
        table_ptr, lens_ptr = block_table.data_ptr(), cache_lens.data_ptr()
    if prefix is not None:
        p_table, p_len = prefix
        p_width = p_table.shape[0] if isinstance(p_table, torch.Tensor) and p_table.dim() == 1 else -1
        _check_i32(p_table, (p_width,), device, "prefix_table")
        _check_i32(p_len, (1,), device, "prefix_len")
        p_table_ptr, p_len_ptr = p_table.data_ptr(), p_len.data_ptr()
    if kv_len == 0 and width == 0 and p_width == 0 and q_len > 0:
        raise ValueError("attention over no keys: k/v are empty and there is no cached page")
    if _elsewhere(device):
        with _on(device):
            return _attend(what, q, k, v, pages, prefix, block_table, cache_lens, block_boundaries,
                           softmax_scale, causal)
    out = torch.empty((b, q_len, heads, dim), device=device, dtype=dtype)
    if b == 0 or q_len == 0:
        return out
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(dim)
    q, *q_at = _rows(q)
    k, *k_at = _rows(k)
    v, *v_at = _rows(v)
    starts_ptr, starts_dt, n_blocks = 0, _lib.DX_I32, 0
    if block_boundaries is not None:
        starts, starts_dt, n_blocks = _starts(block_boundaries, q_len, device)
        starts_ptr = starts.data_ptr()
    code = _lib.dtype_code(dtype)
    ws_bytes = _workspace_bytes(device.index, code, b, q_len, kv_len, heads, kv_heads, dim, rows,
                                width, int(prefix is not None), p_width)
    # From torch's allocator, on the current stream: no other call holds it.
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    o_row = heads * dim
    call = _lib.PAGED_CALL.pack(
        q.data_ptr(), *q_at, k.data_ptr(), *k_at, v.data_ptr(), *v_at,
        out.data_ptr(), q_len * o_row, o_row, dim,
        pages.data_ptr(), s0, s1, s2, s3, n_pages, rows, table_ptr, t_sb, width, lens_ptr,
        p_table_ptr, p_width, p_len_ptr, code, b, q_len, kv_len, heads, kv_heads, dim,
        starts_ptr, starts_dt, n_blocks, 1 if causal else 0, scale,
        0 if ws is None else ws.data_ptr(), ws_bytes, _lib.stream_handle(device))
    lib = _lib.load()
    rc = (lib.dx_paged_attention if prefix is None else lib.dx_shared_prefix_attention)(call)
    if rc:
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
