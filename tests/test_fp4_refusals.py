"""Calls that the 4-bit cache's operators, and those that keep its heaviest rows, refuse before
anything is launched (no GPU)."""

from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

from dexter_amd.ops.gfx950 import _lib, keep, paged, paged_fp4

HEADER = Path(__file__).resolve().parents[1] / "include" / "dexter_gfx950.h"
BF, F16, F32, I32, FP4 = _lib.DX_BF16, _lib.DX_F16, _lib.DX_F32, _lib.DX_I32, _lib.DX_FP4


def _message(lib, rc, code=_lib.DX_EINVAL):
    assert rc == code, rc
    return lib.dx_last_error().decode()


def _append(lib, *, k=16, k_sl=256, pages=16, p_sp=4096, dtype=BF, n_pages=4, rows=16, b=1, n=1, h=2,
            d=128, table=16, starts=16, width=4):
    return lib.dx_kv_page_append_fp4(k, 256, k_sl, 128, 16, 256, 256, 128, pages, 1 << 20, p_sp, 2048, dtype,
                                     n_pages, rows, table, 4, width, starts, None, b, n, h, d, None)


def _read(lib, *, pages=16, p_sp=4096, dtype=BF, n_pages=4, rows=16, b=1, n=1, h=2, d=128, table=16,
          starts=16, width=4, k=16):
    return lib.dx_kv_page_read_fp4(pages, 1 << 20, p_sp, 2048, dtype, n_pages, rows, table, 4, width, starts,
                                   None, k, 16, b, n, h, d, None)


def test_write_and_read_refusals(built_lib):
    lib = _lib.load()
    assert "strides" in _message(lib, _append(lib, k_sl=4))
    for call in (_append, _read):
        def bad(**kw):
            return _message(lib, call(lib, **kw))
        assert call(lib, b=0) == call(lib, n=0) == _lib.DX_OK
        assert "dtype code 2" in bad(dtype=F32)
        assert "head_dim 32" in bad(d=32)
        assert "head_dim 96" in bad(d=96)
        assert "bad shape" in bad(h=0)
        assert "pages of 24 rows" in bad(rows=24)
        assert "pages of 2048 rows" in bad(rows=2048)
        assert "pages of 0 rows" in bad(rows=0)
        assert "null pointer" in bad(table=None)
        assert "null pointer" in bad(starts=None)
        assert "null pointer" in bad(k=None)
        assert "null pages" in bad(pages=None)
        assert "pointers must be 16-byte aligned" in bad(pages=24)
        assert "strides" in bad(p_sp=4088)
        assert "below 2^31" in bad(n_pages=1 << 31)
        assert "below 2^31" in bad(n=1 << 31)
        assert "exceed one launch" in bad(b=1 << 20, n=1 << 12)
        assert "exceed one launch" in bad(n=1 << 30, h=4)


def _attend(lib, name, lse=16, *, dtype=BF, d=128, rows=16, p_sp=4096, p_sh=2048, pages=16, ws=0, ws_bytes=0,
            h=4, hkv=2, lk=4):
    call = _lib.PAGED_CALL.pack(
        16, 2048, 512, 128, 16, 1024, 256, 128, 16, 1024, 256, 128, 16, 2048, 512, 128,
        pages, 1 << 20, p_sp, 3, p_sh, 8, rows, 16, 3, 3, 16, 16, 2, 16, dtype, 2, 4, lk, h, hkv, d, 0, I32, 0,
        0, 1.0, ws, ws_bytes, 0)
    return getattr(lib, name)(call, lse)


def test_attention_refusals(built_lib):
    lib = _lib.load()
    for name in ("dx_paged_attention_fp4", "dx_shared_prefix_attention_fp4"):
        def bad(**kw):
            return _message(lib, _attend(lib, name, **kw))
        assert "null call" in _message(lib, getattr(lib, name)(None, None))
        assert "dtype code 2" in bad(dtype=F32)
        assert "head_dim 96" in bad(d=96)
        assert "pages of 24 rows" in bad(rows=24)
        assert "strides" in bad(p_sp=4088)
        assert "strides" in bad(p_sh=2056)
        assert "aligned" in bad(pages=24)
        assert "null pages" in bad(pages=0)
        assert "lse" in bad(lse=18)
        assert "not a multiple" in bad(h=4, hkv=3)
    # A pool's row stride is the format's, not the call's: this one passes to the workspace check.
    assert "needed" in _message(lib, _attend(lib, "dx_shared_prefix_attention_fp4"), _lib.DX_EWORKSPACE)
    for name in ("dx_paged_attention_lse", "dx_shared_prefix_attention_lse"):
        assert "null call" in _message(lib, getattr(lib, name)(None, 16))
        for lse in (None, 18):
            call = _lib.PAGED_CALL.pack(
                16, 2048, 512, 128, 16, 1024, 256, 128, 16, 1024, 256, 128, 16, 2048, 512, 128,
                16, 1 << 20, 4096, 256, 128, 8, 16, 16, 3, 3, 16, 16, 2, 16, BF, 2, 4, 4, 4, 2, 128, 0, I32, 0,
                0, 1.0, 0, 0, 0)
            assert "lse" in _message(lib, getattr(lib, name)(call, lse))


def _weights(lib, *, q=16, lse=16, q_sl=512, pages=16, p_sr=256, n_pages=8, rows=16, table=16, width=3, lens=16,
             weights=16, dtype=BF, fp4=0, b=2, lq=4, h=4, hkv=2, d=128, scale=1.0):
    z = lambda x: 0 if x is None else x  # noqa: E731
    return lib.dx_paged_key_weights(_lib.WEIGHTS_CALL.pack(
        z(q), 2048, q_sl, 128, z(lse), z(pages), 4096, p_sr, 128, n_pages, rows, z(table), 3, width, z(lens),
        z(weights), 96, 48, dtype, fp4, b, lq, h, hkv, d, 0, scale, 0))


def test_weights_refusals(built_lib):
    lib = _lib.load()
    assert "null call" in _message(lib, lib.dx_paged_key_weights(None))
    assert _weights(lib, b=0) == _weights(lib, width=0) == _lib.DX_OK

    def bad(**kw):
        return _message(lib, _weights(lib, **kw))
    assert "dtype code 2" in bad(dtype=F32, fp4=1)
    assert "dtype code 7" in bad(dtype=7)
    assert "head_dim 96" in bad(d=96)
    assert "head_dim 256" in bad(d=256, dtype=F32)
    assert "not a multiple" in bad(h=4, hkv=3)
    assert "bad shape" in bad(h=0)
    assert "pages of 24 rows" in bad(rows=24)
    assert "fewer than 2^30" in bad(width=1 << 27)
    assert "fewer than 2^30" in bad(lq=1 << 28)
    assert "exceed one launch" in bad(b=1 << 15)
    assert "exceeds one launch" in bad(width=1 << 25, b=1000)
    assert "finite" in bad(scale=float("nan"))
    assert "finite" in bad(scale=3e38)
    assert "null q or lse" in bad(q=None)
    assert "null q or lse" in bad(lse=None)
    for name in ("table", "lens", "weights"):
        assert "null pointer" in bad(**{name: None})
    assert "null pages" in bad(pages=None)
    assert "aligned" in bad(q=24)
    assert "strides" in bad(q_sl=4)
    assert "strides" in bad(p_sr=4)


def test_packed_weights_call_matches_the_header():
    text = HEADER.read_text()
    body = text[text.index("typedef struct dx_weights_call {"):text.index("} dx_weights_call;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    kinds = []
    for part in body.split(";"):
        words = part.replace("*", " ").split()
        if words:
            kinds += ["d" if "double" in words else "q"] * (part.count(",") + 1)
    fmt = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", _lib.WEIGHTS_CALL.format))
    assert fmt == "".join(kinds) and _lib.WEIGHTS_CALL.size == 8 * len(kinds)


def test_keep_and_gather_refusals(built_lib):
    lib = _lib.load()

    def rows(*, w=16, width=100, lens=16, k=5, recent=0, out=16, b=2, h=3):
        return lib.dx_kv_keep_rows(w, 300, 100, width, lens, k, recent, out, b, h, None)
    assert rows(b=0) == rows(k=0) == _lib.DX_OK
    assert "bad shape" in _message(lib, rows(h=0))
    assert "bad shape" in _message(lib, rows(recent=-1))
    assert "2^30" in _message(lib, rows(width=1 << 30))
    assert "exceed one launch" in _message(lib, rows(b=1 << 21, h=8))
    for name in ("w", "lens", "out"):
        assert "null pointer" in _message(lib, rows(**{name: None}))

    def gather(*, pages=16, p_sr=256, dtype=BF, n_pages=8, rows=16, src=16, width=3, dst=16, d_width=3, at=16,
               k=5, w=None, b=2, h=3, d=128):
        return lib.dx_kv_page_gather(pages, 1 << 20, 4096, p_sr, 128, dtype, n_pages, rows, src, 3, width, dst, 3,
                                     d_width, at, k, w, 300, 100, 100, b, h, d, None)
    assert gather(b=0) == gather(k=0) == _lib.DX_OK
    assert "dtype code 3" in _message(lib, gather(dtype=I32))
    assert "bad shape" in _message(lib, gather(rows=0))
    assert "head_dim 96" in _message(lib, gather(dtype=FP4, d=96))
    assert "pages of 24 rows" in _message(lib, gather(dtype=FP4, rows=24))
    assert "16-byte chunks" in _message(lib, gather(d=4))
    assert "2^30" in _message(lib, gather(width=1 << 27))
    assert "exceed one launch" in _message(lib, gather(b=1 << 15))
    for name in ("src", "dst", "at"):
        assert "null pointer" in _message(lib, gather(**{name: None}))
    assert "null pages" in _message(lib, gather(pages=None))
    assert "aligned" in _message(lib, gather(pages=24))
    assert "strides" in _message(lib, gather(p_sr=4))


# ---------------------------------------------------------------------------
# The Python layer
# ---------------------------------------------------------------------------
def _tensors(b=2, lq=3, heads=4, kv=2, dim=64, rows=16, dtype=torch.bfloat16):
    return dict(q=torch.zeros(b, lq, heads, dim, dtype=dtype), k=torch.zeros(b, lq, kv, dim, dtype=dtype),
                v=torch.zeros(b, lq, kv, dim, dtype=dtype),
                pages=torch.zeros(2, 5, kv, rows * (dim // 2 + dim // 32), dtype=torch.uint8),
                table=torch.zeros(b, 4, dtype=torch.int32), lens=torch.zeros(b, dtype=torch.int32))


POOLS = [
    (torch.zeros(2, 5, 2, 16 * 34), "uint8"),
    (torch.zeros(2, 5, 16, 2, 34, dtype=torch.uint8), "uint8"),
    (torch.zeros(3, 5, 2, 16 * 34, dtype=torch.uint8), "uint8"),
    (torch.zeros(2, 5, 2, 16 * 34 - 2, dtype=torch.uint8), "multiple of 16"),
    (torch.zeros(2, 5, 2, 8 * 34, dtype=torch.uint8), "multiple of 16"),
    (torch.zeros(2, 5, 2, 0, dtype=torch.uint8), "multiple of 16"),
    (torch.zeros(2, 1, 1, 1040 * 34, dtype=torch.uint8), "multiple of 16"),
    (torch.zeros(2, 1, 2, 16 * 34, dtype=torch.uint8).expand(2, 5, 2, 16 * 34), "expanded"),
    (torch.zeros(2, 5, 2, 16 * 34 + 8, dtype=torch.uint8)[..., :16 * 34], "16-byte aligned"),
    (torch.zeros(2, 5, 16 * 34, 2, dtype=torch.uint8).transpose(2, 3), "16-byte aligned"),
]


@pytest.mark.parametrize("pool,message", POOLS)
def test_pools(pool, message):
    t = _tensors()
    for call in (lambda: paged_fp4.kv_page_append_fp4(pool, t["k"], t["v"], t["table"], t["lens"]),
                 lambda: paged_fp4.kv_page_read_fp4(pool, t["table"], t["lens"], 3, 64, torch.bfloat16),
                 lambda: paged_fp4.paged_attention_fp4(t["q"], t["k"], t["v"], pool, t["table"], t["lens"], None, None)):
        with pytest.raises(ValueError, match=message):
            call()


def test_argument_checks():
    t = _tensors()

    def attend(**change):
        a = {**t, **change}
        paged_fp4.paged_attention_fp4(a["q"], a["k"], a["v"], a["pages"], a["table"], a["lens"], None, None)
    f32 = _tensors(dtype=torch.float32)
    with pytest.raises(ValueError, match="bf16 and f16"):
        attend(**{n: f32[n] for n in "qkv"})
    with pytest.raises(ValueError, match="3 heads for 2"):
        attend(pages=torch.zeros(2, 5, 3, 16 * 34, dtype=torch.uint8))
    d32 = _tensors(dim=32)
    with pytest.raises(ValueError, match="head_dim 32"):
        attend(**{n: d32[n] for n in "qkv"})
    with pytest.raises(ValueError, match="go together"):
        attend(lens=None)
    with pytest.raises(ValueError, match="cache_lens must be int32"):
        attend(lens=t["lens"].long())

    def append(**change):
        a = {**t, "status": None, **change}
        paged_fp4.kv_page_append_fp4(a["pages"], a["k"], a["v"], a["table"], a["lens"], a["status"])
    for change, message in [
            (dict(v=t["v"][:, :1]), "k and v must both be"), (dict(v=t["v"].half()), "both be bf16 or f16"),
            (dict(k=f32["k"], v=f32["v"]), "both be bf16 or f16"), (dict(table=t["table"].long()), "block_table"),
            (dict(lens=7), "starts must be int32"), (dict(status=torch.zeros(2, dtype=torch.int32)), "status"),
            (dict(k=t["q"], v=t["q"]), "2 heads for 4")]:
        with pytest.raises(ValueError, match=message):
            append(**change)

    def read(pages=t["pages"], table=t["table"], starts=t["lens"], n=3, dim=64, dtype=torch.float16):
        paged_fp4.kv_page_read_fp4(pages, table, starts, n, dim, dtype)
    for change, message in [(dict(dtype=torch.float32), "read as bf16 or f16"), (dict(n=-1), "cannot read"),
                            (dict(dim=96), "head_dim 96"), (dict(starts=t["lens"].long()), "starts"),
                            (dict(starts=[0, 0]), "starts"), (dict(table=t["table"][:1]), "block_table")]:
        with pytest.raises(ValueError, match=message):
            read(**change)


def test_keep_argument_checks():
    t = _tensors()
    lse, w = torch.zeros(2, 3, 4), torch.zeros(2, 2, 64)

    def weigh(**change):
        a = {**t, "lse": lse, "w": w, **change}
        keep.paged_key_weights(a["q"], a["lse"], a["w"], a["pages"], a["table"], a["lens"], None)
    p16 = torch.zeros(2, 5, 16, 2, 64, dtype=torch.bfloat16)
    for change, message in [
            (dict(lse=lse.double()), "lse must be"), (dict(lse=lse[:, :2]), "lse must be"), (dict(lse=None), "lse must be"),
            (dict(w=w.double()), "weights must be"), (dict(w=w[..., :63]), "weights must be"),
            (dict(w=torch.zeros(2, 64, 2).transpose(1, 2)), "contiguous rows"),
            (dict(w=torch.zeros(1, 2, 64).expand(2, 2, 64)), "expanded"),
            (dict(pages=p16.half()), "pages"), (dict(pages=p16[..., :32].contiguous()), "pages"),
            (dict(pages=torch.zeros(2, 5, 8, 2, 64, dtype=torch.bfloat16)), "multiple of 16"),
            (dict(pages=torch.zeros(2, 5, 3, 16 * 34, dtype=torch.uint8)), "do not divide"),
            (dict(pages=t["pages"][..., :-2]), "multiple of 16"),
            (dict(table=t["table"].long()), "block_table"), (dict(lens=t["lens"][:1]), "cache_lens"),
            (dict(q=t["q"][0]), "q must be")]:
        with pytest.raises(ValueError, match=message):
            weigh(**change)

    for args, message in [((w[0], t["lens"], 3), "weights must be"), ((w.double(), t["lens"], 3), "float32"),
                          ((w.transpose(1, 2), t["lens"], 3), "contiguous rows"), ((w, t["lens"].long(), 3), "cache_lens"),
                          ((w, t["lens"], -1), "cannot keep"), ((w, t["lens"], 3, -1), "cannot keep")]:
        with pytest.raises(ValueError, match=message):
            keep.kv_keep_rows(*args)

    rows = torch.zeros(2, 2, 5, dtype=torch.int32)

    def gather(**change):
        a = {**t, "rows": rows, "dst": None, "w": None, "dim": 64, **change}
        keep.kv_page_gather(a["pages"], a["table"], a["rows"], a["dst"], a["w"], a["dim"])
    for change, message in [
            (dict(dim=None), "head_dim is needed"), (dict(dim=96), "head_dim 96"), (dict(rows=rows.long()), "rows must be"),
            (dict(rows=rows[:, :1]), "rows must be"), (dict(rows=[[0]]), "rows must be"), (dict(dst=t["table"][:1]), "dst_table"),
            (dict(w=w[:, :1]), "weights must be"), (dict(w=w.half()), "weights must be"),
            (dict(pages=p16, dim=128), "head_dim 128"), (dict(pages=p16.double()), "pages"), (dict(table=None), "block_table")]:
        with pytest.raises(ValueError, match=message):
            gather(**change)


def test_tensors_off_the_gpu_are_refused():
    """A pinned implementation is called without its predicate: it checks the device itself."""
    t = _tensors()
    for call in (
            lambda: paged_fp4.kv_page_append_fp4(t["pages"], t["k"], t["v"], t["table"], t["lens"]),
            lambda: paged_fp4.kv_page_read_fp4(t["pages"], t["table"], t["lens"], 3, 64, torch.bfloat16),
            lambda: paged_fp4.paged_attention_fp4(t["q"], t["k"], t["v"], t["pages"], t["table"], t["lens"], None, None),
            lambda: keep.paged_key_weights(t["q"], torch.zeros(2, 3, 4), None, t["pages"], t["table"], t["lens"], None),
            lambda: keep.kv_keep_rows(torch.zeros(2, 2, 9), t["lens"], 3),
            lambda: keep.kv_page_gather(t["pages"], t["table"], torch.zeros(2, 2, 5, dtype=torch.int32), head_dim=64),
            lambda: paged._attend("paged_attention", t["q"], t["k"], t["v"], torch.zeros(2, 5, 16, 2, 64, dtype=torch.bfloat16),
                                  None, t["table"], t["lens"], None, None, False, True)):
        with pytest.raises(ValueError, match="GPU"):
            call()
