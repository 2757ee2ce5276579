"""Calls that the paged cache's operators refuse, before anything is launched (no GPU)."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

from dexter_amd.ops.gfx950 import _lib, paged

HEADER = Path(__file__).resolve().parents[1] / "include" / "dexter_gfx950.h"
BF, F32, I32 = _lib.DX_BF16, _lib.DX_F32, _lib.DX_I32


def _message(lib, rc, code=_lib.DX_EINVAL):
    assert rc == code, rc
    return lib.dx_last_error().decode()


def _append(lib, *, k=16, k_sl=256, pages=16, p_sr=256, dtype=BF, n_pages=4, rows=16, b=1, n=1, h=2,
            d=128, table=16, starts=16):
    return lib.dx_kv_page_append(k, 256, k_sl, 128, 16, 256, 256, 128, pages, 1 << 20, 4096, p_sr,
                                 128, dtype, n_pages, rows, table, 4, 4, starts, None, b, n, h, d,
                                 None)


def test_append_refusals(built_lib):
    lib = _lib.load()
    assert _append(lib, b=0) == _append(lib, n=0) == _lib.DX_OK  # nothing to do
    assert "dtype code 9" in _message(lib, _append(lib, dtype=9))
    assert "16-byte chunks" in _message(lib, _append(lib, d=4))
    assert "bad shape" in _message(lib, _append(lib, rows=0))
    assert "null pointer" in _message(lib, _append(lib, table=None))
    assert "null pointer" in _message(lib, _append(lib, starts=None))
    assert "null pages" in _message(lib, _append(lib, pages=None))
    assert "pointers must be 16-byte aligned" in _message(lib, _append(lib, k=20))
    assert "strides" in _message(lib, _append(lib, k_sl=4))
    assert "strides" in _message(lib, _append(lib, p_sr=4))
    assert "exceed one launch" in _message(lib, _append(lib, b=1 << 20, n=1 << 12))
    assert "below 2^31" in _message(lib, _append(lib, n_pages=1 << 31))


def _copy(lib, src, dst, *, pools=(16,), n_pages=8, dtype=BF, d=128, rows=16, p_sp=4096, h=2):
    arr = (ctypes.c_void_p * max(len(pools), 1))(*pools)
    ids = ctypes.c_int64 * max(len(src), 1)
    return lib.dx_kv_page_copy(arr, len(pools), 1 << 20, p_sp, 256, 128, dtype, n_pages, rows, h, d,
                               ids(*src), ids(*dst), len(src), None)


def test_copy_refusals(built_lib):
    lib = _lib.load()
    assert _copy(lib, [], []) == _lib.DX_OK
    assert _copy(lib, [1], [2], pools=()) == _lib.DX_OK
    assert "page 8 -> 1 outside a pool of 8" in _message(lib, _copy(lib, [8], [1]))
    assert "outside" in _message(lib, _copy(lib, [0], [-1]))
    assert "page 3 is written twice" in _message(lib, _copy(lib, [0, 1], [3, 3]))
    assert "page 2 is both read and written" in _message(lib, _copy(lib, [1, 2], [2, 3]))
    assert "page 5 is both read and written" in _message(lib, _copy(lib, [5], [5]))
    assert "16-byte aligned" in _message(lib, _copy(lib, [0], [1], pools=(16, 8)))
    assert "dtype code" in _message(lib, _copy(lib, [0], [1], dtype=I32))
    assert "16-byte chunks" in _message(lib, _copy(lib, [0], [1], d=3))
    assert "strides" in _message(lib, _copy(lib, [0], [1], p_sp=2))
    assert "fewer than 2^31" in _message(lib, _copy(lib, [0], [1], rows=1 << 30, h=1 << 10))


def _attend(lib, prefix=False, *, q=16, out=16, pages=16, dtype=BF, b=2, lq=4, lk=4, h=4, hkv=2,
            d=128, rows=16, width=3, table=16, lens=16, n_blocks=0, starts=None, causal=0, scale=1.0,
            ws=None, ws_bytes=0, p_sr=256, q_sl=512, p_width=2, p_table=16, p_len=16):
    z = lambda x: 0 if x is None else x  # noqa: E731
    call = _lib.PAGED_CALL.pack(
        z(q), 2048, q_sl, 128, 16, 1024, 256, 128, 16, 1024, 256, 128, z(out), 2048, 512, 128,
        z(pages), 1 << 20, 4096, p_sr, 128, 8, rows, z(table), width, width, z(lens),
        z(p_table), p_width, z(p_len), dtype, b, lq, lk, h, hkv, d, z(starts), I32, n_blocks,
        causal, scale, z(ws), ws_bytes, 0)
    return (lib.dx_shared_prefix_attention if prefix else lib.dx_paged_attention)(call)


def test_attention_refusals(built_lib):
    lib = _lib.load()
    assert "null call" in _message(lib, lib.dx_paged_attention(None))
    for prefix in (False, True):
        def bad(**kw):
            return _message(lib, _attend(lib, prefix, **kw))
        assert _attend(lib, prefix, b=0) == _attend(lib, prefix, lq=0, lk=0) == _lib.DX_OK
        assert "dtype code" in bad(dtype=7)
        assert "head_dim 96" in bad(d=96)
        assert "head_dim 256" in bad(d=256, dtype=F32)
        assert "not a multiple" in bad(h=4, hkv=3)
        assert "pages of 24 rows" in bad(rows=24)
        assert "pages of 2048 rows" in bad(rows=2048)
        assert "fewer than 2^30 rows" in bad(width=1 << 27)
        assert "must equal q length" in bad(lk=5, causal=1)
        assert "null block starts" in bad(n_blocks=3)
        assert "null pointer" in bad(q=None)
        assert "null block table" in bad(table=None)
        assert "null block table" in bad(lens=None)
        assert "null pages" in bad(pages=None)
        assert "aligned" in bad(out=20)
        assert "strides" in bad(q_sl=4)
        assert "row stride" in bad(p_sr=1 << 25)
        assert "finite" in bad(scale=float("inf"))
        assert "finite" in bad(scale=float("nan"))
        assert "finite" in bad(scale=3e38)  # times log2 e
    assert "null prefix table" in _message(lib, _attend(lib, True, p_table=None))
    assert "null prefix length" in _message(lib, _attend(lib, True, p_len=None))
    # A shared prefix always joins parts: its workspace has to be there.
    need = lib.dx_paged_attention_workspace_bytes(BF, 2, 4, 4, 4, 2, 128, 16, 3, 1, 2)
    assert need > 0
    assert str(need) in _message(lib, _attend(lib, True), _lib.DX_EWORKSPACE)
    assert lib.dx_paged_attention_workspace_bytes(BF, 2, 4, 4, 4, 3, 128, 16, 3, 1, 2) == -_lib.DX_EINVAL


def _tensors(b=2, lq=3, heads=4, kv=2, dim=64, rows=16, dtype=torch.bfloat16):
    return dict(q=torch.zeros(b, lq, heads, dim, dtype=dtype),
                k=torch.zeros(b, lq, kv, dim, dtype=dtype), v=torch.zeros(b, lq, kv, dim, dtype=dtype),
                pages=torch.zeros(2, 5, rows, kv, dim, dtype=dtype),
                table=torch.zeros(b, 4, dtype=torch.int32), lens=torch.zeros(b, dtype=torch.int32))


def _call(t, prefix=None, bb=None, causal=False, scale=None):
    return paged._attend("paged_attention", t["q"], t["k"], t["v"], t["pages"], prefix, t["table"],
                         t["lens"], bb, scale, causal)


@pytest.mark.parametrize("change,message", [
    (dict(lens=torch.zeros(2, dtype=torch.int64)), "cache_lens must be int32"),
    (dict(lens=torch.zeros(3, dtype=torch.int32)), "cache_lens must be int32 \\[2\\]"),
    (dict(lens=[0, 0]), "cache_lens must be int32"),
    (dict(lens=None), "go together"),
    (dict(table=torch.zeros(2, 4, dtype=torch.int64)), "block_table must be int32"),
    (dict(table=torch.zeros(3, 4, dtype=torch.int32)), "block_table must be int32"),
    (dict(table=torch.zeros(4, 2, dtype=torch.int32).t()), "contiguous rows"),
    (dict(pages=torch.zeros(2, 5, 16, 3, 64, dtype=torch.bfloat16)), "pages must be"),
    (dict(pages=torch.zeros(2, 5, 16, 2, 64)), "pages must be"),
    (dict(pages=torch.zeros(5, 16, 2, 64, dtype=torch.bfloat16)), "pages must be"),
    (dict(pages=torch.zeros(2, 5, 24, 2, 64, dtype=torch.bfloat16)), "multiple of 16"),
    (dict(pages=torch.zeros(2, 5, 0, 2, 64, dtype=torch.bfloat16)), "hold no rows"),
    (dict(pages=torch.zeros(2, 1, 16, 2, 64, dtype=torch.bfloat16).expand(2, 5, 16, 2, 64)),
     "must not be expanded"),
    (dict(pages=torch.zeros(2, 5, 16, 2, 68, dtype=torch.bfloat16)[..., :64]), "16-byte aligned"),
    (dict(k=torch.zeros(2, 3, 3, 64, dtype=torch.bfloat16),
          v=torch.zeros(2, 3, 3, 64, dtype=torch.bfloat16)), "must divide"),
    (dict(k=torch.zeros(2, 3, 2, 64), v=torch.zeros(2, 3, 2, 64)), "dtypes"),
])
def test_attention_argument_checks(change, message):
    with pytest.raises(ValueError, match=message):
        _call({**_tensors(), **change})


def test_attention_mask_and_prefix_checks():
    t = _tensors()
    short = {**t, "k": t["k"][:, :2], "v": t["v"][:, :2]}
    with pytest.raises(ValueError, match="must equal q length"):
        _call(short, causal=True)
    with pytest.raises(ValueError, match="must equal q length"):
        _call(short, bb=torch.tensor([0]))
    table, one = torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="prefix_len must be int32"):
        _call(t, prefix=(table, 7))
    with pytest.raises(ValueError, match="prefix_len must be int32"):
        _call(t, prefix=(table, table))
    with pytest.raises(ValueError, match="prefix_table must be int32"):
        _call(t, prefix=(table.long(), one))
    with pytest.raises(ValueError, match="prefix_table must be int32"):
        _call(t, prefix=(table[None], one))
    none = torch.zeros(2, 0, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no keys"):
        _call({**t, "k": none, "v": none, "table": torch.zeros(2, 0, dtype=torch.int32)})


def test_append_argument_checks():
    t = _tensors()

    def call(**change):
        a = {**t, "status": None, **change}
        paged.kv_page_append(a["pages"], a["k"], a["v"], a["table"], a["lens"], a["status"])
    for change, message in [
            (dict(table=t["table"].long()), "block_table must be int32"),
            (dict(lens=t["lens"].float()), "starts must be int32"),
            (dict(lens=7), "starts must be int32"),
            (dict(status=torch.zeros(2, dtype=torch.int32)), "status must be int32"),
            (dict(v=t["v"][:, :1]), "k and v must both be"),
            (dict(pages=t["pages"][:, :, :, :1]), "pages must be"),
            (dict(pages=t["pages"][:1]), "pages must be")]:
        with pytest.raises(ValueError, match=message):
            call(**change)


def test_tensors_off_the_gpu_are_refused():
    """A pinned implementation is called without its predicate: it checks the device itself."""
    t = _tensors()
    with pytest.raises(ValueError, match="GPU"):
        _call(t)
    with pytest.raises(ValueError, match="GPU"):
        paged.kv_page_append(t["pages"], t["k"], t["v"], t["table"], t["lens"])
    with pytest.raises(ValueError, match="GPU"):
        paged.kv_page_copy([t["pages"]], [0], [1])


def test_packed_call_matches_the_header():
    """PAGED_CALL has a field for each of struct dx_paged_call's, in its order."""
    text = HEADER.read_text()
    body = text[text.index("typedef struct dx_paged_call {"):text.index("} dx_paged_call;")]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    kinds = []
    for part in body.split(";"):
        words = part.replace("*", " ").split()
        if words:
            kinds += ["d" if "double" in words else "q"] * (part.count(",") + 1)
    fmt = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([qd])", _lib.PAGED_CALL.format))
    assert fmt == "".join(kinds) and _lib.PAGED_CALL.size == 8 * len(kinds)


def test_copy_argument_checks():
    pool = _tensors()["pages"]
    with pytest.raises(ValueError, match="2 source pages for 1"):
        paged.kv_page_copy([pool], [0, 1], [2])
    with pytest.raises(OverflowError):
        paged.kv_page_copy([pool], [2 ** 64 + 1], [2])
    with pytest.raises(TypeError):
        paged.kv_page_copy([pool], [1.0], [2])
    with pytest.raises(ValueError, match="needs a pool"):
        paged.kv_page_copy([], [0], [2])
    with pytest.raises(ValueError, match="must agree"):
        paged.kv_page_copy([pool, pool[:, :4]], [0], [2])
    with pytest.raises(ValueError, match="must agree"):
        paged.kv_page_copy([pool, pool.half()], [0], [2])
