"""Workspaces of attention over pages with log-sum-exps (no GPU: planned for 256 compute units)."""

from __future__ import annotations

import pytest

from dexter_amd.ops.gfx950 import _lib

BF, F16, F32, I32 = _lib.DX_BF16, _lib.DX_F16, _lib.DX_F32, _lib.DX_I32
# B, Lq, Lk, H, Hkv, D, rows of a page, width, has prefix, prefix width: cut lines, split ones, both.
SHAPES = [(2, 4, 4, 4, 2, 128, 16, 100, 0, 0), (1, 83, 83, 24, 24, 128, 128, 256, 0, 0),
          (8, 83, 83, 24, 24, 64, 64, 6, 1, 129), (3, 1, 1, 8, 2, 64, 16, 3, 1, 2)]


@pytest.mark.parametrize("shape", SHAPES)
def test_second_sums_are_part_of_it(built_lib, shape):
    """A partial row of D sums, a maximum and a sum has one more number in 16 bits; in fp32 the one
    sum serves both."""
    lib, dim = _lib.load(), shape[5]
    for dtype in (BF, F16, F32):
        plain = lib.dx_paged_attention_workspace_bytes(dtype, *shape)
        with_lse = lib.dx_paged_attention_lse_workspace_bytes(dtype, *shape)
        assert plain > 0
        if dtype == F32:
            assert with_lse == plain
            continue
        rows = (with_lse - plain) // 4
        assert rows > 0 and (with_lse - plain) % (4 * 32) == 0
        records = plain - rows * (4 * dim + 8)  # what is no partial row: 16 bytes for each item
        assert records >= 0 and records % 16 == 0
    assert lib.dx_paged_attention_lse_workspace_bytes(BF, 2, 4, 4, 4, 3, 128, 16, 3, 1, 2) == -_lib.DX_EINVAL
    assert lib.dx_paged_attention_lse_workspace_bytes(BF, 0, *SHAPES[0][1:]) == 0


def _call(lib, name, dtype, fp4, ws_bytes, lse):
    page = 2048 if fp4 else 4096
    call = _lib.PAGED_CALL.pack(
        16, 2048, 512, 128, 16, 1024, 256, 128, 16, 1024, 256, 128, 16, 2048, 512, 128,
        16, 1 << 20, page, 256, 128 if not fp4 else 1088, 8, 16, 16, 100, 100, 16, 16, 2, 16, dtype, 2, 4, 4,
        4, 2, 128, 0, I32, 0, 0, 1.0, 16, ws_bytes, 0)
    return getattr(lib, name)(call, lse)


@pytest.mark.parametrize("fp4", [False, True])
def test_a_plain_workspace_is_too_small(built_lib, fp4):
    """Refused before anything is launched, with what is needed."""
    lib = _lib.load()
    for prefix, name in enumerate(("dx_paged_attention", "dx_shared_prefix_attention")):
        shape = (2, 4, 4, 4, 2, 128, 16, 100, prefix, 2 * prefix)
        plain = lib.dx_paged_attention_workspace_bytes(BF, *shape)
        need = lib.dx_paged_attention_lse_workspace_bytes(BF, *shape)
        name += "_fp4" if fp4 else "_lse"
        assert need > plain
        assert _call(lib, name, BF, fp4, plain, 16) == _lib.DX_EWORKSPACE
        assert f"workspace of {plain} bytes, {need} needed" in lib.dx_last_error().decode()
        if fp4:  # without an lse a byte less than the plain one is what is missing
            assert _call(lib, name, BF, fp4, plain - 1, None) == _lib.DX_EWORKSPACE
            assert f"{plain} needed" in lib.dx_last_error().decode()
