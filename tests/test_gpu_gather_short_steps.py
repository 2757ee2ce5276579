"""kv_page_gather where its columns are many (MI355X): workgroups of 256 threads, whose steps are
short, against the oracle. Each case computes which form it takes.

A workgroup moves a column of 64 bytes (of less where a row has less) of one (sequence, head,
plane); 4-bit pools have one more column, of scales. Up to two columns to a compute unit a step is
of 1,024 rows, above that of 256.
"""

from __future__ import annotations

import pytest
import torch

from test_gpu_keep import _gather_case

pytestmark = pytest.mark.gpu
BF, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def _columns(dtype, dim, in4):
    chunks = dim // 32 if in4 else dim * dtype.itemsize // 16
    slice_ = min(4, chunks)
    while slice_ & (slice_ - 1):
        slice_ -= 1
    return 2 * (-(-chunks // slice_) + in4)


def _lens(batch, low, high):
    return [low + (high - low) * (7 * b % batch) // batch for b in range(batch)]


def _many(device, dtype, dim, in4, batch, heads):
    cus = torch.cuda.get_device_properties(device).multi_processor_count
    assert _columns(dtype, dim, in4) * batch * heads > 2 * cus


FORMS = [(BF, 128, False, 22, 3), (BF, 256, False, 11, 3), (F32, 72, False, 18, 3), (BF, 8, False, 64, 5),
         (U8, 64, True, 43, 3), (U8, 128, True, 43, 3), (U8, 256, True, 29, 3)]
IDS = [f"{str(t)[6:]}-{d}" for t, d, *_ in FORMS]


@pytest.mark.parametrize("dtype,dim,in4,batch,heads", FORMS, ids=IDS)
@pytest.mark.parametrize("new", [False, True])
def test_rows_and_weights(device, built_lib, dtype, dim, in4, batch, heads, new):
    """Three steps of rows, the last one short; weights over more than one step of theirs (2,048)."""
    _many(device, dtype, dim, in4, batch, heads)
    lens = [0, 1, 613, 614, 256] + _lens(batch - 5, 500, 1300)
    _gather_case(device, dtype, dim, in4, lens=lens, k=613, recent=50, heads=heads, new=new, rows=32,
                 extra_w=2000)


@pytest.mark.parametrize("dtype,dim,in4,batch,heads", FORMS[:1] + FORMS[5:], ids=IDS[:1] + IDS[5:])
@pytest.mark.parametrize("new", [False, True])
def test_each_row_one_place_down(device, built_lib, dtype, dim, in4, batch, heads, new):
    """Each step reads what lies just behind what it writes, across the steps' borders."""
    _many(device, dtype, dim, in4, batch, heads)
    down = torch.arange(1, 771, dtype=torch.int32).expand(batch, heads, 770).contiguous()
    _gather_case(device, dtype, dim, in4, lens=[771] * batch, k=770, heads=heads, new=new, rows=48, picked=down,
                 views=True)
