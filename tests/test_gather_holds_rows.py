"""kv_page_gather's own copy of row numbers that are not contiguous lives until its launch (no GPU:
the library's entry point is replaced)."""

from __future__ import annotations

import torch

from dexter_amd.ops.gfx950 import _lib, keep


def test_a_copy_of_the_rows_outlives_the_call(monkeypatch):
    seen = []

    class Library:
        def dx_kv_page_gather(self, *args):
            ptr, count = args[14], args[15]
            # What another call of the same size would be given now, had the copy been freed.
            others = [torch.empty(2, 3, count, dtype=torch.int32) for _ in range(8)]
            seen.append((ptr, [t.data_ptr() for t in others]))
            return 0
    monkeypatch.setattr(keep, "_elsewhere", lambda device: False)
    monkeypatch.setattr(_lib, "load", Library)
    monkeypatch.setattr(_lib, "stream_handle", lambda device: 0)
    pool = torch.zeros(2, 5, 16, 3, 64, dtype=torch.bfloat16)
    table = torch.zeros(2, 4, dtype=torch.int32)
    wide = torch.zeros(2, 3, 80, dtype=torch.int32)
    for _ in range(4):
        keep.kv_page_gather(pool, table, wide[..., :40])
    keep.kv_page_gather(pool, table, wide)
    for ptr, others in seen[:4]:
        assert ptr != wide.data_ptr() and ptr not in others
    assert seen[4][0] == wide.data_ptr()  # contiguous ones are read in place
