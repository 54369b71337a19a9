"""A batch's row counts past the 32 bits of the struct are refused, not cut to what fits. On the CPU: they are looked at first."""
from __future__ import annotations

import pytest

import crosslane_amd as xl

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows,max_rows", [(2 ** 32 + 5, None), (5, 2 ** 32 + 1), (5, 2 ** 31), (-2 ** 32 + 5, 5), (0, None), (5, 0), (5, -1)])
def test_refused(rows, max_rows):
    i = torch.zeros((2, 4), dtype=torch.int32)
    cache = torch.zeros((3, 2, 32 * 160), dtype=torch.uint8)
    with pytest.raises(xl.XLError, match="rows"):
        xl.KVBatch(cache, i, i[:, 0], i[0, :3], rows, 128, max_rows)
    with pytest.raises(xl.XLError, match="not on the GPU"):   # (what is looked at next)
        xl.KVBatch(cache, i, i[:, 0], i[0, :3], 5, 128, 5)
