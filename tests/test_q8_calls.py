"""Calls of the 8-bit cache that need no GPU: the ABI's refusals."""
import pytest
import torch

from flashinfer_mlsys2026_dsa_b200 import _native


def evict(acc, acc_stride, rows, max_len, budget, new, new_stride, new_cols):
    return _native.load().dsa_evict_positions(acc, acc_stride, 1 << 20, rows, max_len, budget, 0, 0, 1 << 21, budget,
                                              1 << 22, new, new_stride, new_cols, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are not the GPU's")
def test_new_totals_over_the_old_ones_are_refused():
    """Addresses in bytes, strides in floats: refused before any CUDA call."""
    a = 1 << 30
    assert evict(a, 100, 3, 100, 10, a, 100, 100) == 1
    assert evict(a, 100, 3, 100, 10, a + 4, 10, 10) == 1
    assert evict(a, 100, 3, 100, 10, a + 4 * 99, 10, 10) == 1
    assert evict(a, 100, 3, 100, 10, a + 4 * 250, 10, 10) == 1       # in the last row
    assert evict(a, 100, 3, 100, 10, a - 4 * 25, 10, 10) == 1        # its last row in the first
    assert evict(a, 200, 3, 100, 10, a + 4 * 95, 200, 10) == 1       # rows of one buffer, five columns shared
    assert evict(a, 200, 3, 100, 10, a + 4 * 100, 190, 90) == 1      # apart in row 0, not in row 1
    assert evict(a, 0, 5, 100, 10, a + 4 * 99, 10, 10) == 1          # one row for all
