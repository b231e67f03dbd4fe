"""Calls of the 8-bit cache that need no GPU: the ABI's refusals and the documented serving step."""
import os
import re

import pytest
import torch

from flashinfer_mlsys2026_dsa_b200 import _native, build


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


def test_the_documented_serving_step_counts_the_new_tokens():
    """The step of INTEGRATION.md, run with stand-ins for the calls: the eviction is given lengths
    that include what the append has written, and returns the lengths that the next append takes."""
    text = open(os.path.join(build.REPO_DIR, "INTEGRATION.md")).read()
    step, = [s for s in re.findall(r"```python\n(.*?)```", text, re.S) if "append_q8(" in s]
    seen = {}

    def append_q8(ckv, kpe, row_offsets, starts, *_):
        seen["starts"] = starts.tolist()

    def evict_positions(acc, lengths, budget, **_):
        seen["lengths"] = lengths.tolist()
        return None, lengths.clamp(max=budget)

    names = dict.fromkeys(("ckv", "kpe", "page_table", "ckv_q8", "ckv_scale", "kpe_cache", "q_nope", "q_pe",
                           "positions", "sm_scale", "output", "lse", "weights", "acc", "new_acc", "keep",
                           "new_page_table"))
    names.update(append_q8=append_q8, evict_positions=evict_positions, budget=64,
                 row_offsets=torch.tensor([0, 1, 1, 4], dtype=torch.int32),
                 lengths=torch.tensor([7, 0, 90], dtype=torch.int32))
    for name in ("kernel_q8_paged", "accumulate_weights", "compact_q8"):
        names[name] = lambda *_, **__: None
    exec(step, names)
    assert seen["starts"] == [7, 0, 90]
    assert seen["lengths"] == [8, 0, 93]
    assert names["lengths"].tolist() == [8, 0, 64] and names["lengths"].dtype == torch.int32
