"""The 8-bit cache's entry points without a GPU: refusals, and the 64-bit reference itself."""
import numpy as np
import pytest
import torch

import q8_reference as ref
from flashinfer_mlsys2026_dsa_b200 import (_native, accumulate_weights, append_q8, compact_q8,
                                           evict_positions, kernel_q8, kernel_q8_paged)


def test_reference_rounding_is_e4m3s():
    """Every e4m3 value, the midpoints between neighbours and points beside them, against
    torch's own conversion."""
    grid = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    grid = grid[grid.isfinite()].sort().values.unique()
    mid = (grid[1:] + grid[:-1]) / 2
    x = torch.cat([grid, mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1)])
    np.testing.assert_array_equal(ref.e4m3(x.double().numpy()),
                                  x.to(torch.float8_e4m3fn).double().numpy())


@pytest.mark.parametrize("amax,scale", [(0.0, 2.0 ** -126), (448.0, 1.0), (448.5, 2.0), (1.75, 2.0 ** -8),
                                        (1.7578125, 2.0 ** -7), (1e-38, 2.0 ** -126)])
def test_reference_scale(amax, scale):
    assert ref.scale_for(amax) == scale


def test_calls_without_a_gpu_are_refused():
    q8, scale, kpe = ref.pools(2, 16, 8, 1, device="cpu")
    i32 = dict(dtype=torch.int32)
    q, qp = torch.zeros(1, 16, 512, dtype=torch.bfloat16), torch.zeros(1, 16, 64, dtype=torch.bfloat16)
    idx, table = torch.zeros(1, 4, **i32), torch.zeros(1, 1, **i32)
    out, lse = torch.empty(1, 16, 512, dtype=torch.bfloat16), torch.empty(1, 16)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_q8(q, qp, q8, scale, kpe, idx, 0.1, out, lse)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_q8_paged(q, qp, q8, scale, kpe, table, idx, 0.1, out, lse)
    with pytest.raises(ValueError, match="CUDA"):
        append_q8(q[0, :1], qp[0, :1], torch.tensor([0, 1], **i32), idx[0, :1], table, q8, scale, kpe)
    with pytest.raises(ValueError, match="CUDA"):
        accumulate_weights(torch.zeros(1, 4), idx, torch.zeros(1, 9))
    with pytest.raises(ValueError, match="CUDA"):
        evict_positions(torch.zeros(1, 9), idx[0, :1], 4)
    with pytest.raises(ValueError, match="CUDA"):
        compact_q8(idx, table, table, q8, scale, kpe)


# Host-side checks of the C ABI return before any CUDA call; 16 stands for an aligned pointer.
CACHE = [16, 512, 16, 64, 16, 64, 640]
TABLE = [16, 4, 4]


def _decode(heads=16, topk=64, cache=CACHE, table=(None, 0, 0), page=64, weights=(None, 0),
            scratch=(None, 0), ws=16, tokens=2):
    return _native.load().dsa_sparse_mla_decode_q8(
        16, 512 * heads, 512, 16, 64 * heads, 64, *cache, *table, page, 16, topk, 0.1,
        16, 512 * heads, 512, 16, heads, 1, *weights, tokens, heads, topk, *scratch, ws, None)


def test_decode_arguments():
    assert _decode(tokens=0) == 0
    assert _decode(heads=8) == 2
    assert _decode(topk=0) == 1
    assert _decode(ws=None) == 4
    for i, bad, code in ((0, None, 1), (0, 24, 3), (1, 511, 1), (1, 520, 3), (2, None, 1), (3, 48, 1),
                         (3, 512, 1), (4, 8, 3), (5, 63, 1), (5, 65, 3), (6, 0, 1), (6, 1 << 31, 1)):
        cache = list(CACHE)
        cache[i] = bad
        assert _decode(cache=cache) == code, (i, bad)
    assert _decode(table=(16, 4, 0)) == 1
    assert _decode(table=TABLE, page=48) == 1
    assert _decode(table=TABLE, page=32) == 1          # a block of 64 does not fit a page
    assert _decode(weights=(16, 63), scratch=(16, 1 << 30)) == 1
    assert _decode(weights=(16, 64)) == 4              # no scratch
    assert _decode(weights=(16, 64), scratch=(16, 64)) == 4
    assert _native.load().dsa_q8_scratch_size(2, 8, 64) == 0
    assert _native.load().dsa_q8_scratch_size(2, 16, 64) > 64


def test_append_arguments():
    lib = _native.load()

    def call(tokens=3, rows=2, ckv=16, sb=512, offsets=16, cache=CACHE, table=TABLE, page=64, ws=16):
        return lib.dsa_append_q8(ckv, sb, 16, 64, tokens, offsets, 16, rows, *table, page, *cache,
                                 ws, None)

    assert call(tokens=0) == 0 and call(rows=0) == 0
    assert call(tokens=-1) == 1 and call(rows=-1) == 1 and call(offsets=None) == 1
    assert call(ckv=18) == 3 and call(sb=516) == 3
    assert call(ws=None) == 4
    assert call(page=32) == 1 and call(table=[None, 4, 4]) == 1
    assert call(table=[16, 4, 1 << 26]) == 1           # positions past int32


def test_accumulate_evict_and_compact_arguments():
    lib = _native.load()

    def add(tokens=3, topk=4, rows=3, cols=10, sr=10, offsets=None, ws=16):
        return lib.dsa_accumulate_weights(16, 4, 16, 4, tokens, topk, 16, sr, cols, rows, offsets,
                                          ws, None)

    assert add(tokens=0) == 0 and add(rows=0) == 0
    assert add(topk=0) == 1 and add(rows=2) == 1 and add(sr=9) == 1 and add(ws=None) == 4

    def evict(rows=2, max_len=9, budget=4, sinks=1, recent=3, acc=16, ks=4, new=(None, 0, 0)):
        return lib.dsa_evict_positions(acc, 9, 16, rows, max_len, budget, sinks, recent, 32, ks, 48,
                                       *new, None)

    assert evict(rows=0) == 0
    assert evict(budget=0) == 1 and evict(recent=4) == 1 and evict(sinks=-1) == 1
    assert evict(acc=None) == 1 and evict(ks=3) == 1
    assert evict(new=(16, 4, 4)) == 1                  # the totals themselves
    assert evict(new=(64, 4, 3)) == 1 and evict(new=(64, 3, 4)) == 1

    def compact(rows=2, cols=4, cache=CACHE, old=TABLE, new=TABLE, page=64, ws=16):
        return lib.dsa_compact_q8(16, 4, rows, cols, *old, *new, page, *cache, ws, None)

    assert compact(rows=0) == 0 and compact(cols=0) == 0
    assert compact(cols=-1) == 1 and compact(page=32) == 1 and compact(new=[None, 4, 4]) == 1
    assert compact(ws=None) == 4 and compact(cols=1 << 23) == 1


def test_scratch_of_a_decode_with_weights():
    """Scores of at most 256 rows at a time: [rows, heads, whole tiles] fp32 and a tile number each."""
    lib = _native.load()
    size = lib.dsa_q8_scratch_size
    assert size(1, 16, 1) == (16 * 96 + 1) * 4
    assert size(256, 16, 2048) == 256 * 22 * (16 * 96 + 1) * 4
    assert size(1 << 20, 16, 2048) == size(256, 16, 2048)
    assert size(3, 128, 129) == 3 * 2 * (128 * 128 + 4) * 4
    assert size(0, 16, 2048) == size(1, 48, 2048) == size(1, 16, 0) == size(-1, 16, 1) == 0
