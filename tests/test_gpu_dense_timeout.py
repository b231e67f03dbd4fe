"""Dense attention whose waits run out: the call returns, the timeout bit is set, and what a CTA pair
gave up on is NaN, in output and lse; everything else keeps the bits of a call whose waits do not.

The limit of the waits is shortened (dsa_set_wait_limit) until sound waits run out: no fault or hang
is involved, every wait returns by itself.  With a limit of one cycle the warps that wait for the
first unit give up long before it is known.  The longer limits run out in some pairs, at other
points of their work, or in none, as the GPU's speed has it: what must hold, holds for each.
"""
import math

import pytest
import torch

import dense_reference as ref
from flashinfer_mlsys2026_dsa_b200 import (DSAError, _native, kernel_shared, kernel_window,
                                           read_device_errors, set_strict)

pytestmark = pytest.mark.gpu
SM = 1 / math.sqrt(192.0)
LIMITS = (1, 1, 1000, 3000, 5000, 8000, 12000, 20000, 40000)


def offsets(counts, first=0):
    return torch.tensor([first] + [first + sum(counts[:i + 1]) for i in range(len(counts))],
                        dtype=torch.int32, device="cuda")


def calls():
    """name -> (tokens, heads, call(output, lse)); tokens 0 and 1 of the ragged ones are of no row."""
    lens = [(37 * r) % 700 + 60 for r in range(64)]
    table, pages = ref.tables([-(-n // 64) for n in lens], 1)
    ckv, kpe = ref.pools(pages, 64, 2)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new = [23 + r % 3 for r in range(64)]
    total = 2 + sum(new)
    many, off = ref.queries(total, 128, 3), offsets(new, 2)
    one = ref.queries(64, 16, 4)
    few = ref.queries(2, 128, 5)
    long_table, pages = ref.tables([128], 6)
    long_pools = ref.pools(pages, 64, 7)
    long_n = torch.tensor([8000], dtype=torch.int32, device="cuda")
    return {
        # several units a pair, most of them whole
        "prompts": (total, 128, lambda o, z: kernel_window(*many, ckv, kpe, table, n, SM, o, z, 100, 4, row_offsets=off)),
        # a pair for each row, no join
        "rows": (64, 16, lambda o, z: kernel_window(*one, ckv, kpe, table, n, SM, o, z, 300)),
        # one unit cut over many pairs
        "long": (2, 128, lambda o, z: kernel_window(*few, *long_pools, long_table, long_n, SM, o, z, row_offsets=offsets([2]))),
        "shared": (total, 128, lambda o, z: kernel_shared(
            *many, ckv, kpe, table[:3], n[:3], table, n, SM, o, z, row_offsets=off,
            group_offsets=offsets([20, 0, 30]))),
        "shared rows": (64, 16, lambda o, z: kernel_shared(*one, ckv, kpe, table[5:6], n[5:6], table, n, SM, o, z)),
    }


def run(tokens, heads, call):
    out = torch.full((tokens, heads, 512), 7.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((tokens, heads), 7.0, device="cuda")
    call(out, lse)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("name", ["prompts", "rows", "long", "shared", "shared rows"])
def test_what_a_pair_gives_up_on_is_nan(name):
    case = calls()[name]
    read_device_errors(clear=True)
    want = run(*case)
    keep = want[1] == 7  # tokens of no row
    assert read_device_errors(clear=True) == 0 and want[1].isfinite().all()
    lib = _native.load()
    for limit in LIMITS:
        prev = lib.dsa_set_wait_limit(limit)
        try:
            out, lse = run(*case)
            word = read_device_errors(clear=True)
        finally:
            lib.dsa_set_wait_limit(prev)
        gone = lse.isnan()
        assert torch.equal(out[~gone], want[0][~gone]) and torch.equal(lse[~gone], want[1][~gone]), limit
        assert out[gone].isnan().all() and not gone[keep].any(), limit
        if gone.any() or (limit == 1 and name in ("prompts", "shared")):  # pairs of more units than the walker is ahead
            assert word & _native.DEVERR_TIMEOUT and gone.any(), limit
        # the next call is whole again
        out, lse = run(*case)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert read_device_errors(clear=True) == 0


def test_strict_mode_raises():
    lib = _native.load()
    read_device_errors(clear=True)
    for name in ("prompts", "shared"):
        case = calls()[name]
        was, prev = set_strict(True), lib.dsa_set_wait_limit(1)
        try:
            with pytest.raises(DSAError, match="ran out"):
                run(*case)
        finally:
            lib.dsa_set_wait_limit(prev)
            set_strict(was)
            read_device_errors(clear=True)
        run(*case)
        assert read_device_errors(clear=True) == 0
