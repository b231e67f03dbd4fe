"""The dense operators without a GPU: refusals, host checks of the C ABI, the 64-bit reference."""
import ctypes
import math
import random

import pytest
import torch

import dense_reference as ref
import dense_targets as aimed
from flashinfer_mlsys2026_dsa_b200 import _native, kernel_shared, kernel_window, merge_states


def test_reference_window_is_softmax_over_the_visible_positions():
    """attend() against torch.softmax with the rule written as loops."""
    ckv, kpe = ref.pools(3, 8, 1, "cpu")
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    qn, qp = ref.queries(3, 16, 2, "cpu")
    n, win, sinks = 19, 5, 2
    out, lse, _, _ = ref.window(qn, qp, ckv, kpe, table, [n], [3], 0.1, win, sinks, 8)
    keys = torch.cat([torch.cat([ckv[i], kpe[i]], 1) for i in (2, 0, 1)])[:n].double()
    for j in range(3):
        p = n - 3 + j
        some = [i for i in range(n) if i <= p and (i < sinks or i > p - win)]
        x = torch.cat([qn[j], qp[j]], 1).double() @ keys[some].T * 0.1
        torch.testing.assert_close(out[j], torch.softmax(x, 1) @ keys[some][:, :512])
        torch.testing.assert_close(lse[j], torch.logsumexp(x, 1) / math.log(2))


def test_reference_shared_is_the_window_over_joined_pages():
    ckv, kpe = ref.pools(6, 4, 3, "cpu")
    qn, qp = ref.queries(3, 16, 4, "cpu")
    pre, own = torch.tensor([[5, 1]], dtype=torch.int32), torch.tensor([[0, 2], [4, 3]], dtype=torch.int32)
    got = ref.shared(qn, qp, ckv, kpe, pre, [8], [2], own, [5, 7], [1, 2], 0.1, 4)
    whole = torch.cat([pre.expand(2, -1), own], 1)
    want = ref.window(qn, qp, ckv, kpe, whole, [13, 15], [1, 2], 0.1, None, 0, 4)
    torch.testing.assert_close(got[0], want[0])
    torch.testing.assert_close(got[1], want[1])


def test_reference_merge_joins_parts_of_one_softmax():
    ckv, kpe = ref.pools(4, 8, 5, "cpu")
    q = torch.cat(ref.queries(2, 16, 6, "cpu"), 2)
    keys = ref.sequence(ckv, kpe, torch.arange(4), 30, 8)
    seen = torch.ones(2, 30, dtype=torch.bool)
    first = torch.arange(30) < 11
    whole = ref.attend(q, keys, seen, 0.1)
    parts = [ref.attend(q, keys, seen & first, 0.1), ref.attend(q, keys, seen & ~first, 0.1)]
    out, lse, _, _ = ref.merge([x[0] for x in parts], [x[1] for x in parts])
    torch.testing.assert_close(out, whole[0])
    torch.testing.assert_close(lse, whole[1])


def test_calls_without_a_gpu_are_refused():
    ckv, kpe = ref.pools(2, 16, 1, "cpu")
    qn, qp = ref.queries(1, 16, 2, "cpu")
    out, lse = torch.empty_like(qn), torch.empty(1, 16)
    table, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_window(qn, qp, ckv, kpe, table, n, 0.1, out, lse, 4)
    with pytest.raises(ValueError, match="CUDA"):
        kernel_shared(qn, qp, ckv, kpe, table, n, table, n, 0.1, out, lse)
    with pytest.raises(ValueError, match="CUDA"):
        merge_states([out, out], [lse, lse], out, lse)
    for bad in (dict(window=-1), dict(sinks=-1)):
        with pytest.raises(ValueError, match=">= 0"):
            kernel_window(qn, qp, ckv, kpe, table, n, 0.1, out, lse, **bad)
    for outs, lses in (([], []), ([out] * 9, [lse] * 9), ([out], [lse, lse])):
        with pytest.raises(ValueError, match="parts"):
            merge_states(outs, lses, out, lse)


# Host checks return before any CUDA call; 16 stands for an aligned pointer.
Q = [16, 16 * 512, 512, 16, 16 * 64, 64]
POOLS = [16, 512, 16, 64, 640]
TABLE = [16, 4, 4]


def _window(q=Q, pools=POOLS, page=64, table=TABLE, lengths=16, offsets=None, rows=2, window=8,
            sinks=1, out=(16, 16 * 512, 512), lse=(16, 16, 1), tokens=2, heads=16, scratch=16,
            nbytes=1 << 40, ws=16):
    return _native.load().dsa_mla_decode_window(
        *q, *pools, page, *table, lengths, offsets, rows, window, sinks, 0.1, *out, *lse, tokens,
        heads, scratch, nbytes, ws, None)


def _shared(prefix=TABLE, plens=16, goffs=None, groups=1, tokens=2, rows=2, table=TABLE, page=64,
            ws=16, scratch=16):
    return _native.load().dsa_mla_decode_shared(
        *Q, *POOLS, page, *prefix, plens, goffs, groups, *table, 16, None, rows, 0.1,
        16, 16 * 512, 512, 16, 16, 1, tokens, 16, scratch, 1 << 40, ws, None)


def _with(values, i, x):
    values = list(values)
    values[i] = x
    return values


def test_window_arguments():
    assert _window(tokens=0, rows=0) == 0 and _window(tokens=0) == 0
    assert _window(heads=8) == 2 and _window(tokens=-1) == 1 and _window(rows=-1) == 1
    assert _window(rows=3) == 1                        # a token a row
    assert _window(window=-1) == 1 and _window(sinks=-1) == 1
    assert _window(page=0) == 1 and _window(page=48) == 1
    assert _window(lengths=None) == 1 and _window(ws=None) == 4
    assert _window(tokens=1 << 40, rows=2, offsets=16) == 1
    for i, bad, code in ((0, None, 1), (0, 24, 3), (1, 8193, 3), (2, 513, 3), (3, None, 1), (4, 1026, 3)):
        assert _window(q=_with(Q, i, bad)) == code, (i, bad)
    for i, bad, code in ((0, None, 1), (1, 511, 1), (1, 516, 3), (2, 8, 3), (3, 63, 1), (4, 0, 1),
                         (4, 1 << 31, 1)):
        assert _window(pools=_with(POOLS, i, bad)) == code, (i, bad)
    for i, bad in ((0, None), (1, 3), (2, 0), (2, 1 << 26)):
        assert _window(table=_with(TABLE, i, bad)) == 1, (i, bad)
    assert _window(out=(24, 16 * 512, 512)) == 3 and _window(out=(None, 1, 1)) == 1
    assert _window(lse=(None, 16, 1)) == 1
    assert _window(scratch=None) == 4 and _window(scratch=24) == 3


def test_lines_past_32_bits_are_refused():
    """A call's tiles are counted in 32 bits: 2^22 rows behind 2^19 positions pass them, with a
    window that leaves a tile of each they do not (and reach the device, which is not there)."""
    many = dict(tokens=1 << 22, rows=1 << 22, table=(16, 1 << 13, 1 << 13))
    assert _window(**many, window=1 << 30) == 1
    if not torch.cuda.is_available():
        assert _window(**many, window=10) == 5
    # a prefix of 2^26 positions for as many tokens as the call takes
    assert _shared(tokens=1 << 22, rows=1 << 22, prefix=(16, 1 << 20, 1 << 20)) == 1


def test_shared_arguments():
    assert _shared(tokens=0, rows=0) == 0
    assert _shared(groups=0) == 1 and _shared(groups=2) == 1 and _shared(plens=None) == 1
    assert _shared(prefix=[None, 4, 4]) == 1 and _shared(prefix=[16, 3, 4]) == 1
    assert _shared(prefix=[16, 1 << 26, 1 << 26]) == 1
    assert _shared(rows=1) == 1 and _shared(ws=None) == 4 and _shared(page=3) == 1


def test_scratch_size():
    size = _native.load().dsa_dense_scratch_size
    for bad in ((1, 8, 0), (-1, 16, 0), (1 << 40, 16, 1), (0, 16, 1)):
        assert size(*bad) == 0


def _merge(parts=2, outs=(1 << 20, 2 << 20), strides=(8192, 512) * 2, lses=(3 << 20, 4 << 20),
           lse_strides=(16, 1) * 2, out=(5 << 20, 8192, 512), lse=(6 << 20, 16, 1), tokens=3, heads=16):
    n = len(outs)
    return _native.load().dsa_merge_states(
        parts, (ctypes.c_void_p * n)(*outs), (ctypes.c_int64 * (2 * n))(*strides),
        (ctypes.c_void_p * n)(*lses), (ctypes.c_int64 * (2 * n))(*lse_strides), *out, *lse, tokens,
        heads, None)


def test_merge_arguments():
    assert _merge(tokens=0) == 0
    assert _merge(parts=0) == 1 and _merge(parts=9) == 1 and _merge(tokens=-1) == 1 and _merge(heads=0) == 1
    assert _merge(outs=(None, 16)) == 1 and _merge(lses=(16, None)) == 1
    assert _merge(outs=(24, 1 << 20)) == 3 and _merge(strides=(8192, 513, 8192, 512)) == 3
    assert _merge(out=(24, 8192, 512)) == 3 and _merge(out=(None, 1, 1)) == 1


def test_merge_refuses_a_result_that_overlaps_a_part():
    """A row of 16 heads is 16,384 bytes here, a token's lse 64."""
    first = 1 << 20
    for shift in (16, 1008, 1024, 16384, 2 * 16384, -1024, -16):
        assert _merge(out=(first + shift, 8192, 512)) == 1, shift
    for shift in (4, 60, 64, 128, -4):
        assert _merge(lse=((3 << 20) + shift, 16, 1)) == 1, shift
    # other strides over the same memory
    assert _merge(out=(first, 16384, 512)) == 1
    # interleaved with a part (rows between its rows, one of which would be met)
    assert _merge(strides=(16384, 512) * 2, out=(first + 16384 + 512, 16384, 512)) == 1


def test_merge_refuses_a_result_over_the_other_kind_of_part():
    """An lse inside a part's output, and an output over a part's lse."""
    first, z = 1 << 20, 3 << 20
    for at in (first, first + 512, first + 3 * 16384 - 4, (2 << 20) + 1024):
        assert _merge(lse=(at, 16, 1)) == 1, at
    for at in (z, z - 1008, z - 3 * 16384 + 16, (4 << 20) + 176):
        assert _merge(out=(at, 8192, 512)) == 1, at
    # beside each other in one buffer of 16 x (1024 + 16) bytes a token: the lse of the next head
    packed = dict(outs=(first, 2 << 20), strides=(8320, 520) * 2)
    assert _merge(**packed, lse=(first + 1020, 4160, 260)) == 1
    assert _merge(**packed, lse=(first + 1040 + 1020, 4160, 260)) == 1
    if not torch.cuda.is_available():  # what is no overlap reaches the device, which is not there
        assert _merge(lse=(first - 192, 16, 1)) == 5 and _merge(lse=(first + 3 * 16384, 16, 1)) == 5
        assert _merge(out=(z - 3 * 16384, 8192, 512)) == 5 and _merge(out=(z + 192, 8192, 512)) == 5
        assert _merge(**packed, lse=(first + 1024, 4160, 260)) == 5
        # a token's lses behind its outputs
        assert _merge(outs=(first, 2 << 20), strides=(8224, 512) * 2, lse=(first + 16384, 4112, 1)) == 5


def test_merge_takes_a_part_whose_unused_strides_differ():
    """With one token or one head, that stride says nothing."""
    first, z = 1 << 20, 3 << 20
    for tokens, heads, out, lse in ((1, 16, (first, 9999 * 8, 512), (z, 5, 1)), (3, 1, (first, 8192, 8), (z, 16, 77)),
                                    (1, 1, (first, 8, 16), (z, 9, 9))):
        if not torch.cuda.is_available():
            assert _merge(tokens=tokens, heads=heads, out=out, lse=lse) == 5
        assert _merge(tokens=tokens, heads=heads, out=(out[0] + 16, *out[1:])) == 1


def test_merge_overlaps_against_every_byte():
    """Random layouts near one another: what shares a byte is refused; with equal strides nothing else is."""
    if torch.cuda.is_available():
        pytest.skip("calls that are taken would run")
    rng = random.Random(1)
    taken = 0

    def rows(p, sb, sh, tokens, heads, width):
        return {p + t * sb + h * sh + i for t in range(tokens) for h in range(heads) for i in range(0, width, 4)}

    for _ in range(1500):
        tokens, heads = rng.choice((1, 2, 3)), rng.choice((1, 2, 3))
        sh = rng.choice((512, 520, 1040, 16)) if rng.random() < 0.8 else 3 * 520
        sb = rng.choice((512, heads * 520, heads * 1040 + 520, 520, 64))
        lse_at = (1 << 20) + 4 * rng.randrange(-400, 1200 * tokens)
        lb, lh = rng.choice(((sb // 2, sh // 2), (heads, 1), (sb // 2, 1), (3, 7)))
        got = _merge(parts=1, outs=(1 << 20,), strides=(sb, sh), lses=(8 << 20,), lse_strides=(lb, lh),
                     out=(16 << 20, sb, sh), lse=(lse_at, lb, lh), tokens=tokens, heads=heads)
        a = rows(1 << 20, 2 * sb, 2 * sh, tokens, heads, 1024)
        meets = not a.isdisjoint(rows(lse_at, 4 * lb, 4 * lh, tokens, heads, 4))
        assert got == (1 if meets else 5) or (got == 1 and (lb, lh) != (sb // 2, sh // 2))
        out_at = (1 << 20) + 16 * rng.randrange(-200, 300 * tokens)
        other = _merge(parts=1, outs=(1 << 20,), strides=(sb, sh), lses=(8 << 20,), lse_strides=(lb, lh),
                       out=(out_at, sb, sh), lse=(8 << 20, lb, lh), tokens=tokens, heads=heads)
        meets = not a.isdisjoint(rows(out_at, 2 * sb, 2 * sh, tokens, heads, 1024))
        assert other == (1 if meets and out_at != 1 << 20 else 5)
        taken += (got == 5) + (other == 5)
    assert taken > 500


def test_aimed_queries_show_a_value_from_a_wrong_place():
    """With a query for every eighth position, a chunk of 32 values that is left out, read as zero or
    taken from elsewhere is far outside the bound, and a chunk counted twice outside lse's."""
    n = 4096
    ckv, kpe = ref.pools(n // 64, 64, 1, "cpu")
    keys = ref.sequence(ckv, kpe, torch.arange(n // 64), n, 64)
    at = aimed.spread(n // 8, n)
    assert len(set(at.tolist())) == n // 8 and len(set((at // 32).tolist())) == n // 32
    qn, qp = aimed.aim(keys, at.view(1, n // 8))
    q = torch.cat([qn, qp], 2)
    sm = 1 / math.sqrt(192.0)
    out, lse, otol, ltol = ref.attend(q, keys, torch.ones(1, n, dtype=torch.bool), sm)
    p = torch.softmax(q[0].double() @ keys.T * sm, 1)
    assert p.gather(1, at[:, None]).min() > 0.9
    for a in (0, 32 * 77, n - 32):
        for values in (torch.zeros(32, 512, dtype=torch.float64), keys[(a + 192) % n:][:32, :512]):
            wrong = (out[0] + p[:, a:a + 32] @ (values - keys[a:a + 32, :512])).to(torch.bfloat16)
            off = ((wrong.double() - out[0]).abs() / otol[0]).amax(1)
            assert (off > 10).sum() >= 2, a
        twice = lse[0] + torch.log2(1 + p[:, a:a + 32].sum(1))
        assert (((twice - lse[0]) / ltol[0]) > 10).sum() >= 2
