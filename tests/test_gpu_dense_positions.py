"""Long sequences in which each query rests on one position of its own (tests/dense_targets.py):
values from a wrong place, at any turn of the ring, tile, chunk or cut, are far outside the bounds."""
import math

import pytest
import torch

import dense_reference as ref
import dense_targets as aimed
from flashinfer_mlsys2026_dsa_b200 import kernel_shared, kernel_window, read_device_errors

pytestmark = pytest.mark.gpu
SM = 1 / math.sqrt(192.0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(counts):
    return i32([sum(counts[:i]) for i in range(len(counts) + 1)])


def outputs(tokens, heads):
    return (torch.full((tokens, heads, 512), 7.0, dtype=torch.bfloat16, device="cuda"),
            torch.full((tokens, heads), 7.0, device="cuda"))


def compare(out, lse, want):
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")
    assert read_device_errors() == 0


def window_queries(ckv, kpe, table, lens, new, heads, page, win, sinks):
    """Query i of a row's tokens x heads rests on one of the positions that all its tokens see."""
    parts = []
    for r, (n, m) in enumerate(zip(lens, new)):
        keys = ref.sequence(ckv, kpe, table[r], n, page)
        seen = ref.seen_window(n - m, n, win, sinks) & ref.seen_window(n - 1, n, win, sinks)
        some = torch.nonzero(seen)[:, 0]
        at = some[aimed.spread(m * heads, len(some), 7 * r)]
        parts.append(aimed.aim(keys, at.view(m, heads)))
    return tuple(torch.cat(x) for x in zip(*parts))


@pytest.mark.parametrize("lens,new,heads,page,win,sinks", [
    ([20011], [40], 128, 64, None, 0),              # one row over the whole GPU
    ([20011], [320], 16, 8, None, 0),
    ([9000, 130, 6000], [40, 1, 60], 64, 16, 5000, 64),
    ([5000] * 74, [1] * 74, 128, 64, 3000, 4),      # a pair for each row
    ([5000, 4100, 800], [1, 1, 1], 128, 1, None, 0),
], ids=["20011_h128", "20011_h16", "window_h64", "rows_h128", "pages_of_1"])
def test_window(lens, new, heads, page, win, sinks):
    table, pages = ref.tables([-(-n // page) for n in lens], 1)
    ckv, kpe = ref.pools(pages, page, 2)
    qn, qp = window_queries(ckv, kpe, table, lens, new, heads, page, win, sinks)
    out, lse = outputs(sum(new), heads)
    kernel_window(qn, qp, ckv, kpe, table, i32(lens), SM, out, lse, win, sinks, row_offsets=offsets(new))
    compare(out, lse, ref.window(qn, qp, ckv, kpe, table, lens, new, SM, win, sinks, page))


@pytest.mark.parametrize("pre,sizes,lens,new,heads,page", [
    # decode behind a long system prompt: 4,096 query rows, one for every eighth position
    ([32768], [256], [(29 * r) % 300 + 1 for r in range(256)], [1] * 256, 16, 64),
    ([8000, 5001], [9, 12], [(29 * r) % 300 + 8 for r in range(21)], [1 + r % 8 for r in range(21)], 128, 32),
    # new questions of hundreds of tokens behind a prefix
    ([3000], [3], [1700, 900, 700], [700, 900, 33], 16, 64),
    ([1500, 600], [1, 2], [400, 300, 260], [260, 300, 1], 128, 16),
], ids=["32768_b256", "two_groups_h128", "prompts_h16", "prompts_h128"])
def test_shared(pre, sizes, lens, new, heads, page):
    pre_table, n0 = ref.tables([-(-n // page) for n in pre], 1, spare=0)
    table, n1 = ref.tables([-(-n // page) for n in lens], 8)
    table = torch.where(table >= 0, table + n0, -1)
    ckv, kpe = ref.pools(n0 + n1, page, 3)
    prefixes = [ref.sequence(ckv, kpe, pre_table[g], n, page) for g, n in enumerate(pre)]
    parts, used = [], [0] * len(pre)
    row = 0
    for g, size in enumerate(sizes):
        for r in range(row, row + size):
            n, m = lens[r], new[r]
            own = ref.sequence(ckv, kpe, table[r], n, page)
            # four of five queries rest on the prefix, one on what all the row's tokens see of its own
            pick = aimed.aim(prefixes[g], aimed.spread(m * heads, pre[g], used[g]).view(m, heads))
            if n > m:
                near = aimed.aim(own, aimed.spread(m * heads, n - m + 1, r).view(m, heads))
                for a, b in zip(pick, near):
                    a.view(m * heads, -1)[::5] = b.view(m * heads, -1)[::5]
            used[g] += 3 * r + 1
            parts.append(pick)
        row += size
    qn, qp = (torch.cat(x) for x in zip(*parts))
    out, lse = outputs(sum(new), heads)
    kernel_shared(qn, qp, ckv, kpe, pre_table, i32(pre), table, i32(lens), SM, out, lse,
                  row_offsets=offsets(new), group_offsets=offsets(sizes))
    compare(out, lse, ref.shared(qn, qp, ckv, kpe, pre_table, pre, sizes, table, lens, new, SM, page))


def test_rows_before_and_behind_the_groups_have_no_prefix():
    """Groups that begin behind the first row and end before the last; some without rows."""
    pre, lens, new, heads, page = [700, 300, 90], [33, 200, 64, 9, 150, 400, 77], [1, 3, 2, 1, 9, 2, 1], 32, 64
    pre_table, n0 = ref.tables([-(-n // page) for n in pre], 1, spare=0)
    table, n1 = ref.tables([-(-n // page) for n in lens], 8)
    table = torch.where(table >= 0, table + n0, -1)
    ckv, kpe = ref.pools(n0 + n1, page, 3)
    qn, qp = ref.queries(sum(new), heads, 4)
    out, lse = outputs(sum(new), heads)
    kernel_shared(qn, qp, ckv, kpe, pre_table, i32(pre), table, i32(lens), SM, out, lse,
                  row_offsets=offsets(new), group_offsets=i32([2, 4, 4, 6]))
    t = [sum(new[:r]) for r in range(len(new) + 1)]
    for a, b, g in ((0, 2, None), (2, 4, 0), (4, 6, 2), (6, 7, None)):
        x = slice(t[a], t[b])
        some = (qn[x], qp[x], ckv, kpe)
        rest = (table[a:b], lens[a:b], new[a:b], SM)
        want = ref.window(*some, *rest, None, 0, page) if g is None else \
            ref.shared(*some, pre_table[g:g + 1], pre[g:g + 1], [b - a], *rest, page)
        compare(out[x], lse[x], want)
