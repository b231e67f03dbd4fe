"""The dense operators on the GPU against tests/dense_reference.py in 64 bits."""
import math

import pytest
import torch

import dense_reference as ref
from flashinfer_mlsys2026_dsa_b200 import (_native, kernel, kernel_shared, kernel_window, merge_states,
                                           read_device_errors)

pytestmark = pytest.mark.gpu
SM = 1 / math.sqrt(192.0)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(counts, first=0):
    return i32([first] + [first + sum(counts[:i + 1]) for i in range(len(counts))])


def outputs(tokens, heads):
    """Buffers that hold something else before the call."""
    return (torch.full((tokens, heads, 512), 7.0, dtype=torch.bfloat16, device="cuda"),
            torch.full((tokens, heads), 7.0, device="cuda"))


def union(n, m, window, sinks):
    """Positions that any of a row's m tokens sees."""
    some = torch.zeros(n, dtype=torch.bool, device="cuda")
    for j in range(m):
        some |= ref.seen_window(n - m + j, n, window, sinks, "cuda")
    return some


def window_case(lens, new, heads, page, win, sinks, seed=1, poison=True, scale=SM):
    table, pages = ref.tables([-(-n // page) for n in lens], seed)
    ckv, kpe = ref.pools(pages, page, seed + 1)
    if poison:
        ref.poison(ckv, kpe, [table], [[union(n, m, win, sinks) for n, m in zip(lens, new)]], page)
    qn, qp = ref.queries(sum(new), heads, seed + 2)
    want = ref.window(qn, qp, ckv, kpe, table, lens, new, scale, win, sinks, page)
    return (qn, qp, ckv, kpe, table, i32(lens)), want


def run_window(lens, new, heads, page, win, sinks, seed=1, scale=SM):
    args, want = window_case(lens, new, heads, page, win, sinks, seed, scale=scale)
    out, lse = outputs(sum(new), heads)
    off = None if all(m == 1 for m in new) else offsets(new)
    kernel_window(*args, scale, out, lse, win, sinks, row_offsets=off)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")
    assert read_device_errors() == 0


@pytest.mark.parametrize("heads", [16, 32, 64, 128])
@pytest.mark.parametrize("win,sinks", [(1, 0), (32, 0), (33, 1), (200, 4), (640, 33), (None, 0), (0, 5)])
def test_window_one_token(heads, win, sinks):
    run_window([1, 2, 31, 32, 33, 191, 192, 193, 700, 1500], [1] * 10, heads, 64, win, sinks)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 64, 128, 256])
def test_window_pages(page):
    run_window([1, 7, 150, 517], [1, 3, 9, 2], 32, page, 100, 5)


@pytest.mark.parametrize("heads", [16, 32, 64, 128])
@pytest.mark.parametrize("win,sinks", [(1, 0), (50, 0), (100, 7), (300, 40), (None, 0), (0, 3)])
def test_window_many_tokens(heads, win, sinks):
    """Rows of 0 to 60 tokens, some of them the whole sequence."""
    run_window([5, 300, 0, 60, 411, 33, 130], [5, 1, 0, 60, 17, 8, 9], heads, 64, win, sinks)


def test_window_prompt_from_its_first_token():
    run_window([700], [700], 16, 64, 128, 4)
    run_window([230, 97], [230, 97], 128, 16, None, 0)


@pytest.mark.parametrize("rows", [1, 73, 74, 75, 148, 300])
def test_window_row_counts(rows):
    run_window([(37 * r) % 900 + 1 for r in range(rows)], [1] * rows, 16, 64, 333, 3)


def test_window_long_row_split_over_the_gpu():
    """One row whose positions are spread over all SMs, and two of unequal length."""
    run_window([20011], [1], 16, 64, None, 0)
    run_window([20011, 130], [2, 1], 128, 64, 15000, 64)


def test_window_of_everything_and_more():
    """A window or sinks past the sequence's length, up to the largest."""
    for win, sinks in ((10 ** 9, 0), (2 ** 31 - 1, 2 ** 31 - 1), (0, 10 ** 9), (5, 500)):
        args, want = window_case([90, 400], [2, 1], 16, 64, None if win > 400 or sinks > 400 else win, sinks)
        out, lse = outputs(3, 16)
        kernel_window(*args, SM, out, lse, win, sinks, row_offsets=offsets([2, 1]))
        ref.check(out, want[0], want[2], f"output {win} {sinks}")
        ref.check(lse, want[1], want[3], "lse")


def test_rows_of_length_zero_see_nothing():
    args, _ = window_case([0, 40, 0], [1, 1, 1], 16, 64, 10, 0, poison=False)
    out, lse = outputs(3, 16)
    kernel_window(*args, SM, out, lse, 10)
    assert not out[0].any() and not out[2].any() and (lse[0] == -math.inf).all() and (lse[2] == -math.inf).all()
    assert lse[1].isfinite().all()


def test_more_tokens_than_positions():
    """Tokens before the sequence's first position see nothing; the others what they would."""
    lens, new = [3], [5]
    table, pages = ref.tables([1], 1)
    ckv, kpe = ref.pools(pages, 64, 2)
    qn, qp = ref.queries(5, 16, 3)
    out, lse = outputs(5, 16)
    kernel_window(qn, qp, ckv, kpe, table, i32(lens), SM, out, lse, 10, row_offsets=offsets(new))
    want = ref.window(qn[2:], qp[2:], ckv, kpe, table, [3], [3], SM, 10, 0, 64)
    assert not out[:2].any() and (lse[:2] == -math.inf).all()
    ref.check(out[2:], want[0], want[2], "output")
    ref.check(lse[2:], want[1], want[3], "lse")


@pytest.mark.parametrize("scale", [0.0, -0.05, 1.0, 8.0])
def test_window_scales(scale):
    """Flat, turned round and sharp softmaxes (scores of hundreds in log2)."""
    run_window([300, 900], [1, 9], 32, 64, 500, 4, scale=scale)


def test_scores_that_grow_and_fall():
    """Keys aligned with the query whose size grows, falls or jumps along the sequence: the running
    maximum rises in every tile, never after the first, or once."""
    n = 1200
    table, pages = ref.tables([-(-n // 64)] * 3, 4)
    ckv, kpe = ref.pools(pages, 64, 5)
    qn, qp = ref.queries(3, 16, 6)
    at = torch.arange(n, device="cuda")
    for r, size in enumerate((at / n * 3, 3 - at / n * 3, (at == 777) * 5.0)):
        slot = table[r].long()[at // 64] * 64 + at % 64
        flat = ckv.view(-1, 512)
        flat[slot] += (size[:, None] * qn[r, 0].float()).to(torch.bfloat16)
    out, lse = outputs(3, 16)
    lens = [n] * 3
    kernel_window(qn, qp, ckv, kpe, table, i32(lens), SM, out, lse)
    want = ref.window(qn, qp, ckv, kpe, table, lens, [1] * 3, SM, None, 0, 64)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")


def test_a_nan_that_a_token_sees_reaches_it_and_no_other_row():
    args, want = window_case([200, 200, 200], [1, 1, 1], 16, 64, 100, 0, poison=False)
    ckv, table = args[2], args[4]
    ckv[int(table[1, 2]), 10, 3] = math.nan  # position 138 of row 1
    out, lse = outputs(3, 16)
    kernel_window(*args, SM, out, lse, 100)
    assert out[1].isnan().all() and lse[1].isnan().all()
    for r in (0, 2):
        ref.check(out[r], want[0][r], want[2][r], "output")
        ref.check(lse[r], want[1][r], want[3][r], "lse")


# ---------------------------------------------------------------------------- shared prefixes


def shared_case(pre, sizes, lens, new, heads, page, seed=1, poison=True):
    pre_table, n0 = ref.tables([-(-n // page) for n in pre], seed, spare=0)
    table, n1 = ref.tables([-(-n // page) for n in lens], seed + 7)
    order = torch.randperm(n0 + n1, generator=torch.Generator().manual_seed(seed)).to(torch.int32).cuda()
    pre_table = torch.where(pre_table >= 0, order[pre_table.long().clamp(min=0)], -1)
    table = torch.where(table >= 0, order[(table.long() + n0).clamp(max=n0 + n1 - 1)], -1)
    ckv, kpe = ref.pools(n0 + n1, page, seed + 1)
    if poison:
        full = [[torch.ones(n, dtype=torch.bool, device="cuda") for n in x] for x in (pre, lens)]
        ref.poison(ckv, kpe, [pre_table, table], full, page)
    qn, qp = ref.queries(sum(new), heads, seed + 2)
    want = ref.shared(qn, qp, ckv, kpe, pre_table, pre, sizes, table, lens, new, SM, page)
    return (qn, qp, ckv, kpe, pre_table, i32(pre), table, i32(lens)), want


def run_shared(pre, sizes, lens, new, heads, page=64, seed=1):
    args, want = shared_case(pre, sizes, lens, new, heads, page, seed)
    out, lse = outputs(sum(new), heads)
    off = None if all(m == 1 for m in new) else offsets(new)
    groups = None if len(pre) == 1 and sizes[0] == len(lens) else offsets(sizes)
    kernel_shared(*args, SM, out, lse, row_offsets=off, group_offsets=groups)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")
    assert read_device_errors() == 0


@pytest.mark.parametrize("heads", [16, 32, 64, 128])
@pytest.mark.parametrize("prefix", [1, 63, 192, 193, 1000, 5000])
def test_shared_one_group(heads, prefix):
    run_shared([prefix], [9], [1, 2, 64, 100, 191, 192, 193, 400, 33], [1] * 9, heads)


@pytest.mark.parametrize("heads", [16, 32, 64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_shared_groups_and_many_tokens(heads, page):
    """Groups of 1 to 6 rows, one without rows, rows without tokens and rows of no group."""
    run_shared([700, 5, 300, 64], [3, 1, 0, 6], [9, 40, 1, 20, 200, 3, 8, 70, 31, 64, 12, 90],
               [1, 4, 1, 9, 0, 3, 8, 2, 1, 20, 1, 2], heads, page)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 128])
def test_shared_pages(page):
    run_shared([150, 33], [2, 2], [7, 40, 9, 65], [1, 2, 9, 1], 16, page)


@pytest.mark.parametrize("rows", [1, 2, 8, 9, 100])
def test_shared_row_counts(rows):
    run_shared([400], [rows], [(29 * r) % 150 + 1 for r in range(rows)], [1] * rows, 16)


def test_shared_rows_of_length_zero_see_the_prefix_alone():
    args, _ = shared_case([333], [2], [1, 5], [1, 1], 16, 64, poison=False)
    qn, qp, ckv, kpe, pre_table, pre, table, lens = args
    out, lse = outputs(2, 16)
    kernel_shared(qn, qp, ckv, kpe, pre_table, pre, table, i32([0, 5]), SM, out, lse)
    whole = ref.window(qn[:1], qp[:1], ckv, kpe, pre_table, [333], [1], SM, None, 0, 64)
    ref.check(out[:1], whole[0], whole[2], "output")
    ref.check(lse[:1], whole[1], whole[3], "lse")


def test_shared_prefix_of_length_zero():
    args, _ = shared_case([5], [2], [100, 5], [1, 1], 16, 64, poison=False)
    qn, qp, ckv, kpe, pre_table, pre, table, lens = args
    out, lse = outputs(2, 16)
    kernel_shared(qn, qp, ckv, kpe, pre_table, i32([0]), table, i32([100, 0]), SM, out, lse)
    whole = ref.window(qn[:1], qp[:1], ckv, kpe, table, [100], [1], SM, None, 0, 64)
    ref.check(out[:1], whole[0], whole[2], "output")
    ref.check(lse[:1], whole[1], whole[3], "lse")
    assert not out[1].any() and (lse[1] == -math.inf).all()


# ----------------------------------------------------------------------------- how it is called


def test_tokens_of_no_row_are_left_as_they_are():
    lens, new = [40, 300], [3, 2]
    args, want = window_case(lens, new, 16, 64, 100, 2, poison=False)
    qn, qp, rest = args[0], args[1], args[2:]
    pad = lambda x: torch.cat([x[:2] * math.nan, x, x[:4] * math.nan])  # noqa: E731
    out, lse = outputs(11, 16)
    kernel_window(pad(qn), pad(qp), *rest, SM, out, lse, 100, 2, row_offsets=offsets(new, 2))
    assert (out[:2] == 7).all() and (out[7:] == 7).all() and (lse[:2] == 7).all() and (lse[7:] == 7).all()
    ref.check(out[2:7], want[0], want[2], "output")
    ref.check(lse[2:7], want[1], want[3], "lse")
    args, want = shared_case([100], [2], lens, new, 16, 64, poison=False)
    out, lse = outputs(11, 16)
    kernel_shared(pad(args[0]), pad(args[1]), *args[2:], SM, out, lse, row_offsets=offsets(new, 2))
    assert (out[:2] == 7).all() and (out[7:] == 7).all() and (lse[:2] == 7).all() and (lse[7:] == 7).all()
    ref.check(out[2:7], want[0], want[2], "output")
    ref.check(lse[2:7], want[1], want[3], "lse")


@pytest.mark.parametrize("inner", [False, True])
def test_strides(inner):
    """One [tokens, heads, 576] query, one [slots, 576] cache, strided outputs, tables and lengths;
    with `inner`, no unit inner stride anywhere but in the cache."""
    lens, new = [200, 77, 500], [1, 4, 2]
    args, want = window_case(lens, new, 32, 64, 130, 9, poison=False)
    qn, qp, ckv, kpe, table, n = args
    q = torch.cat([qn, qp], 2)
    cache = torch.cat([ckv, kpe], 2)
    T = sum(new)
    out = torch.full((T, 2, 32, 512), 7.0, dtype=torch.bfloat16, device="cuda")[:, 1]
    lse = torch.full((32, T), 7.0, device="cuda").t()
    qa, qb, tab = q[..., :512], q[..., 512:], torch.stack([table, table], 1)[:, 0]
    off = offsets(new)
    if inner:
        qa, qb = (x.permute(2, 0, 1).contiguous().permute(1, 2, 0) for x in (qa, qb))
        out = torch.full((512, T, 32), 7.0, dtype=torch.bfloat16, device="cuda").permute(1, 2, 0)
        tab = table.t().contiguous().t()
        n = torch.stack([n, n], 1)[:, 0]
        off = torch.stack([off, off], 1)[:, 0]
    kernel_window(qa, qb, cache[..., :512], cache[..., 512:], tab, n, SM, out, lse, 130, 9, row_offsets=off)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")


def test_flat_pools_and_page_size():
    args, want = window_case([100, 250], [1, 1], 16, 32, 90, 2)
    qn, qp, ckv, kpe, table, n = args
    for size in (32, None):
        out, lse = outputs(2, 16)
        a = (qn, qp, ckv.view(-1, 512), kpe.view(-1, 64), table, n, SM, out, lse, 90, 2)
        if size is None:
            with pytest.raises(ValueError, match="page_size"):
                kernel_window(*a)
            continue
        kernel_window(*a, page_size=size)
        ref.check(out, want[0], want[2], "output")


@pytest.mark.parametrize("page", [4, 16, 64])
def test_positions_without_a_page_are_left_out_and_flagged(page):
    lens = [300, 300, 300]
    args, _ = window_case(lens, [1, 1, 1], 16, page, None, 0, poison=False)
    qn, qp, ckv, kpe, table, n = args
    table = table.clone()
    hole = 128 // page
    table[0, hole] = -1                       # a page missing in the middle
    table[1, hole] = ckv.shape[0]             # a page outside the pool
    read_device_errors()
    out, lse = outputs(3, 16)
    kernel_window(qn, qp, ckv, kpe, table, n, SM, out, lse)
    assert read_device_errors() == 1
    keys = ref.sequence(ckv, kpe, args[4][0], 300, page), ref.sequence(ckv, kpe, args[4][1], 300, page)
    at = torch.arange(300, device="cuda") // page
    for r in (0, 1):
        q = torch.cat([qn[r:r + 1], qp[r:r + 1]], 2)
        want = ref.attend(q, keys[r], (at != hole)[None], SM)
        ref.check(out[r:r + 1], want[0], want[2], "output")
        ref.check(lse[r:r + 1], want[1], want[3], "lse")
    # a length past the table
    out, lse = outputs(3, 16)
    have = args[4].shape[1] * page
    kernel_window(qn, qp, ckv, kpe, args[4], i32([300, have + 77, 2 ** 31 - 1]), SM, out, lse)
    assert read_device_errors() == 1
    want = ref.window(qn[:1], qp[:1], ckv, kpe, args[4], [300], [1], SM, None, 0, page)
    ref.check(out[:1], want[0], want[2], "output")


def test_offsets_past_32_bits():
    """Slots whose byte offsets pass 2^32 and whose element offsets pass 2^31."""
    page, pages = 64, 70000
    ckv = torch.empty(pages, page, 512, dtype=torch.bfloat16, device="cuda")
    kpe = torch.empty(pages, page, 64, dtype=torch.bfloat16, device="cuda")
    table = i32([[69999, 3, 69990, 65535, 65536], [0, 69998, 32768, 2, 69000]])
    for t in table.flatten().tolist():
        a, b = ref.pools(1, page, t)
        ckv[t], kpe[t] = a[0], b[0]
    qn, qp = ref.queries(2, 16, 3)
    out, lse = outputs(2, 16)
    kernel_window(qn, qp, ckv, kpe, table, i32([300, 310]), SM, out, lse)
    want = ref.window(qn, qp, ckv, kpe, table, [300, 310], [1, 1], SM, None, 0, page)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")


def test_same_bits_in_every_run():
    w, _ = window_case([3000, 50, 700], [1, 9, 33], 16, 64, 2000, 4, poison=False)
    s, _ = shared_case([3000, 90], [20, 13], [(17 * r) % 300 + 3 for r in range(33)], [1 + r % 3 for r in range(33)],
                       16, 64, poison=False)
    first = None
    for _ in range(4):
        a, b = outputs(43, 16), outputs(sum(1 + r % 3 for r in range(33)), 16)
        kernel_window(*w, SM, *a, 2000, 4, row_offsets=offsets([1, 9, 33]))
        kernel_shared(*s, SM, *b, row_offsets=offsets([1 + r % 3 for r in range(33)]),
                      group_offsets=offsets([20, 13]))
        got = [x.clone() for x in (*a, *b)]
        first = first or got
        for x, y in zip(first, got):
            assert torch.equal(x, y)


def test_graphs_follow_lengths_and_offsets():
    lens, new = [130, 400, 64], [1, 3, 2]
    w, _ = window_case([700] * 3, [3, 3, 3], 16, 64, 100, 2, poison=False)
    s, _ = shared_case([500], [3], [700] * 3, [3, 3, 3], 16, 64, poison=False)
    off, wl, sl, pl = offsets([3, 3, 3]), w[5].clone(), s[7].clone(), s[5].clone()
    a, b, c = outputs(9, 16), outputs(9, 16), outputs(9, 16)

    def step():
        kernel_window(*w[:5], wl, SM, *a, 100, 2, row_offsets=off)
        kernel_shared(*s[:5], pl, s[6], sl, SM, *b, row_offsets=off)
        merge_states([a[0], b[0]], [a[1], b[1]], *c)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        # the capture's stream has a workspace of its own
        step()
    off.copy_(offsets(new))
    wl.copy_(i32(lens))
    sl.copy_(i32(lens))
    pl.copy_(i32([77]))
    for x in (*a, *b, *c):
        x.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    T = sum(new)
    want = ref.window(w[0][:T], w[1][:T], *w[2:5], lens, new, SM, 100, 2, 64)
    ref.check(a[0][:T], want[0], want[2], "output")
    ref.check(a[1][:T], want[1], want[3], "lse")
    want = ref.shared(s[0][:T], s[1][:T], *s[2:5], [77], [3], s[6], lens, new, SM, 64)
    ref.check(b[0][:T], want[0], want[2], "output")
    ref.check(b[1][:T], want[1], want[3], "lse")
    want = ref.merge([a[0][:T], b[0][:T]], [a[1][:T], b[1][:T]])
    ref.check(c[0][:T], want[0], want[2], "output")
    assert (a[0][T:] == 7).all() and (b[0][T:] == 7).all()


def test_streams_overlap():
    """Calls on two streams at once, each with its own scratch."""
    w, want = window_case([3000, 50, 700], [1, 9, 33], 16, 64, 2000, 4, poison=False)
    s, want2 = shared_case([2000], [9], [100] * 9, [1] * 9, 32, 64, poison=False)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    got, off = [], offsets([1, 9, 33])
    torch.cuda.synchronize()
    for _ in range(5):
        a, b = outputs(43, 16), outputs(9, 32)
        other.wait_stream(torch.cuda.current_stream())
        kernel_window(*w, SM, *a, 2000, 4, row_offsets=off)
        with torch.cuda.stream(other):
            kernel_shared(*s, SM, *b)
        got.append((a, b))
    torch.cuda.synchronize()
    for a, b in got:
        ref.check(a[0], want[0], want[2], "output")
        ref.check(b[0], want2[0], want2[2], "output")


@pytest.mark.parametrize("rows", [33, 513, 1025, 1600])
def test_window_many_rows(rows):
    """More rows than lanes, than threads and than twice that; every ninth sees nothing."""
    lens = [0 if r % 9 == 4 else (53 * r) % 400 + 1 for r in range(rows)]
    args, want = window_case([max(n, 1) for n in lens], [1] * rows, 16, 64, 150, 2)
    out, lse = outputs(rows, 16)
    kernel_window(*args[:5], i32(lens), SM, out, lse, 150, 2)
    live = torch.tensor([n > 0 for n in lens], device="cuda")
    ref.check(out[live], want[0][live], want[2][live], "output")
    ref.check(lse[live], want[1][live], want[3][live], "lse")
    assert not out[~live].any() and (lse[~live] == -math.inf).all()


@pytest.mark.parametrize("groups", [20, 40, 300, 700])
def test_shared_many_groups(groups):
    """Groups of 0 to 3 rows of 1 to 3 tokens; 40 and more with their rows are over 32 entries."""
    sizes = [g % 4 for g in range(groups)]
    rows = sum(sizes)
    run_shared([(29 * g) % 330 + 1 for g in range(groups)], sizes, [(37 * r) % 90 + 3 for r in range(rows)],
               [1 + r % 3 for r in range(rows)], 32, 32)


def test_queries_and_tables_that_rows_share():
    """Strides of 0: one token's query and one page list for all rows."""
    args, _ = window_case([400], [1], 16, 64, 120, 3, poison=False)
    qn, qp, ckv, kpe, table, _ = args
    lens = [400, 1, 77, 300]
    q = qn.expand(4, -1, -1), qp.expand(4, -1, -1)
    out, lse = outputs(4, 16)
    kernel_window(*q, ckv, kpe, table.expand(4, -1), i32([400]).expand(4).clone(), SM, out, lse, 120, 3)
    want = ref.window(*q, ckv, kpe, table.expand(4, -1), [400] * 4, [1] * 4, SM, 120, 3, 64)
    ref.check(out, want[0], want[2], "output")
    kernel_window(*q, ckv, kpe, table.expand(4, -1), i32(lens), SM, out, lse, 120, 3)
    want = ref.window(*q, ckv, kpe, table.expand(4, -1), lens, [1] * 4, SM, 120, 3, 64)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")


def test_slots_behind_the_last_whole_page():
    """A flat pool of three pages and a half: what lies behind the third is no page."""
    ckv, kpe = (x.view(-1, w)[:3 * 64 + 32] for x, w in zip(ref.pools(4, 64, 3), (512, 64)))
    qn, qp = ref.queries(1, 16, 4)
    read_device_errors()
    out, lse = outputs(1, 16)
    kernel_window(qn, qp, ckv, kpe, i32([[2, 3, 0]]), i32([192]), SM, out, lse, page_size=64)
    assert read_device_errors() == 1
    pools = ckv[:192].view(3, 64, 512), kpe[:192].view(3, 64, 64)
    keys = ref.sequence(*pools, i32([2, 0, 0]), 192, 64)
    seen = torch.arange(192, device="cuda") // 64 != 1
    want = ref.attend(torch.cat([qn, qp], 2), keys, seen[None], SM)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")


def test_two_graphs_at_once():
    """Two graphs captured on one stream, replayed in turn on it and side by side on two."""
    w, want = window_case([3000, 50, 700], [1, 9, 33], 16, 64, 2000, 4, poison=False)
    s, want2 = shared_case([2000], [9], [100] * 9, [1] * 9, 32, 64, poison=False)
    off = offsets([1, 9, 33])
    a, b = outputs(43, 16), outputs(9, 32)
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()

    def one():
        kernel_window(*w, SM, *a, 2000, 4, row_offsets=off)

    def two():
        kernel_shared(*s, SM, *b)

    torch.cuda.synchronize()
    graphs = []
    with torch.cuda.stream(stream):
        for step in (one, two):
            step()
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=stream):
                step()
    torch.cuda.synchronize()
    for apart in (False, True):
        for x in (*a, *b):
            x.fill_(7)
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(stream):
                graphs[0].replay()
            with torch.cuda.stream(other if apart else stream):
                graphs[1].replay()
        torch.cuda.synchronize()
        for got, exp in ((a, want), (b, want2)):
            ref.check(got[0], exp[0], exp[2], "output")
            ref.check(got[1], exp[1], exp[3], "lse")


def test_scratch_that_is_too_small_is_refused():
    lib = _native.load()
    args, _ = window_case([100], [1], 16, 64, 10, 0, poison=False)
    qn, qp, ckv, kpe, table, n = args
    out, lse = outputs(1, 16)
    ws = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    for shared in (0, 1):
        size = lib.dsa_dense_scratch_size(1, 16, shared)
        assert size > 0
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        for nbytes in (size - 1, 0):
            head = (qn.data_ptr(), 8192, 512, qp.data_ptr(), 1024, 64, ckv.data_ptr(), 512,
                    kpe.data_ptr(), 64, ckv.shape[0] * 64, 64)
            own = (table.data_ptr(), table.stride(0), table.shape[1], n.data_ptr(), None, 1)
            tail = (0.1, out.data_ptr(), 8192, 512, lse.data_ptr(), 16, 1, 1, 16, scratch.data_ptr(),
                    nbytes, ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
            if shared:
                rc = lib.dsa_mla_decode_shared(*head, *own[:4], None, 1, *own, *tail)
            else:
                rc = lib.dsa_mla_decode_window(*head, *own, 10, 0, *tail)
            assert rc == 4
    torch.cuda.synchronize()
    assert (out == 7).all() and (lse == 7).all()


# --------------------------------------------------------------------------------- the join


@pytest.mark.parametrize("parts", [1, 2, 3, 8])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (3, 16), (70, 128), (33, 7)])
def test_merge(parts, tokens, heads):
    g = torch.Generator(device="cuda").manual_seed(parts * 100 + tokens)
    outs = [torch.randn(tokens, heads, 512, generator=g, device="cuda").to(torch.bfloat16) for _ in range(parts)]
    lses = [torch.randn(tokens, heads, generator=g, device="cuda") * 6 for _ in range(parts)]
    gone = torch.rand(parts, tokens, heads, generator=g, device="cuda") < 0.3
    for i in range(parts):
        outs[i][gone[i]] = math.nan  # a part without weight may hold anything
        lses[i][gone[i]] = -math.inf
    want = ref.merge(outs, lses)
    out, lse = outputs(tokens, heads)
    merge_states(outs, lses, out, lse)
    ref.check(out, want[0], want[2], "output")
    ref.check(lse, want[1], want[3], "lse")
    # into a part's own place, strided
    both = torch.stack(outs, 1)
    zs = torch.stack(lses, 2)
    merge_states([both[:, i] for i in range(parts)], [zs[..., i] for i in range(parts)],
                 both[:, parts - 1], zs[..., 0])
    ref.check(both[:, parts - 1], want[0], want[2], "output in place")
    ref.check(zs[..., 0], want[1], want[3], "lse in place")


def test_merge_of_far_lses_and_nan():
    outs = [torch.full((4, 1, 512), float(i + 1), dtype=torch.bfloat16, device="cuda") for i in range(2)]
    lses = [torch.tensor([[500.0], [-500.0], [3e38], [math.nan]], device="cuda"),
            torch.tensor([[-500.0], [500.0], [-3e38], [1.0]], device="cuda")]
    out, lse = outputs(4, 1)
    merge_states(outs, lses, out, lse)
    assert (out[0] == 1).all() and (out[1] == 2).all() and (out[2] == 1).all()
    assert lse[:3, 0].tolist() == [500.0, 500.0, torch.tensor(3e38).item()]
    assert out[3].isnan().all() and lse[3].isnan().all()


def test_merge_refusals():
    out, lse = outputs(4, 16)
    a, b = outputs(4, 16)
    buf = torch.zeros(5, 16, 512, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        merge_states([buf[:4], a], [b, b], buf[1:], lse)
    z = torch.zeros(5, 16, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        merge_states([a, a], [z[1:], b], out, z[:4])
    with pytest.raises(TypeError, match="bfloat16"):
        merge_states([a.float()], [b], out, lse)
    with pytest.raises(ValueError, match="part 1"):
        merge_states([a, a[:3]], [b, b[:3]], out, lse)
    with pytest.raises(ValueError, match="CUDA"):
        merge_states([a, a.cpu()], [b, b], out, lse)


def test_refusals():
    args, _ = window_case([100, 100], [1, 1], 16, 64, 10, 0, poison=False)
    qn, qp, ckv, kpe, table, n = args
    out, lse = outputs(2, 16)

    def call(i=None, x=None, **kw):
        a = [qn, qp, ckv, kpe, table, n, SM, out, lse, 10]
        if i is not None:
            a[i] = x
        kernel_window(*a, **kw)

    call()
    for i, x, error in ((0, qn.float(), TypeError), (0, qn[..., :500], ValueError), (1, qp[:1], ValueError),
                        (2, ckv.float(), TypeError), (2, ckv[..., :64], ValueError), (3, kpe[:1], ValueError),
                        (4, table.long(), TypeError), (4, table[:1], ValueError), (5, n.long(), TypeError),
                        (5, n.cpu(), ValueError), (5, n[:1], ValueError), (7, out[:1], ValueError),
                        (7, out.float(), TypeError), (8, lse.double(), TypeError), (4, None, TypeError),
                        (5, [100, 100], TypeError), (9, -1, ValueError)):
        with pytest.raises(error):
            call(i, x)
    with pytest.raises(ValueError, match="row_offsets"):
        call(row_offsets=i32([0, 2]))
    with pytest.raises(ValueError, match="power of two"):
        call(page_size=48)
    with pytest.raises(ValueError, match="num_heads"):
        call(0, qn[:, :8])
    s, _ = shared_case([70, 80], [1, 1], [100, 100], [1, 1], 16, 64, poison=False)
    with pytest.raises(ValueError, match="group_offsets"):
        kernel_shared(*s, SM, out, lse)
    with pytest.raises(ValueError, match="group_offsets"):
        kernel_shared(*s, SM, out, lse, group_offsets=i32([0, 2]))
    with pytest.raises(ValueError, match="prefix_table"):
        kernel_shared(*s[:4], s[4][:1], *s[5:], SM, out, lse, group_offsets=i32([0, 1, 2]))
    torch.cuda.synchronize()


def test_empty_batches():
    args, _ = window_case([100], [1], 16, 64, 10, 0, poison=False)
    out, lse = outputs(0, 16)
    kernel_window(args[0][:0], args[1][:0], *args[2:4], args[4][:0], args[5][:0], SM, out, lse, 10)
    merge_states([out], [lse], out, lse)


def test_sparse_and_window_attention_joined():
    """A step of a model that attends to its window and sinks and, before them, to selected
    positions: `kernel` over the selection, the window, and the join, against one softmax."""
    lens, heads, page, win, sinks, topk = [900, 1500, 260, 40], 32, 64, 200, 4, 64
    args, _ = window_case(lens, [1] * 4, heads, page, None, 0, poison=False)
    qn, qp, ckv, kpe, table, n = args
    g = torch.Generator().manual_seed(5)
    picked = []
    for length in lens:
        middle = list(range(sinks, max(sinks, length - win)))
        order = torch.randperm(len(middle), generator=g)[:topk].sort().values.tolist()
        picked.append([middle[i] for i in order])
    idx = torch.full((4, topk), -1, dtype=torch.int32, device="cuda")
    for r, pos in enumerate(picked):
        if pos:
            p = torch.tensor(pos, device="cuda")
            idx[r, :len(pos)] = (table[r].long()[p // page] * page + p % page).to(torch.int32)
    sparse, near, out = outputs(4, heads), outputs(4, heads), outputs(4, heads)
    kernel(qn, qp, ckv, kpe, idx, SM, *sparse)
    kernel_window(qn, qp, ckv, kpe, table, n, SM, *near, win, sinks)
    merge_states([sparse[0], near[0]], [sparse[1], near[1]], *out)
    for r, length in enumerate(lens):
        seen = ref.seen_window(length - 1, length, win, sinks, "cuda")
        seen[picked[r]] = True
        keys = ref.sequence(ckv, kpe, table[r], length, page)
        want = ref.attend(torch.cat([qn[r:r + 1], qp[r:r + 1]], 2), keys, seen[None], SM)
        # each part's output was rounded to bf16 before the join: 2^-8 of the values' weighted size
        k = keys[seen]
        p = torch.softmax(torch.cat([qn[r], qp[r]], 1).double() @ k.T * SM, 1)
        more = 2.0 ** -8 * (p @ k[:, :512].abs())
        ref.check(out[0][r:r + 1], want[0], want[2] + more + 2.0 ** -18, "output")
        ref.check(out[1][r:r + 1], want[1], want[3] + 2.0 ** -18, "lse")


def test_merge_in_place_through_another_view_and_in_one_buffer():
    """One token whose part has another (unused) stride; outputs and lses of a token in one row."""
    for tokens in (1, 5):
        g = torch.Generator(device="cuda").manual_seed(tokens)
        outs = [torch.randn(tokens, 16, 512, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
        lses = [torch.randn(tokens, 16, generator=g, device="cuda") for _ in range(2)]
        want = ref.merge(outs, lses)
        buf = torch.zeros(tokens, 16, 520, dtype=torch.bfloat16, device="cuda")
        out, lse = buf[..., :512], buf.view(torch.float32)[..., 256]
        merge_states(outs, lses, out, lse)
        ref.check(out, want[0], want[2], "output")
        ref.check(lse, want[1], want[3], "lse")
        out.copy_(outs[0])
        lse.copy_(lses[0])
        own = out.as_strided(out.shape, (8 * 999, *out.stride()[1:])) if tokens == 1 else out
        merge_states([own, outs[1]], [lse, lses[1]], out, lse)
        ref.check(out, want[0], want[2], "output in place")
        ref.check(lse, want[1], want[3], "lse in place")
        with pytest.raises(ValueError, match="overlap"):
            merge_states([out, outs[1]], lses, out, out[..., 0:2].view(torch.float32)[..., 0])


def test_page_sizes_below_one_are_refused():
    """By the direct route of a second call too, which writes "the pools' page size" as -1."""
    args, _ = window_case([100], [1], 16, 64, 10, 0, poison=False)
    s, _ = shared_case([70], [1], [100], [1], 16, 64, poison=False)
    out, lse = outputs(1, 16)
    kernel_window(*args, SM, out, lse, 10)
    for size in (0, -1, -64):
        with pytest.raises(ValueError, match="power of two"):
            kernel_window(*args, SM, out, lse, 10, page_size=size)
        with pytest.raises(ValueError, match="power of two"):
            kernel_shared(*s, SM, out, lse, page_size=size)
