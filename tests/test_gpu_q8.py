"""The 8-bit cache's kernels against their definitions in 64 bits (tests/q8_reference.py)."""
import math

import numpy as np
import pytest
import torch

import q8_reference as ref
from flashinfer_mlsys2026_dsa_b200 import (DSAError, _native, accumulate_weights, append_q8,
                                           compact_q8, evict_positions, kernel_q8,
                                           kernel_q8_paged, read_device_errors)

pytestmark = pytest.mark.gpu
SM = 1.0 / math.sqrt(192.0)
NAN = float("nan")


@pytest.fixture(autouse=True)
def clean_errors():
    read_device_errors(clear=True)
    yield
    read_device_errors(clear=True)


def queries(B, H, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed + 100)
    q = torch.randn(B, H, 576, generator=g).mul(size).to(torch.bfloat16).cuda()
    return q[..., :512].contiguous(), q[..., 512:].contiguous()


def selection(B, topk, slots, seed=0, short=True):
    """Distinct slots per row; rows cut to 0, 1 and odd counts, with padding in the middle."""
    g = torch.Generator().manual_seed(seed + 200)
    idx = torch.stack([torch.randperm(slots, generator=g)[:topk] if topk <= slots else
                       torch.randint(0, slots, (topk,), generator=g) for _ in range(B)]).to(torch.int32)
    if short:
        for b in range(B):
            if b % 4 == 1:
                idx[b, topk // 3:] = -1
            if b % 4 == 2:
                idx[b, torch.randperm(topk, generator=g)[:topk // 2]] = -1
            if b % 4 == 3:
                idx[b] = -1
        if B > 4:
            idx[4, 1:] = -1
    return idx.cuda()


def run(q, cache, idx, table=None, weights=True, sm=SM):
    B, H, _ = q[0].shape
    out = torch.full((B, H, 512), NAN, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((B, H), NAN, device="cuda")
    w = torch.full(idx.shape, NAN, device="cuda") if weights else None
    if table is None:
        kernel_q8(*q, *cache, idx, sm, out, lse, weights=w)
    else:
        kernel_q8_paged(*q, *cache, table, idx, sm, out, lse, weights=w)
    torch.cuda.synchronize()
    return (out, lse, w) if weights else (out, lse)


def check(got, q, cache, slots, sm=SM):
    out, lse, w, out_tol, lse_tol = ref.attend(*q, *cache, slots, sm)
    dead = ~torch.isfinite(lse)
    g = got[1].cpu().double()
    assert torch.equal(g[dead], lse[dead])
    assert (g - lse)[~dead].abs().le(lse_tol[~dead]).all()
    assert (got[0].cpu().double() - out).abs().le(out_tol + 1e-30).all()
    if len(got) > 2:
        tol = w * (lse_tol.amax(1)[:, None] * 2 + 2.0 ** -18) + 1e-30
        assert (got[2].cpu().double() - w).abs().le(tol).all()


@pytest.mark.parametrize("topk", [1, 2, 31, 32, 33, 95, 96, 97, 128, 191, 193, 300, 1001, 2048])
@pytest.mark.parametrize("heads", [16, 32, 64, 128])
def test_attend(heads, topk):
    cache = ref.pools(40, 64, 16, topk)
    q, idx = queries(6, heads, topk), selection(6, topk, 40 * 64, topk)
    got = run(q, cache, idx)
    check(got, q, cache, idx)
    assert read_device_errors() == 0
    assert torch.equal(got[2][idx < 0], torch.zeros_like(got[2][idx < 0]))
    again = run(q, cache, idx, weights=False)
    assert torch.equal(got[0].view(torch.int16), again[0].view(torch.int16))
    assert torch.equal(got[1], again[1])


@pytest.mark.parametrize("page,block", [(1, 1), (16, 1), (16, 16), (64, 64), (128, 128), (256, 256), (64, 8)])
def test_attend_blocks_and_pages(page, block):
    pages = 2048 // page
    cache = ref.pools(pages, page, block, block, spread=1.5)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).to(torch.int32).cuda().view(4, -1)
    pos = selection(4, 211, 512, 5)
    slots = torch.where(pos >= 0, table.gather(1, (pos.clamp(min=0) // page).long()) * page + pos % page, -1)
    q = queries(4, 16, block)
    got = run(q, cache, pos, table)
    check(got, q, cache, slots)
    flat = run(q, cache, slots.to(torch.int32))
    for a, b in zip(got, flat):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,heads,topk", [(1, 16, 4096), (3, 64, 2500), (200, 16, 130), (150, 32, 97),
                                             (80, 128, 100), (300, 16, 1)])
def test_attend_row_counts(rows, heads, topk):
    """From one long row to more rows than SMs."""
    cache = ref.pools(80, 64, 64, rows)
    q, idx = queries(rows, heads, rows), selection(rows, topk, 80 * 64, rows)
    check(run(q, cache, idx), q, cache, idx)
    check(run(q, cache, idx, weights=False), q, cache, idx)


@pytest.mark.parametrize("heads", [16, 64])
def test_attend_many_rows_most_of_them_empty(heads):
    """Twenty rows and more per SM, in runs of empty ones (also an SM's first and last)."""
    rows, topk = 3100, 230
    cache = ref.pools(8, 64, 16, heads)
    g = torch.Generator().manual_seed(heads)
    idx = torch.randint(0, 512, (rows, topk), generator=g, dtype=torch.int32)
    cut = torch.where(torch.rand(rows, generator=g) < 0.2, torch.randint(0, topk + 1, (rows,), generator=g), 0)
    cut[:150] = 0
    cut[-40:] = 0
    cut[1200:1900] = 0
    idx[torch.arange(topk)[None] >= cut[:, None]] = -1
    idx = idx.cuda()
    q = queries(rows, heads, heads)
    check(run(q, cache, idx), q, cache, idx)
    check(run(q, cache, idx, weights=False), q, cache, idx)


def test_attend_repeated_slots_and_long_selections():
    """A slot named twice counts twice; topk past the pool, and past 16 bits."""
    cache = ref.pools(4, 64, 32, 9)
    q, idx = queries(2, 16, 9), selection(2, 70001, 256, 9, short=False)
    check(run(q, cache, idx), q, cache, idx)


def test_attend_scales_of_very_different_size():
    """Scales from 2^-100 to 2^60 in one row, zero among them: the large ones decide."""
    q8, scale, kpe = ref.pools(32, 64, 16, 4)
    e = torch.linspace(-100, 60, scale.numel()).round()[torch.randperm(scale.numel(), generator=torch.Generator().manual_seed(1))]
    small = torch.exp2(e).clamp(max=2.0 ** -9).view_as(scale).cuda()
    small[3] = 0
    q, idx = queries(4, 16, 4), selection(4, 700, 2048, 4)
    check(run(q, (q8, small, kpe), idx), q, (q8, small, kpe), idx)
    # the same cache scaled by 2^60 against queries scaled down: exact powers of two
    big = small * 2.0 ** 60
    qs = (q[0] * 2.0 ** -60, q[1])
    check(run(qs, (q8, big, kpe), idx), qs, (q8, big, kpe), idx)


@pytest.mark.parametrize("heads", [16, 32, 128])
def test_attend_scales_and_scores_that_grow(heads):
    """Every tile raises the running maximum or the running scale: each is carried over."""
    q8, scale, kpe = ref.pools(32, 64, 32, 6)
    scale = torch.exp2(torch.arange(scale.numel()).float() / 8).view_as(scale).cuda() * 2.0 ** -12
    idx = torch.arange(2048, dtype=torch.int32).repeat(3, 1).cuda()
    idx[1] = idx[1].flip(0)
    idx[2, 1::2] = -1
    q = queries(3, heads, 6, 0.3)
    check(run(q, (q8, scale, kpe), idx), q, (q8, scale, kpe), idx)
    # scores of a few hundred: one entry takes nearly all of a head's weight
    cache = ref.pools(32, 64, 32, 7)
    q = queries(3, heads, 7, 30.0)
    check(run(q, cache, idx), q, cache, idx)


def test_attend_a_heavy_entry_over_many_equal_ones():
    """One entry with half the weight and 2047 equal small ones that share the rest."""
    q8 = torch.zeros(32, 64, 512, dtype=torch.float8_e4m3fn, device="cuda")
    raw = q8.view(torch.uint8)
    raw[..., 1:] = 0x35                                   # 0.8125 in every value but the first
    raw[0, 0, 0], raw[0, 0, 1:] = 0x78, 0xB5              # the heavy one: 256, and -0.8125
    scale = torch.full((32, 2), 1.0, device="cuda")
    kpe = torch.zeros(32, 64, 64, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 16, 512, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = math.log(2047.0) / 256 / SM
    q = (q, torch.zeros(1, 16, 64, dtype=torch.bfloat16, device="cuda"))
    idx = torch.arange(2048, dtype=torch.int32, device="cuda")[None]
    for order in (idx, idx.flip(1)):
        check(run(q, (q8, scale, kpe), order), q, (q8, scale, kpe), order)


def test_attend_queries_of_any_size():
    """Query rows of zeros, of one large value beside tiny ones, and up to 2^60."""
    cache = ref.pools(8, 64, 16, 3)
    cache = (cache[0], cache[1] * 2.0 ** -62, cache[2])
    q = queries(2, 16, 3)
    qn = q[0].clone()
    qn[0, 0] = 0
    qn[0, 1] *= 2.0 ** -30
    qn[0, 2] *= 2.0 ** 60
    qn[0, 3, 1:] *= 2.0 ** -20
    qn[1] *= 2.0 ** 40
    idx = selection(2, 333, 512, 3, short=False)
    check(run((qn, q[1]), cache, idx), (qn, q[1]), cache, idx)


def test_attend_nan_and_infinity_stay_where_they_are():
    q8, scale, kpe = ref.pools(8, 64, 16, 2)
    q, idx = queries(4, 16, 2), selection(4, 100, 256, 2, short=False)
    clean = run(q, (q8, scale, kpe), idx)
    # behind no index: NaN and infinities in the other half of every pool change nothing
    q8.view(torch.uint8)[4:] = 0x7F
    scale[4:] = NAN
    kpe[4:] = math.inf
    idx[0, 50:] = -1
    dirty = run(q, (q8, scale, kpe), idx)
    for a, b in zip(clean, dirty):
        assert torch.equal(a[1:], b[1:]) and torch.isfinite(b.float()).all()
    # behind one index of row 2: that row alone
    idx[2, 7] = 300
    bad = run(q, (q8, scale, kpe), idx)
    assert torch.isnan(bad[0][2].float()).all() and torch.isnan(bad[1][2]).all()
    for a, b in zip(dirty, bad):
        assert torch.equal(a[[0, 1, 3]], b[[0, 1, 3]])
    # a query row: that head alone
    idx[2, 7] = 0
    dirty = run(q, (q8, scale, kpe), idx)
    for value in (NAN, math.inf):
        q2 = (q[0].clone(), q[1])
        q2[0][1, 5, 9] = value
        bad = run(q2, (q8, scale, kpe), idx)
        assert torch.isnan(bad[0][1, 5].float()).all() and torch.isnan(bad[1][1, 5])
        keep = torch.ones(4, 16, dtype=torch.bool)
        keep[1, 5] = False
        assert torch.equal(dirty[0][keep], bad[0][keep]) and torch.equal(dirty[1][keep], bad[1][keep])


def test_attend_entries_without_a_slot_are_flagged_and_left_out():
    cache = ref.pools(4, 64, 16, 8)
    q, idx = queries(2, 16, 8), selection(2, 40, 256, 8, short=False)
    idx[0, 3], idx[0, 9], idx[1, 39] = 256, -2, 2 ** 31 - 1
    got = run(q, cache, idx)
    assert read_device_errors() == _native.DEVERR_BAD_INDEX
    left = idx.masked_fill((idx < 0) | (idx >= 256), -1)
    check(got, q, cache, left)
    table = torch.tensor([[2, 0, 9, -1], [1, 3, 2, 0]], dtype=torch.int32, device="cuda")
    pos = torch.tensor([[5, 70, 130, 200, 256, -7, -1]] * 2, dtype=torch.int32, device="cuda")
    got = run(q, cache, pos, table)
    assert read_device_errors() == _native.DEVERR_BAD_INDEX
    slots = torch.tensor([[133, 6, -1, -1, -1, -1, -1], [69, 198, 130, 8, -1, -1, -1]], dtype=torch.int32)
    check(got, q, cache, slots.cuda())


def test_attend_strides():
    """One pool of 640-byte slots, queries as one [B, H, 576], transposed heads, wide outputs,
    one page table and one selection for all rows."""
    q8, scale, kpe = ref.pools(16, 64, 32, 5)
    both = torch.zeros(16, 64, 640, dtype=torch.uint8, device="cuda")
    both[..., :512] = q8.view(torch.uint8)
    both[..., 512:] = kpe.view(torch.uint8)
    joint = (both[..., :512].view(torch.float8_e4m3fn), scale, both[..., 512:].view(torch.bfloat16))
    q = queries(3, 32, 5)
    cat = torch.cat(q, 2)
    idx = selection(3, 150, 1024, 5)
    want = run(q, (q8, scale, kpe), idx)
    wide = torch.full((3, 40, 600), NAN, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((32, 3), NAN, device="cuda").t()
    w = torch.full((3, 150, 2), NAN, device="cuda")
    kernel_q8(cat[..., :512], cat[..., 512:], *joint, idx, SM, wide[:, 4:36, 8:520], lse, weights=w[..., 0])
    assert torch.equal(wide[:, 4:36, 8:520], want[0]) and torch.equal(lse, want[1])
    assert torch.equal(w[..., 0], want[2]) and torch.isnan(w[..., 1]).all()
    wide[:, 4:36, 8:520] = NAN
    assert torch.isnan(wide.float()).all()
    qt = (q[0].transpose(0, 1).contiguous().transpose(0, 1), q[1].transpose(0, 1).contiguous().transpose(0, 1))
    got = run(qt, joint, idx.t().contiguous().t())
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    table = torch.arange(15, -1, -1, dtype=torch.int32, device="cuda")[None].expand(3, 16)
    pos = idx[:1].expand(3, 150)
    got = run(q, joint, pos, table)
    slots = torch.where(pos >= 0, (15 - pos // 64) * 64 + pos % 64, -1)
    check(got, q, (q8, scale, kpe), slots)


def test_attend_slots_past_32_bit_offsets():
    """Slots whose byte offsets pass 2^31 and 2^32."""
    pages = 133_000  # 8.5 million slots: 4.4 GB of latent rows
    q8 = torch.zeros(pages, 64, 512, dtype=torch.float8_e4m3fn, device="cuda")
    kpe = torch.zeros(pages, 64, 64, dtype=torch.bfloat16, device="cuda")
    scale = torch.ones(pages, 2, device="cuda")
    small = ref.pools(3, 64, 32, 12)
    at = [0, 66_000, pages - 1]
    for i, p in enumerate(at):
        q8[p], scale[p], kpe[p] = small[0][i], small[1][i], small[2][i]
    idx = selection(2, 150, 192, 12, short=False)
    far = torch.tensor(at, device="cuda")[(idx // 64).long()] * 64 + idx % 64
    q = queries(2, 16, 12)
    a, b = run(q, small, idx), run(q, (q8, scale, kpe), far.to(torch.int32))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("heads", [16, 128])
def test_attend_same_bits_on_streams_and_in_graphs(heads):
    """Two graphs captured on one stream and replayed on two others at once, beside eager calls."""
    cache = ref.pools(64, 64, 64, 11)
    sets = [(queries(20, heads, s), selection(20, 900, 4096, s)) for s in (0, 1)]
    want = [run(q, cache, idx) for q, idx in sets]
    outs, graphs = [], []
    cap = torch.cuda.Stream()
    for q, idx in sets:
        o = (torch.empty(20, heads, 512, dtype=torch.bfloat16, device="cuda"),
             torch.empty(20, heads, device="cuda"), torch.empty(20, 900, device="cuda"))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(cap):
            kernel_q8(*q, *cache, idx, SM, o[0], o[1], weights=o[2])
            cap.synchronize()
            with torch.cuda.graph(g, stream=cap):
                kernel_q8(*q, *cache, idx, SM, o[0], o[1], weights=o[2])
        outs.append(o)
        graphs.append(g)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for o in outs:
            for t in o:
                t.fill_(NAN)
        torch.cuda.synchronize()
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        eager = run(*[sets[0][0], cache, sets[0][1]])
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            for a, b in zip(w, o):
                assert torch.equal(a, b)
        for a, b in zip(want[0], eager):
            assert torch.equal(a, b)


def test_attend_refusals():
    cache = ref.pools(4, 64, 16, 8)
    q, idx = queries(2, 16, 8), selection(2, 40, 256, 8)
    out, lse = torch.empty(2, 16, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 16, device="cuda")
    ok = dict(q_nope=q[0], q_pe=q[1], ckv_q8=cache[0], ckv_scale=cache[1], kpe_cache=cache[2],
              sparse_indices=idx, sm_scale=SM, output=out, lse=lse)
    kernel_q8(**ok)
    for name, value, error in (
            ("q_nope", q[0].half(), TypeError), ("q_nope", q[0][..., :500], ValueError),
            ("q_nope", q[0][:, :8], ValueError), ("q_pe", q[1][:1], ValueError),
            ("ckv_q8", cache[0].view(torch.uint8), TypeError), ("ckv_q8", cache[0].float(), TypeError),
            ("ckv_q8", cache[0].view(256, 512), ValueError), ("ckv_q8", cache[0][:, ::2], ValueError),
            ("ckv_scale", cache[1][:, :3], ValueError), ("ckv_scale", cache[1].double(), TypeError),
            ("ckv_scale", cache[1].t().contiguous().t(), ValueError),
            ("kpe_cache", cache[2].float(), TypeError), ("kpe_cache", cache[2][:3], ValueError),
            ("sparse_indices", idx.long(), TypeError), ("sparse_indices", idx[:1], ValueError),
            ("sparse_indices", idx[:, :0], ValueError), ("sparse_indices", idx.cpu(), ValueError),
            ("sparse_indices", None, TypeError), ("output", out.float(), TypeError),
            ("lse", lse[:, :3], ValueError), ("weights", lse, ValueError),
            ("weights", idx, TypeError)):
        with pytest.raises(error):
            kernel_q8(**{**ok, name: value})
    odd = torch.empty(4 * 64 * 512 + 8, dtype=torch.uint8, device="cuda")[8:].view(torch.float8_e4m3fn)
    with pytest.raises(DSAError, match="16 bytes"):
        kernel_q8(**{**ok, "ckv_q8": odd.view(4, 64, 512)})
    with pytest.raises(TypeError):
        kernel_q8_paged(*q, *cache, None, idx, SM, out, lse)
    with pytest.raises(ValueError):
        kernel_q8_paged(*q, *cache, idx[:1], idx, SM, out, lse)
    three = ref.pools(2, 48, 16, 8)
    with pytest.raises(ValueError, match="power of two"):
        kernel_q8_paged(*q, *three, idx[:, :2].contiguous(), idx, SM, out, lse)
    check(run(q, three, idx.remainder(96)), q, three, idx.remainder(96))  # flat ids need no page size
    kernel_q8(q[0][:0], q[1][:0], *cache, idx[:0], SM, out[:0], lse[:0])
    assert read_device_errors() == 0


# ------------------------------------------------------------------------------------ append


def tables(rows, cols, pages, seed=0):
    p = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:rows * cols]
    return p.to(torch.int32).view(rows, cols)


def same_pools(cache, want):
    for t, w in zip(cache, want):
        np.testing.assert_array_equal(t.cpu().float().double().numpy().reshape(w.shape), w)


def tokens(n, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed + 300)
    x = torch.randn(n, 512, generator=g) * torch.exp(spread * torch.randn(n, 1, generator=g))
    return x.to(torch.bfloat16), torch.randn(n, 64, generator=g).to(torch.bfloat16)


@pytest.mark.parametrize("page,block", [(1, 1), (16, 1), (16, 4), (64, 64), (64, 16), (256, 256), (128, 32)])
def test_append(page, block):
    """Rows of 0, 1 and odd counts that start inside and at the edge of blocks; tokens before
    the first row and behind the last are left alone."""
    counts = [1, 0, 5, block, block + 1, 300, 2, 63, 1]
    starts = torch.tensor([0, 7, block - 1, block, 3, 11, 2 * block - 1, 40, 299], dtype=torch.int32)
    cols = -(-700 // page)
    cache = ref.pools(len(counts) * cols + 2, page, block, page + block)
    table = tables(len(counts), cols, cache[0].shape[0], block)
    off = np.cumsum([3] + counts).tolist()
    x, k = tokens(off[-1] + 9, block)
    want = ref.append(x, k, off, starts, table.numpy(), *cache)
    args = (x.cuda(), k.cuda(), torch.tensor(off, dtype=torch.int32).cuda(), starts.cuda(), table.cuda())
    append_q8(*args, *cache)
    same_pools(cache, want)
    append_q8(*args, *cache)  # the same tokens again: nothing left to grow
    same_pools(cache, want)
    assert read_device_errors() == 0


def test_append_a_token_at_a_time_grows_the_scale():
    """A block filled one token per call, each larger than the last, then smaller ones."""
    cache = ref.pools(2, 64, 64, 1)
    table = torch.tensor([[1]], dtype=torch.int32)
    x, k = tokens(64, 2, spread=0.0)
    x = (x.float() * torch.exp2(torch.cat([torch.arange(40) * 0.7 - 12, torch.zeros(24)]))[:, None]).to(torch.bfloat16)
    pools = [t.clone() for t in cache]
    for i in range(64):
        start = torch.tensor([i], dtype=torch.int32)
        want = ref.append(x[i:i + 1], k[i:i + 1], [0, 1], start, table.numpy(), *pools)
        append_q8(x[i:i + 1].cuda(), k[i:i + 1].cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(),
                  start.cuda(), table.cuda(), *pools)
        same_pools(pools, want)


def test_append_zeros_infinities_and_nan():
    cache = ref.pools(4, 16, 8, 3)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    x, k = tokens(32, 4)
    x[:8] = 0
    x[9, 3], x[9, 4], x[10, 5] = math.inf, -math.inf, NAN
    x[16:24] = NAN
    x[25] = 3.3e38
    x[26] = 1e-38
    off = [0, 32]
    want = ref.append(x, k, off, torch.tensor([0]), table.numpy(), *cache)
    append_q8(x.cuda(), k.cuda(), torch.tensor(off, dtype=torch.int32).cuda(),
              torch.tensor([0], dtype=torch.int32).cuda(), table.cuda(), *cache)
    same_pools(cache, want)
    assert cache[1].view(-1)[4 * 1 + 0] == 2.0 ** -126  # the block of zeros


def test_append_positions_without_a_page_are_flagged():
    cache = ref.pools(4, 16, 8, 3)
    table = torch.tensor([[2, -1, 9], [0, 1, 3]], dtype=torch.int32)
    x, k = tokens(80, 5)
    starts, off = torch.tensor([3, 30], dtype=torch.int32), [0, 50, 80]
    want = ref.append(x, k, off, starts, table.numpy(), *cache)
    append_q8(x.cuda(), k.cuda(), torch.tensor(off, dtype=torch.int32).cuda(), starts.cuda(), table.cuda(), *cache)
    same_pools(cache, want)
    assert read_device_errors(clear=True) == _native.DEVERR_BAD_INDEX
    # offsets past the tokens, descending ones and a negative start leave the pools alone or in bounds
    before = [t.clone() for t in cache]
    append_q8(x.cuda(), k.cuda(), torch.tensor([0, 5, 5], dtype=torch.int32).cuda(),
              torch.tensor([-4, 0], dtype=torch.int32).cuda(), table.cuda(), *cache)
    for a, b in zip(before, cache):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert read_device_errors(clear=True) == _native.DEVERR_BAD_INDEX
    for off in ([0, 90, 200], [7, 3, 100], [-5, -2, 80], [80, 40, 0]):
        append_q8(x.cuda(), k.cuda(), torch.tensor(off, dtype=torch.int32).cuda(),
                  torch.tensor([0, 2 ** 31 - 1], dtype=torch.int32).cuda(), table.cuda(), *cache)
    torch.cuda.synchronize()


def test_append_many_rows_strides_and_refusals():
    """A step of 1500 sequences; tokens as slices of one [tokens, 576]; a joint pool."""
    rows = 1500
    both = torch.zeros(1600, 16, 640, dtype=torch.uint8, device="cuda")
    cache = (both[..., :512].view(torch.float8_e4m3fn), torch.ones(1600, 2, device="cuda"),
             both[..., 512:].view(torch.bfloat16))
    x, k = tokens(rows, 6)
    cat = torch.cat([x, k], 1).cuda()
    table = tables(rows, 1, 1600)
    starts = (torch.arange(rows) % 16).to(torch.int32)
    off = torch.arange(rows + 1, dtype=torch.int32)
    want = ref.append(x, k, off.tolist(), starts, table.numpy(), *cache)
    args = [cat[:, :512], cat[:, 512:], off.cuda(), starts.cuda(), table.cuda(), *cache]
    append_q8(*args)
    same_pools(cache, want)
    for i, bad, error in ((0, cat, ValueError), (0, cat[:, :512].float(), TypeError), (1, cat[1:, 512:], ValueError),
                          (2, off.cuda()[:-1], ValueError), (2, off.long().cuda(), TypeError),
                          (3, starts, ValueError), (4, table.cuda()[1:], ValueError), (4, None, TypeError),
                          (6, cache[1][:, :0], ValueError)):
        with pytest.raises(error):
            append_q8(*(args[:i] + [bad] + args[i + 1:]))
    append_q8(cat[:0, :512], cat[:0, 512:], off.cuda() * 0, *args[3:])
    same_pools(cache, want)


@pytest.mark.parametrize("rows,live,most,block", [(70000, 300, 5, 2), (70000, 300, 5, 16), (400, 380, 29, 16),
                                                  (1000, 150, 29, 64)])
def test_append_rows_without_a_token(rows, live, most, block):
    """Many rows, some or most of them without a new token, the first and the last among them;
    tokens before the first offset and behind the last."""
    page, cols = max(16, block), 64 // max(16, block) + 1
    g = torch.Generator().manual_seed(block)
    counts = torch.zeros(rows, dtype=torch.long)
    some = torch.randperm(rows - 2, generator=g)[:live] + 1
    counts[some] = torch.randint(1, most + 1, (live,), generator=g)
    off = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]) + 3
    n = int(off[-1]) + 5
    table = torch.full((rows, cols), -1, dtype=torch.int32)
    table[some] = tables(live, cols, live * cols + 9, block)
    starts = torch.randint(0, 34, (rows,), generator=g, dtype=torch.int32)
    cache = ref.pools(live * cols + 9, page, block, 4)
    x, k = tokens(n, 8)
    want = ref.append(x, k, off.tolist(), starts, table.numpy(), *cache)
    append_q8(x.cuda(), k.cuda(), off.to(torch.int32).cuda(), starts.cuda(), table.cuda(), *cache)
    same_pools(cache, want)
    assert read_device_errors() == 0


# ------------------------------------------------------------------- accumulate, evict, compact


@pytest.mark.parametrize("rows,per,topk,cols", [(1, 1, 1, 1), (5, 1, 700, 900), (3, 4, 257, 300), (2, 9, 1500, 1500),
                                                (2, 17, 2500, 2600), (30, 8, 1025, 1100), (60, 2, 33, 100), (90, 3, 64, 64)])
def test_accumulate(rows, per, topk, cols):
    g = torch.Generator().manual_seed(topk)
    n = rows * per
    pos = torch.stack([torch.randperm(cols, generator=g)[:topk] for _ in range(n)]).to(torch.int32)
    pos[torch.rand(n, topk, generator=g) < 0.2] = -1
    w, acc = torch.rand(n, topk, generator=g), torch.rand(rows, cols, generator=g)
    want = acc.double()
    off = [0] + [per] * rows if per == 1 else [0] + [per + (1 if r == 0 else -1 if r == 1 else 0) for r in range(rows)]
    off = np.cumsum(off).tolist()
    for r in range(rows):
        for t in range(off[r], off[r + 1]):
            at = pos[t] >= 0
            want[r, pos[t, at].long()] += w[t, at].double()
    got = []
    for _ in range(2):
        a = acc.cuda()
        accumulate_weights(w.cuda(), pos.cuda(), a, None if per == 1 else torch.tensor(off, dtype=torch.int32).cuda())
        got.append(a)
    assert torch.equal(*got)
    # at most per + 1 additions of values below per + 2 each
    assert (got[0].cpu().double() - want).abs().max() <= (per + 2) * (per + 2) * 2.0 ** -24
    assert read_device_errors() == 0


def test_accumulate_repeated_and_outside_positions():
    acc = torch.zeros(2, 8, device="cuda")
    pos = torch.tensor([[3, 3, 3, -1, 8, -2], [0, 7, 0, 7, -1, -1]], dtype=torch.int32, device="cuda")
    w = torch.tensor([[1.0, 2, 4, 100, 100, 100], [1, 2, 4, 8, 100, 100]], device="cuda")
    accumulate_weights(w, pos, acc)
    assert acc.tolist() == [[0, 0, 0, 7, 0, 0, 0, 0], [5, 0, 0, 0, 0, 0, 0, 10]]
    assert read_device_errors(clear=True) == _native.DEVERR_BAD_INDEX
    # rows of a wider buffer; the tokens behind the last row are not added
    wide = torch.zeros(1, 12, device="cuda")
    accumulate_weights(w, pos, wide[:, 2:10], torch.tensor([1, 2], dtype=torch.int32, device="cuda"))
    assert wide.tolist() == [[0, 0, 5, 0, 0, 0, 0, 0, 0, 10, 0, 0]]
    accumulate_weights(w, pos, wide[:, 2:10], torch.tensor([5, 9], dtype=torch.int32, device="cuda"))
    assert wide.sum() == 15
    for args, error in (((w, pos, acc[:1]), ValueError), ((w, pos.long(), acc), TypeError),
                        ((w, pos[:, :3], acc), ValueError), ((w, pos, acc.t()), ValueError),
                        ((w, pos, acc[:1].expand(2, 8)), ValueError), ((w.half(), pos, acc), TypeError),
                        ((w, pos, acc, torch.zeros(2, dtype=torch.int32, device="cuda")), ValueError)):
        with pytest.raises(error):
            accumulate_weights(*args)
    accumulate_weights(w[:, :0], pos[:, :0], acc)
    accumulate_weights(w[:0], pos[:0], acc[:0])


@pytest.mark.parametrize("max_len,budget,sinks,recent", [
    (1, 1, 0, 0), (50, 50, 4, 9), (51, 50, 4, 9), (700, 64, 0, 0), (700, 64, 64, 0), (700, 64, 0, 64),
    (5000, 1000, 4, 128), (20001, 2048, 7, 333), (60000, 513, 1, 1)])
@pytest.mark.parametrize("rows", [3, 100])
def test_evict_positions(rows, max_len, budget, sinks, recent):
    if rows * max_len > 1_000_000:
        rows = 10
    g = torch.Generator().manual_seed(max_len + budget)
    acc = torch.rand(rows, max_len, generator=g).pow(6)
    acc[acc < 0.05] = 0                      # ties
    acc[0, ::7] = NAN                        # below every number
    acc[-1, ::5] = math.inf
    lens = torch.randint(0, max_len + 1, (rows,), generator=g, dtype=torch.int32)
    lens[0], lens[-1] = max_len, max_len + 5  # past the end counts as the end
    new = torch.full((rows, budget + 3), NAN, device="cuda")
    keep, n = evict_positions(acc.cuda(), lens.cuda(), budget, sinks=sinks, recent=recent, new_acc=new)
    want, want_n, totals = ref.evict(acc, lens, budget, sinks, recent)
    assert n.tolist() == want_n
    assert keep.tolist() == want
    for r in range(rows):
        np.testing.assert_array_equal(new[r, :want_n[r]].cpu().numpy(), np.float32(totals[r]))
        assert (new[r, want_n[r]:] == 0).all()
    alone, m = evict_positions(acc.cuda(), lens.cuda(), budget, sinks=sinks, recent=recent)
    assert torch.equal(alone, keep) and torch.equal(m, n)


def test_evict_refusals():
    acc, lens = torch.rand(2, 9, device="cuda"), torch.tensor([9, 3], dtype=torch.int32, device="cuda")
    for kw, error in ((dict(budget=0), ValueError), (dict(budget=4, sinks=2, recent=3), ValueError),
                      (dict(budget=4, sinks=-1), ValueError), (dict(budget=4, new_acc=acc), ValueError),
                      (dict(budget=4, new_acc=acc[:, :3].contiguous()), ValueError),
                      (dict(budget=4, new_acc=acc.double()), TypeError)):
        with pytest.raises(error):
            evict_positions(acc, lens, **kw)
    with pytest.raises(TypeError):
        evict_positions(acc, lens.long(), 4)
    with pytest.raises(ValueError):
        evict_positions(acc, lens[:1], 4)
    keep, n = evict_positions(acc[:, :0], lens, 4)
    assert (keep == -1).all() and (n == 0).all()
    keep, n = evict_positions(acc[:0], lens[:0], 4)
    assert keep.shape == (0, 4) and n.shape == (0,)


@pytest.mark.parametrize("page,block", [(1, 1), (16, 4), (64, 64), (64, 16), (256, 256), (128, 32)])
@pytest.mark.parametrize("budget", [1, 63, 200, 513])
def test_compact(page, block, budget):
    rows, length = 5, 700
    cols, new_cols = -(-length // page), -(-budget // page)
    cache = ref.pools(rows * (cols + new_cols) + 1, page, block, budget, spread=2.0)
    table = tables(rows, cols + new_cols, cache[0].shape[0], budget)
    old, new = table[:, :cols], table[:, cols:]
    g = torch.Generator().manual_seed(budget)
    keep = torch.full((rows, budget), -1, dtype=torch.int32)
    for r, n in enumerate((budget, budget, max(1, budget // 2), 0, budget - 1)):
        keep[r, :n] = torch.randperm(length, generator=g)[:n].sort().values
    want = ref.compact(keep.tolist(), old.numpy(), new.numpy(), *cache)
    compact_q8(keep.cuda(), table.cuda()[:, :cols], new.cuda(), *cache)
    same_pools(cache, want)
    assert read_device_errors() == 0


def test_compact_odd_entries_and_refusals():
    cache = ref.pools(10, 16, 8, 3, spread=2.0)
    cache[1][2:4] = 0                                     # blocks of zero scale
    table = torch.tensor([[1, 2, -1], [3, 4, 77]], dtype=torch.int32)
    new = torch.tensor([[5, 6], [7, -1]], dtype=torch.int32)
    # -1 in between, a missing page on either side, a position past the table, an order that is
    # not ascending, and a position twice
    keep = torch.tensor([[5, -1, 30, 30, 33, 48, 0, -3] + [17] * 12, [40, 3, 2, 1, 0, 9, 9, 20] + [31] * 12],
                        dtype=torch.int32)
    want = ref.compact(keep.tolist(), table.numpy(), new.numpy(), *cache)
    args = [keep.cuda(), table.cuda(), new.cuda(), *cache]
    compact_q8(*args)
    same_pools(cache, want)
    assert read_device_errors(clear=True) == _native.DEVERR_BAD_INDEX
    for i, bad, error in ((0, keep.cuda()[:1], ValueError), (0, keep.long().cuda(), TypeError),
                          (1, table.cuda()[:, :0], ValueError), (2, None, TypeError),
                          (3, cache[0].view(torch.uint8), TypeError), (4, cache[1][:1], ValueError)):
        with pytest.raises(error):
            compact_q8(*(args[:i] + [bad] + args[i + 1:]))
    compact_q8(keep.cuda()[:, :0], *args[1:])
    compact_q8(keep.cuda()[:0], table.cuda()[:0], new.cuda()[:0], *cache)
    same_pools(cache, want)


def test_compact_scales_of_minus_zero():
    """A block of scale -0 beside one of a positive scale: the values keep what they stand for."""
    cache = ref.pools(3, 16, 4, 5)
    cache[1][0, 0] = -0.0
    keep = torch.tensor([[1, 5, 9, 2]], dtype=torch.int32)
    table, new = torch.tensor([[0]], dtype=torch.int32), torch.tensor([[2]], dtype=torch.int32)
    before = ref.values(*cache[:2])
    compact_q8(keep.cuda(), table.cuda(), new.cuda(), *cache)
    after = ref.values(*cache[:2])
    assert cache[1][2, 0] == cache[1][0, 1:3].max()
    # one more rounding to e4m3: 2^-4 of the value, or half its smallest step, 2^-10 scales
    want = before[keep[0].long()]
    assert ((after[32:36] - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * float(cache[1][2, 0])).all()


def test_a_step_in_a_graph_on_another_stream():
    """Append, decode with weights, accumulate, evict and compact, captured as one graph from a
    stream that owns none of the tensors, and replayed; the same bits as the eager calls."""
    rows, page, block, length = 6, 16, 4, 150
    cols = 16
    table = tables(rows, 2 * cols, 2 * rows * cols, 9)
    old, new = table[:, :cols].contiguous().cuda(), table[:, cols:].contiguous().cuda()
    x, k = (t.cuda() for t in tokens(2 * rows, 77))
    q = queries(2 * rows, 16, 5)
    off = (2 * torch.arange(rows + 1)).to(torch.int32).cuda()
    starts = torch.full((rows,), length, dtype=torch.int32).cuda()
    lens = starts + 2
    g = torch.Generator().manual_seed(3)
    pos = torch.stack([torch.randperm(length + 2, generator=g)[:100] for _ in range(2 * rows)]).to(torch.int32).cuda()
    per_token = old.repeat_interleave(2, 0)

    def step(cache, acc):
        out = torch.empty(2 * rows, 16, 512, dtype=torch.bfloat16, device="cuda")
        lse, w = torch.empty(2 * rows, 16, device="cuda"), torch.empty(2 * rows, 100, device="cuda")
        new_acc = torch.empty(rows, 64, device="cuda")
        append_q8(x, k, off, starts, old, *cache)
        kernel_q8_paged(*q, *cache, per_token, pos, SM, out, lse, weights=w)
        accumulate_weights(w, pos, acc, off)
        keep, n = evict_positions(acc, lens, 64, sinks=2, recent=8, new_acc=new_acc)
        compact_q8(keep, old, new, *cache)
        return out, lse, w, keep, n, new_acc

    def fresh():
        return ref.pools(2 * rows * cols, page, block, 21), torch.zeros(rows, 200, device="cuda")

    cache, acc = fresh()
    want = [t.clone() for t in step(cache, acc)] + [acc] + [t.clone() for t in cache]
    cache, acc = fresh()
    start = [t.clone() for t in (*cache, acc)]
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(cache, acc)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = step(cache, acc)
    other = torch.cuda.Stream()
    for _ in range(3):
        for t, s in zip((*cache, acc), start):
            t.view(torch.uint8).copy_(s.view(torch.uint8))
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*got, acc, *cache), want):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert read_device_errors() == 0


# ------------------------------------------------------------------------------ all together


def test_prompt_decode_evict_decode():
    """A serving loop: prompts appended, steps decoded with their weights added up, the cache cut
    to a budget, and the next step decoded over what was kept."""
    B, H, page, block, budget = 3, 16, 64, 16, 256
    lens = [700, 401, 150]
    pool = (torch.zeros(60, page, 512, dtype=torch.float8_e4m3fn, device="cuda"),
            torch.zeros(60, page // block, device="cuda"),
            torch.zeros(60, page, 64, dtype=torch.bfloat16, device="cuda"))
    table = tables(B, 16, 60).cuda()
    x, k = tokens(sum(lens), 1, spread=0.5)
    off = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    append_q8(x.cuda(), k.cuda(), off, torch.zeros(B, dtype=torch.int32, device="cuda"), table, *pool)
    acc = torch.zeros(B, 1024, device="cuda")
    total = torch.zeros(B, 1024, dtype=torch.float64)
    for step in range(3):
        x1, k1 = tokens(B, 50 + step, spread=0.5)
        n = torch.tensor([v + step for v in lens], dtype=torch.int32).cuda()
        append_q8(x1.cuda(), k1.cuda(), torch.arange(B + 1, dtype=torch.int32, device="cuda"), n, table, *pool)
        pos = torch.full((B, 320), -1, dtype=torch.int32)
        for b in range(B):
            m = min(320, lens[b] + step + 1)
            pos[b, :m] = torch.randperm(lens[b] + step + 1, generator=torch.Generator().manual_seed(9 * b + step))[:m].sort().values
        pos = pos.cuda()
        q = queries(B, H, step)
        got = run(q, pool, pos, table)
        slots = torch.where(pos >= 0, table.gather(1, (pos.clamp(min=0) // page).long()) * page + pos % page, -1)
        check(got, q, pool, slots)
        accumulate_weights(got[2], pos, acc)
        w = ref.attend(*q, *pool, slots, SM)[2]
        for b in range(B):
            at = pos[b].cpu() >= 0
            total[b, pos[b].cpu()[at].long()] += w[b, at]
    assert (acc.cpu().double() - total).abs().max() <= 16 * 3 * 2.0 ** -14
    lengths = torch.tensor([v + 3 for v in lens], dtype=torch.int32, device="cuda")
    new_acc = torch.empty(B, 1024, device="cuda")
    keep, n = evict_positions(acc, lengths, budget, sinks=4, recent=32, new_acc=new_acc)
    assert keep.tolist() == ref.evict(acc.cpu(), lengths.cpu(), budget, 4, 32)[0]
    assert n.tolist() == [256, 256, 153]
    fresh = torch.tensor(sorted(set(range(60)) - set(table.flatten().tolist()))[:12], dtype=torch.int32)
    new_table = fresh.view(B, 4).cuda()
    want = ref.compact(keep.tolist(), table.cpu().numpy(), new_table.cpu().numpy(), *pool)
    compact_q8(keep, table, new_table, *pool)
    same_pools(pool, want)
    q = queries(B, H, 99)
    j = torch.arange(budget, dtype=torch.int32, device="cuda").expand(B, budget)
    pos = torch.where(j < n[:, None], j, -1)
    got = run(q, pool, pos, new_table)
    slots = torch.where(pos >= 0, new_table.gather(1, (pos.clamp(min=0) // page).long()) * page + pos % page, -1)
    check(got, q, pool, slots)
    assert read_device_errors() == 0
