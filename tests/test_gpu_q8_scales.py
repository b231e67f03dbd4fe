"""The 8-bit decode where the scales of one selection differ widely, against tests/q8_bounds.py."""
import math

import pytest
import torch

import q8_bounds
from flashinfer_mlsys2026_dsa_b200 import kernel_q8, read_device_errors

pytestmark = pytest.mark.gpu
SM = 1.0 / math.sqrt(192.0)
LOG2E = math.log2(math.e)
SLOTS = 4096
# rows, heads, entries: in splits of several tiles, and unsplit
SHAPES = [(3, 16, 2400), (150, 16, 500), (2, 32, 2400), (3, 128, 700), (40, 128, 500)]
NAN = float("nan")


def e4m3(x):
    return x.clamp(-448, 448).to(torch.float8_e4m3fn).view(-1, 16, 512).cuda()


def run(q, cache, idx):
    B, H, _ = q[0].shape
    out = torch.full((B, H, 512), NAN, dtype=torch.bfloat16, device="cuda")
    lse, w = torch.full((B, H), NAN, device="cuda"), torch.full(idx.shape, NAN, device="cuda")
    kernel_q8(*q, *cache, idx, SM, out, lse, weights=w)
    alone = (torch.full_like(out, NAN), torch.full_like(lse, NAN))
    kernel_q8(*q, *cache, idx, SM, *alone)
    assert torch.equal(out.view(torch.int16), alone[0].view(torch.int16)) and torch.equal(lse, alone[1])
    assert read_device_errors() == 0
    return out, lse, w


def rope(scores):
    """(kpe rows, q_pe element) whose product is about the given scores in log2 units, exact in
    the reference: the bf16 values of scores / (SM log2 e) behind a one in the query."""
    k = torch.zeros(len(scores), 64)
    k[:, 0] = scores / (SM * LOG2E)
    return k.to(torch.bfloat16).view(-1, 16, 64).cuda()


def rope_queries(B, H):
    qp = torch.zeros(B, H, 64, dtype=torch.bfloat16, device="cuda")
    qp[..., 0] = 1
    return qp


@pytest.mark.parametrize("growth", [4, 6, 8, 10, 12, 14, 16, 20, 28, 40])
@pytest.mark.parametrize("rows,heads,topk", SHAPES)
def test_one_slot_of_a_far_larger_scale(rows, heads, topk, growth):
    """Each row holds a slot whose scale is 2^growth times the others', at a place of its own from the
    first tile to the last; heads give it nearly all of their weight, some, or none."""
    g = torch.Generator().manual_seed(growth)
    x = torch.rand(SLOTS, 512, generator=g) * 300 + 100  # of one sign, so that outputs do not cancel
    x[0] *= torch.where(torch.rand(512, generator=g) < 0.5, -1.0, 1.0)
    q8 = e4m3(x)
    scale = torch.full((SLOTS,), 2.0 ** -9)
    scale[0] = 2.0 ** (growth - 9)
    kpe = (torch.randn(SLOTS // 16, 16, 64, generator=g) * 0.5).to(torch.bfloat16).cuda()
    cache = (q8, scale.view(-1, 16).cuda(), kpe)
    idx = torch.stack([torch.randperm(SLOTS - 1, generator=g)[:topk] + 1 for _ in range(rows)]).to(torch.int32)
    at = torch.linspace(0, topk - 1, rows).long() if rows > 3 else torch.tensor([2, topk // 2 + 30, topk - 1])[:rows]
    idx[torch.arange(rows), at] = 0
    big = q8.view(-1, 512)[0].float().cpu() * scale[0]
    q = 0.02 * torch.randn(rows, heads, 512, generator=g)
    q -= (q @ big / (big @ big))[..., None] * big
    aim = torch.linspace(-60, 20, rows * heads).view(rows, heads)
    q += (aim / (SM * LOG2E * (big @ big)))[..., None] * big
    q = (q.to(torch.bfloat16).cuda(), torch.randn(rows, heads, 64, generator=g).to(torch.bfloat16).cuda())
    idx = idx.cuda()
    q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)


@pytest.mark.parametrize("growth", [6, 12, 20, 40, 60, 80])
@pytest.mark.parametrize("rows,heads,topk", SHAPES)
def test_small_scales_with_the_weight(rows, heads, topk, growth):
    """Entries of a small scale, in the first tiles, whose weight makes up for it: they and the
    later ones share the output."""
    g = torch.Generator().manual_seed(growth)
    q8 = e4m3(torch.rand(SLOTS, 512, generator=g) * 300 + 100)
    scale = torch.full((SLOTS,), 2.0 ** -growth)
    scale[SLOTS // 2:] = 1
    score = torch.rand(SLOTS, generator=g) * 2
    score[:SLOTS // 2] += growth
    cache = (q8, scale.view(-1, 16).cuda(), rope(score))
    q = (torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device="cuda"), rope_queries(rows, heads))
    idx = torch.stack([torch.randperm(SLOTS, generator=g)[:topk].sort().values for _ in range(rows)]).to(torch.int32)
    idx[0] = idx[0].flip(0)
    idx = idx.cuda()
    q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)


@pytest.mark.parametrize("late", [2.0 ** -60, 0.5, 1.0, 2.0, 4.0, 2.0 ** 20, 2.0 ** 60, 2.0 ** 90])
@pytest.mark.parametrize("rows,heads,topk", SHAPES)
def test_tokens_of_zeros_first(rows, heads, topk, late):
    """The first tiles hold tokens of zeros, which an append gives the scale 2^-126, or a scale of 0;
    later ones any scale."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(SLOTS, 512, generator=g) * 100 + 30
    zeros = topk * 5 // 8
    x[:zeros] = 0
    q8 = e4m3(x)
    scale = torch.full((SLOTS,), 2.0 ** -126)
    scale[zeros // 2:zeros] = 0
    scale[zeros:] = late
    cache = (q8, scale.view(-1, 16).cuda(), (torch.randn(SLOTS // 16, 16, 64, generator=g) * 0.5).to(torch.bfloat16).cuda())
    q = torch.randn(rows, heads, 576, generator=g)
    q = ((q[..., :512] * 0.02 / late).to(torch.bfloat16).cuda(), q[..., 512:].to(torch.bfloat16).cuda())
    idx = torch.arange(topk, dtype=torch.int32).repeat(rows, 1)
    idx[1, ::2] = torch.arange(SLOTS - topk // 2, SLOTS, dtype=torch.int32)  # among the others
    idx = idx.cuda()
    q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)


@pytest.mark.parametrize("rows,heads,topk", SHAPES)
def test_scales_that_grow_from_tile_to_tile(rows, heads, topk):
    """Every 64 entries the scale grows, from 2^-126 to 2^24 in all, and a last one falls again."""
    g = torch.Generator().manual_seed(5)
    q8 = e4m3(torch.randn(SLOTS, 512, generator=g) * 100 + 30)
    steps = torch.linspace(-126, 24, -(-topk // 64)).round()
    scale = torch.ones(SLOTS)
    for i, e in enumerate(steps.tolist()):
        scale[64 * i:64 * i + 64] = 2.0 ** e
    scale[topk - 20:] = 2.0 ** -20
    kpe = (torch.randn(SLOTS // 16, 16, 64, generator=g) * 0.5).to(torch.bfloat16).cuda()
    cache = (q8, scale.view(-1, 16).cuda(), kpe)
    q = torch.randn(rows, heads, 576, generator=g)
    q = ((q[..., :512] * 2.0 ** -30).to(torch.bfloat16).cuda(), q[..., 512:].to(torch.bfloat16).cuda())
    idx = torch.arange(topk, dtype=torch.int32).repeat(rows, 1)
    idx[1] = idx[1].flip(0)
    idx = idx.cuda()
    q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)


@pytest.mark.parametrize("drop", [0.05, 0.3, 0.77, 1.4, 3.3, 6.9, 9.1])
@pytest.mark.parametrize("heads", [16, 32])
def test_outputs_that_cancel_pin_all_terms_of_a_probability(heads, drop):
    """Half of the entries weigh 2^-drop of the others and carry values of the other sign, in all
    pairs of sizes, so that in some columns the output nearly cancels and only the error of the
    probabilities is left: two e4m3 terms (2^-8) would not do."""
    x = torch.zeros(SLOTS, 512)
    i = torch.arange(512)
    up = (8 + i % 8) * 2.0 ** 4               # 128 .. 240
    down = (8 + i // 8 % 8) * 2.0 ** (i // 64)  # 8 .. 1920
    x[0::2], x[1::2] = up, -down.clamp(max=448)
    score = torch.zeros(SLOTS)
    score[1::2] = -drop
    cache = (e4m3(x), torch.ones(SLOTS // 16, 16, device="cuda"), rope(score))
    q = (torch.zeros(3, heads, 512, dtype=torch.bfloat16, device="cuda"), rope_queries(3, heads))
    idx = torch.randperm(SLOTS, generator=torch.Generator().manual_seed(1))[:800].to(torch.int32).repeat(3, 1).cuda()
    worst = q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)
    assert worst[0] > 2.0 ** -12  # the bound is of the output's size somewhere


@pytest.mark.parametrize("rows,heads,topk", SHAPES + [(64, 16, 2048)])
def test_ordinary_caches(rows, heads, topk):
    """Sizes as a cache has them: within the kernel's own 12 bits, not only bf16's."""
    g = torch.Generator().manual_seed(topk)
    x = torch.randn(SLOTS, 512, generator=g) * torch.exp(0.5 * torch.randn(SLOTS, 1, generator=g))
    scale = torch.exp2(torch.ceil(torch.log2(x.view(-1, 16, 512).abs().amax((1, 2)) / 448)))
    cache = (e4m3(x / scale.repeat_interleave(16)[:, None]), scale.view(-1, 1).cuda(),
             torch.randn(SLOTS // 16, 16, 64, generator=g).to(torch.bfloat16).cuda())
    q = torch.randn(rows, heads, 576, generator=g).to(torch.bfloat16).cuda()
    q = (q[..., :512].contiguous(), q[..., 512:].contiguous())
    idx = torch.stack([torch.randperm(SLOTS, generator=g)[:topk] for _ in range(rows)]).to(torch.int32).cuda()
    q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)


@pytest.mark.parametrize("above", [20, 80, 95, 110, 200])
@pytest.mark.parametrize("rows,heads,topk", SHAPES)
def test_zero_tokens_with_the_weight(rows, heads, topk, above):
    """Zero tokens (scale 2^-126) whose scores lie 2^above over the others': the output is small, and off by
    2^-107 of the others' values a slot at most; rows of padding and padded ones beside them."""
    g = torch.Generator().manual_seed(above)
    x = torch.rand(SLOTS, 512, generator=g) * 300 + 100
    zero = torch.rand(SLOTS, generator=g) < 0.5
    x[zero] = 0
    scale = torch.where(zero, 2.0 ** -126, 0.25)
    cache = (e4m3(x), scale.view(-1, 16).cuda(), rope(torch.where(zero, float(above), 0.0) + torch.rand(SLOTS, generator=g)))
    q = (torch.zeros(rows, heads, 512, dtype=torch.bfloat16, device="cuda"), rope_queries(rows, heads))
    idx = torch.stack([torch.randperm(SLOTS, generator=g)[:topk] for _ in range(rows)]).to(torch.int32)
    idx[1, topk // 3:] = -1
    idx[1, ::3] = -1
    if rows > 2:
        idx[2] = -1
    idx = idx.cuda()
    q8_bounds.check(run(q, cache, idx), q, cache, idx, SM)
