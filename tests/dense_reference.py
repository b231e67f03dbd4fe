"""Dense attention over a latent cache in 64 bits, with bounds that follow each rounding.

Works on any device, one row at a time; the pools may hold NaN wherever no token of a row looks.
"""
import math

import torch

LOG2E = math.log2(math.e)
D = torch.float64


def sequence(ckv, kpe, page_row, n, page):
    """The keys [n, 576] of a sequence's first n positions (float64)."""
    at = torch.arange(n, device=ckv.device)
    slot = page_row.long()[at // page] * page + at % page
    return torch.cat([ckv.reshape(-1, 512)[slot], kpe.reshape(-1, 64)[slot]], 1).to(D)


def seen_window(p, n, window, sinks, device=None):
    """Which of n positions the token at position p sees."""
    q = torch.arange(n, device=device)
    near = q > p - window if window is not None else torch.ones_like(q, dtype=torch.bool)
    return (q <= p) & ((q < sinks) | near)


def attend(q, keys, seen, sm_scale):
    """(output, lse, output's bound, lse's bound) of queries q [m, h, 576] over keys [n, 576];
    seen [m, n].

    * A score is a sum of 576 products in fp32 and a few scalings: 600 roundings of 2^-24 of
      sum |q v| at most: dz, in log2 units.
    * A probability: dz ln 2, 2^-21 for the exponential of a rounded difference, and bf16: 2^-8.
      Numerator and denominator each carry the first two, the numerator alone the last.
    * Sums over n entries: one rounding of 2^-23 for each 16 entries, and some for rescaling and
      joining splits: 2^-23 (n / 16 + 128) in all.
    * The output is rounded to bf16: 2^-8 of its value.
    * lse = m + log2 l: dz, the relative error of l over ln 2, 2^-21 for the logarithm and a
      rounding 2^-23 of its own size and of m's.
    """
    m, h, _ = q.shape
    out = torch.zeros(m, h, 512, dtype=D, device=q.device)
    lse = torch.full((m, h), -math.inf, dtype=D, device=q.device)
    otol, ltol = torch.full_like(out, 1e-37), torch.full_like(lse, 1e-37)
    for i in range(m):
        k = keys[seen[i]]
        if not len(k):
            continue
        x = q[i].to(D)
        z = x @ k.T * (sm_scale * LOG2E)
        dz = 600 * 2.0 ** -24 * (x.abs() @ k.abs().T) * abs(sm_scale) * LOG2E
        top = z.amax(1, keepdim=True)
        w = torch.exp2(z - top)
        total = w.sum(1, keepdim=True)
        p = w / total
        v = k[:, :512]
        out[i], lse[i] = p @ v, (top + torch.log2(total))[:, 0]
        rel = torch.expm1(dz * math.log(2)) + 2.0 ** -21
        sums = 2.0 ** -23 * (len(k) / 16 + 128)
        mean = (p * rel).sum(1, keepdim=True)  # the denominator's relative error
        otol[i] = (p * (rel + 2.0 ** -8 + mean + 2 * sums)) @ v.abs() * (1 + 2.0 ** -7) + 2.0 ** -8 * out[i].abs() + 1e-37
        ltol[i] = (dz.amax(1) + (mean[:, 0] + sums) * LOG2E + 2.0 ** -21
                   + 2.0 ** -23 * (lse[i].abs() + z.abs().amax(1)))
    return out, lse, otol, ltol


def window(q_nope, q_pe, ckv, kpe, table, lens, new, sm_scale, win, sinks, page):
    """The whole call: lens and new are host lists, tokens packed in row order."""
    parts, t = [], 0
    for r, (n, m) in enumerate(zip(lens, new)):
        q = torch.cat([q_nope[t:t + m], q_pe[t:t + m]], 2)
        keys = sequence(ckv, kpe, table[r], n, page)
        seen = torch.stack([seen_window(n - m + j, n, win, sinks, ckv.device) for j in range(m)]) \
            if m else torch.zeros(0, n, dtype=torch.bool, device=ckv.device)
        parts.append(attend(q, keys, seen, sm_scale))
        t += m
    return tuple(torch.cat(x) for x in zip(*parts))


def shared(q_nope, q_pe, ckv, kpe, pre_table, pre_lens, sizes, table, lens, new, sm_scale, page):
    """sizes: rows of each group; rows behind the last group have no prefix."""
    owner = [g for g, n in enumerate(sizes) for _ in range(n)] + [None] * (len(lens) - sum(sizes))
    parts, t = [], 0
    for r, (n, m) in enumerate(zip(lens, new)):
        q = torch.cat([q_nope[t:t + m], q_pe[t:t + m]], 2)
        keys = sequence(ckv, kpe, table[r], n, page)
        before = 0
        if owner[r] is not None:
            before = pre_lens[owner[r]]
            keys = torch.cat([sequence(ckv, kpe, pre_table[owner[r]], before, page), keys])
        at = torch.arange(len(keys), device=ckv.device) - before
        seen = at <= torch.arange(n - m, n, device=ckv.device)[:, None]
        parts.append(attend(q, keys, seen, sm_scale))
        t += m
    return tuple(torch.cat(x) for x in zip(*parts))


def merge(outputs, lses):
    """(output, lse, bounds): fp32 weights of 2^-21, their sums, and the rounding to bf16."""
    z = torch.stack([x.to(D) for x in lses])
    top = z.amax(0)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    w = torch.exp2(z - top)
    total = w.sum(0)
    some = total > 0
    share = torch.where(some, w / total.clamp(min=1e-300), 0.0)
    out = torch.zeros_like(outputs[0], dtype=D)
    size = torch.zeros_like(out)
    for o, s in zip(outputs, share):
        x = torch.where(s[..., None] > 0, o.to(D), 0.0)
        out += x * s[..., None]
        size += x.abs() * s[..., None]
    lse = torch.where(some, top + torch.log2(total.clamp(min=1e-300)), -math.inf)
    # a weight: the difference of the lses is rounded (2^-24 of up to the difference, times ln 2 in
    # the weight; shares below 2^-64 of the row play no part), the exponential 2^-22
    rel = 2.0 ** -24 * 64 + 2.0 ** -20
    return out, lse, 2.0 ** -8 * out.abs() + 2 * rel * size + 1e-37, \
        2.0 ** -19 + 2.0 ** -23 * lse.abs().nan_to_num(posinf=0.0)


def pools(pages, page, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    ckv = torch.randn(pages, page, 512, generator=g, device=device).mul_(0.6).to(torch.bfloat16)
    kpe = torch.randn(pages, page, 64, generator=g, device=device).mul_(0.6).to(torch.bfloat16)
    return ckv, kpe


def queries(tokens, heads, seed, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(tokens, heads, 512, generator=g, device=device).to(torch.bfloat16),
            torch.randn(tokens, heads, 64, generator=g, device=device).to(torch.bfloat16))


def tables(counts, seed, device="cuda", spare=3):
    """Page tables of sequences of `counts` pages from a shuffled pool, -1 behind them."""
    total = sum(counts) + spare
    perm = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    out = torch.full((len(counts), max(1, max(counts))), -1, dtype=torch.int32)
    a = 0
    for r, n in enumerate(counts):
        out[r, :n] = perm[a:a + n]
        a += n
    return out.to(device), total


def poison(ckv, kpe, table, keep, page):
    """NaN and infinities wherever no position in `keep` (per row: bool over positions) lies."""
    used = torch.zeros(ckv.shape[0] * page, dtype=torch.bool, device=ckv.device)
    for t, rows in zip(table, keep):
        for r, mask in enumerate(rows):
            at = torch.nonzero(mask)[:, 0]
            used[t[r].long()[at // page] * page + at % page] = True
    bad = torch.tensor([math.nan, math.inf, -math.inf], device=ckv.device)
    for pool in (ckv, kpe):
        flat = pool.view(-1, pool.shape[-1])
        fill = bad[torch.arange(flat.shape[0], device=ckv.device) % 3].to(pool.dtype)
        flat[~used] = fill[~used][:, None]


def check(got, want, tol, what):
    """Every value within its bound; infinities and NaN in the same places."""
    got = got.to(D)
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and not got[~inf].isinf().any(), f"{what}: infinities"
    fine = want.isfinite()
    over = ((got - want).abs() / tol)[fine]
    assert not over.numel() or over.max() <= 1, f"{what}: {over.max().item():.3g} times the bound"
