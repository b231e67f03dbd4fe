"""The 8-bit cache operators in 64 bits, from their definitions, and inputs for their tests."""
import math

import numpy as np
import torch

LOG2E = math.log2(math.e)
D = torch.float64


def e4m3(v):
    """float64 values rounded to the nearest e4m3 value (ties to even); NaN stays NaN."""
    v = np.asarray(v, dtype=np.float64)
    e = np.maximum(np.frexp(np.abs(v))[1], -5)
    step = np.ldexp(1.0, e - 4)
    return np.clip(np.rint(v / step) * step, -448.0, 448.0)


def scale_for(amax):
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    e = -126
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def pools(pages, page, block, seed, device="cuda", spread=0.5):
    """A cache with random contents: (ckv_q8, ckv_scale, kpe_cache)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, page // block, block * 512, generator=g)
    x *= torch.exp(spread * torch.randn(pages, page // block, 1, generator=g))
    s = torch.tensor([[scale_for(float(a)) for a in row] for row in x.abs().amax(2)])
    q8 = (x / s[..., None]).to(torch.float8_e4m3fn).view(pages, page, 512)
    kpe = torch.randn(pages, page, 64, generator=g).to(torch.bfloat16)
    return q8.to(device), s.float().to(device), kpe.to(device)


def values(q8, scale):
    """The latent values a cache stands for, [slots, 512] float64 on the CPU."""
    block = q8.shape[1] // scale.shape[1]
    s = scale.cpu().to(D).view(-1).repeat_interleave(block)
    return q8.cpu().float().to(D).view(-1, 512) * s[:, None]


def attend(q_nope, q_pe, q8, scale, kpe, slots, sm_scale):
    """(output, lse, weights, output tolerance, lse tolerance) in float64 on the CPU.

    Tolerances, all from roundings.  A score is a sum of 576 products in fp32 whose rounding
    errors add up to at most 600 * 2^-24 of sum |q v| (the products of 8-bit and bf16 operands
    are exact; the 24 beyond 576 cover the scalings), and q itself is kept to 2^-20 of its
    row's largest value; lse adds the log's and the sum's own roundings (2^-20, and 2^-22 of
    its value).  The probabilities enter the second product with 8 significant bits or more
    (2^-8 each, the smallest with 2^-19 of the largest), and the output is rounded to bf16
    (2^-8 of its value).
    """
    B, H, _ = q_nope.shape
    val, pe = values(q8, scale), kpe.cpu().to(D).view(-1, 64)
    qn, qp, idx = q_nope.cpu().to(D), q_pe.cpu().to(D), slots.cpu().long()
    c = sm_scale * LOG2E
    out = torch.zeros(B, H, 512, dtype=D)
    lse = torch.full((B, H), -math.inf, dtype=D)
    weights = torch.zeros(idx.shape, dtype=D)
    out_tol, lse_tol = torch.zeros(B, H, 512, dtype=D), torch.zeros(B, H, dtype=D)
    for b in range(B):
        at = torch.nonzero((idx[b] >= 0) & (idx[b] < val.shape[0]))[:, 0]
        if not len(at):
            continue
        v, k = val[idx[b, at]], pe[idx[b, at]]
        z = (qn[b] @ v.T + qp[b] @ k.T) * c
        size = (qn[b].abs() @ v.abs().T + qp[b].abs() @ k.abs().T) * abs(c)
        m = z.amax(1, keepdim=True)
        p = torch.exp2(z - m)
        total = p.sum(1, keepdim=True)
        p = p / total
        out[b], lse[b] = p @ v, (m + torch.log2(total))[:, 0]
        weights[b, at] = p.sum(0)
        qerr = 2.0 ** -20 * qn[b].abs().amax(1, keepdim=True) * v.abs().sum(1) * abs(c)
        dz = (600 * 2.0 ** -24 * size + qerr).amax(1)
        lse_tol[b] = 2 * dz + 2.0 ** -20 + 2.0 ** -22 * lse[b].abs()
        rel = (2.0 ** -8 + 4 * lse_tol[b])[:, None]
        floor = 2.0 ** -19 * p.amax(1, keepdim=True) * v.abs().sum(0)
        out_tol[b] = 2.0 ** -8 * out[b].abs() + rel * (p @ v.abs()) + floor
    return out, lse, weights, out_tol, lse_tol


def append(ckv, kpe, offsets, starts, table, q8, scale, kpe_cache):
    """What dsa_append_q8 leaves in the pools: (q8, scale, kpe) as float64 arrays on the CPU."""
    page, block = q8.shape[1], q8.shape[1] // scale.shape[1]
    q = q8.cpu().float().double().numpy().reshape(-1, 512).copy()
    s = scale.cpu().double().numpy().reshape(-1).copy()
    k = kpe_cache.cpu().double().numpy().reshape(-1, 64).copy()
    x, xk = ckv.cpu().double().numpy(), kpe.cpu().double().numpy()
    for r, start in enumerate(starts.tolist()):
        a, b = offsets[r], offsets[r + 1]
        done = 0
        while done < b - a:
            p = start + done
            n = min(block - p % block, b - a - done)
            pg = p // page
            done += n
            if pg >= table.shape[1] or table[r, pg] < 0 or (table[r, pg] + 1) * page > len(q):
                continue
            slot = int(table[r, pg]) * page + p % page
            new = x[a + done - n:a + done]
            fin = np.abs(new[np.isfinite(new)])
            sc = scale_for(fin.max() if fin.size else 0.0)
            i = slot // block
            if p % block:
                sc = max(sc, s[i])
                old = slice(i * block, slot)
                q[old] = e4m3(np.float32(q[old]) * np.float32(s[i] / sc))
            q[slot:slot + n] = e4m3(np.where(np.isfinite(new), new, np.nan) / sc)
            k[slot:slot + n] = xk[a + done - n:a + done]
            s[i] = sc
    return q, s, k


def evict(acc, lengths, budget, sinks, recent):
    """(keep, new lengths, totals) as nested lists, by sorting."""
    keep, lens, totals = [], [], []
    for row, n in zip(acc.tolist(), lengths.tolist()):
        n = max(0, min(n, len(row)))
        if n > budget:
            fixed = {p for p in range(n) if p < sinks or p >= n - recent}
            key = lambda p: (p not in fixed, -row[p] if row[p] == row[p] else math.inf, p)  # noqa: E731
            got = sorted(sorted(range(n), key=key)[:budget])
        else:
            got = list(range(n))
        keep.append(got + [-1] * (budget - len(got)))
        lens.append(len(got))
        totals.append([row[p] for p in got])
    return keep, lens, totals


def compact(keep, table, new_table, q8, scale, kpe_cache):
    """What dsa_compact_q8 leaves in the pools, as float64 arrays on the CPU."""
    page, block = q8.shape[1], q8.shape[1] // scale.shape[1]
    q0 = q8.cpu().float().double().numpy().reshape(-1, 512)
    s0 = scale.cpu().double().numpy().reshape(-1)
    k0 = kpe_cache.cpu().double().numpy().reshape(-1, 64)
    q, s, k = q0.copy(), s0.copy(), k0.copy()

    def slot(t, r, p):
        if p < 0 or p // page >= t.shape[1] or t[r, p // page] < 0:
            return -1
        x = int(t[r, p // page]) * page + p % page
        return x if x < len(q) else -1

    for r in range(len(keep)):
        for j0 in range(0, len(keep[r]), block):
            moves = []
            for j in range(j0, min(j0 + block, len(keep[r]))):
                if keep[r][j] != -1:
                    a, b = slot(table, r, keep[r][j]), slot(new_table, r, j)
                    if a >= 0 and b >= 0:
                        moves.append((a, b))
            if not moves:
                continue
            big = max(s0[a // block] for a, _ in moves)
            s[moves[0][1] // block] = big
            for a, b in moves:
                ratio = np.float32(s0[a // block]) / np.float32(big) if big > 0 else np.float32(0)
                q[b] = e4m3(np.float32(q0[a]) * ratio)
                k[b] = k0[a]
    return q, s, k
