"""The 8-bit decode in 64 bits, with bounds that follow each rounding of the kernel.

Unlike q8_reference.attend, whose tolerance holds the values unweighted, every part here goes with
the weight that an entry has, so that a slot of a far larger scale hides nothing.
"""
import math

import torch

LOG2E = math.log2(math.e)
D = torch.float64


def attend(q_nope, q_pe, q8, scale, kpe, slots, sm_scale):
    """(output, lse, weights) and their tolerances, float64 on the cache's device.

    * A score is a sum of 576 products in fp32: 600 roundings of 2^-24 of sum |q v| at most (24 for
      the scalings); the query is kept to 2^-20 of its row's largest value.  Both give an
      interval of each score, and the intervals of all scores one of each probability and of lse.
    * A probability times its scale is three e4m3 terms: each keeps 4 significant bits of what the
      one before left, 2^-12 in all, and the last one's step, 2^-9 / 2^8, rounds off at most
      2^-18, where the largest of the row is 3.5 or more: 2^-19 of the largest (p scale).  Only where
      the weight lies on scales below 2^-88 of the largest one is the row's largest less; the sum of
      the probabilities is then 2^88 or more: 2^-18 / 3.5 / 2^88 < 2^-107 of that scale.
    * Sums over the entries: a step of 32 entries adds a rounding of 2^-23 for itself and three for
      its products; exponentials (2^-22) and up to a rescale a tile: 2^-23 (topk / 8 + 64) in all.
    * lse is m + log2(l): each with 2^-22 of its size (log2 l is at most 100), 2^-20 for the sum.
    * The output is rounded to bf16: 2^-8 of its value.
    """
    B, H, _ = q_nope.shape
    topk = slots.shape[1]
    dev = q8.device
    block = q8.shape[1] // scale.shape[1]
    raw = q8.float().to(D).view(-1, 512)
    s = scale.to(D).view(-1).repeat_interleave(block)
    pe = kpe.to(D).view(-1, 64)
    qn, qp, idx = q_nope.to(D), q_pe.to(D), slots.long()
    c = abs(sm_scale) * LOG2E
    out = torch.zeros(B, H, 512, dtype=D, device=dev)
    lse = torch.full((B, H), -math.inf, dtype=D, device=dev)
    weights = torch.zeros(B, topk, dtype=D, device=dev)
    # where there is nothing: the value itself
    out_tol, lse_tol, w_tol = (torch.full_like(t, 1e-37) for t in (out, lse, weights))
    for b in range(B):
        at = torch.nonzero((idx[b] >= 0) & (idx[b] < raw.shape[0]))[:, 0]
        if not len(at):
            continue
        x8, sk, k = raw[idx[b, at]], s[idx[b, at]], pe[idx[b, at]]
        v = x8 * sk[:, None]
        z = (qn[b] @ v.T + qp[b] @ k.T) * sm_scale * LOG2E
        size = (qn[b].abs() @ v.abs().T + qp[b].abs() @ k.abs().T) * c
        dz = 600 * 2.0 ** -24 * size + 2.0 ** -20 * qn[b].abs().amax(1, keepdim=True) * v.abs().sum(1) * c
        up, low = z + dz, z - dz
        m = up.amax(1, keepdim=True)

        def total(t):
            return torch.exp2(t - m).sum(1, keepdim=True)

        def share(own, rest_of, rest_own):  # own / (own + the others), the others at their other end
            rest = (total(rest_of) - torch.exp2(rest_own - m)).clamp(min=0)
            e = torch.exp2(own - m)
            return torch.where(e > 0, e / (e + rest).clamp(min=1e-300), torch.zeros_like(e))

        mid = z.amax(1, keepdim=True)
        p = torch.exp2(z - mid)
        sums = p.sum(1, keepdim=True)
        p = p / sums
        err = torch.maximum(share(up, low, low) - p, p - share(low, up, up)).clamp(min=0)
        out[b], lse[b] = p @ v, (mid + torch.log2(sums))[:, 0]
        weights[b, at] = p.sum(0)
        high = torch.logsumexp(up * math.log(2.0), 1) / math.log(2.0)
        lows = torch.logsumexp(low * math.log(2.0), 1) / math.log(2.0)
        lse_own = 2.0 ** -20 + 2.0 ** -22 * (lse[b].abs() + 100)
        lse_tol[b] = torch.maximum(high - lse[b], lse[b] - lows) + lse_own
        rel = 2.0 ** -12 + (topk / 8 + 64) * 2.0 ** -23
        last = (2.0 ** -19 * (p * sk).amax(1, keepdim=True) + 2.0 ** -107 * sk.max()) * x8.abs().sum(0)
        near = err @ v.abs() + rel * (p @ v.abs()) + last
        out_tol[b] = near + 2.0 ** -8 * (out[b].abs() + near) + 1e-37
        # a weight is 2^(score - lse): the exponential, the difference's rounding and lse's own
        w_tol[b, at] = (err + p * (2.0 ** -20 + lse_own[:, None] + 2.0 ** -23 * (z.abs() + lse[b].abs()[:, None]))).sum(0) + 1e-37
    return (out, lse, weights), (out_tol, lse_tol, w_tol)


def check(got, q, cache, slots, sm_scale):
    """Asserts that (output, lse[, weights]) lie within the bounds; returns the worst ratios."""
    want, tol = attend(*q, *cache, slots, sm_scale)
    worst = []
    for name, g, w, t in zip(("output", "lse", "weights"), got, want, tol):
        dead = ~torch.isfinite(w)
        assert torch.equal(g.to(D)[dead], w[dead]), name
        over = ((g.to(D) - w).abs() / t)[~dead]
        assert not torch.isnan(over).any(), f"{name}: NaN"
        worst.append(float(over.max()) if over.numel() else 0.0)
        assert worst[-1] <= 1, f"{name}: {worst[-1]:.3g} times its bound, {(over > 1).sum()} of {over.numel()}"
    return worst
