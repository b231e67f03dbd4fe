"""Queries that each rest on one position, so that every position of a long sequence matters.

Over random keys a softmax of n positions is flat, and an output's bound (2^-8 of sum p |v|) exceeds
what one position adds to it.  A query equal to a key q = k scores |k|^2 sm there: with k of 576
values of size 0.6 about 15 (natural logarithm) above the others, whose weights add up to n e^0.2.
So for n up to 32768 the position holds nearly all of the weight, the output is its value within
about 1 %, and a value that is missing, counted twice or taken from elsewhere is off by some tens of
times the bound.
"""
import math

import torch


def spread(count, n, first=0):
    """count positions below n, evenly spread and all different while count <= n: steps of the golden
    section, made prime to n."""
    step = max(1, round(n * 0.618))
    while math.gcd(step, n) > 1:
        step += 1
    return (first + step * torch.arange(count)) % n


def aim(keys, at):
    """bf16 (q_nope, q_pe) [.., 512], [.., 64]: the keys [n, 576] at the positions `at`."""
    q = keys[at.to(keys.device)].to(torch.bfloat16)
    return q[..., :512].contiguous(), q[..., 512:].contiguous()
