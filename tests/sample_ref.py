"""float64 restatement of ``sample_tokens`` on the CPU, a row at a time."""

import math

import torch


def kept(x, T, k, p, m):
    """(indexes that the cuts keep, in the order of the logits; their float64 weights)."""
    v = x.double().tolist()
    order = sorted((i for i, a in enumerate(v) if a > -math.inf), key=lambda i: (-v[i], i))
    if not order:
        return [], []
    if not T > 0:
        return order[:1], [1.0]
    top = v[order[0]]
    w = [1.0 if v[i] == top else math.exp((v[i] - top) / T) if (v[i] - top) / T > -800 else 0.0 for i in order]
    if k and k > 0:
        order, w = order[:k], w[:k]
    if p is not None and p < 1:
        need, run, n = p * math.fsum(w), 0.0, 0
        while n == 0 or run < need:
            if n == len(w):
                break
            run += w[n]
            n += 1
        order, w = order[:n], w[:n]
    both = [(i, a) for i, a in zip(order, w) if a >= (m or 0.0)]
    return [i for i, _ in both], [a for _, a in both]


def draw(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """The token and how near the draw was to another: the distance of u times the sum from
    the borders of the token's weight, in sums."""
    idx, w = kept(x, T, k, p, m)
    if not idx:
        return -1, 1.0
    by_index = sorted(zip(idx, w))
    total = math.fsum(w)
    goal, run = u * total, 0.0
    for i, a in by_index:
        if run + a > goal and a > 0:
            return i, min(goal - run, run + a - goal) / total
        run += a
    return [i for i, a in by_index if a > 0][-1], 0.0
