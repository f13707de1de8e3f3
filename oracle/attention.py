"""Attention-side oracle: head norms + rotation, tree attention over a cache
and eviction, from their definitions in 64 bits (torch CPU, loops)."""

from __future__ import annotations

import math

import torch


def norm_rope(x, pos, freqs, *, rot, layout="half", factor=1.0, weight=None, eps=1e-6, zero_centered=False):
    """x (T, H, D), pos (T): normed and rotated in float64."""
    x = x.double()
    D = x.shape[-1]
    if weight is not None:
        w = weight.double() + (1.0 if zero_centered else 0.0)
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + eps) * w
    y = x.clone()
    for t, p in enumerate(pos.tolist()):
        for i in range(rot // 2):
            a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
            # the angle modulo a turn with whole numbers: exact far into a context
            turns = round(freqs[i] / (2 * math.pi) * 2 ** 80)
            ang = (p * turns % 2 ** 80) / 2 ** 80 * 2 * math.pi
            c, s = factor * math.cos(ang), factor * math.sin(ang)
            y[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
            y[t, :, b] = x[t, :, a] * s + x[t, :, b] * c
    return y


def tree_sees(parents) -> torch.Tensor:
    """(n, n) bool: row i sees token j.  A -2 token sees nothing and is nobody's parent."""
    n = len(parents)
    see = torch.zeros((n, n), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p == -2:
            continue
        if 0 <= p < i and parents[p] != -2:
            see[i] = see[p]
        see[i, i] = True
    return see


def tree_depth(parents) -> list[int]:
    return [int(r.sum()) - 1 for r in tree_sees(parents)]


def attention(q, kn, vn, sees, k, v, scale, token_weight=None):
    """One request: q (n, Hq, D), kn / vn (n, H, D) new, k / v (H, L, D) cached,
    sees (n, n).  Returns out (n, Hq, D), lse (n, Hq), weight sums (H, L + n)."""
    n, hq, D = q.shape
    H, L, _ = k.shape
    g = hq // H
    out = torch.zeros((n, hq, D), dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    sums = torch.zeros((H, L + n), dtype=torch.float64)
    for i in range(n):
        if not sees[i, i]:
            continue
        at = list(range(L)) + [L + j for j in range(n) if sees[i, j]]
        for h in range(hq):
            kk = torch.cat((k[h // g], kn[:, h // g])).double()[at]
            vv = torch.cat((v[h // g], vn[:, h // g])).double()[at]
            z = kk @ q[i, h].double() * scale
            lse[i, h] = torch.logsumexp(z, 0)
            p = torch.exp(z - lse[i, h])
            out[i, h] = p @ vv
            sums[h // g, at] += p * (1.0 if token_weight is None else float(token_weight[i]))
    return out, lse, sums


def kept(weights, length, budget, sinks, recent) -> list[int]:
    """Positions one head keeps, ascending.  Equal weights: the lower position; NaN is the largest."""
    if length <= budget:
        return list(range(length))
    lo, hi = sinks, length - recent
    mid = sorted(range(lo, hi), key=lambda s: (0, 0.0, s) if math.isnan(weights[s]) else (1, -weights[s], s))
    return sorted(list(range(lo)) + mid[: budget - sinks - recent] + list(range(hi, length)))
