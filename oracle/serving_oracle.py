"""CPU oracle, in 64 bits, for rotary positions and the paged-cache operators.

TEST INFRASTRUCTURE ONLY: only ``tests/`` may import it.  None of it has a counterpart in the
reference; it restates the operators' formulas sequence by sequence, slot by slot, on dense rows.
"""
from __future__ import annotations

import math

import torch


def rotary(x, positions, inv_freq, axes, interleaved=False, scale=1.0, inverse=False):
    """x [..., L, D] with positions [A, ..., L]: pair i of a row, as a complex number, times
    ``scale * exp(i theta)``.  Returns float64."""
    y = x.detach().to("cpu", torch.float64).clone()
    n = inv_freq.numel()
    pos = positions.to("cpu", torch.float64)
    inv = inv_freq.to("cpu", torch.float64)
    for i in range(n):
        theta = pos[axes[i]] * inv[i] * (-1 if inverse else 1)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, n + i)
        u, w = y[..., a].clone(), y[..., b].clone()
        y[..., a] = scale * (u * theta.cos() - w * theta.sin())
        y[..., b] = scale * (w * theta.cos() + u * theta.sin())
    return y


def visible(n, window, sinks):
    """Slots that the newest of n tokens sees."""
    return [j for j in range(n) if n - 1 - j < window or j < sinks]


def decode(q, k, v, n, window, sinks, scale=None, logits=None):
    """One sequence: q [Hq, D], k and v [Hkv, >= n, D].  Returns float64 (o [Hq, D], lse [Hq] in
    base 2, p [Hq, n] with 0 where a slot is not visible, amount [Hq, D] = sum p |v|, and
    delta [Hq] = the largest sum |q k| * scale, by which 32-bit scores may be off)."""
    hq, d = q.shape
    g = hq // k.shape[0]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    vis = visible(n, window, sinks)
    o, amount = torch.zeros(hq, d, dtype=torch.float64), torch.zeros(hq, d, dtype=torch.float64)
    lse = torch.full((hq,), -math.inf, dtype=torch.float64)
    p = torch.zeros(hq, n, dtype=torch.float64)
    delta = torch.zeros(hq, dtype=torch.float64)
    q = q.to("cpu", torch.float64)
    for h in range(hq):
        kk, vv = (t[h // g].to("cpu", torch.float64)[vis] for t in (k, v))
        s = (kk @ q[h]) * scale
        both = s if logits is None else torch.cat([s, logits[h:h + 1].to("cpu", torch.float64)])
        if both.numel() == 0 or bool((both == -math.inf).all()):
            continue
        total = torch.logsumexp(both, 0)
        e = torch.exp(s - total)
        p[h, vis] = e
        o[h], amount[h] = e @ vv, e @ vv.abs()
        lse[h] = total / math.log(2)
        if vis:
            delta[h] = (kk.abs() @ q[h].abs()).max() * abs(scale)
    return o, lse, p, amount, delta


def evict(weights, positions, n, seen, keep, sinks, recent):
    """One KV head of one sequence of n > keep slots: (free, movers), the slots below keep that
    come free and the kept slots from keep on that fill them, both in order."""
    w = [float(x) for x in weights[:n]]
    pos = [int(x) for x in positions[:n]]

    def rank(j):
        held = pos[j] < sinks or pos[j] >= seen - recent
        x = -math.inf if math.isnan(w[j]) else w[j]
        return (0 if held else 1, 0.0 if held else -x, j)

    kept = set(sorted(range(n), key=rank)[:keep])
    return [j for j in range(keep) if j not in kept], sorted(j for j in kept if j >= keep)
