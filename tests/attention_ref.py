"""Plain 64-bit forms of prompt attention, attention weights and eviction, and
the error bounds that follow from the kernels' roundings."""
from __future__ import annotations

import math

import numpy as np
import torch

U32 = 2.0 ** -24


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def cumulative(lens):
    return [0] + np.cumsum(lens).tolist()


def attention(q, k, v, ahead: int, causal: bool, scale: float):
    """One sequence in float64: (out, lse, bound on |out error|, bound on |lse error|).
    q [m, Hq, D], k, v [n, Hkv, D]; query i sees keys j <= i + ahead."""
    m, hq, d = q.shape
    n, hkv = k.shape[:2]
    u = half_step(q.dtype)
    qf, kf, vf = (t.detach().cpu().double() for t in (q, k, v))
    out, otol = torch.zeros(m, hq, d, dtype=torch.float64), torch.zeros(m, hq, d, dtype=torch.float64)
    lse = torch.full((m, hq), -math.inf, dtype=torch.float64)
    ltol = torch.zeros(m, hq, dtype=torch.float64)
    for i in range(m):
        c = max(0, min(n, i + ahead + 1)) if causal else n
        if c == 0:
            continue
        for h in range(hkv):
            g = slice(h * hq // hkv, (h + 1) * hq // hkv)
            s = qf[i, g] @ kf[:c, h].T * scale
            top = s.max(1, keepdim=True).values
            e = torch.exp(s - top)
            z = e.sum(1, keepdim=True)
            p = e / z
            out[i, g] = p @ vf[:c, h]
            lse[i, g] = (top + z.log())[:, 0]
            # Scores: d fp32 additions of exact products, then one rounding each of
            # the scaled score and the running maximum; the exponential 2^-21.
            mag = (qf[i, g].abs() @ kf[:c, h].abs().T).max() * scale
            rel = float(d * U32 * mag + 4 * U32 * s.abs().max() * 1.45 + 2.0 ** -21 + c * U32)
            # p is rounded to the element type (half a step; in fp16 below its
            # smallest normal by at most 2^-25 of the row's largest p), the products
            # and their sums are fp32, the result is rounded once more.
            a = p @ vf[:c, h].abs()
            tiny = 2.0 ** -25 * c * vf[:c, h].abs().max() if q.dtype == torch.float16 else 0.0
            otol[i, g] = a * (u + 2 * rel + c * U32) * 1.01 + (u * 1.01) * out[i, g].abs() + tiny
            otol[i, g] += torch.finfo(q.dtype).tiny
            ltol[i, g] = rel + 4 * U32 * (lse[i, g].abs() + 1)
    return out, lse, otol, ltol


def weights(q, lse, k, ahead: int, causal: bool, scale: float):
    """One request in float64: (weights [Hkv, n], bound on their error)."""
    m, hq, d = q.shape
    n, hkv = k.shape[:2]
    qf, kf, lf = (t.detach().cpu().double() for t in (q, k, lse))
    w = torch.zeros(hkv, n, dtype=torch.float64)
    tol = torch.zeros(hkv, n, dtype=torch.float64)
    rows = m * hq // hkv
    for i in range(m):
        c = max(0, min(n, i + ahead + 1)) if causal else n
        for j in range(hq):
            h = j * hkv // hq
            if c == 0 or lf[i, j] == -math.inf:
                continue
            s = kf[:c, h] @ qf[i, j] * scale
            e = torch.exp(s - lf[i, j])
            w[h, :c] += e
            mag = (kf[:c, h].abs() @ qf[i, j].abs()) * scale
            rel = d * U32 * mag + 4 * U32 * (s.abs() + lf[i, j].abs()) * 1.45 + 2.0 ** -21
            tol[h, :c] += e * (rel + rows * U32)
    return w, tol


def evict(score, place, n: int, keep: int, recent: int, end: int):
    """(destination slots, source slots) of one sequence and head: score and
    place (positions) of its n tokens, in slot order."""
    if n <= keep:
        return [], []
    def rank(t):
        s = float(score[t])
        return (0 if place[t] >= end - recent else 1,
                -math.inf if math.isnan(s) else 0 if s == math.inf else 1,
                -s if not (math.isnan(s) or s == math.inf) else 0.0, t)
    stays = set(sorted(range(n), key=rank)[:keep])
    return ([t for t in range(keep) if t not in stays],
            [t for t in range(keep, n) if t in stays])


def assert_within(got, ref, tol, what=""):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    assert torch.equal(got[~fin & ~torch.isnan(ref)], ref[~fin & ~torch.isnan(ref)]), what
    over = (got - ref).abs()[fin] - tol[fin]
    assert over.numel() == 0 or over.max() <= 0, \
        f"{what}: {int((over > 0).sum())} values beyond their bound, by up to {over.max():.3e}"
