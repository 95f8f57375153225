"""Plain 64-bit forms of the quantised cache (codes, values, attention) and the error
bounds that follow from the kernels' roundings."""
from __future__ import annotations

import math

import numpy as np
import torch

from attention_ref import U32, half_step

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
CODECS = [E4M3, INT8]


def e4m3_table() -> np.ndarray:
    """Value of each of the 256 codes (NaN for 0x7f and 0xff)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, (1 + m / 8) * 2.0 ** (e - 7), m / 8 * 2.0 ** -6)
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


def values(codes: np.ndarray, codec) -> np.ndarray:
    """float64 values of uint8 codes (before the scale)."""
    return codes.view(np.int8).astype(np.float64) if codec is INT8 else e4m3_table()[codes]


def encode(x: torch.Tensor, codec):
    """(uint8 codes, fp32 scales) of rows ``[..., D]``; the codes of rows that are not finite
    mean nothing."""
    most = torch.finfo(x.dtype).max
    x = x.detach().cpu().float().numpy()
    amax = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0, x)
    amax = np.maximum(np.where(bad, 0, amax), np.float32(2.0 ** -100)).astype(np.float32)
    if codec is INT8:
        scale, inverse = amax / np.float32(127), np.float32(127) / amax
        codes = np.rint(x * inverse[..., None]).astype(np.int8).view(np.uint8)
    else:
        # the least power of two that brings amax to 448 or below
        e = np.ceil(np.log2(amax.astype(np.float64) / 448))
        e = np.where(amax / 2.0 ** e > 448, e + 1, e)
        e = np.where(amax / 2.0 ** (e - 1) <= 448, e - 1, e)
        scale = (2.0 ** e).astype(np.float32)
        y = x.astype(np.float64) / scale[..., None].astype(np.float64)
        table = e4m3_table()[:127]           # 0 .. 448, ascending
        a = np.abs(y)
        up = np.searchsorted(table, a).clip(0, 126)
        down = np.maximum(up - 1, 0)
        low, high = a - table[down], table[up] - a
        pick = np.where((low < high) | ((low == high) & (down % 2 == 0)), down, up)
        # a code whose value the rows' type cannot hold is the one below
        pick = np.where(table[pick] * scale[..., None].astype(np.float64) > most, pick - 1, pick)
        codes = (pick + np.where(np.signbit(y), 128, 0)).astype(np.uint8)
    return codes, np.where(bad, np.float32(np.nan), scale).astype(np.float32)


def attention(q, k, ks, v, vs, scale: float, dtype: torch.dtype):
    """One query of ``q [group, D]`` over ``k``, ``v [n, D]`` (float64 code values) with row scales
    ``ks``, ``vs [n]``: (out, lse, bound on |out error|, bound on |lse error|)."""
    q, k, ks, v, vs = (t.double() for t in (q, k, ks, v, vs))
    n, d = k.shape
    g = q.shape[0]
    if n == 0:
        zero = torch.zeros(g, d, dtype=torch.float64, device=q.device)
        return zero, torch.full((g,), -math.inf, dtype=torch.float64, device=q.device), zero, zero[:, 0]
    x = (q @ k.T) * ks * scale
    top = x.max(1, keepdim=True).values
    e = torch.exp(x - top)
    z = e.sum(1, keepdim=True)
    p = e / z
    val = v * vs[:, None]
    out = p @ val
    lse = (top + z.log())[:, 0]
    # Scores: d exact products summed in fp32 (each addition off by a step at most), three
    # roundings of the scaled score and its distance from the running maximum; the
    # exponential 2^-21.
    mag = ((q.abs() @ k.abs().T) * ks.abs()).max(1, keepdim=True).values * scale
    spread = (top - x.min(1, keepdim=True).values + x.abs().max(1, keepdim=True).values)
    rel = (d + 8) * 2 * U32 * mag + 4 * U32 * spread * 1.45 + 2.0 ** -21
    # Each weight with its V row's scale becomes a pair of bf16 (what the first rounding leaves,
    # 2^-8 of it at most, is rounded again); sums over n tokens and the joins are fp32; the result is
    # rounded once.
    w = 2.0 ** -15
    sums = 2 * (n + 64) * U32
    u = half_step(dtype)
    otol = (p @ val.abs()) * (w + 2 * rel + 2 * sums) * 1.01 + u * 1.01 * out.abs()
    # fp32 has no normal numbers below 2^-126: a weight, its product with its scale, or either
    # when it is rescaled, may count as zero there, or as a step of 2^-126 more.  The largest weight is
    # at least 1/2 when the last maximum stands, so this is off by at most 4 * 2^-126 per token, times
    # its value or (after the scale) its code, of at most 448.
    otol = otol + n * 2.0 ** -124 * (val.abs().max() + 448) + torch.finfo(dtype).tiny
    ltol = (rel + sums)[:, 0] + 4 * U32 * (lse.abs() + 1)
    return out, lse, otol, ltol
