"""Routing by groups, rotary positions and attention in 64 bits, from their definitions, on the CPU."""
from __future__ import annotations

import math

import numpy as np
import torch


def grouped_topk(logits, topk, num_groups=1, topk_groups=1, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    """(weights float64 [M, topk], ids int32 [M, topk]), a token at a time."""
    x = logits.double().numpy()
    M, E = x.shape
    size = E // num_groups
    weights, ids = np.zeros((M, topk)), np.zeros((M, topk), dtype=np.int32)
    with np.errstate(over="ignore"):
        for t in range(M):
            l = np.where(np.isnan(x[t]), -np.inf, x[t])
            if scoring == "sigmoid":
                s = 1.0 / (1.0 + np.exp(-l))
            else:
                top = l.max()
                s = np.array([1.0 if v == top else math.exp(v - top) for v in l])
                s = s / s.sum()
            c = l if bias is None else s + bias.double().numpy()
            c = np.where(np.isnan(c), -np.inf, c)
            worth = []
            for g in range(num_groups):
                best = sorted(c[g * size:(g + 1) * size], reverse=True)
                w = best[0] if bias is None or size == 1 else best[0] + best[1]
                worth.append(-np.inf if np.isnan(w) else w)
            kept = sorted(range(num_groups), key=lambda g: (-worth[g], g))[:topk_groups]
            order = sorted((e for g in kept for e in range(g * size, (g + 1) * size)), key=lambda e: (-c[e], e))[:topk]
            ids[t], w = order, s[order]
            if renormalize:
                w = w / w.sum() if w.sum() > 0 else np.zeros(topk)
            weights[t] = w * scale
    return torch.from_numpy(weights), torch.from_numpy(ids)


def rotary(x, positions, freq, interleaved=False, factor=1.0):
    """Rows x [T, H, D] turned, float64; angles in 80-bit floats."""
    angle = positions.numpy().astype(np.longdouble)[:, None] * freq.double().numpy().astype(np.longdouble)[None, :]
    cos, sin = (torch.from_numpy((f(angle) * factor).astype(np.float64))[:, None, :] for f in (np.cos, np.sin))
    n, out = 2 * freq.numel(), x.double().clone()
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    a, b = x.double()[..., first], x.double()[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    return out


def attention(q, k, v, seen, scale):
    """Rows q [n, H, D] over keys k, v [m, G, D], row i seeing keys where seen [n, m]: (out float64 [n, H, D], error float64 [n, H, D]).

    error: how far a computation may be off that sums in 32 bits and rounds the softmax's terms to q's type for the second product; the
    result's own rounding is not in it.  With u half a step of the type and |.| taken of every factor:
      scores: D / 16 sums of exact products, a rounding or truncation (2^-23) each, four more for scale, difference and exponential: d = 2^-23 (D / 16 + 4) max |s|,
              which the terms have as a relative error, above and below the line: 2 d; the exponential itself 2^-21
      terms rounded once: u;  sums of m terms: 2^-23 (m / 16 + 4), above and below the line
    all of it times the sum of |p v|."""
    n, H, D = q.shape
    m, G, _ = k.shape
    out, error = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    u = torch.finfo(q.dtype).eps / 2
    for h in range(H):
        kh, vh, qh = k[:, h // (H // G)].double(), v[:, h // (H // G)].double(), q[:, h].double()
        for i in range(n):
            at = seen[i].nonzero()[:, 0]
            if at.numel() == 0:
                continue
            s = scale * (kh[at] @ qh[i])
            p = torch.exp(s - s.max())
            p = p / p.sum()
            out[i, h] = p @ vh[at]
            d = 2.0 ** -23 * (D / 16 + 4) * float((kh[at].abs() @ qh[i].abs()).max()) * scale
            error[i, h] = (p @ vh[at].abs()) * (u + 2 * d + 2.0 ** -20 + 2.0 ** -22 * (at.numel() / 16 + 4))
    return out, error
