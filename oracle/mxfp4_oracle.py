"""MXFP4 in 64 bits on the CPU, from the definition of the format (OCP microscaling: e2m1 elements, a power-of-two
scale for each 32 of them).  TEST INFRASTRUCTURE ONLY."""
from __future__ import annotations

import numpy as np
import torch

from .moe_oracle import gating_topk

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _rows64(x) -> np.ndarray:
    return x.double().numpy() if isinstance(x, torch.Tensor) else np.asarray(x, dtype=np.float64)


def mxfp4_exponent(amax: np.ndarray) -> np.ndarray:
    """Scale bytes of blocks with these largest magnitudes."""
    _, e = np.frexp(np.where(np.isfinite(amax), amax, 1.0))  # amax = m 2^e, m in [1/2, 1)
    b = np.clip(e - 1 - 2 + 127, 0, 254)
    b = np.where(amax == 0, 127, b)
    return np.where(np.isfinite(amax), b, 255).astype(np.int64)


def mxfp4_round(v: np.ndarray) -> np.ndarray:
    """Index into LEVELS of the nearest value of |v| (ties to the even index, above 6: 6)."""
    a = np.abs(v)
    borders = np.append((LEVELS[:-1] + LEVELS[1:]) / 2, np.inf)
    low = np.searchsorted(borders[:-1], a, side="left")  # a on a border: the lower level's index
    return np.where((a == borders[low]) & (low % 2 == 1), low + 1, low)


def mxfp4_quant_rows(x):
    """codes uint8 [rows, K / 2] and scale bytes uint8 [rows, K / 32] of rows [rows, K]."""
    x = _rows64(x)
    rows, K = x.shape
    blocks = x.reshape(rows, K // 32, 32)
    with np.errstate(invalid="ignore"):
        amax = np.abs(blocks).max(axis=2)
    b = mxfp4_exponent(amax)
    bad = (b == 255)[..., None]
    v = np.where(bad, 0.0, blocks) * 2.0 ** (127.0 - np.where(bad, 127, b[..., None]))
    code = mxfp4_round(v) + 8 * (np.signbit(v) & ~bad)
    code = code.reshape(rows, K // 2, 2).astype(np.uint8)
    return code[..., 0] | (code[..., 1] << 4), b.astype(np.uint8)


def mxfp4_values(codes, scales) -> np.ndarray:
    """What codes [.., K / 2] and scale bytes [.., K / 32] stand for, in 64 bits."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    nibble = np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[:-1] + (scales.shape[-1], 32))
    v = LEVELS[nibble & 7] * np.where(nibble & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(codes.shape[:-1] + (codes.shape[-1] * 2,))


def mxfp4_held(x) -> np.ndarray:
    """Rows as the format holds them, in 64 bits."""
    return mxfp4_values(*mxfp4_quant_rows(x))


def _held_with_exponent(x: np.ndarray, b: np.ndarray) -> np.ndarray:
    unit = 2.0 ** (b - 127.0)[..., None]
    return LEVELS[mxfp4_round(x / unit)] * np.sign(x) * unit


def mxfp4_doubt(x: np.ndarray, err: np.ndarray) -> np.ndarray:
    """How far, element by element, the held value of rows known to within +- err may lie from that of x: an element next to
    a border between two levels may take either, a block whose largest magnitude is next to a power of two either scale."""
    rows, K = x.shape
    xb, eb = x.reshape(rows, K // 32, 32), err.reshape(rows, K // 32, 32)
    mag = np.abs(xb)
    amax, up, down = mag.max(axis=2), (mag + eb).max(axis=2), np.maximum(mag - eb, 0).max(axis=2)
    ref = _held_with_exponent(xb, mxfp4_exponent(amax))
    worst = np.zeros_like(xb)
    for b in (mxfp4_exponent(up), mxfp4_exponent(down)):
        for y in (xb, xb + eb, xb - eb):
            worst = np.maximum(worst, np.abs(_held_with_exponent(y, b) - ref))
    return worst.reshape(rows, K)


def fused_moe_mxfp4(hidden_states, w1, w1_scale, w2, w2_scale, logits, topk: int, renormalize: bool = True):
    """The layer in 64 bits: (out [M, H], doubt [M, H]).  doubt bounds what 32-bit sums may change by way of the activated
    rows' quantisation: a gate or up sum of K products is taken to be off by at most (K / 64 + 4) 2^-24 of the sum of the
    products' magnitudes (a rounding per 64 products, four more where these are summed), the activated value by that through silu'(g) <= 1.1
    and |silu(g)| <= |g|, plus 2^-20 of itself for the exponential and the quotient.  Everything else is
    summed in 32 bits, which doubt leaves to the caller."""
    x = mxfp4_held(hidden_states)
    weights, ids = gating_topk(logits, topk, renormalize)
    weights, ids = _rows64(weights), ids.numpy() if isinstance(ids, torch.Tensor) else np.asarray(ids)
    out, doubt = np.zeros_like(x), np.zeros_like(x)
    for e in range(w1.shape[0]):
        token, slot = np.nonzero(ids == e)
        if token.size == 0:
            continue
        m1, m2 = mxfp4_values(w1[e], w1_scale[e]), mxfp4_values(w2[e], w2_scale[e])
        F = m1.shape[0] // 2
        g, u = x[token] @ m1[:F].T, x[token] @ m1[F:].T
        act = g / (1.0 + np.exp(-g)) * u
        off = (x.shape[1] / 64 + 4) * 2.0 ** -24 * (np.abs(x[token]) @ np.abs(m1).T) + 2.0 ** -100
        err = 1.1 * off[:, :F] * (np.abs(u) + off[:, F:]) + np.abs(g) * off[:, F:] + np.abs(act) * 2.0 ** -20
        share = weights[token, slot][:, None]
        rows = (mxfp4_held(act) @ m2.T) * share
        np.add.at(out, token, rows)
        np.add.at(doubt, token, (mxfp4_doubt(act, err) @ np.abs(m2).T) * share)
    return out, doubt
