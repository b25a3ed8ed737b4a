"""Plain 64-bit forms of the operators behind the attention, and what their tests share."""
from __future__ import annotations

import math

import numpy as np

from tests.helpers import bf16_to_f32

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
INT4 = np.array([c - 16 * (c > 7) for c in range(16)], dtype=np.float64)
VALUES = {"int4": INT4, "e2m1": E2M1}


def f32_to_bf16(x) -> np.ndarray:
    """Nearest even; NaN stays NaN."""
    f = np.asarray(x, dtype=np.float32)
    u = f.view(np.uint32).astype(np.uint64)
    r = ((u + ((u >> 16) & 1) + 0x7FFF) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7FC0), r)


def f64(bits: np.ndarray) -> np.ndarray:
    return bf16_to_f32(bits).astype(np.float64)


# ---- products with 4-bit weights ------------------------------------------------

def w4_weight(codes: np.ndarray, scales: np.ndarray, group: int, fmt: str) -> np.ndarray:
    """codes [rows][cols / 2], scales bits [rows][cols / group] -> [rows][cols]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[0], -1)
    return VALUES[fmt][c] * np.repeat(f64(scales), group, axis=1)


def w4_bound(x, w, exact, group) -> np.ndarray:
    """The output's own rounding, 2^-8 of it, and f32 sums of `cols` exact products and of
    cols / group scaled sums in any order: each addition off by 2^-23 of what it adds at most
    (a matrix product's additions need not be to nearest), each scaling by 2^-24."""
    cols = x.shape[1]
    steps = cols + cols // group + 2
    return 2.0 ** -8 * np.abs(exact) + steps * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T) + 2.0 ** -133


def random_w4(rng, m, n, k, group):
    x = f32_to_bf16(rng.standard_normal((m, k)) * np.exp(0.7 * rng.standard_normal(k)))
    codes = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    scales = f32_to_bf16(0.01 * np.exp(0.5 * rng.standard_normal((n, k // group))))
    return x, codes, scales


# ---- norms around a block ---------------------------------------------------------

def norm_residual(y, r, *, eps, post_norm, post, gate, pre, a, b, r_eps):
    """(r', x, bounds of both) in 64 bits.  r_eps: half a step of the residual's type.

    A sum of n squares in f32 is off by n 2^-24 of itself at most, its root by half of that; the
    mean, eps, root, division and the products behind them add 2^-24 each (eight in all)."""
    n = y.shape[1]
    e = 2.0 ** -24
    rel = (n / 2 + 8) * e
    t = y / np.sqrt((y * y).mean(1, keepdims=True) + eps) * post if post_norm else y * post
    t = t * gate
    out = a * r + b * t
    err = np.abs(b * t) * (rel + 4 * e) + np.abs(a * r) * 2 * e + np.abs(out) * e
    inv = 1 / np.sqrt((out * out).mean(1, keepdims=True) + eps)
    x = out * inv * pre
    shift = np.sqrt((err * err).mean(1, keepdims=True)) * inv  # of the root, relative
    x_err = (err * inv + np.abs(out) * inv * (shift + rel)) * np.abs(pre) + np.abs(x) * (4 * e + 2.0 ** -8)
    return out, x, err + np.abs(out) * r_eps, x_err


# ---- sampling -----------------------------------------------------------------------

def sample_weights(z, temperature, top_k, top_p, min_p):
    """The weights of a row by index, 0 for what is not kept (z in 64 bits)."""
    z = np.where(np.isnan(z), -np.inf, z)
    alive = z > -np.inf
    w = np.zeros(z.size)
    if not alive.any():
        return w
    top = z.max()
    greedy = not temperature > 0
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        w = np.exp((z - top) / (1.0 if greedy else temperature))
    w = np.where(z == top, 1.0, np.nan_to_num(w, nan=0.0))
    order = np.lexsort((np.arange(z.size), -z))[:int(alive.sum())]
    k = 1 if greedy else top_k
    if 0 < k < order.size:
        order = order[:k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        order = order[:int(np.searchsorted(sums, max(top_p, 0.0) * sums[-1], side="left")) + 1]
    kept = np.zeros(z.size, bool)
    kept[order] = True
    if min_p > 0:
        kept &= (w >= min_p) | (z == top)
    return np.where(kept, w, 0.0)


def sample_token(w, u):
    """(token, distance of u from the next border, as a part of the whole)."""
    sums = np.cumsum(w)
    if sums[-1] == 0:
        return -1, 1.0
    at = (min(max(u, 0.0), 1 - 2.0 ** -24) if not math.isnan(u) else 0.0) * sums[-1]
    i = int(np.searchsorted(sums, at, side="right"))
    alive = np.flatnonzero(w)
    i = min(i, int(alive[-1]))
    borders = np.unique(sums[alive])[:-1]  # the last is the end
    return i, float(np.min(np.abs(borders - at)) / sums[-1]) if borders.size else 1.0
