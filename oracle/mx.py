"""Microscaling formats and 4-bit experts in 64 bits (numpy), from the
definitions: groups of 32 columns share 2^e, e the smallest integer >= -127
that keeps the group's largest magnitude within the format."""

from __future__ import annotations

import math

import numpy as np

GROUP = 32
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _exponent(big: float, top: float) -> int:
    if big == 0.0:
        return -127
    e = math.frexp(big)[1] - math.frexp(top)[1]
    while math.ldexp(top, e) < big:
        e += 1
    while math.ldexp(top, e - 1) >= big:
        e -= 1
    return max(e, -127)


def group_exponents(v: np.ndarray, top: float) -> np.ndarray:
    """e of each group of v [R, K] -> [R, K / 32]."""
    g = np.abs(np.asarray(v, dtype=np.float64)).reshape(v.shape[0], -1, GROUP).max(axis=2)
    return np.vectorize(lambda b: _exponent(float(b), top), otypes=[np.int64])(g) if g.size else g.astype(np.int64)


def _nearest(v: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the nearest grid value of |v|, ties to the even index."""
    a = np.abs(v)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo = hi - 1
    dl, dh = a - grid[lo], grid[hi] - a
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def e4m3_grid() -> np.ndarray:
    """The 127 non-negative e4m3 values in code order."""
    return np.array([math.ldexp(m, -9) if e == 0 else math.ldexp(8 + m, e - 10)
                     for e in range(16) for m in range(8)][:127])


def round_mx8(v: np.ndarray) -> np.ndarray:
    """v [R, K] rounded to MX8, as the values the result stands for."""
    v = np.asarray(v, dtype=np.float64)
    if not v.size:
        return v.copy()
    e = np.repeat(group_exponents(v, 448.0), GROUP, axis=1)
    s = np.ldexp(1.0, e)
    return np.sign(v) * e4m3_grid()[_nearest(v / s, e4m3_grid())] * s


def quantize_mx4(w: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes [R, K / 2], scale bytes [R, K / 32]) of w [R, K]."""
    w = np.asarray(w, dtype=np.float64)
    e = group_exponents(w, 6.0)
    v = w / np.ldexp(1.0, np.repeat(e, GROUP, axis=1))
    c = (_nearest(v, E2M1) | (np.signbit(v) << 3)).astype(np.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4), (e + 127).astype(np.uint8)


def values_mx4(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    c = np.empty((codes.shape[0], codes.shape[1] * 2), dtype=np.uint8)
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    v = np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]
    return v * np.ldexp(1.0, np.repeat(scales.astype(np.int64) - 127, GROUP, axis=1))


def expert(x: np.ndarray, w13: np.ndarray, w2: np.ndarray, mx8: bool) -> tuple[np.ndarray, np.ndarray]:
    """(act, y) of rows x through one expert's weight values; with mx8 act is
    rounded to MX8 before the down product."""
    I = w13.shape[0] // 2
    gate, up = x @ w13[:I].T, x @ w13[I:].T
    act = gate / (1.0 + np.exp(-gate)) * up
    if mx8:
        act = round_mx8(act)
    return act, act @ w2.T


def rms_norm(r: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    r = np.asarray(r, dtype=np.float64)
    return r / np.sqrt((r * r).mean(axis=1, keepdims=True) + eps) * weight
