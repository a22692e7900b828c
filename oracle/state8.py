"""TEST INFRASTRUCTURE ONLY - optimizer states in 8 bits, restated on the CPU in numpy float64.

The form is ``include/ranncgrad.h``'s "optimizer states in 8 bits"; the reference has no counterpart.  Everything is worked
out per tensor, flat, from the definition: the numbers of e4m3 are a table, rounding is a search in it.  Pinned in
``tests/test_state8_host.py`` against torch's own float8 conversion and against values worked out by hand.
"""
from __future__ import annotations

from typing import Dict, Tuple

import numpy as np

BLOCK = 256
PLACE, FIRST, ROOT = 0xD1B54A33, 0xABC98389, 0x8CB92BA7
EPS = 2.0 ** -24           # half a step of fp32, relative

#: e4m3's numbers from 0 to 448, by code
GRID = np.array([f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8)][:-1])


def blocks(x: np.ndarray) -> np.ndarray:
    """[number of blocks, 256], the last one filled up with zeros."""
    x = np.asarray(x)
    n = -(-x.size // BLOCK) * BLOCK
    out = np.zeros(n, dtype=x.dtype)
    out[:x.size] = x.reshape(-1)
    return out.reshape(-1, BLOCK)


def values_of(codes: np.ndarray) -> np.ndarray:
    """The e4m3 numbers of uint8 codes (no NaN codes: the form has none)."""
    codes = np.asarray(codes, dtype=np.uint8)
    assert not ((codes & 0x7F) == 0x7F).any()
    return np.where(codes & 0x80, -1.0, 1.0) * GRID[codes & 0x7F]


def read_back(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """float64 values of flat codes (a second moment's: its root)."""
    k = np.repeat(np.asarray(scales, dtype=np.float64) / 256.0, BLOCK)[:codes.size]
    with np.errstate(invalid="ignore"):
        return values_of(codes) * k


def scale_of(x: np.ndarray) -> np.ndarray:
    """Per block: the largest magnitude, 0 below 2^-100, NaN where something is not finite."""
    with np.errstate(invalid="ignore"):
        s = np.abs(blocks(x)).max(axis=1)
        s = np.where(np.isfinite(s), s, np.nan)
        return np.where(s < 2.0 ** -100, 0.0, s)


def in_range(x: np.ndarray, scales: np.ndarray, root: bool) -> np.ndarray:
    """256 x / s, flat; zero in blocks that hold no numbers.  A root that is not zero is at least e4m3's smallest."""
    s = np.repeat(scales, BLOCK)[:x.size]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        y = np.where(s > 0, 256.0 * (x / s), 0.0)
    return np.where(y > 0, np.maximum(y, GRID[1]), y) if root else y


def neighbours(y: np.ndarray) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Codes (without sign) of the e4m3 numbers around |y|, and where between them |y| lies, from 0 to 1."""
    a = np.minimum(np.abs(y), 448.0)
    low = np.clip(np.searchsorted(GRID, a, side="right") - 1, 0, len(GRID) - 2)
    return low, low + 1, (a - GRID[low]) / (GRID[low + 1] - GRID[low])


def quantize(values: np.ndarray, root: bool) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(codes to nearest, ties to even; scales; distance of each element's part from a tie)."""
    with np.errstate(invalid="ignore"):
        x = np.sqrt(np.asarray(values, dtype=np.float64)) if root else np.asarray(values, dtype=np.float64)
    s = scale_of(x)
    y = in_range(x, s, root)
    low, high, part = neighbours(y)
    up = (part > 0.5) | ((part == 0.5) & (low % 2 == 1))
    codes = np.where(up, high, low) | np.where(np.signbit(y), 0x80, 0)
    return codes.astype(np.uint8), s, np.abs(part - 0.5)


def dither(numel: int, step: int, factor: int, first: int = 0) -> np.ndarray:
    """The 20-bit numbers of a tensor's elements at a step, from its element ``first`` on."""
    i = (np.arange(numel, dtype=np.uint64) + np.uint64(first)) & np.uint64(0xFFFFFFFF)
    u = (i * np.uint64(PLACE) + np.uint64(step % (1 << 32)) * np.uint64(factor)) & np.uint64(0xFFFFFFFF)
    return (u >> np.uint64(12)).astype(np.int64)


def adam_step(p, g, codes1, scales1, codes2, scales2, step, lr, beta1, beta2, eps, weight_decay, decoupled=False,
              maximize=False, grad_scale=1.0, coef=1.0, first=0) -> Dict[str, np.ndarray]:
    """One step on a flat tensor (or on whole blocks of one, from its element ``first`` on), in float64 from the stored codes.  ``codes1`` / ``codes2`` of the result are what the
    dither gives; ``sure1`` / ``sure2`` say where fp32 arithmetic cannot decide otherwise; ``p_tol`` bounds its error of p."""
    with np.errstate(all="ignore"):
        p = np.asarray(p, dtype=np.float64)
        g = np.asarray(g, dtype=np.float64) * grad_scale * coef * (-1.0 if maximize else 1.0)
        # how far fp32 may be off: each fp32 operation (and each rounded factor) adds at most EPS of its result
        g_err = 2 * EPS * np.abs(g)
        p1, p1_err = p, np.zeros_like(p)
        if decoupled:
            p1 = p * (1.0 - lr * weight_decay)
            p1_err = 2 * EPS * np.abs(p1)
        elif weight_decay != 0:
            g = g + weight_decay * p
            g_err = g_err + 2 * EPS * np.abs(weight_decay * p) + EPS * np.abs(g)
        m_old, r_old = read_back(codes1, scales1), read_back(codes2, scales2)
        m = beta1 * m_old + (1 - beta1) * g
        m_err = 3 * EPS * np.abs(beta1 * m_old) + (1 - beta1) * (g_err + 2 * EPS * np.abs(g)) + EPS * np.abs(m)
        v = beta2 * r_old ** 2 + (1 - beta2) * g ** 2
        v_err = 5 * EPS * beta2 * r_old ** 2 + (1 - beta2) * (2 * g_err * np.abs(g) + 3 * EPS * g ** 2) + EPS * v
        r = np.sqrt(v)
        r_err = np.where(r > 0, v_err / (2 * np.maximum(r, 1e-300)), 0.0) + EPS * r
        denom = r / np.sqrt(1 - beta2 ** step) + eps
        d_err = r_err / np.sqrt(1 - beta2 ** step) + 5 * EPS * denom
        update = (-lr / (1 - beta1 ** step)) * m / denom
        u_err = np.abs(update) * (d_err / denom + 6 * EPS) + lr / (1 - beta1 ** step) * m_err / denom
        new_p = p1 + update
        out = {"p": new_p, "p_tol": p1_err + u_err + EPS * np.abs(new_p)}
        for tag, x, x_err, factor in (("1", m, m_err, FIRST), ("2", r, r_err, ROOT)):
            s = scale_of(x)
            y = in_range(x, s, tag == "2")
            low, high, part = neighbours(y)
            u = dither(x.size, step, factor, first)
            up = part * 2.0 ** 20 + u >= 2.0 ** 20
            codes = np.where(up, high, low) | np.where(np.signbit(y), 0x80, 0)
            out["codes" + tag], out["scales" + tag] = codes.astype(np.uint8), s
            # y's error in units of the neighbours' distance: x's own, the scale's (of the element that sets it, at most
            # the largest error in the block, which that element's rounding steps give) and three roundings
            rel = np.repeat(np.where(s > 0, blocks(x_err).max(axis=1) / np.maximum(s, 1e-300), 0.0), BLOCK)[:x.size]
            s_of = np.maximum(np.repeat(s, BLOCK)[:x.size], 1e-300)
            y_err = 256.0 * x_err / s_of + np.abs(y) * (rel + 3 * EPS)
            t_err = y_err / (GRID[high] - GRID[low])
            # the element goes up or down where part + u / 2^20 passes 1 or 0; twice the error where the distance halves
            at, tol = part * 2.0 ** 20 + u, 2 * t_err * 2.0 ** 20 + 2
            out["sure" + tag] = (np.abs(at - 2.0 ** 20) > tol) & (at > tol)
            out["scale_tol" + tag] = blocks(x_err).max(axis=1)
        return out
