"""float64 forms of the 8-bit feed-forward operators: RMS norm with the residual's addition, the gated unit, the rounding
of rows to 8 bits by blocks, and the product of block-scaled operands. Test infrastructure only (see oracle/__init__.py).

The e4m3 values are written down here from the format (4 exponent bits with bias 7, 3 mantissa bits, NaN where all are
set), apart from the package's own; both are compared with torch's in tests/test_f8.py.
"""

from __future__ import annotations

import numpy as np

BLOCK = 128
F8_MAX = 448.0


def e4m3_value(code: np.ndarray) -> np.ndarray:
    """float64 values of e4m3 bit patterns."""
    c = np.asarray(code).astype(np.int64)
    sign = 1.0 - 2.0 * (c >> 7)
    e, f = (c & 0x78) >> 3, (c & 7) / 8.0
    v = sign * np.where(e > 0, np.ldexp(1.0 + f, (e - 7).astype(int)), np.ldexp(f, -6))
    return np.where((c & 0x7F) == 0x7F, np.nan, v)


def e4m3_round(x: np.ndarray) -> np.ndarray:
    """x rounded to the nearest e4m3 value (half to even), magnitudes past 448 to 448."""
    x = np.asarray(x, np.float64)
    _, e = np.frexp(np.maximum(np.abs(x), 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.clip(np.rint(x / step) * step, -F8_MAX, F8_MAX)


def rms_norm(h: np.ndarray, w: np.ndarray | None, eps: float, norm: bool = True) -> np.ndarray:
    h = np.asarray(h, np.float64)
    v = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) if norm else h
    return v if w is None else v * np.asarray(w, np.float64)


def gated(x: np.ndarray, D: int) -> np.ndarray:
    """value * gate / (1 + exp(-gate)) of rows [value | gate]."""
    x = np.asarray(x, np.float64)
    v, g = x[:, :D], x[:, D:2 * D]
    with np.errstate(over="ignore"):
        return v * g / (1.0 + np.exp(-g))


def blocks(v: np.ndarray) -> np.ndarray:
    """Rows as blocks [M][nb][128], zeros behind the last column."""
    M, D = v.shape
    nb = -(-D // BLOCK)
    p = np.zeros((M, nb * BLOCK), v.dtype)
    p[:, :D] = v
    return p.reshape(M, nb, BLOCK)


def block_scales(v: np.ndarray) -> np.ndarray:
    top = np.abs(blocks(v)).max(-1)
    return np.where(top > 0, top / F8_MAX, 1.0)


def row_scales(v: np.ndarray) -> np.ndarray:
    top = np.abs(v).max(-1)
    return np.where(top > 0, top / 127.0, 1.0)


def per_column(s: np.ndarray, D: int) -> np.ndarray:
    """Block scales [M][nb] at each of the D columns."""
    return np.repeat(s, BLOCK, -1)[:, :D]


def dequantised(codes: np.ndarray, s: np.ndarray, rows: int = 1) -> np.ndarray:
    """float64 values of e4m3 codes [N][K] with a scale for each `rows` x 128 block."""
    N, K = codes.shape
    return e4m3_value(codes) * np.repeat(np.repeat(np.asarray(s, np.float64), rows, 0)[:N], BLOCK, 1)[:, :K]


def product(a, sa, w, sw):
    """(A x W^T in float64, the sum of its terms' magnitudes) of block-scaled codes."""
    x, y = dequantised(a, sa), dequantised(w, sw, BLOCK)
    return x @ y.T, np.abs(x) @ np.abs(y).T
