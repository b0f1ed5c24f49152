"""e4m3 values on the host: 8-bit floating point with 4 exponent and 3 mantissa bits (bias 7), no infinities, NaN where
all of them are set, largest value 448. `block_codes` makes the weights that ops.gemm takes with format "f8"."""

from __future__ import annotations

import numpy as np

F8_MAX = 448.0
BLOCK = 128


def to_f8(x: np.ndarray) -> np.ndarray:
    """The bit patterns (uint8) of float32 values, rounded to the nearest e4m3 value (half to even); magnitudes past 448
    become 448, NaN stays NaN."""
    x = np.asarray(x, np.float32)
    bits = x.view(np.uint32)
    mag = np.minimum(np.abs(x), np.float32(F8_MAX))  # NaN stays
    u = np.ascontiguousarray(mag).view(np.uint32)
    # from 2^-6 on: the float's exponent and 3 rounded mantissa bits; below, multiples of 2^-9 (rint; 8 of them is 2^-6)
    normal = ((u + 0x7FFFF + ((u >> 20) & 1)) >> 20).astype(np.int64) - ((127 - 7) << 3)
    small = np.rint(np.nan_to_num(mag) * np.float32(512)).astype(np.int64)
    code = np.where(mag >= np.float32(2.0 ** -6), normal, small)
    code = np.where(np.isnan(x), 0x7F, code)
    return (code.astype(np.uint8) | ((bits >> 24) & 0x80).astype(np.uint8)).reshape(x.shape)


def _table() -> np.ndarray:
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 0x7F) == 0x7F] = np.nan
    return np.where(c & 0x80, -v, v).astype(np.float32)


VALUES = _table()  # the float32 value of each of the 256 bit patterns


def from_f8(codes: np.ndarray) -> np.ndarray:
    """The float32 values of e4m3 bit patterns (uint8)."""
    return VALUES[np.asarray(codes, np.uint8)]


def block_codes(w: np.ndarray, rows: int = BLOCK, cols: int = BLOCK):
    """(codes uint8 [N][K], scales float32 [ceil(N / rows)][ceil(K / cols)]) of a float matrix w [N][K]: each block's scale
    is its largest magnitude / 448 (1 where that is 0), its codes e4m3(w / scale). With rows = 1: activations."""
    w = np.asarray(w, np.float32)
    N, K = w.shape
    nb, kb = -(-N // rows), -(-K // cols)
    pad = np.zeros((nb * rows, kb * cols), np.float32)
    pad[:N, :K] = w
    b = pad.reshape(nb, rows, kb, cols)
    top = np.abs(b).max((1, 3))
    s = np.where(top > 0, top / np.float32(F8_MAX), np.float32(1)).astype(np.float32)
    s = np.maximum(s, np.float32(2.0 ** -126))  # w / s stays finite
    codes = to_f8(b / s[:, None, :, None]).reshape(nb * rows, kb * cols)[:N, :K]
    return np.ascontiguousarray(codes), s
