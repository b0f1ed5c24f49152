"""Rotary frequencies on the host. `frequencies` gives the radians per position of each rotated pair of channels, scaled for
contexts longer than the trained one; `turns` the codes of them that ops.qk_norm_rope_paged takes."""

from __future__ import annotations

import math

import numpy as np

SCALINGS = ("none", "linear", "ntk", "yarn")


def frequencies(rot: int, *, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, trained: int = 0,
                fast: float = 32.0, slow: float = 1.0):
    """(radians per position float64 [rot / 2], the factor on rotated channels) of a head whose first `rot` channels turn.
    Pair j turns by base^(-2 j / rot) a position; for a context `factor` times the trained one

      linear: every frequency / factor (positions interpolated)
      ntk:    the base grows by factor^(rot / (rot - 2)): the fastest pair keeps its frequency, the slowest one is / factor
      yarn:   pairs that turn at least `fast` times over the `trained` positions keep their frequency, those that turn at most
              `slow` times are / factor, between them the share falls linearly with j (bounds at whole pairs, the slow one
              at rot - 1 at most: it may lie behind the last pair, rot / 2 - 1); rotated channels times 0.1 ln(factor) + 1"""
    if rot < 2 or rot % 2:
        raise ValueError(f"rope: rot must be even and positive, got {rot}")
    if not (base > 1 and math.isfinite(base)) or not (factor >= 1 and math.isfinite(factor)):
        raise ValueError(f"rope: base must be above 1 and factor at least 1, got {base}, {factor}")
    if scaling not in SCALINGS:
        raise ValueError(f"rope: scaling must be one of {SCALINGS}, got {scaling!r}")
    j = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2 * j / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling != "yarn":
        return f, 1.0
    if trained < 1 or not fast > slow > 0:
        raise ValueError(f"rope: yarn needs the trained positions and fast > slow > 0, got {trained}, {fast}, {slow}")
    first, last = (rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow))
    first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
    share = 1 - np.clip((j - first) / max(last - first, 1e-3), 0, 1) if last > 0 else 0 * j  # (0: all turn too seldom)
    return f * share + f / factor * (1 - share), 0.1 * math.log(factor) + 1.0


def turns(freq: np.ndarray) -> np.ndarray:
    """uint32 [n][2] (low word, high word): the 2^-64 parts of a turn that each angle grows by per position. The product of
    a code and a position keeps its fraction of a turn in 64-bit integer arithmetic, where a float's product has lost it at
    10^6. A code is a float64 quotient, off by 2^-53 of itself or so: an angle at position P by up to P 2^-56 turns for the
    fastest pair, 2^-25 at 2^31."""
    freq = np.asarray(freq, np.float64)
    if freq.ndim != 1 or not np.isfinite(freq).all():
        raise ValueError(f"rope: frequencies must be a vector of finite numbers, got shape {freq.shape}")
    codes = [int(math.ldexp(math.fmod(f / (2 * math.pi), 1.0), 64)) % (1 << 64) for f in freq.tolist()]
    return np.array([[c & 0xFFFFFFFF, c >> 32] for c in codes], np.uint32).reshape(len(codes), 2)
