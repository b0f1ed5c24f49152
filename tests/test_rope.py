"""Rotary frequencies and their codes on the host (h3metal_amd/rope.py), against exact rational arithmetic."""

import math
from fractions import Fraction

import numpy as np
import pytest

from h3metal_amd import rope

PI = Fraction(31415926535897932384626433832795028841971693993751, 10 ** 49)


@pytest.mark.parametrize("rot", [2, 40, 96, 128])
def test_unscaled_and_linear(rot):
    f, s = rope.frequencies(rot, base=1e6)
    assert s == 1.0 and f.shape == (rot // 2,) and f[0] == 1.0
    for j in range(rot // 2):
        assert math.isclose(f[j], math.exp(-2 * j / rot * math.log(1e6)), rel_tol=1e-13)
    g, s = rope.frequencies(rot, base=1e6, scaling="linear", factor=4.0)
    assert s == 1.0 and np.array_equal(g, f / 4)


def test_ntk_keeps_the_fastest_pair_and_stretches_the_slowest():
    f, _ = rope.frequencies(128, base=1e4)
    g, s = rope.frequencies(128, base=1e4, scaling="ntk", factor=8.0)
    assert s == 1.0 and g[0] == f[0] and math.isclose(g[-1], f[-1] / 8, rel_tol=1e-12)
    assert np.all(g <= f * (1 + 1e-15)) and np.all(g >= f / 8 * (1 - 1e-12))


def test_yarn_keeps_fast_pairs_and_divides_slow_ones():
    rot, base, trained, factor = 128, 1e6, 32768, 4.0
    f, _ = rope.frequencies(rot, base=base)
    g, s = rope.frequencies(rot, base=base, scaling="yarn", factor=factor, trained=trained)
    assert math.isclose(s, 0.1 * math.log(factor) + 1)
    laps = trained * f / (2 * math.pi)
    share = (f / g - 1) / (factor - 1)  # 0 kept, 1 divided
    # a pair is between the bounds for at most one pair more on each side than its laps say (the bounds are whole pairs)
    assert np.all(g[laps >= 32 * base ** (2 / rot)] == f[laps >= 32 * base ** (2 / rot)])
    low = laps <= base ** (-2 / rot)
    assert low.any() and np.allclose(g[low], f[low] / factor, rtol=1e-14)
    assert np.all(np.diff(share) >= -1e-12)


def test_codes_are_parts_of_a_turn():
    """A code differs from 2^64 f / (2 pi) by less than the float64 quotient's rounding (2^-52 of it) and one part, and what
    a position makes of it in 64-bit arithmetic is the fraction of a turn."""
    f, _ = rope.frequencies(128, base=1e6)
    codes = rope.turns(f)
    assert codes.dtype == np.uint32 and codes.shape == (64, 2)
    for j in range(64):
        code = int(codes[j, 0]) | int(codes[j, 1]) << 32
        want = Fraction(float(f[j])) / (2 * PI) * 2 ** 64
        assert abs(code - want) <= want * Fraction(1, 2 ** 52) + 1
        for pos in (1, 12345, 2 ** 31 - 1):
            part = (code * pos) % 2 ** 64
            turn = Fraction(float(f[j])) * pos / (2 * PI)
            off = abs(Fraction(part, 2 ** 64) - (turn - math.floor(turn)))
            assert min(off, 1 - off) <= pos * (turn / pos * Fraction(1, 2 ** 52) + Fraction(1, 2 ** 64))


def test_codes_of_negative_and_many_turns():
    two = rope.turns(np.array([2 * math.pi * 2.5, -2 * math.pi * 0.25, 0.0]))
    assert two.tolist() == [[0, 1 << 31], [0, 3 << 30], [0, 0]]
    assert rope.turns(np.zeros(0)).shape == (0, 2)


@pytest.mark.parametrize("bad", [dict(rot=3), dict(rot=0), dict(rot=4, base=1.0), dict(rot=4, base=float("inf")),
                                 dict(rot=4, factor=0.5), dict(rot=4, scaling="other"), dict(rot=4, scaling="yarn"),
                                 dict(rot=4, scaling="yarn", trained=100, fast=1.0, slow=2.0)])
def test_refusals(bad):
    with pytest.raises(ValueError):
        rope.frequencies(bad.pop("rot"), **bad)


def test_codes_refuse_what_is_no_vector_of_numbers():
    for bad in (np.zeros((2, 2)), np.array([np.nan]), np.array([np.inf])):
        with pytest.raises(ValueError):
            rope.turns(bad)
