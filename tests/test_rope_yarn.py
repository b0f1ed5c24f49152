"""YaRN's frequencies (h3metal_amd/rope.py) against an evaluation of their own: the bounds are found by counting pairs upwards,
where rope.py solves for them, and laps are compared as logarithms of fractions of pi."""

import math

import numpy as np
import pytest

from h3metal_amd import rope


def shares(rot, base, trained, fast, slow):
    """Each pair's share of the division by the factor: 0 up to the last whole pair that turns at least `fast` times, 1 from the
    first whole pair on that turns at most `slow` times (pairs counted on behind the head's last one, to rot - 1), linear between."""
    def log_laps(j):
        return math.log(trained) - math.log(math.tau) - j * math.log(base) * 2 / rot

    j0 = 0
    while log_laps(j0 + 1) >= math.log(fast):
        j0 += 1
    j1 = 0
    while log_laps(j1) > math.log(slow) and j1 < rot - 1:
        j1 += 1
    if j1 == 0:  # even the first pair turns at most `slow` times
        return [1.0] * (rot // 2)
    return [0.0 if j <= j0 else 1.0 if j >= j1 else (j - j0) / (j1 - j0) for j in range(rot // 2)]


@pytest.mark.parametrize("rot,base,trained", [
    (16, 1e4, 32768), (64, 1e4, 65536), (128, 1e4, 131072), (4, 1e6, 32768),  # the slow bound lies behind the last pair
    (128, 1e4, 10 ** 9), (2, 1e4, 4096), (8, 100.0, 10 ** 7),                   # ... and behind rot - 1
    (128, 1e6, 32768), (64, 1e4, 4096), (96, 5e5, 8192), (128, 1e4, 2048)])
@pytest.mark.parametrize("factor,fast,slow", [(4.0, 32.0, 1.0), (32.0, 32.0, 1.0), (2.0, 8.0, 2.0)])
def test_shares_of_the_pairs(rot, base, trained, factor, fast, slow):
    f, _ = rope.frequencies(rot, base=base)
    g, s = rope.frequencies(rot, base=base, scaling="yarn", factor=factor, trained=trained, fast=fast, slow=slow)
    want = np.array(shares(rot, base, trained, fast, slow))
    assert np.allclose(g, f * (1 - want) + f / factor * want, rtol=1e-12, atol=0)
    assert math.isclose(s, 0.1 * math.log(factor) + 1)
    laps = trained * f / (2 * math.pi)
    assert np.all(g[laps > slow * (1 + 1e-9)] > f[laps > slow * (1 + 1e-9)] / factor * (1 + 1e-9))  # not the whole factor


@pytest.mark.parametrize("rot,trained,fast,slow", [(8, 6, 32.0, 1.0), (8, 60, 32.0, 20.0), (2, 1, 32.0, 1.0)])
def test_trained_positions_that_no_pair_turns_often_over(rot, trained, fast, slow):
    """Even the fastest pair turns at most `slow` times: all of them are divided."""
    f, _ = rope.frequencies(rot, base=1e4)
    g, _ = rope.frequencies(rot, base=1e4, scaling="yarn", factor=4.0, trained=trained, fast=fast, slow=slow)
    assert shares(rot, 1e4, trained, fast, slow) == [1.0] * (rot // 2) and np.allclose(g, f / 4, rtol=1e-14, atol=0)
