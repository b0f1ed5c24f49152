"""attention_paged where scores are -infinity for seen keys: a key masked by an infinite channel, as over left padding. Such a key
has the weight 0, whether it fills the first block of a row's keys, of a cut tile's part, or all of a part. Bounds as in
test_gpu_attention_paged."""

import numpy as np
import pytest

from paged_util import as_type
from test_gpu_attention_paged import batch, check, launch

pytestmark = pytest.mark.gpu


def masked(new, keys, levels, *, t="bf16", D=128, H=4, seed=0, **kw):
    """A batch whose first sequence's keys score about their level (log2 units): `levels` is [(first key, level), ..], in order.
    Channel 0 of the queries is 1 and takes a key's mask, channel 1 is 1 and takes its level; the scale is 1."""
    c = batch(new, keys, H=H, KVH=1, D=D, t=t, seed=seed, q_size=0.05, **kw)
    q = np.random.default_rng(seed + 100).standard_normal(c["q"].shape) * 0.05
    q[:, :, :2] = 1.0
    c["q"] = as_type(q, t)[0]
    zero, low = (as_type(np.array([x]), t)[0][0] for x in (0.0, -np.inf))
    for j in range(keys[0]):
        level = [v for at, v in levels if j >= at][-1]
        row = c["kc"][c["table"][0, j // c["page"]], 0, j % c["page"]]
        row[0] = low if level == -np.inf else zero
        row[1] = zero if level == -np.inf else as_type(np.array([level * np.log(2.0)]), t)[0][0]
    return c


@pytest.mark.parametrize("ROWS", [32, 256])
@pytest.mark.parametrize("D,t", [(128, "bf16"), (96, "bf16"), (64, "bf16"), (128, "f16"), (64, "f16")])
@pytest.mark.parametrize("causal", [True, False])
def test_first_keys_score_minus_infinity(gpu, D, t, ROWS, causal):
    """The first 64, 100 or 200 keys are masked; later scores are low, high, or jump; whole tiles and cut ones."""
    for seed, (new, keys) in enumerate([([70], [400]), ([64, 3], [3000, 20]), ([1], [3000])]):
        for first in (64, 100, 200) if keys[0] == 400 else (64, 700):
            for a, b in ((20.0, 60.0), (-200.0, -200.0), (-140.0, -150.0), (5.0, 5.0)):
                c = masked(new, keys, [(0, -np.inf), (first, a), (first + 150, b)], t=t, D=D, seed=seed)
                check(launch(gpu, c, causal=causal, scale=1.0, ROWS=ROWS), c, causal=causal, scale=1.0)


@pytest.mark.parametrize("ROWS", [32, 256])
def test_all_keys_score_minus_infinity(gpu, ROWS):
    """0 / 0 for every row that sees a key, in whole tiles and cut ones."""
    for new, keys in (([70], [70]), ([5], [3000])):
        c = masked(new, keys, [(0, -np.inf)])
        assert np.isnan(check(launch(gpu, c, scale=1.0, ROWS=ROWS), c, scale=1.0)).all()


@pytest.mark.parametrize("ROWS", [32, 256])
@pytest.mark.parametrize("D,t", [(128, "bf16"), (96, "f16"), (64, "bf16")])
def test_seen_values_whose_weight_vanishes(gpu, D, t, ROWS):
    """NaN, or an infinity with a weight below any float, in the value of a seen key: the channel is NaN, also where the key
    lies in a part of a cut tile whose factor is 0."""
    for new, keys in (([1], [3000]), ([64], [3000]), ([70], [400])):
        for level, what in ((300.0, np.nan), (1200.0, np.inf), (1200.0, -np.inf)):
            c = masked(new, keys, [(0, 0.0), (keys[0] // 2, level)], t=t, D=D, seed=3)
            c["vc"][c["table"][0, 0], 0, 3, 10] = as_type(np.array([what]), t)[0][0]
            want = check(launch(gpu, c, scale=1.0, ROWS=ROWS), c, scale=1.0)
            assert np.isnan(want[:, :, 10]).all() and np.isfinite(want[:, :, :10]).all()
