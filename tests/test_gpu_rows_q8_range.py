"""rms_norm_q8 where a row's products, their squares' sum or the residual's sum leave what a float holds: a block's codes and
scale depend on its own values alone."""

import numpy as np
import pytest

from h3metal_amd import ops

pytestmark = pytest.mark.gpu


def run(gpu, x, w, D, *, norm, eps=1e-6):
    M = x.shape[0]
    o, s = gpu.empty((M, D), "f8"), gpu.empty((M, (D + 127) // 128), "f32")
    ops.rms_norm_q8(gpu, gpu.upload(x), gpu.upload(w), o, s, M, D, eps=eps, norm=norm)
    gpu.wait()
    return o.numpy(), s.numpy()


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D", [256, 512, 4096])
@pytest.mark.parametrize("h,g", [(1e-40, 1e-6), (-1e-25, 1e-22), (1e30, 1e20)])
def test_a_block_does_not_depend_on_its_neighbours(gpu, h, g, D, norm):
    """Products h * w below and above what a float holds, beside a block whose quotients are powers of two and beside one
    whose quotients are near ties and below 2^-6 (which takes the exactly rounded path)."""
    print(f"[rms_norm_q8] h={h} w={g} D={D} norm={norm}", flush=True)
    rng = np.random.default_rng(3)
    got = []
    w = np.ones(D, np.float32)
    w[:128] = np.float32(g)
    for noisy in (False, True):
        x = np.ones((3, D), np.float32)
        x[:, :128] = np.float32(h) * rng.uniform(0.5, 1, (3, 128)).astype(np.float32) if not noisy else got[0][2]
        if noisy:
            x[:, 128:256] = np.exp(rng.uniform(-14, 0, (3, 128)))
        got.append(run(gpu, x, w, D, norm=norm) + (x[:, :128].copy(),))
    (c0, s0, _), (c1, s1, _) = got
    assert np.array_equal(c0[:, :128], c1[:, :128])
    if not norm:
        assert np.array_equal(s0[:, 0], s1[:, 0])
    if abs(h) * g < 1e-45:  # a float holds none of these values: zeros
        assert not (c1[:, :128] & 0x7F).any() and np.all(s1[:, 0] == 1)
