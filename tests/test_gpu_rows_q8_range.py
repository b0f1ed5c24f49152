"""rms_norm_q8 where a row's products, their squares' sum or the residual's sum leave what a float holds: a block's codes and
scale depend on its own values alone."""

import numpy as np
import pytest

from h3metal_amd import ops
from oracle import rows_q8 as orq
from oracle.bf16 import from_bf16
from test_gpu_rows_q8 import EXACT, U, as_type, check_codes, norm_case

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


# Bounds of the checks: test_gpu_rows_q8.py's. A scale is off by its roundings and its sum's, and by 2^-149 where it is
# subnormal; e4m3 codes are exactly rounded, int8 ones rounded from within 5 * 2^-24.
CASES = [(h, 1.0, 0.0, True) for h in (1e-44, 1e-41, 3e-38, 1e-30, 3e-23, 1e-20, 1e-16, 1e-12, 1e15, 1e18, 3e19, 1e25, 3e38)] + [
    (1e25, 1.0, 1e-6, True), (1e-30, 1e-20, 0.0, True), (1e-30, 1e20, 0.0, True), (1e25, 1e25, 1e-6, True),
    (1e25, 1e-25, 1e-6, True), (1e-3, 1e-38, 1e-6, True), (1e-3, 3e38, 1e-6, True), (1e-20, 1e-20, 1e-6, False),
    (3e25, 3e14, 1e-6, False), (1e15, 1e15, 1e-6, False), (1e-10, 1e-10, 1e-30, True)]


@pytest.mark.parametrize("out", ["f8", "i8"])
@pytest.mark.parametrize("D", [1, 200, 300, 4096, 16385])
@pytest.mark.parametrize("hm,wm,eps,norm", CASES)
def test_magnitudes(gpu, hm, wm, eps, norm, D, out):
    """Rows and gains from the smallest floats to the largest, whose squares, their sum, products or largest quotient no
    float holds."""
    rng = np.random.default_rng(19)
    M = 3
    x = (rng.uniform(0.3, 1, (M, D)) * rng.choice([-1, 1], (M, D)) * hm).astype(np.float32)
    w = (rng.uniform(0.3, 1, D) * wm).astype(np.float32)
    h, c, s = norm_case(gpu, x, "f32", None, None, w, D, out=out, eps=eps, norm=norm)
    check_range(h, c, s, w, D, out, eps, norm)


def check_range(h, c, s, w, D, out, eps, norm):
    v = orq.rms_norm(h, w, eps, norm)
    top = orq.per_column(np.abs(orq.blocks(v)).max(-1), D) if out == "f8" else np.abs(v).max(-1, keepdims=True)
    v = np.where(top < 2.0 ** -149, 0.0, v)  # an amax below the smallest float counts as 0
    ws = orq.block_scales(v) if out == "f8" else orq.row_scales(v)[:, None]
    tol = (6 + 0.5 * (D / 16 + 12)) * U
    assert np.all(np.abs(s - ws) <= tol * ws + 2.0 ** -149), np.max(np.abs(s - ws) / ws)
    if out == "f8":
        check_codes(c, v / orq.per_column(ws, D), EXACT)
    else:
        q = v / ws
        assert np.all((c >= np.rint(q - np.abs(q) * 5 * U)) & (c <= np.rint(q + np.abs(q) * 5 * U)))


@pytest.mark.parametrize("out", ["f8", "i8"])
@pytest.mark.parametrize("D", [256, 640, 4096])
def test_magnitudes_side_by_side(gpu, D, out):
    """Rows of every magnitude in one call, in bf16 with a residual, blocks of every magnitude in one row, and rows of zeros
    between them."""
    rng = np.random.default_rng(20)
    mags = np.float32([1, 1e-30, 1e30, 0, 3e-23, 1e19, 1e-3, 0, 3e38, 1e-37])
    M = len(mags)
    x = rng.uniform(0.3, 1, (M, D)).astype(np.float32) * mags[:, None] / 2
    w = np.ones(D, np.float32)
    h, c, s = norm_case(gpu, x, "bf16", x / 2, "bf16", w, D, out=out, eps=0.0 if D == 640 else 1e-30, inplace=True)
    live = mags > 0
    check_range(h[live], c[live], s[live], w, D, out, 0.0 if D == 640 else 1e-30, True)
    assert not (c[~live] & 0x7F).any() and np.all(s[~live] == 1)
    w *= np.repeat(np.float32([1, 1e-30, 1e30, 1e-38, 3e38]), 128)[np.arange(D) % 640]
    for norm in (True, False):
        h, c, s = norm_case(gpu, rng.uniform(0.3, 1, (2, D)) * 1e-9, "f32", None, None, w, D, out=out, norm=norm)
        check_range(h, c, s, w, D, out, 1e-6, norm)


def rounded_once(v, t):
    """float64 rounded to bf16's 8 bits (values well inside its range) or to half; half to even."""
    if t == "f16":
        return v.astype(np.float16).astype(np.float64)
    m, e = np.frexp(v)
    return np.ldexp(np.rint(m * 256) / 256, e)


@pytest.mark.parametrize("out", ["f8", "i8"])
@pytest.mark.parametrize("rt,bits", [("bf16", 8), ("f16", 11)])
def test_the_residuals_sum_is_rounded_once(gpu, rt, bits, out):
    """A float x that takes a 16-bit residual beside the middle of two 16-bit values, by less than a float's step of the sum;
    and sums of ordinary values."""
    rng = np.random.default_rng(22)
    M, D = 4, 600
    rh, r = as_type(rng.uniform(1, 2, (M, D)) * rng.choice([-1, 1], (M, D)) * 2.0 ** rng.integers(-3, 4, (M, D)), rt)
    ulp = 2.0 ** (np.floor(np.log2(np.abs(r))) - (bits - 1))  # a step of the residual
    x = (ulp * (rng.choice([-1.5, -0.5, 0.5, 1.5], (M, D)) + rng.choice([-1, 0, 1], (M, D)) * 2.0 ** -20.0)).astype(np.float32)
    x[3] = rng.standard_normal(D)
    want = rounded_once(r.astype(np.float64) + x.astype(np.float64), rt)
    twice = as_type(r + x, rt)[1].astype(np.float64)
    assert np.mean(twice[:3] != want[:3]) > 0.1
    print(f"[rms_norm_q8] {rt} residual of a float x, {out}", flush=True)
    R, O, S = gpu.upload(rh, rt), gpu.empty((M, D), out), gpu.empty((M, 5 if out == "f8" else 1), "f32")
    ops.rms_norm_q8(gpu, gpu.upload(x), None, O, S, M, D, eps=1e-6, res=R)
    gpu.wait()
    got = R.numpy()
    got = (from_bf16(got) if rt == "bf16" else got).astype(np.float64)
    assert np.array_equal(got, want), np.mean(got != want)
    check_range(want, O.numpy(), S.numpy(), None, D, out, 1e-6, True)


def test_a_half_is_added_to_a_bf16_residual_with_one_rounding(gpu):
    """Halves that are the middle of two bf16 values, beside residuals far below a float's step of the sum."""
    rng = np.random.default_rng(23)
    M, D = 3, 700
    x = (rng.integers(128, 256, (M, D)) + 0.5) * 2.0 ** rng.integers(-12, 6, (M, D)) * rng.choice([-1, 1], (M, D))
    xh, xf = as_type(x, "f16")
    assert np.array_equal(xf, x)
    rh, r = as_type(x * rng.choice([-1, 0, 1], (M, D)) * 2.0 ** rng.integers(-40, -26, (M, D)), "bf16")
    want = rounded_once(r.astype(np.float64) + xf.astype(np.float64), "bf16")
    assert np.mean(as_type(r + xf, "bf16")[1] != want) > 0.2
    print("[rms_norm_q8] bf16 residual of a half x", flush=True)
    R, O, S = gpu.upload(rh, "bf16"), gpu.empty((M, D), "f8"), gpu.empty((M, 6), "f32")
    ops.rms_norm_q8(gpu, gpu.upload(xh), None, O, S, M, D, eps=1e-6, res=R)
    gpu.wait()
    assert np.array_equal(from_bf16(R.numpy()), want)
    check_range(want, O.numpy(), S.numpy(), None, D, "f8", 1e-6, True)


def test_sums_of_zeros_infinities_and_the_largest_values(gpu):
    """Signs of zero, infinities, NaN, and sums that no float or no 16-bit value holds, as the float sum rounds them."""
    big = np.float32(3.4028235e38)
    r = np.float32([0.0, -0.0, 1.0, np.inf, -np.inf, np.inf, 3.3e38, -3.3e38, 65504, -65504, 65504, 1.0])
    x = np.float32([-0.0, -0.0, -1.0, 1.0, np.inf, 2.0, big, -big, 16, -16, 8, np.nan])
    for rt in ("bf16", "f16"):
        rh, rf = as_type(r[None], rt)
        with np.errstate(over="ignore", invalid="ignore"):
            sh, want = as_type(rf + x[None], rt)
        print(f"[rms_norm_q8] special sums {rt}", flush=True)
        R = gpu.upload(rh, rt)
        ops.rms_norm_q8(gpu, gpu.upload(x[None]), None, gpu.empty((1, 12), "f8"), gpu.empty((1, 1), "f32"), 1, 12, eps=1e-6, res=R)
        gpu.wait()
        got = R.numpy()
        got = (from_bf16(got) if rt == "bf16" else got).astype(np.float32)
        number = ~np.isnan(want)  # (a NaN's sign means nothing)
        assert np.array_equal(got, want, equal_nan=True) and np.array_equal(np.signbit(got[number]), np.signbit(want[number]))
