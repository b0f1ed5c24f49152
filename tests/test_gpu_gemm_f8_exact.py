"""ops.gemm with weight format f8 and EXACT=1: 16-bit outputs as float sums of exact products, rounded once, like the float
outputs. The same tiles give the float output and the 16-bit one from the same sums, so these agree bit for bit."""

import numpy as np
import pytest

from h3metal_amd import f8, ops
from h3metal_amd.gpu import GpuError
from oracle import rows_q8 as orq
from oracle.bf16 import from_bf16, to_bf16
from test_gpu_gemm_f8 import check, operands, weight

pytestmark = pytest.mark.gpu


def product(gpu, a, sa, w, sw, out, bias=None, pads=(0, 0, 0), **variant):
    """The bits of out [M][N]; A's, W's and the output's rows pads[0], pads[1], pads[2] columns apart; what lies behind
    the output's rows stays."""
    (M, K), N = a.shape, w.shape[0]
    print(f"[gemm f8] M={M} N={N} K={K} out={out} bias={bias is not None} pads={pads} {variant}", flush=True)
    rows = np.full((M, K + pads[0]), 0x7F, np.uint8)
    rows[:, :K] = a
    cs = N + pads[2]
    raw = np.full((M + 2, cs), 3, {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[out])
    O = gpu.upload(raw, out)
    ops.gemm(gpu, gpu.upload(rows, "f8"), weight(gpu, w, sw, bias, K + pads[1] if pads[1] else None), O, M, sa=gpu.upload(sa),
             a_stride=K + pads[0], c_stride=cs, **variant)
    gpu.wait()
    got = O.numpy()
    res = got[:M, :N].copy()
    got[:M, :N] = raw[:M, :N]
    assert np.array_equal(got.view(np.uint8), raw.view(np.uint8)), "written past the rows"
    return res


def rounded(x, out):
    return to_bf16(x) if out == "bf16" else x.astype(np.float16)


@pytest.mark.parametrize("TILE", range(9), ids=["plan", "16", "32", "48", "64", "80", "128", "256x128", "256"])
@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K,bias,pads", [(1, 1, 16, False, (0, 0, 0)), (9, 1001, 400, True, (0, 0, 0)),
                                             (70, 261, 336, True, (16, 48, 3)), (300, 512, 1040, False, (0, 0, 8)),
                                             (520, 640, 128, True, (0, 0, 0))])
def test_16_bit_outputs_are_rounded_float_outputs(gpu, M, N, K, bias, pads, out, TILE):
    rng = np.random.default_rng(M + 7 * K)
    ops4 = operands(rng, M, N, K)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    want = rounded(product(gpu, *ops4, "f32", b, pads, TILE=TILE), out)
    got = product(gpu, *ops4, out, b, pads, TILE=TILE, EXACT=1)
    assert np.array_equal(got.view(np.uint16), want.view(np.uint16))


@pytest.mark.parametrize("TILE", [0, 6, 7], ids=["plan", "128", "256x128"])
@pytest.mark.parametrize("M,N,K", [(4607, 4096, 640), (5000, 2056, 128), (4400, 2304, 272)])
def test_large_products(gpu, M, N, K, TILE):
    """Workgroups that take several tiles, and a last, partly filled round's rows on smaller ones."""
    rng = np.random.default_rng(M)
    ops4 = operands(rng, M, N, K)
    want = rounded(product(gpu, *ops4, "f32", TILE=TILE), "bf16")
    assert np.array_equal(product(gpu, *ops4, "bf16", TILE=TILE, EXACT=1), want)


def test_sums_are_those_of_exact_products(gpu):
    """Of 256 K outputs, those that are not the rounded float64 product. An error e of a row's values, in units of their
    2-norm's mean, moves a normal value v over a tie of bf16 (2^-8 |v| apart at least) with probability min(1, c / |v|),
    c = 2^8 e, which is 0.8 c (1 + ln(1 / c)) over all v. Float sums of about 20 additions are 2.5e-7 off or less
    (20^0.5 steps of 2^-24): 5.5e-4 of the values; the 8-bit instruction's 1.5e-5 is more than ten times as many."""
    rng = np.random.default_rng(21)
    a, sa, w, sw = operands(rng, 256, 1024, 1024)
    want = to_bf16(orq.product(a, sa, w, sw)[0].astype(np.float32))
    off = np.mean(product(gpu, a, sa, w, sw, "bf16", EXACT=1) != want)
    assert off <= 1e-3, off


@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (9, 1001, 2000), (16, 512, 640)])
def test_the_smallest_tiles_take_exact_products(gpu, M, N, K, out):
    """They are bound by the weight's loads, so 16-bit outputs need no choice."""
    rng = np.random.default_rng(K)
    ops4 = operands(rng, M, N, K)
    want = rounded(product(gpu, *ops4, "f32", TILE=1), out)
    assert np.array_equal(product(gpu, *ops4, out, TILE=1).view(np.uint16), want.view(np.uint16))


def test_refusals(gpu):
    for macros in (dict(WFMT=9, EXACT=2), dict(WFMT=9, EXACT=-1), dict(WFMT=4, EXACT=1), dict(WFMT=1, EXACT=0)):
        with pytest.raises(GpuError, match="EXACT"):
            gpu.kernel("gemm", "gemm", **macros)


def off(got, want):
    return np.linalg.norm(got - want), np.linalg.norm(want)


TILES = pytest.mark.parametrize("TILE", range(9), ids=["plan", "16", "32", "48", "64", "80", "128", "256x128", "256"])


@TILES
@pytest.mark.parametrize("M,N,K,bias", [(9, 130, 160, False), (77, 256, 1024, True), (300, 515, 256, False), (520, 640, 2064, True),
                                        (4607, 1024, 640, False)])
def test_residual_takes_exact_products(gpu, M, N, K, bias, TILE):
    """X += gate[rtype] * (v + bias) in the 2-norm: 4e-6 of the added values (float sums are 1e-6 off or less, the 8-bit
    instruction's 1.5e-5) and the roundings of gate * v and of the sum, half a float step each."""
    rng = np.random.default_rng(M + K)
    a, sa, w, sw = operands(rng, M, N, K)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    x, gate = rng.standard_normal((M, N)).astype(np.float32), rng.standard_normal((3, N)).astype(np.float32)
    rt = rng.integers(0, 3, M).astype(np.uint8)
    X = gpu.upload(x)
    print(f"[gemm f8] residual M={M} N={N} K={K} bias={bias} TILE={TILE}", flush=True)
    ops.gemm(gpu, gpu.upload(a, "f8"), weight(gpu, w, sw, b), X, M, sa=gpu.upload(sa), epi=1, rtype=gpu.upload(rt),
             gate=gpu.upload(gate), TILE=TILE)
    gpu.wait()
    v = orq.product(a, sa, w, sw)[0]
    added = gate[rt].astype(np.float64) * (v if b is None else v + b)
    err, size = off(X.numpy(), x + added)
    assert err <= 4e-6 * np.linalg.norm(gate[rt] * v) + 2.0 ** -24 * (2 * np.linalg.norm(added) + size), err / np.linalg.norm(added)


@TILES
@pytest.mark.parametrize("M,N,K", [(9, 1001, 400), (300, 512, 1040), (520, 640, 256)])
def test_half_outputs_are_off_by_their_rounding(gpu, M, N, K, TILE):
    """A half's rounding is 2^-11 / 3^0.5 of the values in the 2-norm at most; 1.5e-5 of the 8-bit instruction's sums and
    2^-25 of subnormal halves beside it are under a twentieth of that."""
    rng = np.random.default_rng(N)
    ops4 = operands(rng, M, N, K)
    for kw in ({}, dict(EXACT=1)):
        err, size = off(product(gpu, *ops4, "f16", TILE=TILE, **kw).astype(np.float64), orq.product(*ops4)[0])
        assert err <= 0.6 * 2.0 ** -11 * size, err / size


@pytest.mark.parametrize("M,D,F", [(1, 200, 72), (37, 2632, 1001), (300, 517, 329)])
def test_widths_that_are_no_multiple_of_16(gpu, M, D, F):
    """Norm, product, gated unit, product, with K rounded up to 16: zero columns behind the weights' codes, rows K apart in
    buffers that start as zeros. Each product against float64 of what it read; the zeros stay."""
    rng = np.random.default_rng(D)
    KD, KF = -(-D // 16) * 16, -(-F // 16) * 16
    print(f"[feed-forward] widths M={M} D={D} F={F}", flush=True)

    def codes(N, K, k):
        c, s = f8.block_codes((rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32))
        return np.pad(c, ((0, 0), (0, k - K))), s

    w1, s1 = codes(2 * F, D, KD)
    w2, s2 = codes(D, F, KF)
    x = to_bf16(rng.standard_normal((M, D)).astype(np.float32))
    A, SA = gpu.empty((M, KD), "f8"), gpu.empty((M, -(-D // 128)), "f32")
    H, B, SB = gpu.empty((M, 2 * F), "bf16"), gpu.empty((M, KF), "f8"), gpu.empty((M, -(-F // 128)), "f32")
    O = gpu.empty((M, D), "f32")
    ops.rms_norm_q8(gpu, gpu.upload(x, "bf16"), None, A, SA, M, D, eps=1e-6, o_stride=KD)
    ops.gemm(gpu, A, weight(gpu, w1, s1), H, M, sa=SA)
    ops.swiglu_f8(gpu, H, B, SB, M, F, o_stride=KF)
    ops.gemm(gpu, B, weight(gpu, w2, s2), O, M, sa=SB)
    gpu.wait()
    a, b = A.numpy(), B.numpy()
    assert not a[:, D:].any() and not b[:, F:].any()
    check(from_bf16(H.numpy()).astype(np.float64), a[:, :D], SA.numpy(), w1[:, :D], s1, "bf16")
    check(O.numpy().astype(np.float64), b[:, :F], SB.numpy(), w2[:, :F], s2, "f32")
