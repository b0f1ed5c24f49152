"""rms_norm_q8 and swiglu_f8 against float64: the residual's sum bit for bit, scales and codes within the float steps'
roundings, at lengths from one column, odd strides and offsets, all type pairs; rows of zeros, tiny and huge values, NaN
and infinities; what lies behind the rows stays; refusals.

Bounds. rms_norm_q8's e4m3 codes are the rounded exact quotients (EXACT: what the oracle's own float64 steps may be off). An
int8 code is right if it is the rounding of some value within 5 * 2^-24 of v / s: h w, 127 / amax (two roundings with amax's
own) and the product; a gated unit's code likewise, its value's own error given apart. A scale is amax times the reciprocal
root over 448: 6 roundings, and half the relative error of the sum of squares, whose positive terms are added on at least 16
lanes (D / 16 additions in a row and 12 across lanes and waves, at most)."""

import numpy as np
import pytest

from h3metal_amd import ops
from h3metal_amd.gpu import GpuError
from oracle import rows_q8 as orq
from oracle.bf16 import from_bf16, to_bf16

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of float, relative to the value
EXACT = 2.0 ** -49


def as_type(x, t):
    """(what is uploaded, its float32 values)"""
    x = np.asarray(x, np.float32)
    if t == "bf16":
        b = to_bf16(x)
        return b, from_bf16(b).astype(np.float32)
    if t == "f16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float32)
    return x, x


def strided(gpu, host, dtype, stride, offset, fill):
    """`host` [M][D] as rows `stride` apart from element `offset` of a buffer whose other elements hold `fill`; the view
    and the whole."""
    M, D = host.shape
    flat = np.full(offset + M * stride + 7, fill, host.dtype)
    flat[offset:offset + M * stride].reshape(M, stride)[:, :D] = host
    whole = gpu.upload(flat, dtype)
    return whole.view((M, stride), offset_elems=offset), whole, flat


def inside(flat, offset, M, stride, D):
    return flat[offset:offset + M * stride].reshape(M, stride)[:, :D]


def check_codes(codes, q, tol):
    """Each code is the rounding of a value within `tol` (relative) of q."""
    got = orq.e4m3_value(codes)
    lo, hi = orq.e4m3_round(q - np.abs(q) * tol), orq.e4m3_round(q + np.abs(q) * tol)
    assert np.all((got >= lo) & (got <= hi)), np.argwhere(~((got >= lo) & (got <= hi)))[:5]


def norm_case(gpu, x, xt, res, rt, w, D, *, out="f8", eps=1e-6, norm=True, inplace=False, pad=0, off=0):
    """Runs rms_norm_q8 on rows with `pad` columns between them from element `off`; checks sum, scales, codes and that
    nothing else was written. Returns codes, scales."""
    M = x.shape[0]
    print(f"[rms_norm_q8] M={M} D={D} x={xt} res={rt} w={w is not None} out={out} norm={norm} pad={pad} off={off}", flush=True)
    xh, xf = as_type(x, xt)
    X, _, _ = strided(gpu, xh, xt, D + pad, off, 0)
    kw = {}
    h = xf
    if rt:
        rh, rf = as_type(res, rt)
        R, Rw, rflat = strided(gpu, rh, rt, D + pad, off, 1)
        with np.errstate(over="ignore", invalid="ignore"):
            sh, h = as_type(rf + xf, rt)
        if inplace:
            kw = dict(res=R, res_stride=D + pad)
            S, Sw, sflat, soff, sstr = R, Rw, rflat, off, D + pad
        else:
            soff, sstr = off + 1, D + pad + 1
            S, Sw, sflat = strided(gpu, np.zeros_like(sh), rt, sstr, soff, 1)
            kw = dict(res=R, res_stride=D + pad, res_out=S, res_out_stride=sstr)
    raw = np.uint8 if out == "f8" else np.int8
    O, Ow, oflat = strided(gpu, np.zeros((M, D), raw), out, D + pad, off, 77)
    ns = (D + 127) // 128 if out == "f8" else 1
    SC, SCw, scflat = strided(gpu, np.zeros((M, ns), np.float32), "f32", ns, off, -5)
    ops.rms_norm_q8(gpu, X, gpu.upload(w) if w is not None else None, O, SC, M, D, eps=eps, norm=norm, x_stride=D + pad,
                    o_stride=D + pad, **kw)
    gpu.wait()
    if rt:
        want = sflat.copy()
        inside(want, soff, M, sstr, D)[:] = sh
        got = Sw.numpy()
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), "the residual's sum"
    ogot, sgot = Ow.numpy(), SCw.numpy()
    codes, scale = inside(ogot, off, M, D + pad, D).copy(), inside(sgot, off, M, ns, ns).copy()
    inside(ogot, off, M, D + pad, D)[:] = 0
    inside(sgot, off, M, ns, ns)[:] = 0
    assert np.array_equal(ogot, oflat) and np.array_equal(sgot, scflat), "written past the rows"
    return h, codes, scale


def check_norm(h, codes, scale, w, D, out, eps=1e-6, norm=True):
    v = orq.rms_norm(h, w, eps, norm)
    ws = orq.block_scales(v) if out == "f8" else orq.row_scales(v)[:, None]
    tol = (6 + 0.5 * (D / 16 + 12)) * U
    assert np.all(np.abs(scale - ws) <= tol * ws), np.max(np.abs(scale - ws) / ws)
    if out == "f8":
        check_codes(codes, v / orq.per_column(ws, D), EXACT)
    else:
        q = v / ws
        lo, hi = np.rint(q - np.abs(q) * 5 * U), np.rint(q + np.abs(q) * 5 * U)
        assert np.all((codes >= lo) & (codes <= hi))


SHAPES = [(1, 1), (3, 7), (2, 8), (5, 127), (1, 128), (4, 129), (33, 200), (7, 512), (3, 1000), (130, 1024), (2, 2047),
          (1, 4096), (19, 4096), (5, 5376), (2, 10240), (1, 16385), (1, 40000)]


@pytest.mark.parametrize("out", ["f8", "i8"])
@pytest.mark.parametrize("M,D", SHAPES)
def test_norm_shapes(gpu, M, D, out):
    rng = np.random.default_rng(M * 31 + D)
    x, r = rng.standard_normal((M, D)) * 2, rng.standard_normal((M, D))
    x[:, ::17] *= 30
    w = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    for pad, off in ((0, 0), (3, 1)):
        h, c, s = norm_case(gpu, x, "bf16", r, "bf16", w, D, out=out, pad=pad, off=off)
        check_norm(h, c, s, w, D, out)


@pytest.mark.parametrize("out", ["f8", "i8"])
@pytest.mark.parametrize("rt", [None, "bf16", "f16", "f32"])
@pytest.mark.parametrize("xt", ["bf16", "f16", "f32"])
def test_norm_types(gpu, xt, rt, out):
    rng = np.random.default_rng(5)
    for M, D, inplace in ((3, 1000, True), (65, 384, False)):
        x, r = rng.standard_normal((M, D)) * 3, rng.standard_normal((M, D)) * 0.01
        h, c, s = norm_case(gpu, x, xt, r, rt, None, D, out=out, inplace=inplace)
        check_norm(h, c, s, None, D, out)


def test_many_rows_have_exact_codes(gpu):
    """Half a million values, of which about ten have a float quotient beyond a tie from the exact one."""
    rng = np.random.default_rng(14)
    M, D = 128, 4096
    x = rng.standard_normal((M, D))
    w = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    h, c, s = norm_case(gpu, x, "f32", None, None, w, D)
    check_norm(h, c, s, w, D, "f8")


@pytest.mark.parametrize("out", ["f8", "i8"])
def test_norm_options(gpu, out):
    """Without the norm (plain rounding to 8 bits), with a gain or none, and a large eps."""
    rng = np.random.default_rng(6)
    M, D = 9, 640
    x = rng.standard_normal((M, D)) * 1e-3
    w = rng.standard_normal(D).astype(np.float32)
    for kw in (dict(norm=False), dict(norm=True, eps=1.0), dict(norm=True, eps=0.0)):
        for g in (None, w):
            h, c, s = norm_case(gpu, x, "f32", x, "f32", g, D, out=out, **kw)
            check_norm(h, c, s, g, D, out, kw.get("eps", 1e-6), kw["norm"])


@pytest.mark.parametrize("out", ["f8", "i8"])
@pytest.mark.parametrize("mag", [1e-44, 1e-41, 3e-38, 1e-35, 1e-20, 1e15, 1e18, 3e38])
def test_extreme_magnitudes(gpu, mag, out):
    """Without the norm, rows from subnormal floats to the largest. A scale below 2^-126 is a multiple of 2^-149."""
    rng = np.random.default_rng(7)
    M, D = 4, 300
    x = (rng.uniform(-1, 1, (M, D)) * mag).astype(np.float32)
    h, c, s = norm_case(gpu, x, "f32", None, None, None, D, out=out, norm=False)
    v = h.astype(np.float64)
    ws = orq.block_scales(v) if out == "f8" else orq.row_scales(v)[:, None]
    assert np.all(np.abs(s - ws) <= 3 * U * ws + 2.0 ** -149)
    if out == "f8":
        check_codes(c, v / orq.per_column(ws, D), EXACT)
    else:
        q = v / ws
        assert np.all((c >= np.rint(q - np.abs(q) * 5 * U)) & (c <= np.rint(q + np.abs(q) * 5 * U)))


def test_zero_blocks_and_rows(gpu):
    rng = np.random.default_rng(8)
    M, D = 4, 700
    x = rng.standard_normal((M, D)).astype(np.float32)
    x[1] = 0
    x[2, 128:256] = 0
    x[3, 640:] = 0
    for out in ("f8", "i8"):
        h, c, s = norm_case(gpu, x, "bf16", np.zeros_like(x), "f32", None, D, out=out)
        check_norm(h, c, s, None, D, out)
        assert not c[1].any() and np.all(s[1] == 1)
    assert s.shape == (M, 1)


def test_nan_and_infinity(gpu):
    """amax passes over NaN; only the row (through its sum, the scales) and the NaN itself are touched. An infinity's block
    has an infinite scale, code 0 elsewhere and NaN at the infinity; without the norm other blocks are as ever."""
    rng = np.random.default_rng(9)
    M, D = 3, 300
    x = rng.standard_normal((M, D)).astype(np.float32)
    x[1, 5], x[2, 200] = np.nan, np.inf
    h, c, s = norm_case(gpu, x, "f32", None, None, None, D, norm=False)
    clean = np.where(np.isfinite(x), x, 0).astype(np.float64)
    ws = orq.block_scales(clean)
    ok = np.ones((M, 3), bool)
    ok[2, 1] = False
    assert np.all(np.abs(s - ws)[ok] <= 3 * U * ws[ok]) and np.isinf(s[2, 1])
    assert c[1, 5] & 0x7F == 0x7F and c[2, 200] & 0x7F == 0x7F
    at = np.repeat(ok, 128, 1)[:, :D].copy()
    at[1, 5] = False
    q = clean / orq.per_column(ws, D)
    check_codes(c[at], q[at], EXACT)
    rest = c[2, 128:256].copy()
    rest[200 - 128] = 0
    assert not (rest & 0x7F).any()
    h, c, s = norm_case(gpu, x, "f32", None, None, None, D, out="i8", norm=False)
    assert c[1, 5] == 0 and np.isinf(s[2, 0]) and np.isfinite(s[:2]).all()
    h, c, s = norm_case(gpu, x, "f32", None, None, None, D)  # with the norm: the NaN's row, the infinity's
    check_norm(x[:1], c[:1], s[:1], None, D, "f8")
    assert np.isnan(s[1]).all() and np.array_equal(s[2, [0, 2]], [0, 0]) and np.isnan(s[2, 1])


def test_no_rows(gpu):
    o, s = gpu.upload(np.full((2, 128), 9, np.uint8), "f8"), gpu.upload(np.full((2, 1), 9, np.float32))
    ops.rms_norm_q8(gpu, gpu.empty((2, 128), "bf16"), None, o, s, 0, 128, eps=1e-6)
    ops.swiglu_f8(gpu, gpu.empty((2, 256), "bf16"), o, s, 0, 128)
    gpu.wait()
    assert np.all(o.numpy() == 9) and np.all(s.numpy() == 9)


def test_sum_may_take_the_place_of_x(gpu):
    rng = np.random.default_rng(10)
    M, D = 6, 520
    xh, xf = as_type(rng.standard_normal((M, D)), "bf16")
    rh, rf = as_type(rng.standard_normal((M, D)), "bf16")
    X, R, O, S = gpu.upload(xh, "bf16"), gpu.upload(rh, "bf16"), gpu.empty((M, D), "f8"), gpu.empty((M, 5), "f32")
    ops.rms_norm_q8(gpu, X, None, O, S, M, D, eps=1e-6, res=R, res_out=X)
    gpu.wait()
    sh, h = as_type(xf + rf, "bf16")
    assert np.array_equal(X.numpy(), sh) and np.array_equal(R.numpy(), rh)
    check_norm(h, O.numpy(), S.numpy(), None, D, "f8")


def test_rows_past_32_bit_offsets(gpu):
    """Rows whose element offsets pass 2^31."""
    rng = np.random.default_rng(11)
    D, stride = 256, 800_000_000
    M = 4  # 3 * stride > 2^31
    X = gpu.empty((3 * stride + D,), "bf16")
    O = gpu.empty((3 * stride + D,), "f8")
    S = gpu.empty((M, 2), "f32")
    xh, xf = as_type(rng.standard_normal((M, D)), "bf16")
    for m in range(M):
        X.write(xh[m], m * stride)
    ops.rms_norm_q8(gpu, X, None, O, S, M, D, eps=1e-6, x_stride=stride, o_stride=stride)
    gpu.wait()
    c = np.stack([O.view((D,), offset_elems=m * stride).numpy() for m in range(M)])
    check_norm(xf, c, S.numpy(), None, D, "f8")


# -- the gated unit --------------------------------------------------------------------------------------------------


def gated_case(gpu, x, xt, D, pad=0, off=0):
    M = x.shape[0]
    print(f"[swiglu_f8] M={M} D={D} x={xt} pad={pad} off={off}", flush=True)
    xh, xf = as_type(x, xt)
    X, _, _ = strided(gpu, xh, xt, 2 * D + pad, off, 0)
    O, Ow, oflat = strided(gpu, np.zeros((M, D), np.uint8), "f8", D + pad, off, 77)
    ns = (D + 127) // 128
    SC, SCw, scflat = strided(gpu, np.zeros((M, ns), np.float32), "f32", ns, off, -5)
    ops.swiglu_f8(gpu, X, O, SC, M, D, x_stride=2 * D + pad, o_stride=D + pad)
    gpu.wait()
    ogot, sgot = Ow.numpy(), SCw.numpy()
    codes, scale = inside(ogot, off, M, D + pad, D).copy(), inside(sgot, off, M, ns, ns).copy()
    inside(ogot, off, M, D + pad, D)[:] = 0
    inside(sgot, off, M, ns, ns)[:] = 0
    assert np.array_equal(ogot, oflat) and np.array_equal(sgot, scflat), "written past the rows"
    return xf, codes, scale


# The gated value: exp(-|g|) within 2 steps of 2^-23 (the exponential's own and its argument's), the sum, quotient and
# products half a step each: 8 * 2^-24, doubled for a hardware reciprocal and exponential that round a whole step off.
GATED = 16 * U


def check_gated(xf, codes, scale, D):
    v = orq.gated(xf, D)
    ws = orq.block_scales(v)
    assert np.all(np.abs(scale - ws) <= (GATED + 3 * U) * ws + 2.0 ** -149), np.max(np.abs(scale - ws) / ws)
    check_codes(codes, v / orq.per_column(ws, D), 2 * GATED + 5 * U)


@pytest.mark.parametrize("xt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,D", SHAPES)
def test_gated_shapes(gpu, M, D, xt):
    rng = np.random.default_rng(M * 37 + D)
    x = rng.standard_normal((M, 2 * D)) * 3
    for pad, off in ((0, 0), (3, 1)):
        xf, c, s = gated_case(gpu, x, xt, D, pad, off)
        check_gated(xf, c, s, D)


@pytest.mark.parametrize("lo,hi", [(-30, 30), (-86, -60), (-100, -88), (80, 120), (-0.01, 0.01)])
def test_gate_ranges(gpu, lo, hi):
    """Gates of one range a block: saturated, far below zero (where exp passes out of the normal floats), near zero. Values
    of up to 1e6 keep their products in range."""
    rng = np.random.default_rng(12)
    M, D = 5, 384
    x = np.concatenate([rng.uniform(0.1, 1, (M, D)) * 1e6, rng.uniform(lo, hi, (M, D))], 1)
    xf, c, s = gated_case(gpu, x, "f32", D)
    check_gated(xf, c, s, D)


@pytest.mark.parametrize("xt", ["bf16", "f32"])
@pytest.mark.parametrize("lo,hi", [(-90, -86), (-130, -90), (-170, -130)])
def test_low_gates_of_huge_values(gpu, lo, hi, xt):
    """value * gate alone passes the largest float, the exponential alone the smallest one."""
    rng = np.random.default_rng(15)
    M, D = 3, 384
    x = np.concatenate([rng.uniform(0.1, 1, (M, D)) * 3.3e38, rng.uniform(lo, hi, (M, D))], 1)
    xf, c, s = gated_case(gpu, x, xt, D)
    check_gated(xf, c, s, D)
    x[:, D:] = rng.uniform(-1000, -250, (M, D))  # no float holds these products: zeros
    xf, c, s = gated_case(gpu, x, xt, D)
    assert not (c & 0x7F).any() and np.all(s == 1)


def test_gated_zero_nan_infinity(gpu):
    rng = np.random.default_rng(13)
    M, D = 4, 256
    x = rng.standard_normal((M, 2 * D)).astype(np.float32)
    x[0, :D] = 0
    x[1, D + 3] = np.nan
    x[2, D + 4], x[2, 4] = np.inf, 2.0
    x[3, D + 5] = -np.inf  # -inf / (1 + inf) is NaN
    xf, c, s = gated_case(gpu, x, "f32", D)
    assert not (c[0] & 0x7F).any() and np.all(s[0] == 1)
    assert c[1, 3] & 0x7F == 0x7F and np.isfinite(s[1]).all()
    assert c[2, 4] & 0x7F == 0x7F and np.isinf(s[2, 0]) and np.isfinite(s[2, 1])
    assert c[3, 5] & 0x7F == 0x7F and np.isfinite(s[3]).all()


# -- refusals (each ends on the host, before a launch) --------------------------------------------------------------------


def test_norm_refusals(gpu):
    M, D = 4, 256
    x, w = gpu.empty((M, D), "bf16"), gpu.empty((D,), "f32")
    r, o, s = gpu.empty((M, D), "f32"), gpu.empty((M, D), "f8"), gpu.empty((M, 2), "f32")

    def call(M=M, D=D, x=x, w=w, o=o, s=s, **kw):
        kw = dict(eps=1e-6) | kw
        ops.rms_norm_q8(gpu, x, w, o, s, M, D, **kw)

    call(res=r)
    for bad, what in ((dict(M=-1), "bad shape"), (dict(D=0), "bad shape"), (dict(D=(1 << 20) + 1), "bad shape"),
                      (dict(x_stride=255), "bad shape"), (dict(o_stride=255), "bad shape"),
                      (dict(res=r, res_stride=255), "bad shape"), (dict(eps=-1.0), "bad shape"),
                      (dict(eps=float("nan")), "bad shape"), (dict(M=5), "needs"), (dict(x_stride=300), "x needs"),
                      (dict(o_stride=300), "out needs"), (dict(w=gpu.empty((D - 1,), "f32")), "w needs"),
                      (dict(s=gpu.empty((M,), "f32")), "scale needs"), (dict(res=gpu.empty((3, D), "f32")), "res needs"),
                      (dict(M=1 << 24, D=1), "rows"),
                      (dict(res=r, res_out=r.view((M, D), offset_elems=0), res_out_stride=300), "res_out needs"),
                      (dict(o=x.view((M, D), "f8")), "shares memory"), (dict(res=r, s=r.view((M, 2))), "shares memory"),
                      (dict(res=r, o=r.view((M, D), "f8")), "shares memory")):
        with pytest.raises(GpuError, match=what):
            call(**bad)
    big = gpu.empty((M * D + D,), "f32")
    with pytest.raises(GpuError, match="shares memory"):  # a shifted residual: rows would be read after they are written
        call(res=big.view((M, D)), res_out=big.view((M, D), offset_elems=D))
    with pytest.raises(GpuError, match="aligned"):
        odd = gpu.empty((M * D * 4 + 4,), "u8")
        call(res=odd.view((M, D), "f32", offset_elems=1))


def test_gated_refusals(gpu):
    M, D = 4, 256
    x, o, s = gpu.empty((M, 2 * D), "bf16"), gpu.empty((M, D), "f8"), gpu.empty((M, 2), "f32")
    for args, kw, what in (((x, o, s, -1, D), {}, "bad shape"), ((x, o, s, M, 0), {}, "bad shape"),
                           ((x, o, s, M, D), dict(x_stride=2 * D - 1), "bad shape"),
                           ((x, o, s, M, D), dict(o_stride=D - 1), "bad shape"), ((x, o, s, M + 1, D), {}, "x needs"),
                           ((x, gpu.empty((M, D - 1), "f8"), s, M, D), {}, "out needs"),
                           ((x, o, gpu.empty((M,), "f32"), M, D), {}, "scale needs"),
                           ((x, x.view((M, D), "f8"), s, M, D), {}, "share")):
        with pytest.raises(GpuError, match=what):
            ops.swiglu_f8(gpu, *args, **kw)


def test_unknown_macros(gpu):
    for fn, macros in (("rms_norm_q8", dict(IN_T="int")), ("rms_norm_q8", dict(OUT_T="f16")), ("rms_norm_q8", dict(RES_T="i8")),
                       ("swiglu_f8", dict(RES_T="half")), ("rms_norm_q8", dict(NSG=8)), ("swiglu_f8", dict(IN_T="none"))):
        with pytest.raises(GpuError):
            gpu.kernel("ops", fn, **macros)
