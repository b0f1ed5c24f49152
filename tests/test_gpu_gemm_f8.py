"""ops.gemm with weight format f8 (e4m3 operands, a scale for each block of 128) against float64: sizes from one row and
column, short last blocks, strides, every output form; NaN stays in its row; what lies behind the rows stays; the
feed-forward run of norm, product, gated unit and product; refusals.

Bound. A block's 128 products are exact; their sum in the matrix unit is off by at most a whole step of float (2^-23: it may
cut instead of round) of the magnitudes' sum for each addition, the blocks' sums (fused with their scale, which has half a
step) by half a step each, partial sums of the waves included: |error| <= (128 + blocks + 20) 2^-23 sum |terms|. A bias and
the residual form's gate and sum add half a float step of the values each. For 16-bit outputs the products may be those of the
8-bit matrix instruction, which aligns the 8 products of a group (8 neighbours in K) to the largest and keeps 13 bits below
its exponent: 7 of them are off by at most 2^-13 of it. Such an output adds half its step."""

import numpy as np
import pytest

from h3metal_amd import f8, ops
from h3metal_amd.gpu import Gpu, GpuError
from oracle import rows_q8 as orq
from oracle.bf16 import from_bf16, to_bf16

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# the plan's own choice; 16 x 16, 32 x 32, 48 x 64, 64 x 64 and 80 x 64 tiles whose waves split K; 128 x 128, 256 x 128 and
# 256 x 256 tiles (256 x 128 again for float outputs)
TILES = pytest.mark.parametrize("TILE", range(9), ids=["plan", "16", "32", "48", "64", "80", "128", "256x128", "256"])


def bound(mag, K, *values):
    return (128 + (K + 127) // 128 + 20) * 2 * U * mag + U * sum(np.abs(v) for v in values)


def aligned(a, sa, w, sw):
    """7 * 2^-13 times a bound of the sum of the groups' largest products."""
    def top(x):
        x = np.abs(x)
        x = np.pad(x, ((0, 0), (0, -x.shape[1] % 8)))
        return x.reshape(x.shape[0], -1, 8).max(-1)
    return 7 * 2.0 ** -13 * (top(orq.dequantised(a, sa)) @ top(orq.dequantised(w, sw, 128)).T)


def operands(rng, M, N, K):
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:, ::29] *= 8
    x *= np.exp(rng.uniform(-3, 3, (M, 1))).astype(np.float32)
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    return f8.block_codes(x, rows=1) + f8.block_codes(w)


def weight(gpu, w, sw, bias=None, ws=None):
    N, K = w.shape
    if ws:
        p = np.full((N, ws), 0x7F, np.uint8)  # NaN between the rows
        p[:, :K] = w
        w = p
    return ops.QWeight("f8", gpu.upload(w, "f8"), gpu.upload(sw), N, K, bias=None if bias is None else gpu.upload(bias), ws=ws)


def run(gpu, a, sa, w, sw, out="f32", bias=None, pads=(0, 0, 0), TILE=0, no_alloc=False):
    """out [M][N], rows pads[2] columns apart; A's and W's rows pads[0], pads[1] apart."""
    (M, K), N = a.shape, w.shape[0]
    print(f"[gemm f8] M={M} N={N} K={K} out={out} bias={bias is not None} pads={pads} TILE={TILE}", flush=True)
    if pads[0]:
        p = np.full((M, K + pads[0]), 0x7F, np.uint8)
        p[:, :K] = a
        a = p
    cs = N + pads[2]
    raw = np.full((M + 2, cs), 3, {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[out])
    O = gpu.upload(raw, out)
    ops.gemm(gpu, gpu.upload(a, "f8"), weight(gpu, w, sw, bias, K + pads[1] if pads[1] else None), O, M, sa=gpu.upload(sa),
             a_stride=K + pads[0], c_stride=cs, no_alloc=no_alloc, **(dict(TILE=TILE) if TILE else {}))
    gpu.wait()
    got = O.numpy()
    res = got[:M, :N].copy()
    got[:M, :N] = raw[:M, :N]
    assert np.array_equal(got.view(np.uint8), raw.view(np.uint8)), "written past the rows"
    return from_bf16(res).astype(np.float64) if out == "bf16" else res.astype(np.float64)


HALF_STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def check(got, a, sa, w, sw, out, bias=None):
    K = a.shape[1]
    want, mag = orq.product(a, sa, w, sw)
    more = ()
    if bias is not None:
        want = want + bias
        more = (want,)
    tol = bound(mag, K, *more)
    if out != "f32":
        tol = tol + aligned(a, sa, w, sw)
    tol = tol + HALF_STEP[out] * (np.abs(want) + tol) + (2.0 ** -25 if out == "f16" else 0.0)
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)
    if out == "f32" and got.size > 50:  # far below the bound, as roundings of either sign are
        assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)
    if out == "bf16" and got.size > 50:  # a rounding's mean square is a third of its bound's
        assert np.linalg.norm(got - want) <= 0.6 * 2.0 ** -8 * np.linalg.norm(want)


SIZES = [(1, 1, 16), (1, 5, 128), (1, 4096, 512), (2, 130, 144), (3, 33, 2000), (9, 1001, 400), (16, 256, 1024), (17, 64, 4096),
         (31, 100, 272), (33, 128, 128), (64, 200, 640), (65, 129, 384), (100, 512, 16), (129, 300, 1040), (200, 257, 256),
         (257, 384, 512), (300, 1024, 768), (513, 640, 896), (1000, 96, 2064)]


@TILES
@pytest.mark.parametrize("M,N,K", SIZES)
def test_sizes(gpu, M, N, K, TILE):
    rng = np.random.default_rng(M * 3 + N * 5 + K)
    ops4 = operands(rng, M, N, K)
    for out in ("f32", "bf16"):
        check(run(gpu, *ops4, out=out, TILE=TILE), *ops4, out)


@TILES
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K,pads", [(7, 264, 384, (0, 0, 0)), (70, 261, 336, (16, 48, 3)), (300, 512, 256, (128, 0, 8))])
def test_outputs_bias_strides(gpu, M, N, K, pads, out, TILE):
    rng = np.random.default_rng(M + N)
    ops4 = operands(rng, M, N, K)
    bias = rng.standard_normal(N).astype(np.float32)
    check(run(gpu, *ops4, out=out, bias=bias, pads=pads, TILE=TILE), *ops4, out, bias)


@TILES
@pytest.mark.parametrize("M,N,K,bias", [(1, 384, 512, True), (9, 130, 160, False), (77, 256, 1024, True), (300, 515, 256, False),
                                        (520, 640, 384, True)])
def test_residual_form(gpu, M, N, K, bias, TILE):
    """X += gate[rtype] * (v + bias); a row type past the gate table's rows takes its last."""
    rng = np.random.default_rng(M + K)
    a, sa, w, sw = operands(rng, M, N, K)
    b = rng.standard_normal(N).astype(np.float32) if bias else None
    x, gate = rng.standard_normal((M + 1, N)).astype(np.float32), rng.standard_normal((3, N)).astype(np.float32)
    rt = rng.integers(0, 5, M).astype(np.uint8)
    X = gpu.upload(x)
    print(f"[gemm f8] residual M={M} N={N} K={K} bias={bias} TILE={TILE}", flush=True)
    ops.gemm(gpu, gpu.upload(a, "f8"), weight(gpu, w, sw, b), X, M, sa=gpu.upload(sa), epi=1, rtype=gpu.upload(rt),
             gate=gpu.upload(gate), **(dict(TILE=TILE) if TILE else {}))
    gpu.wait()
    got = X.numpy()
    assert np.array_equal(got[M], x[M])
    v, mag = orq.product(a, sa, w, sw)
    if bias:
        v = v + b
    g = gate[np.minimum(rt, 2)].astype(np.float64)
    want = x[:M] + g * v
    tol = np.abs(g) * bound(mag, K, v) * 1.001 + 2 * U * (np.abs(g * v) + np.abs(want))
    assert np.all(np.abs(got[:M] - want) <= tol)


@TILES
@pytest.mark.parametrize("M", [13, 130])
def test_scales_of_every_block_are_its_own(gpu, M, TILE):
    """Codes 1 and scales from 2^-3 to 2^3: v is a sum of powers of two, exact in float."""
    N, K = 300, 656
    rng = np.random.default_rng(4)
    one = f8.to_f8(np.float32([1]))[0]
    a, w = np.full((M, K), one, np.uint8), np.full((N, K), one, np.uint8)
    sa = 2.0 ** rng.integers(-3, 4, (M, 6)).astype(np.float32)
    sw = 2.0 ** rng.integers(-3, 4, (3, 6)).astype(np.float32)
    want, _ = orq.product(a, sa, w, sw)
    assert np.array_equal(run(gpu, a, sa, w, sw, TILE=TILE), want)
    assert np.array_equal(run(gpu, a, sa, w, sw, out="f16", TILE=TILE), want.astype(np.float16).astype(np.float64))


@TILES
@pytest.mark.parametrize("M,out", [(15, "f32"), (40, "f32"), (40, "bf16")])
def test_nan_stays_in_its_row(gpu, M, out, TILE):
    rng = np.random.default_rng(5)
    a, sa, w, sw = operands(rng, M, 140, 400)
    clean = run(gpu, a, sa, w, sw, out=out, TILE=TILE)
    a[3, 399] = 0x7F
    sa[M - 2, 1] = np.inf
    got = run(gpu, a, sa, w, sw, out=out, TILE=TILE)
    assert np.isnan(got[3]).all() and not np.isfinite(got[M - 2]).any()
    keep = np.ones(M, bool)
    keep[[3, M - 2]] = False
    assert np.array_equal(got[keep], clean[keep])


@TILES
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("K", [96, 128, 400, 1040])
def test_infinite_last_scales(gpu, K, out, TILE):
    """An infinite scale of K's last block gives infinities of the block sum's sign, not NaN, in its row and its columns."""
    rng = np.random.default_rng(16)
    M, N = 21, 140
    a, sa, w, sw = operands(rng, M, N, K)
    a[:, -1], w[:, -1] = 0x38, 0x38
    block = orq.product(a[:, (K - 1) // 128 * 128:], np.ones((M, 1)), w[:, (K - 1) // 128 * 128:], np.ones((2, 1)))[0]
    clean = run(gpu, a, sa, w, sw, out=out, TILE=TILE)
    sa[3, -1] = sw[1, -1] = np.inf
    got = run(gpu, a, sa, w, sw, out=out, TILE=TILE)
    far = np.abs(block) > 0.1  # (the sums' own error is far smaller)
    hit = np.zeros((M, N), bool)
    hit[3], hit[:, 128:] = True, True
    assert np.array_equal(got[hit & far], np.copysign(np.inf, block)[hit & far])
    assert np.array_equal(got[~hit], clean[~hit])


@TILES
def test_same_call_same_bits(gpu, TILE):
    """Two calls, and the allocation-free entry point, give the same bits: sums have a fixed order."""
    rng = np.random.default_rng(6)
    ops4 = operands(rng, 150, 384, 1536)
    first = run(gpu, *ops4, TILE=TILE)
    assert np.array_equal(run(gpu, *ops4, TILE=TILE), first)
    assert np.array_equal(run(gpu, *ops4, TILE=TILE, no_alloc=True), first)


@pytest.mark.parametrize("TILE", [0, 6, 7, 8], ids=["plan", "128", "256x128", "256"])
@pytest.mark.parametrize("M,N,K,out", [(4700, 4224, 1296, "bf16"), (2500, 4100, 400, "f32"), (5000, 2056, 128, "f16"),
                                       (4400, 2304, 272, "f32"), (4607, 4096, 640, "bf16")])
def test_large_products_on_sampled_rows(gpu, M, N, K, out, TILE):
    """More tiles than compute units: workgroups take several, and a last, partly filled round's rows may run on smaller
    tiles. One, two, three and more blocks of K."""
    rng = np.random.default_rng(M)
    a, sa, w, sw = operands(rng, M, N, K)
    got = run(gpu, a, sa, w, sw, out=out, TILE=TILE)
    rows = np.r_[0:3, 255:258, 2047:2050, 2300, 4095:4100, M - 300:M - 295, M - 2:M]
    rows = rows[rows < M]
    check(got[rows], a[rows], sa[rows], w, sw, out)


@pytest.mark.parametrize("TILE", [0, 6, 7], ids=["plan", "128", "256x128"])
def test_large_residual_form_on_sampled_rows(gpu, TILE):
    """The last rows, on smaller tiles in the plan's choice, take their own row types and rows of X."""
    rng = np.random.default_rng(18)
    M, N, K = 4607, 4096, 1040
    a, sa, w, sw = operands(rng, M, N, K)
    x, gate = rng.standard_normal((M, N)).astype(np.float32), rng.standard_normal((3, N)).astype(np.float32)
    rt = rng.integers(0, 3, M).astype(np.uint8)
    X = gpu.upload(x)
    print(f"[gemm f8] residual M={M} N={N} K={K} TILE={TILE}", flush=True)
    ops.gemm(gpu, gpu.upload(a, "f8"), weight(gpu, w, sw), X, M, sa=gpu.upload(sa), epi=1, rtype=gpu.upload(rt),
             gate=gpu.upload(gate), **(dict(TILE=TILE) if TILE else {}))
    gpu.wait()
    rows = np.r_[0:3, 255:258, 2047:2050, 4090:4100, M - 130:M - 125, M - 2:M]
    v, mag = orq.product(a[rows], sa[rows], w, sw)
    g = gate[rt[rows]].astype(np.float64)
    want = x[rows] + g * v
    tol = np.abs(g) * bound(mag, K) + 2 * U * (np.abs(g * v) + np.abs(want))
    got = X.numpy()[rows]
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) / tol)


def test_output_past_32_bit_offsets(gpu):
    """Output rows whose element offsets pass 2^31."""
    rng = np.random.default_rng(8)
    M, N, K, cs = 4, 100, 256, 800_000_000
    a, sa, w, sw = operands(rng, M, N, K)
    O = gpu.empty((3 * cs + N,), "bf16")
    ops.gemm(gpu, gpu.upload(a, "f8"), weight(gpu, w, sw), O, M, sa=gpu.upload(sa), c_stride=cs)
    gpu.wait()
    got = np.stack([from_bf16(O.view((N,), offset_elems=m * cs).numpy()) for m in range(M)]).astype(np.float64)
    check(got, a, sa, w, sw, "bf16")


@pytest.mark.parametrize("M,D,F", [(1, 512, 768), (37, 384, 640), (300, 1024, 2176)])
def test_feed_forward(gpu, M, D, F):
    """Norm with the residual's addition, product, gated unit, product into the residual, each step's result checked against
    float64 of what it read."""
    rng = np.random.default_rng(M)
    print(f"[feed-forward] M={M} D={D} F={F}", flush=True)
    x, r = to_bf16(rng.standard_normal((M, D)).astype(np.float32)), rng.standard_normal((M, D)).astype(np.float32)
    nw = (1 + 0.1 * rng.standard_normal(D)).astype(np.float32)
    w1, s1 = f8.block_codes((rng.standard_normal((2 * F, D)) / np.sqrt(D)).astype(np.float32))
    w2, s2 = f8.block_codes((rng.standard_normal((D, F)) / np.sqrt(F)).astype(np.float32))
    R, A, SA = gpu.upload(r), gpu.empty((M, D), "f8"), gpu.empty((M, (D + 127) // 128), "f32")
    H, B, SB = gpu.empty((M, 2 * F), "bf16"), gpu.empty((M, F), "f8"), gpu.empty((M, (F + 127) // 128), "f32")
    Y = gpu.empty((M, D), "f32")
    gate = np.float32([[1.0] * D, [0.5] * D])
    rt = (np.arange(M) % 2).astype(np.uint8)
    ops.rms_norm_q8(gpu, gpu.upload(x, "bf16"), gpu.upload(nw), A, SA, M, D, eps=1e-6, res=R)
    ops.gemm(gpu, A, weight(gpu, w1, s1), H, M, sa=SA)
    ops.swiglu_f8(gpu, H, B, SB, M, F)
    R.copy_to(Y)
    ops.gemm(gpu, B, weight(gpu, w2, s2), Y, M, sa=SB, epi=1, rtype=gpu.upload(rt), gate=gpu.upload(gate))
    gpu.wait()
    h = R.numpy()
    assert np.array_equal(h, r + from_bf16(x))
    a, sa, b, sb = A.numpy(), SA.numpy(), B.numpy(), SB.numpy()
    v = orq.rms_norm(h, nw, 1e-6)
    # a code is off by half its step: 2^-4 of the value, 2^-10 scales below 2^-6 of one
    near = np.maximum(np.abs(v) * 2.0 ** -4, orq.per_column(orq.block_scales(v), D) * 2.0 ** -10)
    assert np.all(np.abs(orq.dequantised(a, sa) - v) <= near * 1.001)
    up = from_bf16(H.numpy()).astype(np.float64)
    check(up, a, sa, w1, s1, "bf16")
    g = orq.gated(up, F)
    near = np.maximum(np.abs(g) * 2.0 ** -4, orq.per_column(orq.block_scales(g), F) * 2.0 ** -10)
    assert np.all(np.abs(orq.dequantised(b, sb) - g) <= near * 1.001)
    p, mag = orq.product(b, sb, w2, s2)
    want = h + gate[rt].astype(np.float64) * p
    assert np.all(np.abs(Y.numpy() - want) <= bound(mag, F) + 2 * U * (np.abs(p) + np.abs(want)))


def test_run_in_two_contexts_at_once(gpu):
    """Norm, product, gated unit and product queued on two contexts' streams, one of them through the allocation-free entry
    point, three times in turn: the bits of a run alone."""
    rng = np.random.default_rng(17)
    M, D, F = 300, 512, 640
    print(f"[feed-forward] two contexts M={M} D={D} F={F}", flush=True)
    x = to_bf16(rng.standard_normal((M, D)).astype(np.float32))
    w1, s1 = f8.block_codes((rng.standard_normal((2 * F, D)) / np.sqrt(D)).astype(np.float32))
    w2, s2 = f8.block_codes((rng.standard_normal((D, F)) / np.sqrt(F)).astype(np.float32))

    def state(g):
        return dict(x=g.upload(x, "bf16"), a=g.empty((M, D), "f8"), sa=g.empty((M, 4), "f32"), w1=weight(g, w1, s1),
                    h=g.empty((M, 2 * F), "bf16"), b=g.empty((M, F), "f8"), sb=g.empty((M, 5), "f32"), w2=weight(g, w2, s2),
                    o=g.empty((M, D), "f32"))

    def queue(g, t, no_alloc):
        ops.rms_norm_q8(g, t["x"], None, t["a"], t["sa"], M, D, eps=1e-6, no_alloc=no_alloc)
        ops.gemm(g, t["a"], t["w1"], t["h"], M, sa=t["sa"], no_alloc=no_alloc)
        ops.swiglu_f8(g, t["h"], t["b"], t["sb"], M, F, no_alloc=no_alloc)
        ops.gemm(g, t["b"], t["w2"], t["o"], M, sa=t["sb"], no_alloc=no_alloc)

    first = state(gpu)
    queue(gpu, first, False)
    gpu.wait()
    want = first["o"].numpy()
    other = Gpu()
    second = state(other)
    try:
        for _ in range(3):
            first["o"].write(np.zeros((M, D), np.float32))
            second["o"].write(np.zeros((M, D), np.float32))
            queue(gpu, first, False)
            queue(other, second, True)
            gpu.wait()
            other.wait()
            assert np.array_equal(first["o"].numpy(), want) and np.array_equal(second["o"].numpy(), want)
    finally:
        second.clear()  # its buffers are freed before their context
        other.close()


def test_int8_rows_feed_the_int8_product(gpu):
    """rms_norm_q8's int8 rows are what gemm takes with format q8."""
    rng = np.random.default_rng(9)
    M, D, N = 70, 640, 256
    x = to_bf16(rng.standard_normal((M, D)).astype(np.float32))
    rows = ops.pad_rows(M, 64)
    A, SA, O = gpu.empty((rows, D), "i8"), gpu.empty((rows,), "f32"), gpu.empty((rows, N), "f32")
    wq, sw = rng.integers(-127, 128, (N, D)).astype(np.int8), rng.uniform(1e-4, 1e-3, N).astype(np.float32)
    ops.rms_norm_q8(gpu, gpu.upload(x, "bf16"), None, A, SA, M, D, eps=1e-6)
    ops.gemm(gpu, A, ops.QWeight("q8", gpu.upload(wq), gpu.upload(sw), N, D), O, M, sa=SA)
    gpu.wait()
    v = orq.rms_norm(from_bf16(x), None, 1e-6)
    a, sa = A.numpy()[:M], SA.numpy()[:M]
    assert np.all(np.abs(a * sa[:, None].astype(np.float64) - v) <= 0.501 * sa[:, None])
    want = (a.astype(np.float64) @ wq.astype(np.float64).T) * sa[:, None].astype(np.float64) * sw
    assert np.all(np.abs(O.numpy()[:M] - want) <= 3 * U * np.abs(want))


def test_refusals(gpu):
    M, N, K = 8, 256, 256
    a, w = gpu.empty((M, K), "f8"), gpu.empty((N, K), "f8")
    sa, sw, o = gpu.empty((M, 2), "f32"), gpu.empty((2, 2), "f32"), gpu.empty((M, N), "bf16")
    x, rt, gate = gpu.empty((M, N), "f32"), gpu.empty((M,), "u8"), gpu.empty((1, N), "f32")

    def call(M=M, N=N, K=K, a=a, w=w, sa=sa, sw=sw, o=o, bias=None, ws=None, **kw):
        ops.gemm(gpu, a, ops.QWeight("f8", w, sw, N, K, bias=bias, ws=ws), o, M, sa=sa, **kw)

    call()
    call(M=0)
    for bad, what in ((dict(M=-1), "bad shape"), (dict(K=0), "bad shape"), (dict(K=24), "bad shape"), (dict(N=0), "bad shape"),
                      (dict(a_stride=128), "bad shape"), (dict(a_stride=264), "bad shape"), (dict(ws=264), "bad shape"),
                      (dict(c_stride=128), "bad shape"), (dict(a_stride=1 << 23), "bad shape"), (dict(M=9), "a needs"),
                      (dict(N=257, o=gpu.empty((M, 257), "bf16")), "w needs"), (dict(sa=gpu.empty((M,), "f32")), "sa needs"),
                      (dict(sw=gpu.empty((2,), "f32")), "sw needs"), (dict(o=gpu.empty((M, 255), "bf16")), "out needs"),
                      (dict(bias=gpu.empty((N - 1,), "f32")), "bias needs"),
                      (dict(M=7, a=gpu.empty((M * K,), "f8").view((7, K), offset_elems=8)), "aligned"),
                      (dict(o=x, epi=1), "rtype"), (dict(o=x, epi=1, rtype=rt), "gate"),
                      (dict(o=x, epi=1, rtype=gpu.empty((M - 1,), "u8"), gate=gate), "rtype needs"),
                      (dict(o=x, epi=1, rtype=rt, gate=gate, g_stride=128), "g_stride"), (dict(TILE=9), "TILE"),
                      (dict(o=a.view((4, N), "bf16"), M=4), "shares memory"), (dict(o=w.view((M, N), "bf16")), "shares memory"),
                      (dict(o=x, epi=1, rtype=rt, gate=x.view((1, N))), "shares memory")):
        with pytest.raises(GpuError, match=what):
            call(**bad)
