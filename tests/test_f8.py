"""e4m3 on the host (h3metal_amd/f8.py), its float64 oracle (oracle/rows_q8.py) and torch's float8_e4m3fn agree; block
scales; and the launchers of the 8-bit feed-forward operators: parameter blocks, buffer orders, refusals. No kernel runs."""

import struct

import numpy as np
import pytest
import torch

from h3metal_amd import f8, ops
from h3metal_amd import gpu as G
from oracle import rows_q8 as orq


def torch_values(codes):
    return torch.from_numpy(codes).view(torch.float8_e4m3fn).to(torch.float64).numpy()


def test_values_of_all_codes():
    c = np.arange(256, dtype=np.uint8)
    want = torch_values(c)
    assert np.array_equal(f8.from_f8(c).astype(np.float64), want, equal_nan=True)
    assert np.array_equal(orq.e4m3_value(c), want, equal_nan=True)
    fin = c[(c & 0x7F) != 0x7F]
    assert np.array_equal(f8.to_f8(f8.from_f8(fin)), fin)


def test_rounding_is_to_nearest_even():
    """Random values, every midpoint of two neighbours and the floats beside it, subnormal codes, and values past 448."""
    rng = np.random.default_rng(0)
    v = f8.from_f8(np.arange(0x7F, dtype=np.uint8)).astype(np.float64)
    mid = ((v[1:] + v[:-1]) / 2).astype(np.float32)
    x = np.concatenate([rng.standard_normal(20000).astype(np.float32) * 60, np.exp(rng.uniform(-12, 6.1, 20000)).astype(np.float32),
                        mid, np.nextafter(mid, np.float32(np.inf)), np.nextafter(mid, np.float32(0)),
                        np.float32([0, 2.0 ** -10, 2.0 ** -10 * 1.0001, 448, 463, 1e9, 1e-30])])
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch_values(torch.from_numpy(np.clip(x, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert np.array_equal(f8.from_f8(f8.to_f8(x)).astype(np.float64), want)
    assert np.array_equal(orq.e4m3_round(x), want)
    assert f8.to_f8(np.float32([np.nan]))[0] & 0x7F == 0x7F


@pytest.mark.parametrize("N,K,rows", [(1, 1, 128), (130, 300, 128), (256, 128, 128), (5, 257, 1)])
def test_block_codes(N, K, rows):
    rng = np.random.default_rng(N + K)
    w = rng.standard_normal((N, K)).astype(np.float32)
    w[0, 0] = 0
    w[-1, K // 2:] *= 1e-3
    c, s = f8.block_codes(w, rows)
    assert c.shape == (N, K) and s.shape == (-(-N // rows), -(-K // 128))
    # a code is off by at most half of its step (2^-4 of the value, 2^-10 below 2^-6), the quotient by 2^-24
    at = np.repeat(np.repeat(s.astype(np.float64), rows, 0)[:N], 128, 1)[:, :K]
    assert np.all(np.abs(orq.dequantised(c, s, rows) - w) <= at * (np.maximum(np.abs(w) / at * 2.0 ** -4, 2.0 ** -10) * 1.00001))
    zc, zs = f8.block_codes(np.zeros((3, 200), np.float32))
    assert not zc.any() and np.all(zs == 1)


# -- the launchers --------------------------------------------------------------------------------------------------


class FakeGpu:
    def __init__(self):
        self.kernels, self.launches = [], []

    def kernel(self, file, fn, **macros):
        self.kernels.append((file, fn, macros))

    def launch(self, k, grid, threads, args, params=b"", params_index=None, tg_mem=0, no_alloc=False):
        self.launches.append((args, params, params_index))


def T(shape, dtype):
    return G.Tensor(G.Buffer(0, 0), 0, tuple(shape), dtype)


def test_norm_launcher():
    g = FakeGpu()
    x, r, ro, w = T((9, 300), "bf16"), T((9, 310), "f32"), T((9, 320), "f32"), T((300,), "f32")
    o, s = T((9, 304), "f8"), T((9, 3), "f32")
    ops.rms_norm_q8(g, x, w, o, s, 9, 300, eps=1e-5, res=r, res_out=ro, res_stride=310, res_out_stride=320, o_stride=304)
    ops.rms_norm_q8(g, x, None, T((9, 300), "i8"), T((9,), "f32"), 9, 300, eps=0.0, norm=False)
    ops.rms_norm_q8(g, x, w, o, s, 9, 300, eps=1e-5, res=r, res_stride=310)
    assert g.kernels[0] == ("ops", "rms_norm_q8", {"IN_T": "bfloat", "RES_T": "float", "OUT_T": "f8"})
    assert g.kernels[1][2] == {"IN_T": "bfloat", "RES_T": "none", "OUT_T": "i8"}
    args, params, _ = g.launches[0]
    assert args == [x, r, w, o, s, ro]
    v = struct.unpack("<6ifi", params)
    assert v[:6] == (9, 300, 300, 310, 320, 304) and v[7] == 1
    assert struct.unpack("<6ifi", g.launches[1][1])[7] == 0 and g.launches[1][0][5] is None
    assert g.launches[2][0][5] is r and struct.unpack("<6ifi", g.launches[2][1])[3:5] == (310, 310)  # in place


@pytest.mark.parametrize("bad", [dict(out=T((2, 128), "f16")), dict(out=T((2, 128), "u8")), dict(scale=T((2,), "f16")),
                                 dict(w=T((128,), "bf16")), dict(x=T((2, 128), "i8")), dict(res=T((2, 128), "i32")),
                                 dict(res_out=T((2, 128), "f32")),
                                 dict(res=T((2, 128), "f32"), res_out=T((2, 128), "bf16"))])
def test_norm_launcher_refuses(bad):
    a = dict(x=T((2, 128), "bf16"), w=None, out=T((2, 128), "f8"), scale=T((2, 1), "f32"), res=None, res_out=None)
    a.update(bad)
    g = FakeGpu()
    with pytest.raises(ValueError, match="rms_norm_q8"):
        ops.rms_norm_q8(g, a["x"], a["w"], a["out"], a["scale"], 2, 128, eps=1e-6, res=a["res"], res_out=a["res_out"])
    assert not g.launches


def test_swiglu_launcher():
    g = FakeGpu()
    x, o, s = T((9, 600), "f16"), T((9, 300), "f8"), T((9, 3), "f32")
    ops.swiglu_f8(g, x, o, s, 9, 300)
    assert g.kernels == [("ops", "swiglu_f8", {"IN_T": "half"})]
    assert g.launches[0][0] == [x, o, s] and struct.unpack("<4i", g.launches[0][1]) == (9, 300, 600, 300)
    for bad in (dict(x=T((9, 600), "i8")), dict(o=T((9, 300), "i8")), dict(s=T((9, 3), "bf16"))):
        a = dict(x=x, o=o, s=s, **{}) | bad
        with pytest.raises(ValueError, match="swiglu_f8"):
            ops.swiglu_f8(g, a["x"], a["o"], a["s"], 9, 300)
    assert len(g.launches) == 1


def test_gemm_launcher_f8():
    """Exact row counts (no padding to a tile), scales a row = blocks of K, any N, and refusals."""
    g = FakeGpu()
    a, sa = T((9, 2000), "f8"), T((9, 16), "f32")
    wt = ops.QWeight("f8", T((1001, 2000), "f8"), T((8, 16), "f32"), 1001, 2000)
    out = T((9, 1001), "f32")
    ops.gemm(g, a, wt, out, 9, sa=sa)
    (f, n, m), = g.kernels
    assert (f, n) == ("gemm", "gemm") and m["WFMT"] == 9 and m["OUT_T"] == "float" and m["HAS_BIAS"] == 0
    args, params, pi = g.launches[0]
    assert pi == 8 and args == [a, wt.w, wt.sw, sa, out, None, None, None]
    assert struct.unpack("<8i", params) == (9, 1001, 2000, 2000, 1001, 2000, 16, 1001)
    for bad in (dict(a=T((9, 2000), "i8")), dict(sa=None), dict(wt=ops.QWeight("f8", wt.w, None, 1001, 2000)),
                dict(wt=ops.QWeight("f8", wt.w, wt.sw, 1001, 2000, G=64)), dict(ksplit=2), dict(sa=T((9, 16), "f16")),
                dict(wt=ops.QWeight("f8", T((1001, 2000), "i8"), wt.sw, 1001, 2000)), dict(epi=1, out=T((9, 1001), "bf16")),
                dict(wt=ops.QWeight("f8", wt.w, T((8, 16), "bf16"), 1001, 2000))):
        k = dict(a=a, sa=sa, wt=wt, ksplit=1, epi=0, out=out) | bad
        with pytest.raises(ValueError, match="gemm|split"):
            ops.gemm(g, k["a"], k["wt"], k["out"], 9, sa=k["sa"], ksplit=k["ksplit"], epi=k["epi"])
    assert len(g.launches) == 1


@pytest.mark.parametrize("bad", [dict(bias=T((1001,), "bf16")), dict(out=T((9, 1001), "f8")), dict(out=T((9, 1001), "i32")),
                                 dict(epi=1, rtype=T((9,), "i32")), dict(epi=1, rtype=T((9,), "f32")),
                                 dict(epi=1, gate=T((2, 1001), "bf16")), dict(epi=1, gate=T((2, 1001), "f16"))])
def test_gemm_launcher_f8_refuses_other_types(bad):
    """Buffers that the kernel would read or write as another type than theirs."""
    g = FakeGpu()
    k = dict(bias=T((1001,), "f32"), out=T((9, 1001), "f32"), epi=0, rtype=T((9,), "u8"), gate=T((2, 1001), "f32"))

    def call(bias, out, **kw):
        wt = ops.QWeight("f8", T((1001, 2000), "f8"), T((8, 16), "f32"), 1001, 2000, bias=bias)
        ops.gemm(g, T((9, 2000), "f8"), wt, out, 9, sa=T((9, 16), "f32"), **kw)

    call(**k)
    call(**k | dict(epi=1))
    call(**k | dict(out=T((9, 1001), "bf16")))
    assert len(g.launches) == 3
    with pytest.raises(ValueError, match="gemm"):
        call(**k | bad)
    assert len(g.launches) == 3
