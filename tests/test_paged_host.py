"""The paged operators' launchers on the CPU: what they pack and bind, and what they refuse before any launch. No kernel
runs here."""

import struct

import pytest

from h3metal_amd import gpu as G
from h3metal_amd import ops
from test_host import FakeGpu, T


def cache(dtype="bf16", pages=9, heads=8, page=16, hd=128):
    return T((pages, heads, page, hd), dtype), T((pages, heads, page, hd), dtype)


def rope_args(**kw):
    kc, vc = cache()
    a = dict(qkv=T((5, 48 * 128), "bf16"), wq=T((128,), "f32"), wk=T((128,), "f32"), turns=T((64, 2), "u32"),
             Q=T((5, 4096), "bf16"), kc=kc, vc=vc, table=T((2, 4), "i32"), q_start=T((3,), "i32"), kv_len=T((2,), "i32"),
             M=5, B=2, Hq=32, Hk=8, hd=128, rot=128, eps=1e-6)
    a.update(kw)
    return a


def attn_args(**kw):
    kc, vc = cache()
    a = dict(q=T((5, 4096), "bf16"), kc=kc, vc=vc, out=T((5, 4096), "bf16"), table=T((2, 4), "i32"),
             q_start=T((3,), "i32"), kv_len=T((2,), "i32"), M=5, B=2, H=32, KVH=8, D=128, scale=128 ** -0.5)
    a.update(kw)
    return a


def test_rope_packs_its_parameters():
    g, a = FakeGpu(), rope_args()
    ops.qk_norm_rope_paged(g, **a)
    (f, n, m), = g.kernels
    assert (f, n) == ("ops", "qk_norm_rope_paged")
    assert m == dict(HDIM=128, IN_T="bfloat", OUT_T="bfloat", INTER=0)
    (_, args, params, _), = g.launches
    assert args == [a[k] for k in ("qkv", "wq", "wk", "turns", "Q", "kc", "vc", "table", "q_start", "kv_len")] + [None]
    vals = struct.unpack("<11i2f", params)
    assert vals[:11] == (5, 2, 32, 8, 48 * 128, 4096, 128, 1, 9, 16, 4) and vals[12] == 1.0
    # without keys: no cache; without queries: no Q; positions of their own, pairs side by side
    g = FakeGpu()
    pos = T((5,), "i32")
    ops.qk_norm_rope_paged(g, **rope_args(kc=None, vc=None, table=None, Hk=0, norm=False, wq=None, wk=None, pos=pos,
                                          interleaved=True, in_stride=5000, q_stride=4100))
    ops.qk_norm_rope_paged(g, **rope_args(Q=None, Hq=0, wq=None))
    assert g.kernels[0][2]["INTER"] == 1 and g.launches[0][1][10] is pos
    assert struct.unpack("<11i2f", g.launches[0][2])[2:11] == (32, 0, 5000, 4100, 128, 0, 0, 0, 0)
    assert struct.unpack("<11i2f", g.launches[1][2])[2:4] == (0, 8)


def test_attention_packs_its_parameters():
    g, a = FakeGpu(), attn_args()
    ops.attention_paged(g, **a)
    ops.attention_paged(g, **attn_args(causal=False, max_q=1, max_kv=33, q_stride=4104, o_stride=4100))
    assert g.kernels[0] == ("attention", "attention_paged", dict(HD=128, IN_T="bfloat", CAUSAL=1))
    assert g.kernels[1][2]["CAUSAL"] == 0
    (_, args, params, _), (_, _, second, _) = g.launches
    assert args == [a[k] for k in ("q", "kc", "vc", "out", "table", "q_start", "kv_len")]
    vals = struct.unpack("<11if", params)
    assert vals[:11] == (5, 2, 32, 8, 4096, 4096, 9, 16, 4, 5, 64)
    assert abs(vals[11] - 128 ** -0.5 * 1.4426950408889634) < 1e-7
    assert struct.unpack("<11if", second)[4:11] == (4104, 4100, 9, 16, 4, 1, 33)
    ops.attention_paged(g, **attn_args(max_q=10 ** 12, max_kv=10 ** 12))  # hints of any size
    ops.attention_paged(g, **attn_args(max_q=-1, max_kv=-10 ** 12))
    assert struct.unpack("<11if", g.launches[2][2])[9:11] == (5, 2 ** 31 - 1)
    assert struct.unpack("<11if", g.launches[3][2])[9:11] == (0, 0)


@pytest.mark.parametrize("bad", [
    dict(Q=None), dict(kc=None), dict(vc=None), dict(table=None), dict(Hq=0), dict(Hk=0),  # a side without its half
    dict(Q=None, Hq=0, kc=None, vc=None, table=None, Hk=0),
    dict(Q=T((5, 4096), "f32")), dict(Q=T((5, 4096), "f16")), dict(qkv=T((5, 6144), "i8")),
    dict(kc=cache("f16")[0]), dict(vc=cache("f16")[1]), dict(kc=cache(pages=8)[0]), dict(kc=cache(heads=4)[0]),
    dict(vc=cache(hd=64)[1]), dict(kc=T((9, 8, 16 * 128), "bf16")),
    dict(wq=None), dict(wk=None), dict(wq=T((128,), "bf16")), dict(turns=None), dict(turns=T((64,), "f32")),
    dict(table=T((2, 4), "u32")), dict(table=T((8,), "i32")), dict(q_start=T((3,), "f32")), dict(kv_len=T((2,), "i16")),
    dict(pos=T((5,), "f32")), dict(kc=None, vc=None, table=None, Hk=0, q_start=T((3,), "f32")),
])
def test_rope_refuses(bad):
    g = FakeGpu()
    with pytest.raises(ValueError, match="qk_norm_rope_paged"):
        ops.qk_norm_rope_paged(g, **rope_args(**bad))
    assert not g.launches


@pytest.mark.parametrize("bad", [
    dict(q=T((5, 4096), "f16")), dict(out=T((5, 4096), "f32")), dict(q=T((5, 4096), "f32"), out=T((5, 4096), "f32")),
    dict(kc=cache("f16")[0]), dict(vc=cache("f16")[1]), dict(KVH=4), dict(D=64), dict(table=T((8,), "i32")),
    dict(table=T((2, 4), "f32")), dict(q_start=T((3,), "u32")), dict(kv_len=T((2,), "f32")),
])
def test_attention_refuses(bad):
    g = FakeGpu()
    with pytest.raises(ValueError, match="attention_paged"):
        ops.attention_paged(g, **attn_args(**bad))
    assert not g.launches


def test_parameter_blocks_have_the_kernels_size():
    assert len(G.pack("11i2f", *range(11), 1.0, 2.0)) == 52 and len(G.pack("11if", *range(11), 1.0)) == 48
