"""qk_norm_rope_paged against float64: heads, types, rotary layouts, positions, batches and pages where they can go wrong;
what no row goes to stays bit for bit; refusals.

Bound of a value, in parts of 2^-24 of its pair's size (factor times (|a| + |b|), for turned channels): the sum of squares 12
additions in a row at most, halved by the root, its mean, eps and root 4, the products with the root and the weight 2, cos and sin
2 and their factor 1, the turn's two products and sum 3, the angle at 2^31 positions 4: under 24. Then one rounding to the
output's type."""

import numpy as np
import pytest

from h3metal_amd import ops, rope
from h3metal_amd.gpu import GpuError
from oracle import paged as op
from paged_util import HALF, LEAST, as_type, ints, page_table, q_starts, value

pytestmark = pytest.mark.gpu

PARTS = 24 * 2.0 ** -24


def within(got, want, size, t):
    err = np.abs(got - want)
    tol = PARTS * size + HALF[t] * np.abs(want) * 1.001 + LEAST[t]
    ok = (err <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok.all(), (np.argwhere(~ok)[:5], got[~ok][:5], want[~ok][:5])


def run_case(gpu, new, keys, *, Hq=4, Hk=2, hd=128, rot=128, x="bf16", t="bf16", inter=False, norm=True, page=16,
             scaling="none", factor=1.0, pos=None, pad=0, in_pad=0, q_pad=0, seed=0, width=None, table=None, data=None,
             eps=1e-6, no_alloc=False, scale_w=1.0, skip=0):
    """Runs the operator on a batch and checks queries and the whole cache, which starts out with random bits."""
    rng = np.random.default_rng(seed)
    q_start = q_starts(new) + np.int32(skip)
    M, B = int(q_start[-1]) + pad, len(new)
    slots = Hq + 2 * Hk
    tab, pages = page_table(rng, keys, page, width=width)
    if table is not None:
        tab = table(tab, pages)
    rows = rng.standard_normal((M, slots * hd + in_pad)) * np.exp2(rng.integers(-3, 4, (M, 1)))
    if data is not None:
        rows = data(rows)
    bits, vals = as_type(rows, x)
    freq, rs = rope.frequencies(rot, base=1e4, scaling=scaling, factor=factor, trained=512) if rot else (np.zeros(0), 1.0)
    w = [(scale_w * (1 + 0.2 * rng.standard_normal(hd))).astype(np.float32) for _ in range(2)]
    old = [as_type(rng.standard_normal((pages, Hk, page, hd)), t)[0] for _ in range(2)]
    Q = gpu.upload(as_type(np.full((M, Hq * hd + q_pad), 7.0), t)[0], t) if Hq else None
    C = [gpu.upload(o, t) for o in old] if Hk else [None, None]
    print(f"[rope] new {new} keys {keys} heads {Hq}/{Hk} hd {hd} rot {rot} {x}->{t} inter {inter} page {page}", flush=True)
    ops.qk_norm_rope_paged(gpu, gpu.upload(bits, x), gpu.upload(w[0]), gpu.upload(w[1]),
                           gpu.upload(rope.turns(freq), "u32") if rot else None, Q, *C, ints(gpu, tab) if Hk else None,
                           ints(gpu, q_start), ints(gpu, keys), M=M, B=B, Hq=Hq, Hk=Hk, hd=hd, rot=rot, eps=eps, norm=norm,
                           interleaved=inter, rope_scale=rs, pos=None if pos is None else ints(gpu, pos),
                           in_stride=slots * hd + in_pad, q_stride=Hq * hd + q_pad, no_alloc=no_alloc)
    gpu.wait()
    seq, at = op.places(q_start, keys, M)
    v = vals[:, :slots * hd].reshape(M, slots, hd)
    turned = v[:, :Hq + Hk]
    if norm:
        ww = np.concatenate([np.broadcast_to(w[0].astype(np.float64), (Hq, hd)),
                             np.broadcast_to(w[1].astype(np.float64), (Hk, hd))])
        turned = op.normed(turned, ww, float(np.float32(eps)))
    P = at if pos is None else np.asarray(pos, np.int64)
    want, size = op.rotated(turned, P, freq, rot, inter, float(np.float32(rs)))
    if Hq:
        got = value(Q.numpy(), t)
        live = seq >= 0
        within(got[live, :Hq * hd].reshape(-1, Hq, hd), want[live, :Hq], size[live, :Hq], t)
        assert np.all(got[~live] == 7) and np.all(got[:, Hq * hd:] == 7)
    if Hk:
        for c, o, new_rows, sizes in ((C[0], old[0], want[:, Hq:], size[:, Hq:]),
                                      (C[1], old[1], v[:, Hq + Hk:], 0 * v[:, Hq + Hk:])):
            got, left = c.numpy(), np.ones(o.shape, bool)
            for m in range(M):
                c_at = int(at[m])
                if seq[m] < 0 or c_at < 0 or c_at // page >= tab.shape[1]:
                    continue
                pg = tab[seq[m], c_at // page]
                if 0 <= pg < pages:
                    within(value(got[pg, :, c_at % page], t), new_rows[m], sizes[m], t)
                    left[pg, :, c_at % page] = False
            assert np.array_equal(got[left], o[left])


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("hd,rot,inter", [(128, 128, False), (128, 128, True), (128, 64, False), (128, 6, True), (128, 38, False),
                                          (128, 0, False), (64, 64, False), (64, 40, True), (64, 2, False), (96, 96, False),
                                          (96, 96, True), (96, 16, False), (96, 90, False)])
def test_heads_and_layouts(gpu, hd, rot, inter, t):
    run_case(gpu, [1, 7, 0, 17, 3], [1, 20, 5, 17, 40], hd=hd, rot=rot, inter=inter, t=t, x=t, seed=hd + rot)


@pytest.mark.parametrize("x,t", [("f32", "bf16"), ("f32", "f16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("norm", [True, False])
def test_types(gpu, x, t, norm):
    run_case(gpu, [3, 9], [3, 30], x=x, t=t, norm=norm, seed=3)
    run_case(gpu, [3, 9], [3, 30], x=x, t=t, norm=norm, hd=64, rot=20, seed=4)


@pytest.mark.parametrize("Hq,Hk", [(32, 8), (1, 1), (5, 1), (64, 8), (7, 7), (3, 0), (0, 3)])
def test_head_counts(gpu, Hq, Hk):
    run_case(gpu, [2, 1, 11], [18, 1, 11], Hq=Hq, Hk=Hk, seed=Hq)
    run_case(gpu, [1], [9], Hq=Hq, Hk=Hk, hd=64, rot=64, seed=Hq)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages(gpu, page):
    """Rows that start and end inside pages, at their ends, and across several."""
    run_case(gpu, [page, 1, 2 * page + 1, 5, 1], [page, page + 1, 4 * page, page + 2, 2 * page], page=page, seed=page, Hk=1)


@pytest.mark.parametrize("B", [1, 63, 64, 65, 200])
def test_many_sequences(gpu, B):
    rng = np.random.default_rng(B)
    new = rng.integers(0, 4, B)
    run_case(gpu, new.tolist(), (new + rng.integers(0, 50, B)).tolist(), Hq=2, Hk=1, pad=3, seed=B)


def test_single_tokens(gpu):
    run_case(gpu, [1] * 37, list(range(1, 38)), Hq=8, Hk=2, hd=128, seed=1)


def test_rows_of_no_sequence_stay(gpu):
    run_case(gpu, [4, 2], [4, 9], pad=21, seed=5)
    run_case(gpu, [0, 0], [4, 9], pad=5, seed=5)


def test_rows_before_the_first_sequence_stay(gpu):
    for new, keys in (([4, 2], [4, 9]), ([7], [20])):
        run_case(gpu, new, keys, skip=3, pad=2, seed=15)


def test_without_norm_weights(gpu):
    """norm=False needs no weights, rot=0 no frequencies."""
    x = as_type(np.random.default_rng(16).standard_normal((5, 3 * 64)), "bf16")[0]
    Q, kc, vc = gpu.empty((5, 64), "bf16"), gpu.empty((2, 1, 16, 64), "bf16"), gpu.empty((2, 1, 16, 64), "bf16")
    ops.qk_norm_rope_paged(gpu, gpu.upload(x, "bf16"), None, None, None, Q, kc, vc, ints(gpu, [[1]]), ints(gpu, [0, 5]),
                           ints(gpu, [5]), M=5, B=1, Hq=1, Hk=1, hd=64, rot=0, eps=0.0, norm=False)
    gpu.wait()
    assert np.array_equal(Q.numpy(), x[:, :64]) and np.array_equal(kc.numpy()[1, 0, :5], x[:, 64:128])
    assert np.array_equal(vc.numpy()[1, 0, :5], x[:, 128:]) and not kc.numpy()[0].any() and not vc.numpy()[1, 0, 5:].any()


def test_strides(gpu):
    for in_pad, q_pad in ((1, 3), (8, 16), (130, 0)):
        run_case(gpu, [5, 12], [5, 40], in_pad=in_pad, q_pad=q_pad, seed=in_pad)
        run_case(gpu, [5, 12], [5, 40], in_pad=in_pad, q_pad=q_pad, x="f32", hd=96, rot=96, seed=in_pad)


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 8.0), ("yarn", 4.0)])
def test_far_positions(gpu, scaling, factor):
    """Positions given for each row, to 2^31 - 1 and below 0, where a float's angle is long lost."""
    pos = [0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31 - 1, 2 ** 31 - 2, -1, -2 ** 31, 999983]
    for inter in (False, True):
        run_case(gpu, [4, 5], [4, 30], pos=pos, scaling=scaling, factor=factor, inter=inter, seed=6)


def test_tokens_without_a_place(gpu):
    """More new tokens than tokens in all, places behind the table, page numbers outside the cache: not stored, and their
    queries as always."""
    run_case(gpu, [9, 3], [4, 3], seed=7)
    run_case(gpu, [5, 20], [16 * 4 + 3, 20], width=4, seed=8, table=lambda t, n: t[:, :4])

    def spoil(t, n):
        t = t.copy()
        t[0, 0], t[0, 1], t[1, 0] = n, -1, 2 ** 31 - 1
        return t
    run_case(gpu, [40, 20, 3], [40, 20, 3], seed=9, table=spoil)


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_rows_whose_squares_leave_the_range(gpu, x, eps):
    def data(rows):
        k = np.array([100, -100, 120, -120, 64, -70, 126, -126, 0, 30])
        return rows / np.abs(rows).max(1, keepdims=True) * np.exp2(k[:len(rows), None].astype(np.float64))
    run_case(gpu, [10], [10], x=x, data=data, eps=eps, seed=10)


def test_rows_of_zeros_and_not_numbers(gpu):
    def data(rows):
        rows = rows.copy()
        rows[1] = 0
        rows[2, 5] = np.nan
        rows[3, 130] = np.inf
        return rows
    for norm in (True, False):
        with np.errstate(invalid="ignore"):
            run_case(gpu, [6], [6], data=data, norm=norm, rot=0, seed=11)


def test_long_batch_and_no_alloc(gpu):
    run_case(gpu, [1000, 1, 333], [1000, 1, 400], Hq=4, Hk=1, hd=64, rot=64, page=64, seed=12)
    run_case(gpu, [3, 1], [3, 50], seed=13, no_alloc=True)


def test_no_rows(gpu):
    run_case(gpu, [0], [0], seed=14)
    run_case(gpu, [], [], seed=14)


def args(gpu, **kw):
    """A right call's arguments, some of them replaced."""
    a = dict(qkv=gpu.empty((4, 8 * 128), "bf16"), wq=gpu.empty((128,)), wk=gpu.empty((128,)), turns=gpu.empty((64, 2), "u32"),
             Q=gpu.empty((4, 4 * 128), "bf16"), kc=gpu.empty((3, 2, 16, 128), "bf16"),
             vc=gpu.empty((3, 2, 16, 128), "bf16"), table=gpu.empty((2, 2), "i32"), q_start=gpu.empty((3,), "i32"),
             kv_len=gpu.empty((2,), "i32"), M=4, B=2, Hq=4, Hk=2, hd=128, rot=128, eps=1e-6)
    a.update(kw)
    return a


@pytest.mark.parametrize("what,bad", [
    ("bad shape", dict(M=-1)), ("bad shape", dict(B=-1)), ("bad shape", dict(M=1 << 24)), ("bad shape", dict(in_stride=1023)),
    ("bad shape", dict(q_stride=511)), ("rot", dict(rot=130)), ("rot", dict(rot=3)), ("rot", dict(rot=-2)),
    ("eps", dict(eps=-1.0)), ("eps", dict(eps=float("nan"))), ("rope_scale", dict(rope_scale=float("inf"))),
    ("qkv needs", dict(M=5, q_stride=512)), ("qkv needs", dict(in_stride=1025)), ("Q needs", dict(q_stride=513)),
    ("q_start needs", dict(q_start=("i32", (2,)))), ("turns needs", dict(turns=("u32", (63, 2)))), ("wq needs", dict(wq=("f32", (127,)))),
    ("kv_len needs", dict(kv_len=("i32", (1,)))), ("table needs", dict(table=("i32", (1, 2)))),
    ("pos needs", dict(pos=("i32", (3,)))), ("page", dict(page=24)), ("page", dict(page=8)), ("page", dict(page=512)),
])
def test_refusals(gpu, what, bad):
    bad = dict(bad)
    for k, v in bad.items():
        if isinstance(v, tuple):
            bad[k] = gpu.empty(v[1], v[0])
    if "page" in bad:
        n = bad.pop("page")
        bad.update(kc=gpu.empty((3, 2, n, 128), "bf16"), vc=gpu.empty((3, 2, n, 128), "bf16"))
    with pytest.raises(GpuError, match=what):
        ops.qk_norm_rope_paged(gpu, **args(gpu, **bad))


def test_refuses_shared_memory_and_other_heads(gpu):
    a = args(gpu, qkv=gpu.empty((24, 8 * 128), "bf16"))
    for name, other in (("Q", "qkv"), ("kc", "vc"), ("vc", "qkv"), ("Q", "kc")):
        t = a[other]
        with pytest.raises(GpuError, match="shares memory"):
            ops.qk_norm_rope_paged(gpu, **dict(a, **{name: t.view(a[name].shape)}))
    with pytest.raises(GpuError, match="aligned"):
        t = gpu.empty((3 * 2 * 16 * 128 + 8,), "bf16")
        ops.qk_norm_rope_paged(gpu, **args(gpu, kc=t.view((3, 2, 16, 128), offset_elems=4)))
    with pytest.raises(GpuError, match="not supported"):
        ops.qk_norm_rope_paged(gpu, **args(gpu, hd=32, rot=32, kc=gpu.empty((3, 2, 16, 32), "bf16"),
                                           vc=gpu.empty((3, 2, 16, 32), "bf16")))
    with pytest.raises(GpuError, match="unknown macro"):
        gpu.kernel("ops", "qk_norm_rope_paged", QK8=1)
