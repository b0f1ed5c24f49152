"""attention_paged against float64: heads, types, lengths from none to long, masks that leave rows empty, pages, strides,
what lies in masked places, page numbers outside the cache; and with qk_norm_rope_paged as a layer that grows its cache.

Bound of an output. A weight is rounded to the type once (u: half a step), and the sum that divides is of the rounded weights:
u sum|w (v - out)|. The output's own rounding: u |out|. A score's float sum of D exact products and its exponential: a score is
off by (D + 4) 2^-24 sum|q k| scale at most, an exponential by 2^-22, a sum over L keys by L / 32 + 16 additions in a row
(32 lanes and tiles of keys side by side): as parts of sum|w v|, doubled for numerator and denominator. In half precision a
weight below 2^-14 is off by 2^-25 instead: L 2^-25 max|v| (the largest weight is 1 or more)."""

import itertools

import numpy as np
import pytest

from h3metal_amd import ops, rope
from h3metal_amd.gpu import Gpu, GpuError
from oracle import paged as op
from paged_util import HALF, as_type, ints, page_table, q_starts, value

pytestmark = pytest.mark.gpu

FILL = 7.0


def batch(new, keys, *, H=4, KVH=2, D=128, t="bf16", page=16, seed=0, pad=0, width=None, q_size=1.0):
    rng = np.random.default_rng(seed)
    q_start = q_starts(new)
    M = int(q_start[-1]) + pad
    table, pages = page_table(rng, keys, page, width=width)
    q = as_type(q_size * rng.standard_normal((M, H, D)), t)[0]
    kc, vc = (as_type(rng.standard_normal((pages, KVH, page, D)), t)[0] for _ in range(2))
    return dict(q=q, kc=kc, vc=vc, table=table, q_start=q_start, kv_len=np.asarray(keys, np.int32), M=M, B=len(new), H=H,
                KVH=KVH, D=D, t=t, page=page)


def launch(gpu, c, *, causal=True, q_pad=0, o_pad=0, scale=None, **kw):
    M, H, D, t = c["M"], c["H"], c["D"], c["t"]
    rows = np.zeros((M, H * D + q_pad), c["q"].dtype)
    rows[:, :H * D] = c["q"].reshape(M, H * D)
    out = gpu.upload(as_type(np.full((M, H * D + o_pad), FILL), t)[0], t)
    print(f"[attn] M {M} B {c['B']} keys {c['kv_len'][:6]} heads {H}/{c['KVH']} D {D} {t} page {c['page']} causal {causal} "
          f"{kw}", flush=True)
    ops.attention_paged(gpu, gpu.upload(rows, t), gpu.upload(c["kc"], t), gpu.upload(c["vc"], t), out, ints(gpu, c["table"]),
                        ints(gpu, c["q_start"]), ints(gpu, c["kv_len"]), M=M, B=c["B"], H=H, KVH=c["KVH"], D=D,
                        scale=scale or D ** -0.5, causal=causal, q_stride=H * D + q_pad, o_stride=H * D + o_pad, **kw)
    gpu.wait()
    got = value(out.numpy(), t)
    assert np.all(got[:, H * D:] == FILL)
    return got[:, :H * D].reshape(M, H, D)


def check(got, c, *, causal=True, scale=None):
    t, D = c["t"], c["D"]
    q, kc, vc = (value(c[n], t) for n in ("q", "kc", "vc"))
    scale = float(np.float32(scale or D ** -0.5))
    want, spread, weight = op.attention(q, kc, vc, c["table"], c["q_start"], c["kv_len"], scale, causal)
    live = ~((np.isnan(want) & (op.places(c["q_start"], c["kv_len"], c["M"])[0] < 0)[:, None, None]))
    assert np.all(got[~live] == FILL)
    L = int(max(c["kv_len"].max(initial=0), 1))
    finite = [np.abs(x[np.isfinite(x)]).max(initial=0) for x in (q, kc, vc)]
    score = D * finite[0] * finite[1] * scale
    parts = 2 * ((D + 4) * score + 4 + L / 32 + 16) * 2.0 ** -24
    tol = HALF[t] * (spread + np.abs(want)) * 1.01 + parts * weight + (L * 2.0 ** -25 * finite[2] if t == "f16" else 0)
    ok = (np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want)
    assert ok[live].all(), (np.argwhere(~ok & live)[:5], got[~ok & live][:5], want[~ok & live][:5], tol[~ok & live][:5])
    return want


def variants(c):
    """The choices of tiles: the call's own, and both heights by name."""
    return [{}] + [dict(ROWS=r) for r in (32, 256)]


def both(gpu, c, causal=True, **kw):
    for v in variants(c):
        check(launch(gpu, c, causal=causal, **kw, **v), c, causal=causal, scale=kw.get("scale"))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_batch(gpu, D, t, causal):
    both(gpu, batch([1, 33, 0, 7, 64], [1, 50, 9, 300, 64], D=D, t=t, seed=D), causal)


@pytest.mark.parametrize("H,KVH", [(1, 1), (8, 8), (32, 8), (5, 1), (12, 4), (7, 1), (40, 8), (33, 1), (64, 1), (48, 1)])
def test_head_groups(gpu, H, KVH):
    both(gpu, batch([1, 9, 1], [37, 80, 1], H=H, KVH=KVH, D=64, seed=H))
    both(gpu, batch([70], [201], H=H, KVH=KVH, D=64, seed=H, t="f16"), False)


@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000, 4099])
def test_single_token_lengths(gpu, L):
    both(gpu, batch([1], [L], H=8, KVH=2, seed=L))
    both(gpu, batch([1, 1, 1], [L, 1, L // 2 + 1], H=2, KVH=2, D=64, t="f16", seed=L))


@pytest.mark.parametrize("n", [2, 15, 16, 17, 31, 32, 33, 63, 65, 128, 129, 257, 300])
def test_chunk_lengths(gpu, n):
    """Prompts from their first token, and chunks behind a prefix that ends anywhere."""
    both(gpu, batch([n], [n], H=2, KVH=1, seed=n))
    both(gpu, batch([n, 3, n], [n + 77, 3, n + 16], H=3, KVH=1, D=64, t="f16", seed=n))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages(gpu, page):
    both(gpu, batch([1, 40, 1, 1], [page, page + 41, 2 * page + 1, 5 * page - 1], page=page, seed=page))
    both(gpu, batch([page + 3], [3 * page], page=page, D=96, seed=page), False)


@pytest.mark.parametrize("B", [63, 64, 65, 200])
def test_many_sequences(gpu, B):
    rng = np.random.default_rng(B)
    new = rng.integers(0, 3, B)
    both(gpu, batch(new.tolist(), (new + rng.integers(0, 90, B)).tolist(), H=4, KVH=1, D=64, seed=B, pad=2))
    both(gpu, batch([1] * B, rng.integers(1, 200, B).tolist(), H=4, KVH=1, D=64, seed=B), max_q=1)


def test_mostly_idle_sequences(gpu):
    """Sequences without new tokens around and between those that have some."""
    new, keys = np.zeros(500, int), np.full(500, 40)
    new[[3, 70, 71, 200, 330, 498]] = [1, 100, 1, 30, 1, 7]
    keys[[3, 70, 71, 200, 330, 498]] = [900, 1500, 1, 30, 3000, 700]
    both(gpu, batch(new.tolist(), keys.tolist(), H=4, KVH=1, D=128, seed=22))
    both(gpu, batch(new.tolist(), keys.tolist(), H=4, KVH=1, D=64, seed=22))


@pytest.mark.parametrize("D,t", [(128, "bf16"), (64, "f16")])
def test_long(gpu, D, t):
    both(gpu, batch([1], [20000], H=4, KVH=1, D=D, t=t, page=64, seed=1))
    both(gpu, batch([1, 1], [20000, 7], H=2, KVH=2, D=D, t=t, page=16, seed=2))
    both(gpu, batch([5, 120], [9000, 3000], H=4, KVH=1, D=D, t=t, page=32, seed=3))
    both(gpu, batch([700], [1500], H=8, KVH=2, D=D, t=t, page=16, seed=4))


def test_long_rows(gpu):
    both(gpu, batch([1500], [1500], H=2, KVH=1, D=128, seed=5))
    both(gpu, batch([900, 600], [900, 2000], H=2, KVH=2, D=96, t="f16", seed=6), False)


def test_empty_rows_and_lengths(gpu):
    """No keys at all, fewer keys than new tokens (the first rows see none), rows of no sequence, kv_len below 0."""
    both(gpu, batch([3, 2], [0, 2], seed=1))
    both(gpu, batch([3, 2], [0, 2], seed=1), False)
    both(gpu, batch([40, 2], [7, 2], seed=2))
    both(gpu, batch([40, 2], [7, 2], seed=2), False)
    both(gpu, batch([4, 1], [9, 30], seed=3, pad=50))
    both(gpu, batch([0, 0], [9, 30], seed=3, pad=5))
    both(gpu, batch([2, 2], [-5, 3], seed=4))


def test_nothing_to_do(gpu):
    both(gpu, batch([0], [0], seed=1))
    both(gpu, batch([], [], seed=1))


def test_keys_past_the_table(gpu):
    c = batch([2, 1], [64, 40], seed=5)
    c["kv_len"] = np.array([1000, 40], np.int32)
    both(gpu, c, False)
    both(gpu, c)


@pytest.mark.parametrize("kw", [dict(max_q=1), dict(max_q=1, max_kv=1), dict(max_q=500, max_kv=10 ** 9), dict(max_kv=0, max_q=0)])
def test_hints_do_not_matter(gpu, kw):
    both(gpu, batch([1, 70, 3], [400, 700, 3], H=8, KVH=2, seed=6), **kw)


def test_strides(gpu):
    c = batch([5, 40], [60, 41], seed=7)
    both(gpu, c, q_pad=8, o_pad=4)
    both(gpu, c, q_pad=264, o_pad=132)


def test_scale_and_large_scores(gpu):
    c = batch([3, 50], [300, 70], seed=8, q_size=30.0)
    both(gpu, c, scale=0.5)
    both(gpu, batch([3, 50], [300, 70], seed=8, t="f16"), scale=1e-30)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_not_numbers_where_nothing_looks(gpu, D, t):
    """NaN and infinities behind the sequences' ends, in pages of nobody, and in keys and values of later tokens: the rows that
    do not see them are as without them, those that do have them."""
    spoils = [np.nan, np.inf, -np.inf]
    new, keys = [40, 1, 3], [70, 20, 3]
    for seed, what in enumerate(spoils):
        c = batch(new, keys, D=D, t=t, seed=seed, width=8)
        bits = as_type(np.array([what]), t)[0][0]
        used = np.zeros((len(c["kc"]), 16), bool)
        for b, L in enumerate(keys):
            for j in range(L):
                used[c["table"][b, j // 16], j % 16] = True
        for n in ("kc", "vc"):
            c[n].transpose(0, 2, 1, 3)[~used] = bits
        both(gpu, c)
        both(gpu, c, False)
        for (token, name), v in itertools.product(((55, "vc"), (69, "vc"), (61, "kc")), variants(c)):
            # tokens of sequence 0 that its rows up to token - 1 miss
            clean = launch(gpu, c, **v)
            d = dict(c, **{name: c[name].copy()})
            d[name][c["table"][0, token // 16], 1, token % 16, 5:9] = bits
            got = launch(gpu, d, **v)
            assert np.array_equal(got[:token - 30], clean[:token - 30]) and np.array_equal(got[40:], clean[40:])
            rows = got[token - 30:40, 2:]  # heads 2 and 3 read key/value head 1
            if name == "vc":
                assert not np.isfinite(rows[:, :, 5:9]).any()
                assert np.isfinite(rows[:, :, :5]).all() and np.isfinite(rows[:, :, 9:]).all()


@pytest.mark.parametrize("ROWS", [0, 32, 256])
def test_not_numbers_in_a_query(gpu, ROWS):
    c = batch([20, 2], [40, 9], seed=9)
    c["q"][3, 1, 7] = as_type(np.array([np.nan]), "bf16")[0][0]
    got = launch(gpu, c, ROWS=ROWS)
    assert np.isnan(got[3, 1]).all()
    c["q"][3, 1, 7] = 0
    again = launch(gpu, c, ROWS=ROWS)
    got[3, 1] = again[3, 1]
    assert np.array_equal(got, again)


@pytest.mark.parametrize("D,ROWS", [(128, 32), (128, 256), (96, 256), (64, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_not_numbers_that_are_seen(gpu, D, ROWS, causal):
    """Infinities of both signs in values that every row, or some rows of a tile, or of a cut tile, see."""
    for seed, (new, keys, at) in enumerate([([100], [400], (3, 250, 330, 399)), ([1], [3000], (5, 2999)),
                                            ([300], [1300], (20, 1000, 1200))]):
        c = batch(new, keys, H=2, KVH=1, D=D, seed=seed)
        for i, token in enumerate(at):
            c["vc"][c["table"][0, token // 16], 0, token % 16, 10 * i] = as_type(np.array([(-1) ** i * np.inf]), "bf16")[0][0]
        got = launch(gpu, c, causal=causal, ROWS=ROWS)
        want = check(got, c, causal=causal)
        assert np.isinf(want).any()


@pytest.mark.parametrize("D,ROWS", [(128, 32), (128, 256), (96, 256), (64, 256)])
def test_scores_that_jump(gpu, D, ROWS):
    """Keys whose scores outgrow those before by far, in any block: the running maximum follows."""
    c = batch([70, 1], [900, 700], H=4, KVH=1, D=D, seed=21)
    q = np.ones((c["M"], 4, D)) * 0.5
    c["q"] = as_type(q, "bf16")[0]
    for b, tokens in ((0, (1, 70, 300, 301, 640, 899)), (1, (699,))):
        for i, token in enumerate(tokens):
            c["kc"][c["table"][b, token // 16], 0, token % 16] = as_type(np.full(D, 3.0 * (i + 1)), "bf16")[0]
    check(launch(gpu, c, ROWS=ROWS), c)
    c["q"] = as_type(-q, "bf16")[0]
    check(launch(gpu, c, ROWS=ROWS), c)


def test_page_numbers_outside_the_cache(gpu):
    """Their keys score NaN: the rows that see them are NaN, the others as always."""
    c = batch([50, 3, 1], [80, 40, 300], seed=10)
    c["table"][0, 3], c["table"][1, 2], c["table"][2, 9] = len(c["kc"]), -1, 2 ** 31 - 1
    for v in variants(c):
        want = check(launch(gpu, c, **v), c)
        assert np.isnan(want[18:50]).all() and not np.isnan(want[:18]).any() and np.isnan(want[53]).all()
        check(launch(gpu, c, causal=False, **v), c, causal=False)
    c["kc"], c["vc"] = c["kc"][:0], c["vc"][:0]  # a cache of no pages
    for v in variants(c):
        assert np.isnan(launch(gpu, c, causal=False, **v)).all()


def test_rows_before_the_first_sequence_and_shared_pages(gpu):
    """A batch whose first rows belong to nobody, and sequences that share the pages of their first 48 keys."""
    c = batch([40, 1, 9], [100, 300, 60], H=4, KVH=2, seed=18, pad=5)
    c["q_start"] = c["q_start"] + 5
    c["table"][1:, :3] = c["table"][0, :3]
    both(gpu, c)
    both(gpu, c, False)


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_a_cache_past_32_bits(gpu, t):
    """Pages 4 GiB and more into the cache: keys and values go there and come from there."""
    KVH, D, page, H = 2, 128, 256, 4
    pages = (5 << 30) // (KVH * page * D * 2)
    rng = np.random.default_rng(19)
    new, keys = [300, 1], [300, 700]
    used = np.array([pages - 1, pages // 5 * 4 + 3, pages - 7, 2, pages - 2], np.int32)
    table = np.full((2, 3), -7, np.int32)
    table[0, :2], table[1] = used[:2], used[2:]
    kc, vc = gpu.empty((pages, KVH, page, D), t), gpu.empty((pages, KVH, page, D), t)
    held = [as_type(rng.standard_normal((5, KVH, page, D)), t)[0] for _ in range(2)]
    for c, rows in ((kc, held[0]), (vc, held[1])):
        for i, pg in enumerate(used):
            c.row(int(pg), 1).write(rows[i:i + 1])
    q_start, M = q_starts(new), 301
    qkv = gpu.upload(as_type(rng.standard_normal((M, (H + 2 * KVH) * D)), t)[0], t)
    w, Q = gpu.upload(np.ones(D, np.float32)), gpu.empty((M, H * D), t)
    turns = gpu.upload(rope.turns(rope.frequencies(D)[0]), "u32")
    idx = (ints(gpu, table), ints(gpu, q_start), ints(gpu, keys))
    print(f"[far cache] {pages} pages", flush=True)
    ops.qk_norm_rope_paged(gpu, qkv, w, w, turns, Q, kc, vc, *idx, M=M, B=2, Hq=H, Hk=KVH, hd=D, rot=D, eps=1e-6)
    gpu.wait()
    small = [np.concatenate([c.row(int(pg), 1).numpy() for pg in used]) for c in (kc, vc)]
    rows = as_type(qkv.numpy() if t == "f16" else value(qkv.numpy(), t), t)[0].reshape(M, -1, D)
    for m in range(300):  # the values of the first sequence's rows
        assert np.array_equal(small[1][m // page, :, m % page], rows[m, H + KVH:])
    c = dict(q=Q.numpy().reshape(M, H, D), kc=small[0], vc=small[1], table=np.array([[0, 1, -7], [2, 3, 4]], np.int32),
             q_start=q_start, kv_len=np.array(keys, np.int32), M=M, B=2, H=H, KVH=KVH, D=D, t=t, page=page)
    for v in variants(c):
        out = gpu.empty((M, H * D), t)
        ops.attention_paged(gpu, Q, kc, vc, out, *idx, M=M, B=2, H=H, KVH=KVH, D=D, scale=D ** -0.5, **v)
        gpu.wait()
        check(value(out.numpy(), t).reshape(M, H, D), c)


def test_starts_that_fall_are_harmless(gpu):
    """q_start out of order, negative or past M is no batch: nothing is promised but that only rows of q and out are touched."""
    for q_start in ([0, 5, 2, 8], [-3, 4, 9, 2], [8, 8, 100, 2 ** 31 - 1], [-2 ** 31, -5, 2 ** 31 - 1, -1]):
        c = batch([3, 3, 2], [30, 40, 9], seed=11)
        c["q_start"] = np.array(q_start, np.int32)
        for v in variants(c):
            launch(gpu, c, **v)
            launch(gpu, c, causal=False, max_q=1, **v)


def test_no_alloc_and_repeats(gpu):
    """Both entry points, twice each on the same context with other work between: bit for bit the same."""
    c = batch([1, 200, 1], [3000, 700, 90], H=8, KVH=2, page=32, seed=12)
    other = batch([1], [5000], H=8, KVH=1, seed=13)
    for v in variants(c):
        first = launch(gpu, c, **v)
        check(first, c)
        check(launch(gpu, other, no_alloc=True, **v), other)
        assert np.array_equal(launch(gpu, c, **v), first)
        static = launch(gpu, c, no_alloc=True, **v)
        check(static, c)
        both(gpu, other)
        assert np.array_equal(launch(gpu, c, no_alloc=True, **v), static)


def test_two_contexts_at_once(gpu):
    """Calls queued on two contexts, each with its scratch memory, before either is waited for."""
    other = Gpu()
    try:
        a, b = batch([1, 90], [4000, 2000], H=8, KVH=2, seed=15), batch([3, 400], [900, 1700], H=8, KVH=2, seed=16)
        for v in variants(a):
            tensors, outs = [], []
            for g, c in ((gpu, a), (other, b)):
                M, H, D = c["M"], c["H"], c["D"]
                t = dict(q=g.upload(c["q"].reshape(M, H * D), "bf16"), kc=g.upload(c["kc"], "bf16"), vc=g.upload(c["vc"], "bf16"),
                         out=g.empty((M, H * D), "bf16"), table=ints(g, c["table"]), q_start=ints(g, c["q_start"]),
                         kv_len=ints(g, c["kv_len"]))
                tensors.append(t)
            for _ in range(5):
                for g, c, t in ((gpu, a, tensors[0]), (other, b, tensors[1])):
                    ops.attention_paged(g, t["q"], t["kc"], t["vc"], t["out"], t["table"], t["q_start"], t["kv_len"], M=c["M"],
                                        B=c["B"], H=c["H"], KVH=c["KVH"], D=c["D"], scale=c["D"] ** -0.5, **v)
            for g, c, t in ((gpu, a, tensors[0]), (other, b, tensors[1])):
                g.wait()
                outs.append(t["out"].numpy())
                check(value(outs[-1], "bf16").reshape(c["M"], c["H"], c["D"]), c)
            del tensors, t
    finally:
        other.close()


def test_lengths_that_change_between_calls(gpu):
    """The same buffers with other lengths and pages in them: the next call follows what they hold."""
    c = batch([40, 1, 1], [500, 900, 20], H=8, KVH=2, seed=17, width=64)
    bufs = dict(q=gpu.upload(c["q"].reshape(c["M"], -1), "bf16"), kc=gpu.upload(c["kc"], "bf16"), vc=gpu.upload(c["vc"], "bf16"),
                out=gpu.empty((c["M"], 1024), "bf16"), table=ints(gpu, c["table"]), q_start=ints(gpu, c["q_start"]),
                kv_len=ints(gpu, c["kv_len"]))
    for q_start, kv_len in (([0, 40, 41, 42], [500, 900, 20]), ([0, 1, 41, 42], [3, 900, 17]), ([0, 0, 2, 42], [500, 2, 20])):
        c["q_start"], c["kv_len"] = np.array(q_start, np.int32), np.array(kv_len, np.int32)
        bufs["q_start"].write(c["q_start"])
        bufs["kv_len"].write(c["kv_len"])
        for v in variants(c):
            ops.attention_paged(gpu, *bufs.values(), M=c["M"], B=3, H=8, KVH=2, D=128, scale=128 ** -0.5, **v)
            gpu.wait()
            check(value(bufs["out"].numpy(), "bf16").reshape(c["M"], 8, 128), c)


def test_layer_grows_its_cache(gpu):
    """A batch whose cache grows over several calls, chunks and single tokens mixed, against attention over all of its rows at
    once: each call's queries, keys and values as the first operator leaves them."""
    rng = np.random.default_rng(14)
    H, KVH, D, page, t, B = 8, 2, 128, 16, "bf16", 3
    steps = [[30, 1, 7], [1, 1, 1], [5, 0, 40], [1, 60, 1], [0, 1, 0]]
    total = np.sum(steps, 0)
    table, pages = page_table(rng, total.tolist(), page)
    freq, rs = rope.frequencies(D, base=1e4)
    turns, kc, vc = gpu.upload(rope.turns(freq), "u32"), gpu.empty((pages, KVH, page, D), t), gpu.empty((pages, KVH, page, D), t)
    w = gpu.upload(np.ones(D, np.float32))
    held = np.zeros(B, np.int64)
    for new in steps:
        held += new
        q_start = q_starts(new)
        M = int(q_start[-1])
        qkv = gpu.upload(as_type(rng.standard_normal((M, (H + 2 * KVH) * D)), t)[0], t)
        Q, out = gpu.empty((M, H * D), t), gpu.upload(as_type(np.full((M, H * D), FILL), t)[0], t)
        tab, qs, kl = ints(gpu, table), ints(gpu, q_start), ints(gpu, held)
        print(f"[layer] new {new} held {held}", flush=True)
        ops.qk_norm_rope_paged(gpu, qkv, w, w, turns, Q, kc, vc, tab, qs, kl, M=M, B=B, Hq=H, Hk=KVH, hd=D, rot=D, eps=1e-6,
                               rope_scale=rs)
        ops.attention_paged(gpu, Q, kc, vc, out, tab, qs, kl, M=M, B=B, H=H, KVH=KVH, D=D, scale=D ** -0.5,
                            max_q=max(new), max_kv=int(held.max()))
        gpu.wait()
        c = dict(q=Q.numpy().reshape(M, H, D), kc=kc.numpy(), vc=vc.numpy(), table=table, q_start=q_start,
                 kv_len=held.astype(np.int32), M=M, B=B, H=H, KVH=KVH, D=D, t=t, page=page)
        check(value(out.numpy(), t).reshape(M, H, D), c)


def args(gpu, **kw):
    a = dict(q=gpu.empty((4, 512), "bf16"), kc=gpu.empty((3, 2, 16, 128), "bf16"), vc=gpu.empty((3, 2, 16, 128), "bf16"),
             out=gpu.empty((4, 512), "bf16"), table=gpu.empty((2, 2), "i32"), q_start=gpu.empty((3,), "i32"),
             kv_len=gpu.empty((2,), "i32"), M=4, B=2, H=4, KVH=2, D=128, scale=0.1)
    a.update(kw)
    return a


@pytest.mark.parametrize("what,bad", [
    ("bad shape", dict(M=-1)), ("bad shape", dict(B=-1)), ("bad shape", dict(M=1 << 24)), ("bad shape", dict(H=3)),
    ("bad shape", dict(q_stride=511)), ("bad shape", dict(o_stride=511)), ("scale", dict(scale=0.0)),
    ("scale", dict(scale=-1.0)), ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))),
    ("q needs", dict(M=5)), ("q_start needs", dict(q_start=("i32", (2,)))), ("multiple of 8", dict(q_stride=516, M=3)),
    ("out needs", dict(o_stride=516)), ("multiple of 8", dict(o_stride=514, M=3)),
    ("kv_len needs", dict(kv_len=("i32", (1,)))), ("table needs", dict(table=("i32", (1, 2)))),
    ("page", dict(page=24)), ("page", dict(page=8)), ("page", dict(page=512)),
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
        ops.attention_paged(gpu, **args(gpu, **bad))


def test_refuses_shared_memory_alignment_and_other_heads(gpu):
    a = args(gpu)
    for name in ("q", "kc", "vc"):
        with pytest.raises(GpuError, match="shares memory"):
            ops.attention_paged(gpu, **args(gpu, **{name: a[name], "out": a[name].view((4, 512))}))
    big = gpu.empty((3 * 2 * 16 * 128 + 8,), "bf16")
    for name, shape in (("q", (4, 512)), ("kc", (3, 2, 16, 128)), ("vc", (3, 2, 16, 128)), ("out", (4, 512))):
        with pytest.raises(GpuError, match="aligned"):
            ops.attention_paged(gpu, **args(gpu, **{name: big.view(shape, offset_elems=2)}))
    with pytest.raises(GpuError, match="not supported"):
        ops.attention_paged(gpu, **args(gpu, q=gpu.empty((4, 128), "bf16"), out=gpu.empty((4, 128), "bf16"), D=32,
                                        kc=gpu.empty((3, 2, 16, 32), "bf16"), vc=gpu.empty((3, 2, 16, 32), "bf16")))
    with pytest.raises(GpuError, match="unknown macro"):
        gpu.kernel("attention", "attention_paged", QK8=1)
    for bad in (dict(ROWS=64), dict(ROWS=-1), dict(ROWS=128, HD=64), dict(ROWS="x")):
        with pytest.raises(GpuError, match="ROWS"):
            gpu.kernel("attention", "attention_paged", **bad)
