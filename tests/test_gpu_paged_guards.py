"""The paged operators write nothing but what they are for, whatever the lengths and page numbers hold: outputs and caches lie
inside larger buffers, whose other bytes, like all inputs, are the same bit for bit afterwards."""

import numpy as np
import pytest

from h3metal_amd import ops, rope
from paged_util import as_type, ints
from test_gpu_attention_paged import batch

pytestmark = pytest.mark.gpu

ODD = [([0, 5, 2, 8], 8), ([-3, 4, 9, 2], 8), ([8, 8, 100, 2 ** 31 - 1], 8), ([-2 ** 31, -5, 2 ** 31 - 1, -1], 8),
       ([0, 3, 6, 6], 8), ([300, 7, 290, 41], 300), ([0, 300, 0, 300], 300)]
LENGTHS = [[30, 40, 9], [-5, 2 ** 31 - 1, -2 ** 31], [0, 48, 1000]]
GUARD = 5  # rows, or pages, on either side


def inside(gpu, rows, t):
    """(the whole tensor, a view of all but GUARD leading and trailing slices) of random bits with `rows` in the middle."""
    rng = np.random.default_rng(len(rows))
    edge = [as_type(rng.standard_normal((GUARD,) + rows.shape[1:]), t)[0] for _ in range(2)]
    whole = gpu.upload(np.concatenate([edge[0], rows, edge[1]]), t)
    return whole, whole.row(GUARD, len(rows))


def edges(a):
    return a[:GUARD], a[-GUARD:]


@pytest.mark.parametrize("ROWS", [0, 32, 256])
@pytest.mark.parametrize("q_start,M", ODD)
@pytest.mark.parametrize("kv_len", LENGTHS)
def test_attention(gpu, q_start, M, kv_len, ROWS):
    c = batch([M, 0, 0], [M, 40, 9], H=4, KVH=2, seed=11)
    pad = 4
    out = as_type(np.full((M, 512 + pad), 7.0), "bf16")[0]
    whole, view = inside(gpu, out, "bf16")
    read = [gpu.upload(c["q"].reshape(M, -1), "bf16"), gpu.upload(c["kc"], "bf16"), gpu.upload(c["vc"], "bf16"),
            ints(gpu, c["table"]), ints(gpu, q_start), ints(gpu, kv_len)]
    before, held = whole.numpy(), [x.numpy() for x in read]
    for kw in (dict(), dict(causal=False, max_q=1), dict(max_q=1, max_kv=1, no_alloc=True)):
        print(f"[guards] attention {q_start} M {M} kv_len {kv_len} ROWS {ROWS} {kw}", flush=True)
        ops.attention_paged(gpu, *read[:3], view, *read[3:], M=M, B=3, H=4, KVH=2, D=128, scale=0.1, o_stride=512 + pad,
                            ROWS=ROWS, **kw)
        gpu.wait()
        after = whole.numpy()
        assert all(np.array_equal(a, b) for a, b in zip(edges(after), edges(before)))
        assert np.array_equal(after[:, 512:], before[:, 512:])
        assert all(np.array_equal(x.numpy(), h) for x, h in zip(read, held))


@pytest.mark.parametrize("q_start,M", ODD)
@pytest.mark.parametrize("kv_len", LENGTHS)
def test_rotary(gpu, q_start, M, kv_len):
    rng = np.random.default_rng(M)
    Hq, Hk, hd, page, pages = 4, 2, 64, 16, 40
    named = rng.permutation(pages)[:24].astype(np.int32)
    table = named.reshape(3, 8).copy()
    table[1, 2:5] = pages, -1, 2 ** 31 - 1
    (qw, Q), *caches = (inside(gpu, as_type(rng.standard_normal(s), "f16")[0], "f16")
                        for s in ((M, Hq * hd + 6), (pages, Hk, page, hd), (pages, Hk, page, hd)))
    (kw, kc), (vw, vc) = caches
    w, freq = np.ones(hd, np.float32), rope.frequencies(hd)[0]
    read = [gpu.upload(rng.standard_normal((M, (Hq + 2 * Hk) * hd)).astype(np.float32)), gpu.upload(w), gpu.upload(w),
            gpu.upload(rope.turns(freq), "u32"), ints(gpu, table), ints(gpu, q_start), ints(gpu, kv_len)]
    before, held = [x.numpy() for x in (qw, kw, vw)], [x.numpy() for x in read]
    print(f"[guards] rotary {q_start} M {M} kv_len {kv_len}", flush=True)
    ops.qk_norm_rope_paged(gpu, *read[:4], Q, kc, vc, *read[4:], M=M, B=3, Hq=Hq, Hk=Hk, hd=hd, rot=hd, eps=1e-6,
                           q_stride=Hq * hd + 6)
    gpu.wait()
    after = [x.numpy() for x in (qw, kw, vw)]
    for a, b in zip(after, before):
        assert all(np.array_equal(x, y) for x, y in zip(edges(a), edges(b)))
    assert np.array_equal(after[0][:, Hq * hd:], before[0][:, Hq * hd:])
    other = np.setdiff1d(np.arange(pages), table) + GUARD  # pages that the table does not name
    assert len(other) >= pages - 24
    assert all(np.array_equal(a[other], b[other]) for a, b in zip(after[1:], before[1:]))
    assert all(np.array_equal(x.numpy(), h) for x, h in zip(read, held))
