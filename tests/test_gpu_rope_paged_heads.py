"""qk_norm_rope_paged: a head's queries and keys do not depend on the heads beside it, whose zeros or large values take another
path through the norm."""

import numpy as np
import pytest

from h3metal_amd import ops, rope
from paged_util import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,rot,inter", [(64, 64, False), (96, 96, False), (128, 128, False), (128, 40, False),
                                          (128, 38, False), (128, 128, True)])
def test_heads_do_not_depend_on_their_neighbours(gpu, hd, rot, inter):
    rng = np.random.default_rng(hd + rot)
    M, Hq, Hk, page = 2000, 4, 2, 16
    rows = rng.standard_normal((M, Hq + 2 * Hk, hd)).astype(np.float32)
    w, turns = gpu.upload(np.ones(hd, np.float32)), gpu.upload(rope.turns(rope.frequencies(rot)[0]), "u32")
    idx = (ints(gpu, [np.arange(M // page)]), ints(gpu, [0, M]), ints(gpu, [M]))

    def run(x):
        Q = gpu.empty((M, Hq * hd), "f16")
        kc, vc = (gpu.empty((M // page, Hk, page, hd), "f16") for _ in range(2))
        ops.qk_norm_rope_paged(gpu, gpu.upload(x.reshape(M, -1)), w, w, turns, Q, kc, vc, *idx, M=M, B=1, Hq=Hq, Hk=Hk, hd=hd,
                               rot=rot, eps=1e-6, interleaved=inter)
        gpu.wait()
        return Q.numpy().reshape(M, Hq, hd), kc.numpy()

    q, k = run(rows)
    for value in (0.0, 1e30, np.inf):
        x = rows.copy()
        x[:, [1, Hq]] = value
        q2, k2 = run(x)
        assert np.array_equal(q[:, [0, 2, 3]], q2[:, [0, 2, 3]]) and np.array_equal(k[:, 1], k2[:, 1]), value
