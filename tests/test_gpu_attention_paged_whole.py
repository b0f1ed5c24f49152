"""attention_paged where every workgroup takes a whole tile, 4 waves each: hundreds of tiles of 70 sequences, most of them idle or
short, at both heights, head dims, types and masks; with infinities, NaN and page numbers outside the cache; and through the
allocation-free entry point. test_paged_choice.py checks on the host that these batches take those kernels."""

import numpy as np
import pytest

from paged_util import as_type
from test_gpu_attention_paged import batch, check, launch
from test_paged_choice import WHOLE, whole_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,KVH,D,ROWS,longest", WHOLE)
@pytest.mark.parametrize("t,causal", [("bf16", True), ("f16", True), ("bf16", False)])
def test_whole_tiles(gpu, H, KVH, D, ROWS, longest, t, causal):
    new, keys = whole_batch(longest=longest)
    c = batch(new, keys, H=H, KVH=KVH, D=D, t=t, seed=D + ROWS, pad=3)
    hints = dict(max_q=max(new), max_kv=max(keys), ROWS=ROWS)
    got = launch(gpu, c, causal=causal, o_pad=4, **hints)
    check(got, c, causal=causal)
    assert np.array_equal(launch(gpu, c, causal=causal, no_alloc=True, o_pad=4, **hints), got, equal_nan=True)
    # values that are infinite or NaN, seen by some rows of a tile or by all, and page numbers outside the cache
    for b, token, what in ((20, 380, np.inf), (20, 7, -np.inf), (66, keys[66] - 1, np.nan), (40, 2, np.inf)):
        c["vc"][c["table"][b, token // 16], KVH // 2, token % 16, b // 2] = as_type(np.array([what]), t)[0][0]
    c["table"][5, 1], c["table"][20, 24] = len(c["kc"]), -1
    want = check(launch(gpu, c, causal=causal, **hints), c, causal=causal)
    assert np.isnan(want).any() and np.isinf(want).any()
