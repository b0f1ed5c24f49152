"""ops.attention where the first keys score -infinity (masked by an infinite channel, as left padding is): their weight is 0, and
the rows are those of the other keys alone. Every kernel that runs 16-bit inputs.

Bound: a weight is rounded once to the type (half a step u): u sum |w (v - out)|; a score's float sum of D products and its
exponential: 2 ((D + 4) D max|q| max|k| + 4 + L / 32 + 16) 2^-24 sum |w v|; in half precision a weight below 2^-14 is off by
2^-25: L 2^-25 max|v|. The outputs are float."""

import numpy as np
import pytest

from paged_util import HALF, as_type
from test_gpu_attention import run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("D,causal,variant", [(128, False, dict(GROUPS=1)), (128, False, dict(SMALL=1)),
                                              (128, True, dict(GROUPS=1)), (96, False, {}), (64, False, {})])
def test_first_keys_score_minus_infinity(gpu, t, D, causal, variant):
    rng = np.random.default_rng(D)
    H, Lq, L, off = 2, 300, 1000, 700
    for first, a, b in ((64, 20.0, 60.0), (128, -200.0, -200.0), (200, -140.0, -150.0), (64, 5.0, 5.0)):
        q, k, v = (rng.standard_normal((H, n, D)) for n in (Lq, L, L))
        q *= 0.05
        q[:, :, :2] = 1.0  # channel 0 takes the mask, channel 1 a level (log2 units) that all scores are near
        k[:, :first, 0], k[:, first:, 0], k[:, :first, 1] = -np.inf, 0.0, 0.0
        k[:, first:, 1] = a * np.log(2.0)
        k[:, first + 150:, 1] = b * np.log(2.0)
        (qb, q), (kb, k), (vb, v) = (as_type(x, t) for x in (q, k, v))
        got = run_attention(gpu, qb, kb, vb, dtype=t, Lq=Lq, L=L, H=H, KVH=H, D=D, scale=1.0, causal=causal,
                            off=off if causal else 0, out_dt="f32", **variant)[:Lq].reshape(Lq, H, D)
        parts = 2 * ((D + 4) * D * np.abs(q).max() * np.abs(k[np.isfinite(k)]).max() + 4 + L / 32 + 16) * 2.0 ** -24
        for h in range(H):
            s = q[h] @ k[h].T
            if causal:
                s[np.arange(L)[None] > np.arange(Lq)[:, None] + off] = -np.inf
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            want = w @ v[h]
            spread = np.stack([w[i] @ np.abs(v[h] - want[i]) for i in range(Lq)])
            tol = HALF[t] * spread * 1.01 + parts * (w @ np.abs(v[h])) + (L * 2.0 ** -25 * np.abs(v).max() if t == "f16" else 0)
            assert np.all(np.abs(got[:, h] - want) <= tol + 2.0 ** -23 * np.abs(want)), (first, a, b)
