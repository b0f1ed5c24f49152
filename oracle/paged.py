"""float64 rows and attention over a paged cache, of ops.qk_norm_rope_paged and ops.attention_paged.

Test infrastructure only (see oracle/__init__.py). The angles are reduced with the exact product of position and frequency
(a float64 has 53 bits, a position up to 31: split in two), not with the kernel's integer codes.
"""

from __future__ import annotations

import numpy as np


def angles(pos, freq):
    """pos * freq mod 2 pi in float64, from a split of freq into 26 + 27 bits so that both partial products are exact."""
    pos, freq = np.asarray(pos, np.float64)[:, None], np.asarray(freq, np.float64)[None]
    m, e = np.frexp(freq)
    hi = np.ldexp(np.floor(m * 2.0 ** 22) / 2.0 ** 22, e)
    lo = freq - hi
    return np.fmod(pos * hi, 2 * np.pi) + np.fmod(pos * lo, 2 * np.pi)


def rotated(v, pos, freq, rot, inter, factor):
    """(turned v, the size of each pair: what float errors of a turn are relative to). v [M][heads][hd] float64."""
    out, size = v.copy(), np.abs(v)
    if rot:
        a = angles(pos, freq)[:, None, :]
        first = np.arange(0, rot, 2) if inter else np.arange(rot // 2)
        second = first + (1 if inter else rot // 2)
        x, y = v[..., first], v[..., second]
        out[..., first] = factor * (x * np.cos(a) - y * np.sin(a))
        out[..., second] = factor * (y * np.cos(a) + x * np.sin(a))
        both = abs(factor) * (np.abs(x) + np.abs(y))
        size[..., first], size[..., second] = both, both
    return out, size


def normed(x, w, eps):
    """The RMS norm over the last axis; x / 2^k first, so that squares stay in range."""
    top = np.abs(x).max(-1, keepdims=True)
    k = np.where((top > 0) & np.isfinite(top), np.floor(np.log2(np.where(top > 0, top, 1))), 0.0)
    y = x * np.exp2(-k)
    with np.errstate(divide="ignore", invalid="ignore"):
        return y / np.sqrt((y * y).mean(-1, keepdims=True) + eps * np.exp2(-2 * k)) * w


def places(q_start, kv_len, M):
    """(sequence, place in it) of each row; (-1, 0) for rows of no sequence."""
    seq, at = np.full(M, -1), np.zeros(M, np.int64)
    for b in range(len(kv_len)):
        lo, hi = q_start[b], min(q_start[b + 1], M)
        for m in range(lo, hi):
            seq[m], at[m] = b, int(kv_len[b]) - int(q_start[b + 1]) + m
    return seq, at


def attention(q, kc, vc, table, q_start, kv_len, scale, causal):
    """(out, spread, weight) float64 [M][H][D] of float64 q [M][H][D] and caches [pages][KVH][page][D]: the output, the sum of
    |w (v - out)| and the sum of |w v|, which errors are relative to. Rows of no sequence stay NaN. Only visible keys
    enter any sum; a key whose page lies outside the cache makes its rows NaN."""
    M, H, D = q.shape
    pages, KVH, page, _ = kc.shape
    out, spread, weight = (np.full(q.shape, np.nan) for _ in range(3))
    for b in range(len(kv_len)):
        lo, hi = int(q_start[b]), min(int(q_start[b + 1]), M)
        L = max(0, min(int(kv_len[b]), table.shape[1] * page))
        ids = table[b, :-(-L // page)]
        bad = (ids < 0) | (ids >= pages)
        safe = np.where(bad, 0, ids)
        k = kc[safe].transpose(1, 0, 2, 3).reshape(KVH, -1, D)[:, :L] if L else np.zeros((KVH, 0, D))
        v = vc[safe].transpose(1, 0, 2, 3).reshape(KVH, -1, D)[:, :L] if L else np.zeros((KVH, 0, D))
        lost = np.repeat(bad, page)[:L]
        for m in range(lo, hi):
            end = max(0, min(L, int(kv_len[b]) - int(q_start[b + 1]) + m + 1)) if causal else L
            for h in range(H):
                if not end:
                    out[m, h] = spread[m, h] = weight[m, h] = 0
                    continue
                g = h // (H // KVH)
                with np.errstate(invalid="ignore"):
                    s = k[g, :end] @ q[m, h] * scale
                    s[lost[:end]] = np.nan
                    e = np.exp(s - s.max())
                    e /= e.sum()
                    vv = np.where(e[:, None] > 0, v[g, :end], np.where(np.isfinite(v[g, :end]), 0, v[g, :end]))
                    out[m, h] = e @ vv
                    spread[m, h] = e @ np.abs(vv - out[m, h])
                    weight[m, h] = e @ np.abs(vv)
    return out, spread, weight
