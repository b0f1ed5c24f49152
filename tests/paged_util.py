"""What the tests of the paged operators share: types, batches with their page tables, uploads."""

import numpy as np

from oracle.bf16 import from_bf16, to_bf16

HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a step, relative to the value
LEAST = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}  # half a step of the smallest values


def as_type(x, t):
    """(what is uploaded, its float64 values)"""
    x = np.asarray(x, np.float32)
    if t == "bf16":
        b = to_bf16(x)
        return b, from_bf16(b).astype(np.float64)
    if t == "f16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float64)
    return x, x.astype(np.float64)


def value(bits, t):
    return (from_bf16(bits) if t == "bf16" else bits).astype(np.float64)


def q_starts(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def page_table(rng, keys, page, spare=2, width=None):
    """(table [B][width], pages): every sequence's pages drawn from a shuffled pool; entries behind them name no page."""
    need = [-(-max(L, 0) // page) for L in keys]
    pages = sum(need) + spare
    order, at = rng.permutation(pages).astype(np.int32), 0
    table = np.full((len(keys), max(width or 0, max(need, default=0), 1)), -7, np.int32)
    for b, n in enumerate(need):
        table[b, :n], at = order[at:at + n], at + n
    return table, pages


def ints(gpu, x):
    return gpu.upload(np.ascontiguousarray(x, np.int32), "i32")
