"""Which kernel a call of attention_paged runs on (h3metal_amd/csrc/paged_plan.h: choose), compiled for the host: that the batches
of the tests and of everyday calls reach every variant on a card of 256 compute units."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256
OWN, STATIC = CUS * (2 * 256 * 130 * 4 + 32), 32 << 20  # scratch bytes of a context (at least), of the allocation-free entry point
CODE = r"""
#include "paged_plan.h"
using namespace h3::plan;
extern "C" void choice(const int *c, int d, int causal, int rows, int cus, unsigned long long ws, long long *out) {
  const Choice x = choose(Call{c[0], c[1], c[2], c[3], c[4], c[5]}, d, causal, rows, cus, ws);
  out[0] = x.rows, out[1] = x.waves, out[2] = x.each, out[3] = x.tiles, out[4] = x.most;
}
"""


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "a C++ compiler is needed"
    d = tmp_path_factory.mktemp("choice")
    (d / "choice.cpp").write_text(CODE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "h3metal_amd", "csrc"), str(d / "choice.cpp"), "-o", str(d / "choice.so")], check=True)
    fn = ctypes.CDLL(str(d / "choice.so")).choice
    fn.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 4 + [ctypes.c_ulonglong, ctypes.c_void_p]

    def run(M, B, H, KVH, max_q, max_kv, *, D=128, causal=True, ROWS=0, cus=CUS, ws=OWN):
        call, out = np.array([M, B, H, KVH, max_q, max_kv], np.int32), np.zeros(5, np.int64)
        fn(call.ctypes.data, D, causal, ROWS, cus, ws, out.ctypes.data)
        return dict(zip(("rows", "waves", "each", "tiles", "most"), out.tolist()))
    return run


def whole_batch(seed=0, longest=500):
    """(new tokens, keys) of 70 sequences: idle ones, single tokens, short chunks, one of 300, one with `longest` keys."""
    rng = np.random.default_rng(seed)
    new = rng.integers(0, 4, 70)
    new[[5, 40, 66]] = [40, 33, 70]
    new[[20, 69, 0]] = [300, 1, 0]
    keys = new + rng.integers(0, 100, 70)
    keys[30], keys[20], keys[50] = 0, 410, longest
    return new.tolist(), keys.tolist()


# what test_gpu_attention_paged_whole.py runs: (H, KVH, D, ROWS, most keys), all on whole tiles
WHOLE = [(16, 16, D, ROWS, longest) for D in (64, 96, 128) for ROWS, longest in ((32, 500), (32, 1500), (256, 500), (256, 1500))]
WHOLE += [(32, 8, 128, 32, 1500), (32, 8, 128, 256, 500)]


@pytest.mark.parametrize("H,KVH,D,ROWS,longest", WHOLE)
@pytest.mark.parametrize("ws", [OWN, STATIC])
def test_the_whole_tiles_that_are_tested(choose, H, KVH, D, ROWS, longest, ws):
    new, keys = whole_batch(longest=longest)
    for causal in (True, False):
        c = choose(sum(new), len(new), H, KVH, max(new), max(keys), D=D, causal=causal, ROWS=ROWS, ws=ws)
        assert c["rows"] == ROWS and c["waves"] == 4 and c["each"] and c["tiles"] > CUS


def test_everyday_calls(choose):
    """One token of a short text, of a long one, of 64 texts; prompts; chunks behind a prefix."""
    assert choose(1, 1, 32, 8, 1, 512) == dict(rows=32, waves=8, each=1, tiles=8, most=512)
    assert choose(1, 1, 32, 8, 1, 131072) == dict(rows=32, waves=4, each=0, tiles=8, most=512)
    assert choose(64, 64, 32, 8, 1, 8192) == dict(rows=32, waves=4, each=0, tiles=512, most=512)
    assert choose(1404, 8, 32, 8, 500, 524) == dict(rows=32, waves=4, each=1, tiles=1456, most=512)
    assert choose(8192, 1, 32, 8, 8192, 8192) == dict(rows=256, waves=4, each=1, tiles=1024, most=256)
    assert choose(512, 1, 32, 8, 512, 16384) == dict(rows=256, waves=4, each=0, tiles=64, most=256)


def test_every_call_has_a_choice(choose):
    """The extremes: no hints at all, scratch for less than one slice, one compute unit, the largest numbers."""
    for M, B, H, KVH in ((1, 1, 1, 1), (1, 1 << 23, 4096, 1), ((1 << 24) - 1, (1 << 24) - 1, 4096, 4096), (5, 1, 7, 7)):
        for max_q, max_kv in ((0, 0), (M, 2 ** 31 - 1), (1, 1)):
            for ROWS in (0, 32, 256):
                for cus, ws in ((1, 0), (256, 0), (256, OWN), (256, 1 << 62)):
                    c = choose(M, B, H, KVH, max_q, max_kv, ROWS=ROWS, cus=cus, ws=ws)
                    assert c["rows"] in (32, 256) and c["waves"] in (4, 8) and 1 <= c["most"] <= 2 * cus and c["tiles"] >= 1
                    assert not c["each"] or c["tiles"] <= 1 << 22
                    assert c["waves"] == 4 or (c["each"] and c["rows"] == 32)
