"""The cut of the paged attention's work (h3metal_amd/csrc/paged_plan.h), compiled for the host and walked: every key block of
every tile is done exactly once, every part of a cut tile has a place of its own that its merge finds, whatever the lengths;
and lengths that make no sense stay within the rows and the table."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CODE = r"""
#include "paged_plan.h"
#include <map>
#include <tuple>
#include <vector>
#include <cstdio>
using namespace h3::plan;
struct Tile { int b, v, t, nb; i64 p, w; };
// the tiles in order, as a workgroup walks them
static std::vector<Tile> walk(const Shape &sh, const int *qs, const int *kv, int kb) {
  std::vector<Tile> out;
  i64 p = 0;
  for (int b = 0; b < sh.B; b++) {
    const Seq q = seq_of(sh, qs[b], qs[b + 1], kv[b]);
    for (int v = 0; v < sh.VH; v++)
      for (int t = 0; t < q.K; t++) {
        out.push_back({b, v, t, tile_blocks(sh, q, t, kb), p, tile_weight(q, t)});
        p += tile_weight(q, t);
      }
  }
  return out;
}
extern "C" int check(int M, int B, int TT, int VH, int causal, int cost, long long most, const int *qs, const int *kv,
                     int kb, int most_slices, int least) {
  const Shape sh{M, B, TT, VH, causal, cost, most};
  const std::vector<Tile> tiles = walk(sh, qs, kv, kb);
  i64 total = 0;
  size_t at = 0;
  for (int b = 0; b < B; b++) {
    const Seq q = seq_of(sh, qs[b], qs[b + 1], kv[b]);
    if (q.lo < 0 || q.hi > M || q.lo > q.hi || q.L < 0 || q.L > most || q.K < 0) return 1;
    const i64 w = head_weight(q);
    for (int v = 0; v < VH; v++)
      for (int t = 0; t < q.K; t++, at++) {
        const Tile &c = tiles[at];
        if (c.p != total + w * v + before_tile(q, t) || c.w < 1) return 2;
        for (i64 z : {c.p, c.p + c.w / 2, c.p + c.w - 1}) {  // found again from any weight inside
          const i64 y = z - total;
          if (y / w != v || tile_at(q, y - w * (y / w)) != t) return 3;
        }
        const i64 keys = tile_keys(sh, q, t);
        if (keys < 0 || keys > q.L || (i64)c.nb * kb < keys) return 4;
      }
    total += w * VH;
  }
  if (tiles.empty()) return 0;
  const Cut cut_ = cut(total, (i64)tiles.size(), most_slices, least);
  const int n = cut_.n;
  if (slice_start(cut_, 0) != 0 || slice_start(cut_, n) != total) return 13;
  std::map<int, std::pair<size_t, int>> state;  // place -> tile, blocks
  std::vector<std::vector<int>> done(tiles.size());
  for (size_t k = 0; k < tiles.size(); k++) done[k].assign(tiles[k].nb, 0);
  size_t first = 0;
  for (int i = 0; i < n; i++) {
    const i64 x0 = slice_start(cut_, i), x1 = slice_start(cut_, i + 1);
    while (first < tiles.size() && tiles[first].p + tiles[first].w <= x0) first++;
    for (size_t k = first; k < tiles.size() && tiles[k].p < x1; k++) {
      const Tile &c = tiles[k];
      const int b0 = block_at(x0, c.p, c.w, c.nb), b1 = block_at(x1, c.p, c.w, c.nb);
      if (b0 > b1) return 5;
      for (int j = b0; j < b1; j++) done[k][j]++;
      const bool begun = c.p < x0, whole = !begun && c.p + c.w <= x1;
      if (!whole) {
        const int s = state_of(i, begun);
        if (s < 0 || s >= 2 * n || state.count(s)) return 6;
        state[s] = {k, b1 - b0};
      }
    }
  }
  for (auto &d : done)
    for (int c : d)
      if (c != 1) return 7;
  // the merges: boundary j belongs to the slice in which its tile begins
  std::map<size_t, int> merged;
  size_t used = 0;
  for (int j = 0; j + 1 < n; j++) {
    const i64 x = slice_start(cut_, j + 1);
    size_t k = 0;
    while (k + 1 < tiles.size() && tiles[k + 1].p <= x) k++;
    const Tile &c = tiles[k];
    if (c.p >= x || c.p < slice_start(cut_, j)) continue;
    merged[k]++;
    int blocks = 0;
    for (int i = j; i < n && slice_start(cut_, i) < c.p + c.w; i++) {
      const auto s = state.find(state_of(i, c.p < slice_start(cut_, i)));
      if (s == state.end() || s->second.first != k) return 8;
      if (s->second.second != block_at(slice_start(cut_, i + 1), c.p, c.w, c.nb) -
                                  block_at(slice_start(cut_, i), c.p, c.w, c.nb)) return 9;
      blocks += s->second.second;
      used++;
    }
    if (blocks != c.nb) return 10;
  }
  for (auto &m : merged)
    if (m.second != 1) return 11;
  return used == state.size() ? 0 : 12;
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "a C++ compiler is needed"
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(CODE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-shared", "-fPIC", "-I",
                    os.path.join(ROOT, "h3metal_amd", "csrc"), str(d / "plan.cpp"), "-o", str(d / "plan.so")], check=True)
    fn = ctypes.CDLL(str(d / "plan.so")).check
    fn.argtypes = [ctypes.c_int] * 6 + [ctypes.c_longlong, ctypes.c_void_p, ctypes.c_void_p] + [ctypes.c_int] * 3

    def run(q_start, kv_len, *, TT, VH, causal, cost=64, most=1 << 20, kb=32, slices=512, least=256, M=None):
        qs, kv = np.asarray(q_start, np.int32), np.asarray(kv_len, np.int32)
        M = int(qs[-1]) if M is None else M
        return fn(M, len(kv), TT, VH, causal, cost, most, qs.ctypes.data, kv.ctypes.data, kb, slices, least)
    return run


@pytest.mark.parametrize("seed", range(40))
def test_every_block_is_done_once(check, seed):
    rng = np.random.default_rng(seed)
    B = int(rng.integers(1, 40))
    new = rng.integers(0, [2, 5, 300][seed % 3], B)
    keys = new + rng.integers(0, [10, 700, 9000][seed % 3 - 1], B) - rng.integers(0, 3, B) * (seed % 5 == 0) * 20
    starts = np.concatenate([[0], np.cumsum(new)])
    for TT in (1, 6, 8, 32, 64, 256):
        for causal in (0, 1):
            for slices, least in ((1, 1), (7, 1), (512, 64), (512, 1024), (2048, 1)):
                assert check(starts, keys, TT=TT, VH=int(rng.integers(1, 9)), causal=causal, slices=slices, least=least,
                             kb=int(rng.choice([32, 64, 128]))) == 0


def test_long_and_short_ones(check):
    assert check([0, 1], [131072], TT=8, VH=8, causal=1) == 0
    assert check([0, 8192], [8192], TT=32, VH=8, causal=1, kb=64, slices=256) == 0
    assert check([0, 1], [2 ** 31 - 1], TT=8, VH=1, causal=0, most=2 ** 31 - 1, kb=1 << 16, slices=64) == 0
    assert check([0, 3], [0], TT=8, VH=3, causal=1, least=1) == 0
    assert check([0, 0, 0], [5, 9], TT=8, VH=3, causal=1) == 0
    assert check([0, 50], [7], TT=8, VH=3, causal=1, least=1) == 0


def test_lengths_that_make_no_sense(check):
    for qs in ([0, 5, 2, 8], [-3, 4, 9, 2], [8, 8, 100, 2 ** 31 - 1], [-2 ** 31, -5, 2 ** 31 - 1, -1]):
        for kv in ([30, 40, 9], [-1, -2 ** 31, 2 ** 31 - 1]):
            for causal in (0, 1):
                assert check(qs, kv, TT=8, VH=2, causal=causal, M=8, most=4096) == 0
