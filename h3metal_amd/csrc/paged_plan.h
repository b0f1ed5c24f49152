// How the attention over a paged cache is cut into work, as plain arithmetic (also compiled for the host, where tests walk
// it).
//
// A tile is up to TT consecutive new tokens of one sequence with one group of query heads; a sequence of n new tokens has
// ceil(n / TT) tiles for each of VH groups. Tiles are ordered by sequence, group, token, and each has a weight (about the
// keys it reads); a slice is a run of equal weight of that order, whatever tiles it begins and ends inside of, so every
// workgroup gets as much to do as the others. Where a slice ends inside a tile, the tile's key blocks are cut in the same
// proportion. Weights of a sequence's tiles form an arithmetic series (with a causal mask each reads TT keys more than the
// one before), so a tile is found from its place in the order without a list of tiles.
#pragma once

#include <math.h>

#ifdef __HIPCC__
#define H3_HD __host__ __device__ __forceinline__
#else
#define H3_HD inline
#endif

namespace h3 {
namespace plan {

typedef long long i64;

struct Shape {
  int M, B;     // rows, sequences
  int TT, VH;   // tokens of a tile, head groups
  int causal;
  int cost;     // what a tile costs besides its keys, in keys
  i64 most;     // keys the page table can name
};

// a / b rounded down for 0 <= a, 1 <= b and a quotient below 2^50, by way of doubles (off by one at most): a 64-bit integer
// division is some 150 instructions
H3_HD i64 div(i64 a, i64 b) {
  i64 q = (i64)((double)a / (double)b);
  const i64 r = a - q * b;
  return r < 0 ? q - 1 : r >= b ? q + 1 : q;
}

// A sequence's part of the batch: rows lo .. hi - 1, L keys, row m sees keys up to off + m (with a causal mask); K tiles a head
// group, tile t weighs a + s t.
struct Seq {
  int lo, hi, K;
  i64 L, off, a, s;
};

H3_HD i64 clamp(i64 v, i64 lo, i64 hi) { return v < lo ? lo : v > hi ? hi : v; }

// Whatever the three numbers are, rows stay within 0 .. M and keys within the table.
H3_HD Seq seq_of(const Shape &sh, int q0, int q1, int kv) {
  Seq q;
  q.lo = (int)clamp(q0, 0, sh.M);
  q.hi = (int)clamp(q1, q.lo, sh.M);
  q.K = (q.hi - q.lo + sh.TT - 1) / sh.TT;
  q.L = clamp(kv, 0, sh.most);
  q.off = (i64)kv - q1;
  if (sh.causal) {
    q.a = clamp(q.off + q.lo, 0, q.L) + sh.TT + sh.cost;
    q.s = sh.TT;
  } else {
    q.a = q.L + sh.cost;
    q.s = 0;
  }
  return q;
}

H3_HD i64 before_tile(const Seq &q, i64 t) { return t * q.a + q.s * (t * (t - 1) / 2); }  // weight of tiles 0 .. t - 1
H3_HD i64 head_weight(const Seq &q) { return before_tile(q, q.K); }
H3_HD i64 tile_weight(const Seq &q, int t) { return q.a + q.s * t; }

// The tile of a head group at weight z of it.
H3_HD int tile_at(const Seq &q, i64 z) {
  i64 t;
  if (q.s == 0) {
    t = div(z, q.a);
  } else {
    const double p = (double)q.a - 0.5 * (double)q.s;
    t = (i64)((sqrt(p * p + 2.0 * (double)q.s * (double)z) - p) / (double)q.s);
    t = clamp(t, 0, q.K - 1);
    while (t > 0 && before_tile(q, t) > z) t--;
    while (t < q.K - 1 && before_tile(q, t + 1) <= z) t++;
  }
  return (int)clamp(t, 0, q.K - 1);
}

// Keys that any row of tile t sees, and its blocks of kb keys (one at least: a tile without keys still writes its zeros).
H3_HD i64 tile_keys(const Shape &sh, const Seq &q, int t) {
  if (!sh.causal) return q.L;
  const i64 end = clamp((i64)q.lo + (i64)(t + 1) * sh.TT, 0, q.hi);  // row behind the tile
  return clamp(q.off + end, 0, q.L);
}
H3_HD int tile_blocks(const Shape &sh, const Seq &q, int t, int kb) {
  const i64 n = (tile_keys(sh, q, t) + kb - 1) / kb;
  return n < 1 ? 1 : (int)n;
}

// The cut of a weight into n slices, n below 2^16.
struct Cut {
  i64 each;  // weight of a slice, and what is left over all of them
  int n, left;
};
H3_HD Cut cut_into(i64 total, int n) {
  const i64 e = total / n;
  return Cut{e, n, (int)(total - e * n)};
}
// At most n slices, of `least` each; as many for each tile if there are more slices than tiles, so that tiles of equal weight
// (one token of one sequence: as many tiles as head groups) are cut alike and no slice has pieces of two.
H3_HD Cut cut(i64 total, i64 tiles, int n, int least) {
  const i64 k = clamp(total / (least < 1 ? 1 : least), 1, n);
  return cut_into(total, (int)(tiles > 0 && k > tiles ? k / tiles * tiles : k));
}
// The weight before slice i.
H3_HD i64 slice_start(const Cut &c, int i) {
  return c.each * i + (int)((unsigned)c.left * (unsigned)i / (unsigned)c.n);
}

// The first key block behind weight x of a tile that starts at p, weighs w and has n blocks: where a slice that ends or
// begins at x cuts it (w n below 2^63).
H3_HD int block_at(i64 x, i64 p, i64 w, int n) { return x <= p ? 0 : x >= p + w ? n : (int)div((x - p) * n, w); }

// A partial state's place: 2 i for the tile that slice i found begun, 2 i + 1 for the one it leaves unfinished.
H3_HD int state_of(int i, bool begun) { return 2 * i + (begun ? 0 : 1); }

}  // namespace plan
}  // namespace h3
