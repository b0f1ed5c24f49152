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

// -- on the host: which kernel runs a call, and how its tiles are shared out --------------------------------------------

constexpr int SHORT_ROWS = 32, CHUNK_ROWS = 256;  // rows of a tile: attention_paged.hip, attention_paged_chunk.hip
constexpr int LEFT_BYTES = 32;                    // of what a slice leaves behind besides its two states

// Query heads of a tile: a key/value head's G heads in HS groups of GP (the last may have fewer).
struct Heads {
  int G, HS, GP;
};
inline Heads heads_of(int H, int KVH, int rows) {
  const int G = H / KVH, HS = (G + rows - 1) / rows;
  return Heads{G, HS, (G + HS - 1) / HS};
}

// What the host knows of a call: rows, sequences, heads, and the caller's maxima of new tokens and keys.
struct Call {
  int M, B, H, KVH, max_q, max_kv;
};
// The tiles that a call has at most, whatever its sequences' lengths.
inline i64 most_tiles(const Call &c, const Heads &h, int rows) {
  const i64 TT = rows / h.GP, n = ((i64)c.M + (i64)c.B * (TT - 1)) / TT;
  return (i64)c.KVH * h.HS * (n < c.M ? n : c.M);
}

// Whether workgroups take whole 256-row tiles, in the order of their length: from 2 tiles a compute unit on where tiles differ in
// length (a prompt of 4096 tokens from its start: 24 % shorter than cut), from 4 on where they do not and a last round would
// be short of tiles (24 chunks of 96 tokens over 4000 keys, 1.5 tiles a unit: 259 us cut in equal slices). Cut tiles cost
// their states.
inline bool chunk_each(i64 tiles, int most, const Call &c) {
  return tiles <= 1 << 22 && tiles >= (2ll * c.max_q >= c.max_kv ? 2 : 4) * (i64)most;
}

// Whether a call runs on tiles of 256 rows: where their estimated time (us) is the shorter one. A start, a tile, its blocks (of
// 32 keys, of 64; their time goes with the head dim), and what cutting costs 256-row tiles; fitted to 60 calls of head dim 128 of
// 1 to 64 sequences of 16 to 4096 new tokens over 128 to 32 768 keys with 1, 4 and 16 heads a key/value head, and tried on 64 of
// head dims 64 and 96, where it loses 1 % on average to the better choice. Measured at head dim 128 | 96 | 64 (32 + 8 heads, calls
// in a row), 32 rows -> 256: a prompt of 4096 tokens 218 -> 135 | 195 -> 121 | 117 -> 93 us, of 1024 29 (256: 66) | 26 (55) | 16
// (48), a chunk of 512 over 16 384 keys 188 -> 151 | 168 -> 126 | 137 -> 99, of 64 over 4096 31 (37) | 28 (32) | 24 (27).
// The estimate knows the maxima only: it takes M / max_q sequences of max_q tokens and max_kv keys. Without the maxima 64 single
// tokens over a table of 32 768 keys count as one chunk and take 320 us instead of 208.
inline bool long_chunks(const Call &c, int d, bool causal, int cus) {
  const i64 n = clamp(c.max_q < c.M ? c.max_q : c.M, 1, c.M), seqs = (c.M + n - 1) / n, G = c.H / c.KVH;
  const double behind = c.max_kv - 0.5 * n, half = 0.5 * n;
  const double keys = !causal ? c.max_kv : behind > half ? behind : half;
  auto tiles = [&](int rows) {
    const i64 HS = (G + rows - 1) / rows, TT = rows / ((G + HS - 1) / HS);
    return (double)(c.KVH * HS * seqs * ((n + TT - 1) / TT));
  };
  const double few = tiles(SHORT_ROWS), many = tiles(CHUNK_ROWS);
  const double cut = chunk_each((i64)many, cus, c) ? 0 : 2ll * c.max_q >= c.max_kv ? 30 : 13;
  const double wide = d / 128.0;
  return 18 + many * (0.036 + 0.0085 / 64 * wide * keys) + cut < 10 + few * wide * (0.012 + 0.001 / 32 * keys);
}

struct Choice {
  int rows, waves;  // of a tile, of a workgroup
  bool each;        // whole tiles, a workgroup each, else slices
  i64 tiles;        // most_tiles
  int most;         // slices that compute units and scratch memory allow
};
// rows: 32 or 256, or 0 for what is estimated faster. d: the head dim.
inline Choice choose(const Call &c, int d, bool causal, int rows, int cus, unsigned long long ws_bytes) {
  const bool chunk = rows ? rows == CHUNK_ROWS : long_chunks(c, d, causal, cus);
  const int RT = chunk ? CHUNK_ROWS : SHORT_ROWS;
  const Heads h = heads_of(c.H, c.KVH, RT);
  const i64 tiles = most_tiles(c, h, RT), held = (i64)(ws_bytes / (2ull * RT * (d + 2) * sizeof(float) + LEFT_BYTES));
  const int most = (int)clamp(held, 1, chunk ? cus : 2 * cus);  // one or two workgroups a compute unit
  if (chunk) return Choice{RT, 4, chunk_each(tiles, most, c), tiles, most};
  // Whole tiles or slices. Few tiles of few keys are not worth a second kernel (one token, us whole with 8 waves and sliced: 512
  // keys 13, 19; 2048 21, 19). Tiles that share keys stay whole, side by side, from one a compute unit on (24 chunks of 48 tokens
  // over 2000 keys 86, 178 sliced); others are sliced until there are many, so that uneven lengths cost nothing. The lengths
  // themselves are not known here: 63 single tokens and a chunk of 16, one of them over 131 072 keys, stay whole and take 1160 us,
  // 138 sliced.
  const bool few = tiles <= cus && c.max_kv <= 2048;
  const bool shared = c.max_q > RT / h.GP;
  const bool each = few || (tiles <= 1 << 22 && (c.max_kv <= 512 || tiles >= (shared ? cus : 8 * most)));
  return Choice{RT, few ? 8 : 4, each, tiles, most};
}

}  // namespace plan
}  // namespace h3
