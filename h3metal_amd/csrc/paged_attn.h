// What the attention kernels over a paged cache share: their arguments, how a workgroup finds its share of the batch on the
// device, and the join of tiles that several workgroups worked on.
#pragma once

#include "attention_common.h"
#include "paged.h"
#include "paged_plan.h"

namespace h3 {

using plan::i64;

using plan::Heads;

struct AttnArgs {
  const char *q, *kc, *vc;
  char *out;
  float *ws;   // partial states: O [rows][D], then m and l of each row
  void *left;  // a Left for each slice
  const char *spare;  // memory that loads without a place of their own may read
};

constexpr int CHUNK_ROWS = plan::CHUNK_ROWS;
constexpr int M_MOST = 1 << 24;  // rows of a call are fewer
// Tiles of 256 rows for long chunks (attention_paged_chunk.hip); t: T_BF16 or T_F16.
int launch_attention_chunk(int d, int t, bool causal, const Exec &ex, const AttnArgs &a, const Batch &bt,
                           const PagedAttnParams &p, const plan::Choice &c, std::string *err);

namespace {

// Whether the 16-bit value in the high half is infinite or NaN
template <int T>
__device__ __forceinline__ bool odd16(unsigned v) {
  constexpr unsigned E = T == T_BF16 ? 0x7F800000u : 0x7C000000u;
  return (v & E) == E;
}

// -- finding the work -------------------------------------------------------------------------------------------------

__device__ __forceinline__ i64 wave_sum_to(i64 v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const i64 u = __shfl_up(v, d);
    v += lane >= d ? u : 0;
  }
  return v;
}
__device__ __forceinline__ i64 lane_value(i64 v, int l) {
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)v, l), hi = __builtin_amdgcn_readlane((int)(v >> 32), l);
  return (i64)(((unsigned long long)hi << 32) | lo);
}

// The batch's weight, and the sequence at a weight of it; 64 sequences at a time, one a lane.
struct Order {
  const plan::Shape &sh;
  const Batch &bt;
  int q0, q1, kv;        // of the first 64 sequences: this lane's
  i64 own, upto, first;  // its weight, the sum up to it, their sum
  i64 all, tiles;        // the batch's weight and tiles

  __device__ Order(const plan::Shape &s, const Batch &b) : sh(s), bt(b) {
    int K;
    own = weight(threadIdx.x & 63, &q0, &q1, &kv, &K);
    if (bt.B == 1) {
      upto = own = all = first = lane_value(own, 0);
      tiles = (i64)__builtin_amdgcn_readfirstlane(K) * sh.VH;
      return;
    }
    upto = wave_sum_to(own);
    all = first = lane_value(upto, 63);
    i64 mine = K;
    for (int k = 64; k < bt.B; k += 64) {
      int x, y, z;
      all += lane_value(wave_sum_to(weight(k + (threadIdx.x & 63), &x, &y, &z, &K)), 63);
      mine += K;
    }
    tiles = lane_value(wave_sum_to(mine), 63) * sh.VH;
  }
  __device__ i64 weight(int b, int *s0, int *s1, int *n, int *K) const {
    *s0 = *s1 = *n = 0;
    if (b < bt.B) {
      *s0 = bt.q_start[b];
      *s1 = bt.q_start[b + 1];
      *n = bt.kv_len[b];
    }
    const plan::Seq q = plan::seq_of(sh, *s0, *s1, *n);
    *K = q.K;
    return plan::head_weight(q) * sh.VH;
  }
  // the sequence at weight x, and the weight before it
  __device__ int find(i64 x, i64 *before) const {
    i64 base = 0, w = own, s = upto, sum = first;
    for (int k = 0;; k += 64) {
      const unsigned long long m = __ballot(base + s > x);
      if (m) {
        const int l = __builtin_ctzll(m);
        *before = base + lane_value(s - w, l);
        return __builtin_amdgcn_readfirstlane(k + l);
      }
      if (k + 64 >= bt.B) return -1;
      base += sum;
      int t0, t1, t2, t3;
      w = weight(k + 64 + (threadIdx.x & 63), &t0, &t1, &t2, &t3);
      s = wave_sum_to(w);
      sum = lane_value(s, 63);
    }
  }
  __device__ plan::Seq seq(int b) const {  // one sequence for the wave: scalar values
    if (b < 64)
      return plan::seq_of(sh, __builtin_amdgcn_readlane(q0, b), __builtin_amdgcn_readlane(q1, b),
                          __builtin_amdgcn_readlane(kv, b));
    return plan::seq_of(sh, __builtin_amdgcn_readfirstlane(bt.q_start[b]), __builtin_amdgcn_readfirstlane(bt.q_start[b + 1]),
                        __builtin_amdgcn_readfirstlane(bt.kv_len[b]));
  }
};

// A tile: sequence, head group, place in the group, the weight before it and its own.
struct Tile {
  int b, v, t;
  i64 p, w;
  plan::Seq q;
};
__device__ __forceinline__ bool tile_at(const Order &o, i64 x, Tile *c) {
  i64 before;
  c->b = o.find(x, &before);
  if (c->b < 0) return false;
  c->q = o.seq(c->b);
  const i64 w = plan::head_weight(c->q), y = x - before;
  c->v = __builtin_amdgcn_readfirstlane((int)plan::clamp(plan::div(y, w), 0, o.sh.VH - 1));
  c->t = __builtin_amdgcn_readfirstlane(plan::tile_at(c->q, y - w * c->v));
  c->p = before + w * c->v + plan::before_tile(c->q, c->t);
  c->w = plan::tile_weight(c->q, c->t);
  return true;
}
__device__ __forceinline__ bool next_tile(const Order &o, Tile *c) {
  c->p += c->w;
  if (++c->t == c->q.K) {
    c->t = 0;
    if (++c->v == o.sh.VH) return c->p < o.all && tile_at(o, c->p, c);  // (past any number of sequences without new tokens)
  }
  c->w = plan::tile_weight(c->q, c->t);
  return true;
}

// The same where a workgroup takes a whole tile, in 32 bits: tile x of the batch, *n of them in all (a grid holds no more than
// 2^22; what garbage lengths add up to is clamped).
__device__ __forceinline__ int wave_sum_to(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d);
    v += lane >= d ? u : 0;
  }
  return v;
}
struct Tiles {
  const plan::Shape &sh;
  const Batch &bt;
  int q0, q1, kv, K, upto, all;  // of the first 64 sequences: this lane's, its tiles a head group, tiles up to it; all tiles

  __device__ Tiles(const plan::Shape &s, const Batch &b) : sh(s), bt(b) {
    load(threadIdx.x & 63, &q0, &q1, &kv, &K);
    upto = bt.B == 1 ? __builtin_amdgcn_readfirstlane(K * sh.VH) : wave_sum_to(K * sh.VH);
    all = __builtin_amdgcn_readlane(upto, 63);
    int a, c, d, k;
    for (int i = 64; i < bt.B; i += 64) {
      load(i + (threadIdx.x & 63), &a, &c, &d, &k);
      all += __builtin_amdgcn_readlane(wave_sum_to(k * sh.VH), 63);
    }
  }
  __device__ void load(int b, int *a, int *c, int *n, int *k) const {
    *a = *c = *n = 0;
    if (b < bt.B) {
      *a = bt.q_start[b];
      *c = bt.q_start[b + 1];
      *n = bt.kv_len[b];
    }
    const int lo = min(max(*a, 0), sh.M), hi = min(max(*c, lo), sh.M);
    *k = (hi - lo + sh.TT - 1) / sh.TT;
  }
  __device__ bool tile(int x, Tile *t) const {
    int a = q0, c = q1, n = kv, k = K, s = upto, base = 0;
    for (int i = 0;; i += 64) {
      const unsigned long long m = __ballot(base + s > x);
      if (m) {
        const int l = __builtin_ctzll(m);
        const int kt = __builtin_amdgcn_readlane(k, l);
        const unsigned y = (unsigned)(x - base - (__builtin_amdgcn_readlane(s, l) - kt * sh.VH));
        t->b = i + l;
        t->q = plan::seq_of(sh, __builtin_amdgcn_readlane(a, l), __builtin_amdgcn_readlane(c, l),
                            __builtin_amdgcn_readlane(n, l));
        if (kt < 1) return false;
        t->v = min((int)(y / (unsigned)kt), sh.VH - 1);
        t->t = min((int)(y % (unsigned)kt), kt - 1);
        return true;
      }
      if (i + 64 >= bt.B) return false;
      base += __builtin_amdgcn_readlane(s, 63);
      load(i + 64 + (threadIdx.x & 63), &a, &c, &n, &k);
      s = wave_sum_to(k * sh.VH);
    }
  }
};

// The slice of a workgroup: workgroup b runs on XCD b % 8; each XCD takes a contiguous run of the slices, so that tiles that
// share keys share an L2.
__device__ __forceinline__ int slice_of(int b, int n) {
  const int per = n >> 3, rem = n & 7, xcd = b & 7;
  return (xcd < rem ? xcd * (per + 1) : rem * (per + 1) + (xcd - rem) * per) + (b >> 3);
}

// -- cut tiles ----------------------------------------------------------------------------------------------------------

// The tile that a slice leaves unfinished: its rows (0: there is none), first query row and head, heads per row and those that
// are there, the last key of its first token (what decides whether a row sees any), the slice that finishes it.
struct Left {
  int R, m0, h0, GP, gc, first_last, end, pad;
};
static_assert(sizeof(Left) == plan::LEFT_BYTES, "what the host counts");
__device__ __forceinline__ Left *left_of(const AttnArgs &a, int slice) { return (Left *)a.left + slice; }

// The last slice that has a part of a tile that ends at weight e and begins in slice i.
__device__ __forceinline__ int last_slice(const plan::Cut &cut, int i, i64 e) {
  const int lane = threadIdx.x & 63;
  int n = i + 1;
  for (int in = 64; in == 64; n += in)
    in = __popcll(__ballot(n + lane < cut.n && plan::slice_start(cut, n + lane) < e));
  return n - 1;
}

// A part without key blocks has no outputs: the sign of its sum of 0, and of its factor, says so.
constexpr float NO_PART = -0.0f;

// Joins the parts of cut tiles: o = sum 2^(m_k - m) o_k / sum 2^(m_k - m) l_k. A part whose factor vanishes counts all the
// same: infinities and NaN of its outputs make NaN, as they would if the row had not been cut. Workgroup (j, y): the tile that
// slice j leaves unfinished, rows from 4 RPW y on, RPW a wave; a wave's halves take every other part, 4 channels a lane. It is
// bound by the chain of three loads (the tile, the weights, the outputs), so those of all rows and parts are under way at once.
template <int DG, int T, int RT, int RPW>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnArgs a, int o_stride) {
  const int j = blockIdx.x, lane = threadIdx.x & 63, half = lane >> 5;
  const Left t = *left_of(a, j);
  const int r0 = __builtin_amdgcn_readfirstlane((int)(blockIdx.y * 4 + (threadIdx.x >> 6)) * RPW);
  if (r0 >= t.R) return;
  const int d0 = 4 * (lane & 31), d = min(d0, DG - 4), n = t.end - j + 1;
  auto state = [&](int k) { return a.ws + (size_t)plan::state_of(j + k, k > 0) * (RT * (DG + 2)); };
  float mx[RPW], sum[RPW];
  f32x4 v[RPW];
#pragma unroll
  for (int i = 0; i < RPW; i++) {
    mx[i] = -INFINITY;
    sum[i] = 0.0f;
    v[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int k0 = 0; k0 < n; k0 += 64) {  // 64 parts at a time, one a lane: their weights
    const int parts = min(64, n - k0);
    float2 s[RPW];
    float f[RPW];
#pragma unroll
    for (int i = 0; i < RPW; i++) {
      s[i] = make_float2(-INFINITY, NO_PART);
      if (lane < parts && r0 + i < t.R) s[i] = *(const float2 *)(state(k0 + lane) + RT * DG + 2 * (r0 + i));
    }
#pragma unroll
    for (int i = 0; i < RPW; i++) {
      float top = s[i].x;
#pragma unroll
      for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
      top = fmaxf(top, mx[i]);
      // a sum of 0: nothing was seen (a sum of NaN counts, whatever its maximum)
      const float f0 = sum[i] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(mx[i] - top);
      f[i] = s[i].y == 0.0f ? s[i].y : __builtin_amdgcn_exp2f(s[i].x - top);
      float add = f[i] * s[i].y;
#pragma unroll
      for (int k = 1; k < 64; k *= 2) add += __shfl_xor(add, k);
      mx[i] = top;
      sum[i] = sum[i] * f0 + add;
      v[i] *= f0;
    }
    auto go = [&](auto ahead) {
      constexpr int AHEAD = decltype(ahead)::value;  // loads of a row in flight, of every lane
      for (int k1 = 0; k1 < parts; k1 += 2 * AHEAD) {
        f32x4 u[RPW][AHEAD];
        float fk[RPW][AHEAD];
#pragma unroll
        for (int i = 0; i < RPW; i++)
#pragma unroll
          for (int k = 0; k < AHEAD; k++) {
            const int from = k1 + 2 * k + half;
            fk[i][k] = __shfl(f[i], from);
            u[i][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (from < parts && __builtin_bit_cast(int, fk[i][k]) >= 0)
              u[i][k] = *(const f32x4 *)(state(k0 + from) + (r0 + i) * DG + d);
          }
#pragma unroll
        for (int i = 0; i < RPW; i++)
#pragma unroll
          for (int k = 0; k < AHEAD; k++) v[i] += (k1 + 2 * k + half < parts ? fk[i][k] : 0.0f) * u[i][k];
      }
    };
    if (parts <= 8) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, RPW == 1 ? 16 : 4>{});
  }
#pragma unroll
  for (int i = 0; i < RPW; i++) {
    const int r = r0 + i, rt = (int)((unsigned)r / (unsigned)t.GP), rg = r - rt * t.GP;
    f32x4 x = v[i];
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] += __shfl_xor(x[e], 32);
    // no sum although a key is visible: all scores are -infinity, and 0 / 0
    const float inv = sum[i] != 0.0f ? 1.0f / sum[i] : t.first_last + rt >= 0 ? NAN : 0.0f;
    if (lane < DG / 4 && r < t.R && rg < t.gc)
      store4<T>(a.out + ((size_t)(t.m0 + rt) * o_stride + (size_t)(t.h0 + rg) * DG + d0) * 2, x[0] * inv, x[1] * inv,
                x[2] * inv, x[3] * inv);
  }
}

}  // namespace
}  // namespace h3
