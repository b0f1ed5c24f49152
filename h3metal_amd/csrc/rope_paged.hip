// The per-head norm and rotary embedding of a batch's new queries and keys, written to rows and to a cache's pages in the
// same pass, for gfx950. A row of the input holds Hq query heads, Hk key heads and Hk value heads of HDIM channels ("slots").
//
//   v = x / sqrt(mean(x^2) + eps) * w over a head's channels (queries and keys; with `norm`)
//   pair j of the first `rot` channels, (j, j + rot / 2) or (2 j, 2 j + 1) interleaved, turns by the angle P f_j:
//     (a, b) -> rope_scale (a cos - b sin, b cos + a sin)
//   one rounding, to the type of the queries and the cache; values are rounded and stored as they are
//
// P is pos[m] where positions are given, else the row's place in its sequence, kv_len[b] - n_b + i. The angles' fractions of a
// turn are 64-bit integer products of P and the frequencies' codes (2^-64 turns per position), so they are exact at any
// position; cos and sin are Taylor sums over an eighth of a turn to either side of a quarter (below 2^-24 off). Angles are
// made once per row and workgroup, in LDS.
//
// A lane holds 8 consecutive channels of a slot (16-byte accesses of 16-bit rows) for ROWS rows, all loaded before the first
// is worked on; HDIM / 8 lanes (16 at HDIM 96, 4 of them idle) form a slot, whose sums are DPP steps.
#include "paged.h"

#include <cmath>
#include <cstring>

namespace h3 {
namespace {

enum { PAIR_LANE = 0, PAIR_NEXT = 1, PAIR_ANY = 2 };  // rotary partners: whole lanes apart, side by side, anywhere

constexpr int PL = 8;  // channels per lane

template <int HDIM> struct Slots {
  static constexpr int LPS = HDIM == 64 ? 8 : 16;  // lanes per slot
  static constexpr int SPG = 256 / LPS;            // slots per workgroup
};

struct RopeArgs {
  const char *qkv;
  const float *wq, *wk;
  const unsigned long long *turns;
  char *q, *kc, *vc;
  const int *pos;
};

// Where a row goes: its place in the cache (-1: nowhere), its rotary position, and whether it belongs to a sequence at all.
struct RowAt {
  long long page;  // page of the cache, -1: not stored
  int row, turn, live;
};

template <typename E, int N> struct __attribute__((packed, aligned(sizeof(E)))) Packed { E v[N]; };

// cos and sin of a fraction of a turn in 2^-32: the nearest quarter turn, and an angle within +-pi/4 of it
__device__ __forceinline__ float2 cos_sin(unsigned t) {
  const unsigned quarter = (t + 0x20000000u) >> 30;
  const float x = (float)(int)(t - (quarter << 30)) * 1.46291807926715968e-9f, x2 = x * x;  // 2 pi / 2^32
  const float s = x + x * x2 * (-1.0f / 6 + x2 * (1.0f / 120 + x2 * (-1.0f / 5040 + x2 * (1.0f / 362880))));
  const float c = 1.0f + x2 * (-0.5f + x2 * (1.0f / 24 + x2 * (-1.0f / 720 + x2 * (1.0f / 40320 - x2 * (1.0f / 3628800)))));
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return make_float2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

template <int LPS>
__device__ __forceinline__ float slot_sum(float v) {
  v += xshfl<1>(v);
  v += xshfl<2>(v);
  v += xshfl<4>(v);
  if constexpr (LPS == 16) v += xshfl<8>(v);
  return v;
}
template <int LPS>
__device__ __forceinline__ float slot_max(float v) {
  v = fmaxf(v, xshfl<1>(v));
  v = fmaxf(v, xshfl<2>(v));
  v = fmaxf(v, xshfl<4>(v));
  if constexpr (LPS == 16) v = fmaxf(v, xshfl<8>(v));
  return v;
}

// The sequence of row m and its place, by one wave: sequences that end at or before m are counted 64 at a time.
__device__ __forceinline__ RowAt find_row(int m, const Batch &bt, const int *pos, bool keys) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int k = 0; k < bt.B; k += 64)
    b += __popcll(__ballot(k + lane < bt.B && bt.q_start[k + lane + 1] <= m));
  RowAt r{-1, 0, 0, 0};
  if (b >= bt.B || bt.q_start[b] > m) return r;
  const long long c = (long long)bt.kv_len[b] - bt.q_start[b + 1] + m, pi = c >> bt.lg;
  r.live = 1;
  r.turn = pos ? pos[m] : (int)c;
  if (keys && c >= 0 && pi < bt.width) {
    const int pg = bt.table[(long long)b * bt.width + pi];
    if (pg >= 0 && pg < bt.pages) r.page = pg;
    r.row = (int)(c & ((1 << bt.lg) - 1));
  }
  return r;
}

template <int HDIM, int IT, int OT, int PAIR, int ROWS>
__global__ __launch_bounds__(256) void rope_paged_kernel(RopeArgs a, Batch bt, PagedRopeParams p) {
  using S = Slots<HDIM>;
  using IE = typename PElem<IT>::type;
  using OE = typename PElem<OT>::type;
  __shared__ RowAt at[ROWS];
  __shared__ float2 cs[ROWS][HDIM / 2];
  __shared__ float mix[PAIR == PAIR_ANY ? 256 * PL : 1];
  const int tid = threadIdx.x, l = tid % S::LPS, c0 = l * PL;
  const int slot = blockIdx.y * S::SPG + tid / S::LPS, m0 = blockIdx.x * ROWS;
  const int slots = p.Hq + 2 * p.Hk;
  const bool on = slot < slots && c0 < HDIM, turned = slot < p.Hq + p.Hk;
  const int half = p.rot / 2;

  Packed<IE, PL> x[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; r++)
    if (on && m0 + r < p.M)
      x[r] = *(const Packed<IE, PL> *)((const IE *)a.qkv + (size_t)(m0 + r) * p.in_stride + slot * HDIM + c0);
    else
      for (int i = 0; i < PL; i++) x[r].v[i] = (IE)0.0f;
  float w[PL];
#pragma unroll
  for (int i = 0; i < PL; i++) w[i] = on && turned && p.norm ? (slot < p.Hq ? a.wq : a.wk)[c0 + i] : 1.0f;

  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  for (int r = wave; r < ROWS; r += 4) {
    RowAt f{-1, 0, 0, 0};
    if (m0 + r < p.M) f = find_row(m0 + r, bt, a.pos, p.Hk > 0);
    if ((tid & 63) == 0) at[r] = f;
  }
  __syncthreads();
  for (int i = tid; i < ROWS * half; i += 256) {
    const int r = i / half, j = i - r * half;
    const unsigned long long t = (unsigned long long)(long long)at[r].turn * a.turns[j];
    const float2 f = cos_sin((unsigned)((t + 0x80000000ull) >> 32));
    cs[r][j] = make_float2(f.x * p.rope_scale, f.y * p.rope_scale);
  }
  __syncthreads();

#pragma unroll
  for (int r = 0; r < ROWS; r++) {
    if (m0 + r >= p.M || !at[r].live) continue;  // the same for the whole workgroup
    float v[PL];
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] = (float)x[r].v[i];
    if (p.norm) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < PL; i++) ss = fmaf(v[i], v[i], ss);
      ss = slot_sum<S::LPS>(ss);
      float inv = __builtin_amdgcn_rsqf(ss * (1.0f / HDIM) + p.eps);
      if (__builtin_expect(__any(turned && !(ss > 0x1p-80f && ss < 0x1p+120f)), 0)) {
        // squares that leave a float's range: the row by a power of two that brings its largest value near 1, eps by its
        // square (2^60 at most upwards: below that eps is all of the sum, or 0)
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < PL; i++) top = fmaxf(top, fabsf(v[i]));
        top = slot_max<S::LPS>(top);
        int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
        if (p.eps > 0.0f && e < -60) e = -60;
        float s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < PL; i++) {
          v[i] = turned ? ldexpf(v[i], -e) : v[i];
          s2 = fmaf(v[i], v[i], s2);
        }
        s2 = slot_sum<S::LPS>(s2);
        inv = 1.0f / sqrtf(s2 * (1.0f / HDIM) + ldexpf(p.eps, -2 * e));
      }
      if (turned) {
#pragma unroll
        for (int i = 0; i < PL; i++) v[i] = v[i] * inv * w[i];
      }
    }
    if (PAIR == PAIR_NEXT) {
      if (turned) {
#pragma unroll
        for (int i = 0; i < PL; i += 2) {
          const int j = (c0 + i) / 2;
          if (j < half) {
            const float2 f = cs[r][j];
            const float u = v[i] * f.x - v[i + 1] * f.y, z = v[i + 1] * f.x + v[i] * f.y;
            v[i] = u;
            v[i + 1] = z;
          }
        }
      }
    } else if (PAIR == PAIR_LANE) {
      // half is a multiple of 8: a lane's channels are all in the first or the second half, its partner half / 8 lanes off
      const int hl = half / PL, low = l < hl, pl = low ? l + hl : l - hl;
      const bool in = turned && c0 < p.rot;
      float u[PL];
#pragma unroll
      for (int i = 0; i < PL; i++) u[i] = __shfl(v[i], c0 < p.rot ? pl : l, S::LPS);
      if (in) {
#pragma unroll
        for (int i = 0; i < PL; i++) {
          const float2 f = cs[r][low ? c0 + i : c0 + i - half];
          v[i] = v[i] * f.x + (low ? -u[i] : u[i]) * f.y;
        }
      }
    } else {
      float *mine = mix + tid / S::LPS * (S::LPS * PL);
#pragma unroll
      for (int i = 0; i < PL; i++) mine[c0 + i] = v[i];
      __syncthreads();
      if (turned) {
#pragma unroll
        for (int i = 0; i < PL; i++) {
          const int c = c0 + i;
          if (c < p.rot) {
            const bool low = c < half;
            const float2 f = cs[r][low ? c : c - half];
            const float u = mine[low ? c + half : c - half];
            v[i] = v[i] * f.x + (low ? -u : u) * f.y;
          }
        }
      }
      __syncthreads();
    }
    Packed<OE, PL> o;
#pragma unroll
    for (int i = 0; i < PL; i++) o.v[i] = (OE)v[i];
    if (!on) continue;
    if (slot < p.Hq) {
      *(Packed<OE, PL> *)((OE *)a.q + (size_t)(m0 + r) * p.q_stride + slot * HDIM + c0) = o;
    } else if (at[r].page >= 0) {
      const int h = slot - p.Hq - (turned ? 0 : p.Hk);
      const size_t to = (((size_t)at[r].page * p.Hk + h) * p.page + at[r].row) * HDIM + c0;
      *(Packed<OE, PL> *)((OE *)(turned ? a.kc : a.vc) + to) = o;
    }
  }
}

template <int HDIM, int IT, int OT, int PAIR>
void run(const Exec &ex, const RopeArgs &a, const Batch &bt, const PagedRopeParams &p) {
  const int slots = p.Hq + 2 * p.Hk, ny = (slots + Slots<HDIM>::SPG - 1) / Slots<HDIM>::SPG;
  constexpr int ROWS = 8;
  hipLaunchKernelGGL((rope_paged_kernel<HDIM, IT, OT, PAIR, ROWS>), dim3((unsigned)((p.M + ROWS - 1) / ROWS), (unsigned)ny),
                     dim3(256), 0, ex.stream, a, bt, p);
}

template <int HDIM, int IT, int OT>
int launch(const Pipeline &pl, const Exec &ex, const Arg *a, int nargs, const void *params, uint32_t params_len,
           std::string *err) {
  const bool inter = pl.ival[0] != 0;
  if (params_len != sizeof(PagedRopeParams)) {
    *err = "parameter block of " + std::to_string(params_len) + " bytes, expected " + std::to_string(sizeof(PagedRopeParams));
    return -1;
  }
  PagedRopeParams p;
  memcpy(&p, params, sizeof p);
  const int lg = log2_page(p.page);
  if (p.M < 0 || p.M >= 1 << 24 || p.B < 0 || p.B >= 1 << 24 || p.Hq < 0 || p.Hk < 0 || p.Hq > 4096 || p.Hk > 4096 ||
      p.Hq + p.Hk < 1 || p.in_stride < (p.Hq + 2 * p.Hk) * HDIM || p.q_stride < p.Hq * HDIM) {
    *err = "bad shape: M " + std::to_string(p.M) + " B " + std::to_string(p.B) + " (below 2^24) heads " +
           std::to_string(p.Hq) + "/" + std::to_string(p.Hk) + " (up to 4096) in_stride " + std::to_string(p.in_stride) +
           " q_stride " + std::to_string(p.q_stride);
    return -1;
  }
  if (p.Hk && (lg < 0 || p.pages < 0 || p.width < 0)) {
    *err = "bad cache: " + std::to_string(p.pages) + " pages of " + std::to_string(p.page) +
           " rows (a power of two from 16 to 256), " + std::to_string(p.width) + " in a row of the table";
    return -1;
  }
  if (p.rot < 0 || p.rot > HDIM || p.rot % 2) {
    *err = "rot " + std::to_string(p.rot) + " must be even and at most the head's " + std::to_string(HDIM) + " channels";
    return -1;
  }
  if ((p.norm && !(p.eps >= 0.0f && std::isfinite(p.eps))) || !std::isfinite(p.rope_scale)) {
    *err = "eps must be finite and not negative, rope_scale finite";
    return -1;
  }
  if (nargs < 11) {
    *err = "expected buffers qkv, wq, wk, turns, Q, kc, vc, table, q_start, kv_len, pos";
    return -1;
  }
  if (p.M == 0 || p.B == 0) return 0;
  const uint64_t ie = IT == P_F32 ? 4 : 2, width = p.Hk ? (uint64_t)p.width : 0;
  const uint64_t need[11] = {((uint64_t)(p.M - 1) * p.in_stride + (uint64_t)(p.Hq + 2 * p.Hk) * HDIM) * ie,
                             p.norm && p.Hq ? HDIM * 4ull : 0,
                             p.norm && p.Hk ? HDIM * 4ull : 0,
                             (uint64_t)p.rot / 2 * 8,
                             p.Hq ? ((uint64_t)(p.M - 1) * p.q_stride + (uint64_t)p.Hq * HDIM) * 2 : 0,
                             p.Hk ? (uint64_t)p.pages * p.Hk * p.page * HDIM * 2 : 0,
                             p.Hk ? (uint64_t)p.pages * p.Hk * p.page * HDIM * 2 : 0,
                             (uint64_t)p.B * width * 4,
                             ((uint64_t)p.B + 1) * 4,
                             (uint64_t)p.B * 4,
                             a[10].ptr ? (uint64_t)p.M * 4 : 0};
  static const char *what[11] = {"qkv", "wq", "wk", "turns", "Q", "kc", "vc", "table", "q_start", "kv_len", "pos"};
  const int align[11] = {(int)ie, 4, 4, 8, 2, 16, 16, 4, 4, 4, 4};
  for (int i = 0; i < 11; i++)
    if (need[i] && !paged_fits(a, i, need[i], align[i], what[i], err)) return -1;
  for (int o : {4, 5, 6})
    for (int i = 0; i < 11; i++)
      if (i != o && paged_overlap(a[o], need[o], a[i], need[i])) {
        *err = std::string(what[o]) + " shares memory with " + what[i];
        return -1;
      }
  const RopeArgs g{a[0].ptr, (const float *)a[1].ptr, (const float *)a[2].ptr, (const unsigned long long *)a[3].ptr,
                   a[4].ptr, a[5].ptr, a[6].ptr, (const int *)a[10].ptr};
  const Batch bt{(const int *)a[7].ptr, (const int *)a[8].ptr, (const int *)a[9].ptr, p.B, (int)width, p.Hk ? p.pages : 0,
                 p.Hk ? lg : 4};
  if (inter) run<HDIM, IT, OT, PAIR_NEXT>(ex, g, bt, p);
  else if (p.rot / 2 % PL == 0) run<HDIM, IT, OT, PAIR_LANE>(ex, g, bt, p);
  else run<HDIM, IT, OT, PAIR_ANY>(ex, g, bt, p);
  return 0;
}

template <int HDIM>
LaunchFn pick(int it, int ot) {
  if (ot == P_BF16)
    return it == P_BF16 ? launch<HDIM, P_BF16, P_BF16> : it == P_F16 ? launch<HDIM, P_F16, P_BF16> : launch<HDIM, P_F32, P_BF16>;
  return it == P_BF16 ? launch<HDIM, P_BF16, P_F16> : it == P_F16 ? launch<HDIM, P_F16, P_F16> : launch<HDIM, P_F32, P_F16>;
}

}  // namespace

// Macros: HDIM (64, 96 or 128), IN_T (half | bfloat | float), OUT_T (half | bfloat: the queries and the cache), INTER (1:
// rotary pairs side by side).
bool make_qk_norm_rope_paged(const Macros &m, Pipeline *pl, std::string *err) {
  int hd, inter;
  if (!macro_int(m, "HDIM", 128, &hd, err) || !macro_int(m, "INTER", 0, &inter, err)) return false;
  for (auto &kv : m)
    if (kv.first != "HDIM" && kv.first != "INTER" && kv.first != "IN_T" && kv.first != "OUT_T") {
      *err = "unknown macro " + kv.first;
      return false;
    }
  const int it = paged_type(macro_str(m, "IN_T", "bfloat")), ot = paged_type(macro_str(m, "OUT_T", "bfloat"));
  if (it < 0 || (ot != P_BF16 && ot != P_F16)) {
    *err = "IN_T must be half|bfloat|float, OUT_T half|bfloat";
    return false;
  }
  if (hd != 64 && hd != 96 && hd != 128) {
    *err = "HDIM " + std::to_string(hd) + " not supported (64, 96 or 128)";
    return false;
  }
  pl->launch = hd == 128 ? pick<128>(it, ot) : hd == 96 ? pick<96>(it, ot) : pick<64>(it, ot);
  pl->ival[0] = inter != 0;
  pl->threads = 256;
  return true;
}

}  // namespace h3
