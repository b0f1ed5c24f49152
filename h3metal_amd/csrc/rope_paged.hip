// The per-head norm and rotary embedding of a batch's new queries and keys, written to rows and to a cache's pages in the
// same pass, for gfx950. A row of the input holds Hq query heads, Hk key heads and Hk value heads of HDIM channels ("slots").
//
//   v = x / sqrt(mean(x^2) + eps) * w over a head's channels (queries and keys; with `norm`)
//   pair j of the first `rot` channels, (j, j + rot / 2) or (2 j, 2 j + 1) interleaved, turns by the angle P f_j:
//     (a, b) -> rope_scale (a cos - b sin, b cos + a sin)
//   one rounding, to the type of the queries and the cache; values are rounded and stored as they are
//
// P is pos[m] where positions are given, else the row's place in its sequence, kv_len[b] - n_b + i. The angles' fractions of a
// turn are 64-bit integer products of P and the frequencies' codes (2^-64 turns per position): no position adds an error to
// the codes', which are float64 quotients (at 2^31 positions an angle is some 2^-25 turns off). cos and sin are Taylor sums
// over an eighth of a turn to either side of a quarter: cut off below 2^-24, and with their float steps within 2 x 2^-24. Angles
// are made once per row and workgroup, in LDS.
//
// A lane holds 8 consecutive channels of a slot (16-byte accesses of 16-bit rows) for ROWS rows, all loaded before the first
// is worked on; HDIM / 8 lanes (16 at HDIM 96, 4 of them idle) form a slot, whose sums are DPP steps. Bound by HBM: 8192 rows of
// 32 + 8 + 8 heads of 128 in 33 us from an idle card (6.1 TB/s), 43 among other calls (4.7; a plain copy reaches 4.9).
#include "paged.h"

#include <cmath>
#include <cstring>
#include <type_traits>


namespace h3 {
namespace {

// rotary partners: whole lanes apart, side by side, anywhere, the lanes of the other half (all of a head of 64 or 128)
enum { PAIR_LANE = 0, PAIR_NEXT = 1, PAIR_ANY = 2, PAIR_ALL = 3 };

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

// 16 bytes of a row, whose rows are aligned to their elements only
typedef unsigned Piece __attribute__((ext_vector_type(4), aligned(2)));

template <int T>
__device__ __forceinline__ void load8(float (&v)[PL], const Piece (&x)[T == P_F32 ? 2 : 1]) {
  if constexpr (T == P_F32) {
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] = __builtin_bit_cast(float, (unsigned)x[i / 4][i & 3]);
  } else if constexpr (T == P_BF16) {
#pragma unroll
    for (int i = 0; i < PL; i += 2) {
      v[i] = __builtin_bit_cast(float, (unsigned)x[0][i / 2] << 16);
      v[i + 1] = __builtin_bit_cast(float, (unsigned)x[0][i / 2] & 0xFFFF0000u);
    }
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < PL; i += 2) {
      const f16x2 h = __builtin_bit_cast(f16x2, (unsigned)x[0][i / 2]);
      v[i] = (float)h[0];
      v[i + 1] = (float)h[1];
    }
  }
}
template <int T>
__device__ __forceinline__ Piece pack8(const float (&v)[PL]) {
  using E = typename PElem<T>::type;
  typedef E E2 __attribute__((ext_vector_type(2)));
  Piece o;
#pragma unroll
  for (int i = 0; i < PL; i += 2) o[i / 2] = __builtin_bit_cast(unsigned, E2{(E)v[i], (E)v[i + 1]});
  return o;
}

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

// Where rows go, by one wave, a row a lane: the rotary position, and the row of the cache, pages counted through (-1: not
// stored; -2: the row is of no sequence).
struct RowsAt {
  long long to;
  int turn;
};
template <int ROWS>
__device__ __forceinline__ RowsAt find_rows(int m0, int M, const Batch &bt, const int *pos, bool keys) {
  const int lane = threadIdx.x & 63, m = m0 + lane;
  int b = 0;  // sequences that end at or before the row, counted 64 at a time
  if (bt.B == 1) {
    b = bt.q_start[1] <= m;
  } else {
    for (int k = 0; k < bt.B; k += 64) {
      const int end = k + lane < bt.B ? bt.q_start[k + lane + 1] : 0x7fffffff;
#pragma unroll
      for (int r = 0; r < ROWS; r++) {
        const int n = __popcll(__ballot(end <= m0 + r));
        b += lane == r ? n : 0;
      }
    }
  }
  RowsAt at{-2, 0};
  if (lane >= ROWS || m >= M || b >= bt.B) return at;
  const int first = bt.q_start[b], end = bt.q_start[b + 1], n = bt.kv_len[b], given = pos ? pos[m] : 0;
  if (first > m || end <= m) return at;
  const long long c = (long long)n - end + m, pi = c >> bt.lg;
  at.to = -1;
  at.turn = pos ? given : (int)c;
  if (keys && c >= 0 && pi < bt.width) {
    const int pg = bt.table[(long long)b * bt.width + pi];
    if (pg >= 0 && pg < bt.pages) at.to = ((long long)pg << bt.lg) + (c & ((1 << bt.lg) - 1));
  }
  return at;
}

template <int HDIM, int IT, int OT, int PAIR, int ROWS>
__global__ __launch_bounds__(256) void rope_paged_kernel(RopeArgs a, Batch bt, PagedRopeParams p) {
  using S = Slots<HDIM>;
  constexpr int IB = IT == P_F32 ? 4 : 2, NP = IB / 2;  // bytes of an element, pieces of a lane's channels
  __shared__ __attribute__((aligned(16))) float2 cs[ROWS][HDIM / 2];
  __shared__ float mix[PAIR == PAIR_ANY ? 256 * PL : 1];
  const int tid = threadIdx.x, l = tid % S::LPS, c0 = l * PL;
  const int slot = blockIdx.y * S::SPG + tid / S::LPS, m0 = blockIdx.x * ROWS;
  const int slots = p.Hq + 2 * p.Hk;
  const bool on = slot < slots && c0 < HDIM, turned = slot < p.Hq + p.Hk;
  const int half = p.rot / 2;

  Piece x[ROWS][NP];  // (rows and slots past the last ones read the last again)
  {
    const char *from = a.qkv + ((size_t)min(slot, slots - 1) * HDIM + min(c0, HDIM - PL)) * IB;
#pragma unroll
    for (int r = 0; r < ROWS; r++)
#pragma unroll
      for (int k = 0; k < NP; k++)
        x[r][k] = *(const Piece *)(from + (size_t)min(m0 + r, p.M - 1) * p.in_stride * IB + 16 * k);
  }
  float w[PL];
#pragma unroll
  for (int i = 0; i < PL; i++) w[i] = 1.0f;
  if (p.norm && turned && c0 < HDIM) {
    const float *from = (slot < p.Hq ? a.wq : a.wk) + c0;
#pragma unroll
    for (int i = 0; i < PL; i++) w[i] = from[i];
  }

  const RowsAt at = find_rows<ROWS>(m0, p.M, bt, a.pos, p.Hk > 0);
  for (int i = tid; i < ROWS * HDIM / 2; i += 256) {
    const int r = i / (HDIM / 2), j = i - r * (HDIM / 2);
    const int turn = __shfl(at.turn, r);
    if (j < half) {
      const unsigned long long t = (unsigned long long)(long long)turn * a.turns[j];
      const float2 f = cos_sin((unsigned)((t + 0x80000000ull) >> 32));
      cs[r][j] = make_float2(f.x * p.rope_scale, f.y * p.rope_scale);
    }
  }
  __syncthreads();

#pragma unroll
  for (int r = 0; r < ROWS; r++) {
    const long long to = (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)at.to, r) |
                                     (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(at.to >> 32), r) << 32);
    if (to == -2) continue;  // the same for the whole workgroup
    float v[PL];
    load8<IT>(v, x[r]);
    if (HDIM == 96 && c0 >= HDIM) {  // idle lanes of a slot
#pragma unroll
      for (int i = 0; i < PL; i++) v[i] = 0.0f;
    }
    if (p.norm) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < PL; i++) ss = fmaf(v[i], v[i], ss);
      ss = slot_sum<S::LPS>(ss);
      float inv = __builtin_amdgcn_rsqf(ss * (1.0f / HDIM) + p.eps);
      const bool out = turned && !(ss > 0x1p-80f && ss < 0x1p+120f);
      if (__builtin_expect(__any(out), 0)) {
        // squares that leave a float's range: the head by a power of two that brings its largest value near 1, eps by its
        // square (2^60 at most upwards: below that eps is all of the sum, or 0). The wave's other heads keep what they have.
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < PL; i++) top = fmaxf(top, fabsf(v[i]));
        top = slot_max<S::LPS>(top);
        int e = top > 0.0f && top < INFINITY ? ilogbf(top) : 0;
        if (p.eps > 0.0f && e < -60) e = -60;
        float s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < PL; i++) {
          v[i] = out ? ldexpf(v[i], -e) : v[i];
          s2 = fmaf(v[i], v[i], s2);
        }
        s2 = slot_sum<S::LPS>(s2);
        inv = out ? 1.0f / sqrtf(s2 * (1.0f / HDIM) + ldexpf(p.eps, -2 * e)) : inv;
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
    } else if (PAIR == PAIR_ALL) {
      if (turned) {
        const bool low = l < S::LPS / 2;
        float2 f[PL];
#pragma unroll
        for (int i = 0; i < PL; i += 2)
          *(float4 *)&f[i] = *(const float4 *)&cs[r][(low ? c0 : c0 - HDIM / 2) + i];
#pragma unroll
        for (int i = 0; i < PL; i++) {
          const float u = xshfl<S::LPS / 2>(v[i]);
          v[i] = v[i] * f[i].x + (low ? -u : u) * f[i].y;
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
    if (!on) continue;
    char *dst;
    if (slot < p.Hq) {
      dst = a.q + ((size_t)(m0 + r) * p.q_stride + slot * HDIM + c0) * 2;
    } else {
      if (to < 0) continue;
      const int h = slot - p.Hq - (turned ? 0 : p.Hk);
      const size_t row = ((((size_t)to >> bt.lg) * p.Hk + h) << bt.lg) + ((size_t)to & ((1 << bt.lg) - 1));
      dst = (turned ? a.kc : a.vc) + (row * HDIM + c0) * 2;
    }
    *(Piece *)dst = pack8<OT>(v);
  }
}

template <int HDIM, int IT, int OT, int PAIR>
void run(const Exec &ex, const RopeArgs &a, const Batch &bt, const PagedRopeParams &p) {
  const int slots = p.Hq + 2 * p.Hk, ny = (slots + Slots<HDIM>::SPG - 1) / Slots<HDIM>::SPG;
  // Rows a workgroup: more share its angles, fewer share the chain of its loads (heads 32 + 8 + 8, us with 1, 2, 4 and 8 rows: 64
  // single tokens 3.6, 4.2, 5.4, 7.3; 2048 rows 12.9, 12.0, 12.0, 12.1; 8192 rows 37.7, 32.7, 33.8, 37.9).
  constexpr int ROWS = 2;
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
  else if (HDIM != 96 && p.rot == HDIM) run<HDIM, IT, OT, PAIR_ALL>(ex, g, bt, p);
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
