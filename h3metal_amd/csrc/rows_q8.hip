// Row kernels that make the 8-bit inputs of the matrix products, for gfx950:
//
//  rms_norm_q8: h = res + x, rounded once to the residual's type and stored (or h = x without a residual);
//    v = h / sqrt(mean(h^2) + eps) * w (v = h * w without the norm), and v in 8 bits:
//    * e4m3 codes with a float scale for each row and block of 128 columns (the last one may be short):
//      s = amax|v| / 448 (1 where amax is 0), code = e4m3(v / s), round to nearest even;
//    * or int8 codes with one scale a row: s = amax|v| / 127, code = rint(v / s).
//  swiglu_f8: v = value * gate / (1 + exp(-gate)) in e4m3, value in columns 0 .. D-1 and gate in D .. 2D-1 of a row (as
//    rot_q8's mode 1).
//
// amax passes over NaN; the code of NaN is NaN (e4m3) or 0 (int8). A block that holds an infinity has an infinite scale
// and NaN at the infinity; with the norm, whose root is then infinite, its scale is NaN and the row's other scales are 0.
//
// Range. Sums, maxima and products are float. A row of rms_norm_q8 whose squares' sum or whose largest products (a block's,
// for int8 the row's) pass out of 2^-100 .. the largest float is taken again in double, so any finite row and gain have the
// codes and scales of the formula; an amax below the smallest float counts as 0. An int8 row of zeros takes that path too.
// swiglu_f8's products stay floats: one past the largest is infinite, and of a gate below 2^-126 bits are lost.
//
// The row's root mean square R scales every value of a block and its amax alike, so v / s = (h w) 448 / amax|h w| does
// not need it: the codes of a block are written at once and only the scales wait for the row's sum. So a row takes one
// pass, is never held (e4m3), and may have any length.
#include "h3hip_internal.h"

#include <cmath>
#include <cstring>

namespace h3 {
namespace {

enum { T_NONE = 0, T_BF16 = 1, T_F16 = 2, T_F32 = 3 };

template <int T> struct Elem;
template <> struct Elem<T_BF16> { using type = __bf16; };
template <> struct Elem<T_F16> { using type = _Float16; };
template <> struct Elem<T_F32> { using type = float; };
template <> struct Elem<T_NONE> { using type = float; };

constexpr int FB = 128;  // columns of a block
constexpr int PL = 8;    // columns of a lane: 16 lanes hold a block
constexpr float F8_MAX = 448.0f;

// 8 values from p, which is aligned to its element only (gfx950 loads 16 bytes from any address); those from column n
// on are 0
template <typename E>
__device__ __forceinline__ void load8(float (&v)[PL], const E *p, int n) {
  typedef E V __attribute__((ext_vector_type(PL), aligned(sizeof(E))));
  if (n >= PL) {
    const V x = *(const V *)p;
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] = (float)x[i];
  } else {
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] = i < n ? (float)p[i] : 0.0f;
  }
}
template <typename E>
__device__ __forceinline__ void store8(E *p, const E (&v)[PL], int n) {
  typedef E V __attribute__((ext_vector_type(PL), aligned(sizeof(E))));
  if (n >= PL) {
    V x;
#pragma unroll
    for (int i = 0; i < PL; i++) x[i] = v[i];
    *(V *)p = x;
  } else {
#pragma unroll
    for (int i = 0; i < PL; i++)
      if (i < n) p[i] = v[i];
  }
}

// The largest of 16 neighbouring lanes' values, in each of them
__device__ __forceinline__ float max16(float m) {
  m = fmaxf(m, xshfl<8>(m));
  m = fmaxf(m, xshfl<4>(m));
  m = fmaxf(m, xshfl<2>(m));
  return fmaxf(m, xshfl<1>(m));
}

// The largest of LPR neighbouring lanes' values (LPR at most 64), in each of them
template <int LPR>
__device__ __forceinline__ float max_of(float m) {
  if constexpr (LPR > 32) m = fmaxf(m, __shfl_xor(m, 32));
  if constexpr (LPR > 16) m = fmaxf(m, xshfl<16>(m));
  return max16(m);
}
template <int LPR>
__device__ __forceinline__ float sum_of(float m) {
  if constexpr (LPR > 32) m += __shfl_xor(m, 32);
  m += xshfl<16>(m);
  m += xshfl<8>(m);
  m += xshfl<4>(m);
  m += xshfl<2>(m);
  return m + xshfl<1>(m);
}

// The scale s = m / most of values whose largest magnitude is m (1 where m is 0), and 1 / (s up): values below 2^-100 are
// scaled by `up` before their product with it, which would overflow.
struct Scale {
  float s, inv, up;
};
template <int MOST>
__device__ __forceinline__ Scale scale_of(float m) {
  const float up = m < 0x1p-100f && m > 0.0f ? 0x1p64f : 1.0f;
  const float s = m > 0.0f ? m * up * (1.0f / MOST) : 1.0f;  // a normal float, and so is its reciprocal
  const float r = __builtin_amdgcn_rcpf(s);
  // one Newton step; infinity's 0 stays
  return {m > 0.0f ? m * (1.0f / MOST) : 1.0f, __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r), s, 1.0f), up};
}

__device__ __forceinline__ uint2 pack_f8(const float (&y)[PL]) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return make_uint2((unsigned)lo, (unsigned)hi);
}

// Whether y, a quotient within 8 * 2^-24, may round to another e4m3 value than the exact one: its 20 dropped mantissa bits
// are near one half, or it is a subnormal code's (whose dropped bits are more).
__device__ __forceinline__ bool near_tie(float y) {
  const unsigned u = __builtin_bit_cast(unsigned, y) & 0x7fffffffu;
  return ((u + 8 - 0x80000u) & 0xfffffu) <= 16 || u - 1 < 0x3c800000u - 1;
}

// x in float, rounded to odd: a further rounding to few bits then gives what rounding x itself gives
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  if ((double)f == x || x != x) return f;
  unsigned u = __builtin_bit_cast(unsigned, f);
  if (fabs((double)f) > fabs(x)) u--;
  return __builtin_bit_cast(float, u | 1);
}

__device__ __forceinline__ void store_codes(unsigned char *p, uint2 c, int n) {
  typedef unsigned V __attribute__((ext_vector_type(2), aligned(1)));
  if (n >= PL) {
    V x = {c.x, c.y};
    *(V *)p = x;
  } else {
#pragma unroll
    for (int i = 0; i < PL; i++)
      if (i < n) p[i] = (unsigned char)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
  }
}

// The sum, or with MOST the largest, of LPR neighbouring lanes' values (LPR 256: of the workgroup's, through red), in each
template <int LPR, bool MOST>
__device__ __forceinline__ double over_row(double v, double *red) {
  auto join = [](double a, double b) { return MOST ? fmax(a, b) : a + b; };
#pragma unroll
  for (int k = (LPR < 64 ? LPR : 64) / 2; k > 0; k >>= 1) v = join(v, __shfl_xor(v, k));
  if constexpr (LPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = join(join(red[0], red[1]), join(red[2], red[3]));
  }
  return v;
}

// a + b in float, rounded to odd. The sum of a 16-bit residual and a float has more bits than a float, whose rounding may make a
// tie of what the residual's type would round up or down (1 + (2^-8 + 2^-30) to bf16). So may a half's sum with bf16, which has
// fewer bits. Other pairs do not need it: neither value has a bit that is half a step of their sum next to values that far below.
__device__ __forceinline__ float sum_to_odd(float a, float b) {
  const float s = a + b, t = s - a, e = (a - (s - t)) + (b - t);  // s + e is the sum, exactly
  unsigned u = __builtin_bit_cast(unsigned, s);
  if (e != 0.0f && fabsf(e) < INFINITY) {  // (the largest floats' sums: e may be NaN, and s is infinite in any 16-bit type)
    if ((e < 0.0f) != (s < 0.0f)) u -= !(u & 1);
    u |= 1;
  }
  return __builtin_bit_cast(float, u);
}

// Whether s may be the middle of two values of type T: only then does a bit that the float sum lost decide (rounding every sum
// to odd: 16896 x 4096 floats into a bf16 residual 127 us, 120 so).
template <int T>
__device__ __forceinline__ bool maybe_tie(float s) {
  const unsigned u = __builtin_bit_cast(unsigned, s);
  return T == T_BF16 ? (u & 0xffffu) == 0x8000u : (u & 0xfffu) == 0;  // (half: those of the subnormal ones too)
}

// Floats from here on keep their products' and squares' sums exact to a float's steps: the square of what is lost below is
// nothing beside it.
constexpr float LOW = 0x1p-100f;

struct NormArgs {
  const char *x, *res;
  const float *w;
  unsigned char *out;
  float *scale;
  char *res_out;
};

// LPR lanes a row: 256 / LPR rows a workgroup. The e4m3 codes are the exactly rounded ones: where a float quotient is near a
// tie or a subnormal code's (5% of the waves' steps on normal rows, 12% where every 64th column is 8 times larger), its
// products and the largest of them are taken again in double.
template <int XT, int RT, bool I8, int LPR>
__global__ __launch_bounds__(256) void rms_norm_q8_kernel(NormArgs a, NormQ8Params p) {
  using XE = typename Elem<XT>::type;
  using RE = typename Elem<RT>::type;
  constexpr int STEP = LPR * PL, HELD = I8 ? 4 : 1;  // int8: this many steps of a row stay in registers until its amax is known
  extern __shared__ float tops[];  // e4m3: the blocks' largest magnitudes
  __shared__ float red[8];
  __shared__ double red2[8];
  const int tid = threadIdx.x, lane = tid % LPR, wave = tid >> 6;
  const int nb = (p.D + FB - 1) / FB, end = nb * FB;
  size_t m = (size_t)blockIdx.x * (256 / LPR) + tid / LPR;
  const bool there = m < (size_t)p.M;
  if (LPR > 64 && !there) return;
  m = there ? m : p.M - 1;  // (lanes past the last row go along with it and write nothing)
  const XE *xr = (const XE *)a.x + m * p.x_stride;
  const RE *rr = (const RE *)a.res + m * p.r_stride;
  RE *ro = (RE *)a.res_out + m * p.ro_stride;
  unsigned char *out = a.out + m * p.o_stride;
  float *top = tops + tid / LPR * nb;

  // h of 8 columns; the first time the sum is made and stored
  auto load = [&](int c, float (&h)[PL]) __attribute__((always_inline)) {
    const int n = p.D - c;
    load8(h, xr + c, n);
    if constexpr (RT != T_NONE) {
      float r[PL];
      load8(r, rr + c, n);
      float t[PL];
      RE s[PL];
#pragma unroll
      for (int i = 0; i < PL; i++) t[i] = r[i] + h[i];
      if constexpr ((XT == T_F32 && RT != T_F32) || (XT == T_F16 && RT == T_BF16)) {
        bool tie = false;
#pragma unroll
        for (int i = 0; i < PL; i++) tie |= maybe_tie<RT>(t[i]);
        if (tie)
#pragma unroll
          for (int i = 0; i < PL; i++) t[i] = sum_to_odd(r[i], h[i]);
      }
#pragma unroll
      for (int i = 0; i < PL; i++) {
        s[i] = (RE)t[i];
        h[i] = (float)s[i];
      }
      if (there) store8(ro + c, s, n);
    }
  };
  auto reload = [&](int c, float (&h)[PL]) __attribute__((always_inline)) {
    if constexpr (RT != T_NONE) load8(h, (const RE *)ro + c, p.D - c);
    else load8(h, xr + c, p.D - c);
  };
  auto gain = [&](int c, float (&g)[PL]) __attribute__((always_inline)) {
    if (a.w) {
      load8(g, a.w + c, p.D - c);
    } else {
#pragma unroll
      for (int i = 0; i < PL; i++) g[i] = 1.0f;
    }
  };

  float sq = 0.0f, rowmax = 0.0f, held[HELD][PL];
  auto step = [&](int c, float (&t)[PL]) __attribute__((always_inline)) {
    float h[PL], g[PL];
    load(c, h);
    gain(c, g);
    float mx = 0.0f;
#pragma unroll
    for (int i = 0; i < PL; i++) {
      sq = __builtin_fmaf(h[i], h[i], sq);
      t[i] = h[i] * g[i];
      mx = fmaxf(mx, fabsf(t[i]));
    }
    if constexpr (!I8) {
      mx = max16(mx);
      const Scale v = scale_of<448>(mx);
      float y[PL];
      const bool out_of_range = !(mx >= LOW && mx < INFINITY);
      bool tie = out_of_range;
#pragma unroll
      for (int i = 0; i < PL; i++) {
        y[i] = t[i] * v.inv;
        tie |= near_tie(y[i]);
      }
      if (__any(tie)) {
        double d[PL], dm = 0.0;
#pragma unroll
        for (int i = 0; i < PL; i++) {
          d[i] = (double)h[i] * g[i];
          dm = fmax(dm, fabs(d[i]));
        }
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) dm = fmax(dm, __shfl_xor(dm, k));
        // (float quotients of zeros, NaN and infinities are as they should be)
        if (out_of_range) {
          if (dm > 0.0 && dm < (double)INFINITY) sq = INFINITY;  // the row again
        } else
#pragma unroll
          for (int i = 0; i < PL; i++) y[i] = to_odd(d[i] * (double)F8_MAX / dm);
      }
      if (there) store_codes(out + c, pack_f8(y), p.D - c);
      if ((lane & 15) == 0) top[c / FB] = mx;
    }
    rowmax = fmaxf(rowmax, mx);
  };
  int c = lane * PL;
  if constexpr (I8) {
#pragma unroll
    for (int k = 0; k < HELD; k++)
      if (c + k * STEP < end) step(c + k * STEP, held[k]);
    c += HELD * STEP;
  }
  for (; c < end; c += STEP) {
    float t[PL];
    step(c, t);
  }
  sq = sum_of<LPR < 64 ? LPR : 64>(sq);
  if constexpr (I8) rowmax = max_of<LPR < 64 ? LPR : 64>(rowmax);
  if constexpr (LPR > 64) {
    if ((tid & 63) == 0) red[wave] = sq, red[4 + wave] = rowmax;
    __syncthreads();
    sq = (red[0] + red[1]) + (red[2] + red[3]);
    rowmax = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
  } else {
    __syncthreads();  // the blocks' largest magnitudes are there
  }
  const float ms = sq / (float)p.D + p.eps;
  if (!(sq < INFINITY) || (p.norm && ms < LOW) || (I8 && !(rowmax >= LOW && rowmax < INFINITY))) {
    double s2 = 0.0, t2 = 0.0;
    for (c = lane * PL; c < end; c += STEP) {
      float h[PL], g[PL];
      reload(c, h);
      gain(c, g);
#pragma unroll
      for (int i = 0; i < PL; i++) {
        s2 = __builtin_fma((double)h[i], (double)h[i], s2);
        if constexpr (I8) t2 = fmax(t2, fabs((double)h[i] * g[i]));
      }
    }
    s2 = over_row<LPR, false>(s2, red2);
    if constexpr (I8) t2 = over_row<LPR, true>(t2, red2 + 4);
    constexpr double CODES = I8 ? 127.0 : (double)F8_MAX;
    const double r = p.norm ? 1.0 / sqrt(s2 / p.D + p.eps) : 1.0;
    for (c = lane * PL; c < end; c += STEP) {
      float h[PL], g[PL];
      double d[PL], most = t2;
      reload(c, h);
      gain(c, g);
#pragma unroll
      for (int i = 0; i < PL; i++) {
        d[i] = (double)h[i] * g[i];
        if constexpr (!I8) most = fmax(most, fabs(d[i]));
      }
      if constexpr (!I8)
#pragma unroll
        for (int k = 8; k > 0; k >>= 1) most = fmax(most, __shfl_xor(most, k));
      // a largest value below the smallest float is 0 (unless an infinite root made it so)
      const bool none = !(most > 0.0) || (r > 0.0 && most * r < 0x1p-149), some = !none && most < (double)INFINITY;
#pragma unroll
      for (int i = 0; i < PL; i++) d[i] = some ? d[i] * CODES / most : d[i] * 0.0;  // NaN and infinities: NaN
      if constexpr (I8) {
        unsigned char q[PL];
#pragma unroll
        for (int i = 0; i < PL; i++) q[i] = d[i] == d[i] ? (unsigned char)(int)rint(d[i]) : 0;
        if (there) store8(out + c, q, p.D - c);
      } else {
        float y[PL];
#pragma unroll
        for (int i = 0; i < PL; i++) y[i] = to_odd(d[i]);
        if (there) store_codes(out + c, pack_f8(y), p.D - c);
      }
      if (there && (I8 ? c == 0 : (lane & 15) == 0)) a.scale[I8 ? m : m * nb + c / FB] = none ? 1.0f : (float)(most * r / CODES);
    }
    return;
  }
  const float r = p.norm ? 1.0f / sqrtf(ms) : 1.0f;
  auto scaled = [&](float most, float codes) {  // (most * r alone may pass the largest float)
    return most * r < INFINITY ? most * r / codes : most * (r / codes);
  };
  if constexpr (!I8) {
    if (there)
      for (int b = lane; b < nb; b += LPR) a.scale[m * nb + b] = top[b] > 0.0f ? scaled(top[b], F8_MAX) : 1.0f;
  } else {
    const Scale v = scale_of<127>(rowmax);
    auto codes = [&](int c, const float (&t)[PL]) __attribute__((always_inline)) {
      unsigned char q[PL];
#pragma unroll
      for (int i = 0; i < PL; i++) q[i] = (unsigned char)(int)rintf(t[i] * v.inv);
      if (there) store8(out + c, q, p.D - c);
    };
    c = lane * PL;
#pragma unroll
    for (int k = 0; k < HELD; k++)
      if (c + k * STEP < end) codes(c + k * STEP, held[k]);
    for (c += HELD * STEP; c < end; c += STEP) {
      float h[PL], g[PL];
      reload(c, h);
      gain(c, g);
#pragma unroll
      for (int i = 0; i < PL; i++) h[i] *= g[i];
      codes(c, h);
    }
    if (lane == 0 && there) a.scale[m] = scaled(rowmax, 127.0f);
  }
}

// value * gate / (1 + exp(-gate)) for gates from GATE_MIN, where 1 + exp(-gate) and its reciprocal are normal floats. The
// exponent -gate log2(e) is taken with its rounding error and the constant's second part, put back to first order; the
// hardware reciprocal gets one Newton step (14 instructions a value; 25 from exp(-|gate|) and a corrected division: 16896 x
// 10240 values 187 us then, 145 now with the block's division below as a product).
constexpr float GATE_MIN = -86.0f;
__device__ __forceinline__ float gated(float v, float g) {
  constexpr float L = 1.44269504088896340736f, L2 = 1.92596303e-8f, LN2 = 0.693147180559945309417f;
  const float n = fminf(g, 100.0f), t = n * -L;  // exp(-100) is nothing beside 1
  const float lo = __builtin_fmaf(n, -L2, __builtin_fmaf(n, -L, -t));
  const float e0 = __builtin_amdgcn_exp2f(t);
  const float d = 1.0f + __builtin_fmaf(e0, lo * LN2, e0);
  const float r = __builtin_amdgcn_rcpf(d);
  return v * (g * __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r));
}
// The same below GATE_MIN, where 1 + exp(gate) is 1: value gate exp(gate), the exponential as the square of
// 2^-64 (2^64 exp(gate / 2)), whose factors go to the value and the gate so that neither product leaves the normal floats
// while the result is one, for values up to the largest.
__device__ __forceinline__ float gated_low(float v, float g) {
  constexpr float L = 1.44269504088896340736f, L2 = 1.92596303e-8f, LN2 = 0.693147180559945309417f;
  const float t = g * L;
  const float lo = __builtin_fmaf(g, L2, __builtin_fmaf(g, L, -t));
  const float h = __builtin_amdgcn_exp2f(fmaxf(t, -500.0f) * 0.5f + 64.0f);  // 0 from gates whose result no float holds
  const float e = g > -300.0f ? __builtin_fmaf(lo, LN2, 1.0f) : 1.0f;
  return v * 0x1p-90f * h * (g * h * 0x1p-38f) * e;
}

// b / nb for b < 2^28 as a product: magic = ceil(2^(32 + shift) / nb), 2^shift the power of two from nb / 16 on (nb = 1: b)
struct Divide {
  unsigned nb, magic, shift;
};

// 16 lanes per block of 128 columns, blocks in row order
template <int XT>
__global__ __launch_bounds__(256) void swiglu_f8_kernel(const char *x, unsigned char *out, float *scale, SwigluF8Params p, Divide d) {
  using XE = typename Elem<XT>::type;
  const unsigned b = blockIdx.x * 16 + threadIdx.x / 16, m = d.nb == 1 ? b : __umulhi(b, d.magic) >> d.shift;
  if (m >= (unsigned)p.M) return;
  const int c = (int)(b - m * d.nb) * FB + (threadIdx.x & 15) * PL, n = p.D - c;
  const XE *row = (const XE *)x + (size_t)m * p.x_stride;
  float v[PL], g[PL];
  load8(v, row + c, n);
  load8(g, row + p.D + c, n);
  float low = g[0], mx = 0.0f;
#pragma unroll
  for (int i = 1; i < PL; i++) low = fminf(low, g[i]);
  if (__builtin_expect(__any(low < GATE_MIN), 0)) {
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] = g[i] < GATE_MIN ? gated_low(v[i], g[i]) : gated(v[i], g[i]);
  } else {
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] = gated(v[i], g[i]);
  }
#pragma unroll
  for (int i = 0; i < PL; i++) mx = fmaxf(mx, fabsf(v[i]));
  mx = max16(mx);
  const Scale s = scale_of<448>(mx);
  if (__builtin_expect(__any(s.up != 1.0f), 0))
#pragma unroll
    for (int i = 0; i < PL; i++) v[i] *= s.up;
#pragma unroll
  for (int i = 0; i < PL; i++) v[i] *= s.inv;
  store_codes(out + (size_t)m * p.o_stride + c, pack_f8(v), n);
  if ((threadIdx.x & 15) == 0) scale[b] = s.s;
}

int esize(int t) { return t == T_F32 ? 4 : 2; }

// the bytes of M rows of `cols` elements, `stride` apart
uint64_t extent(int M, int stride, int cols, int size) { return ((uint64_t)(M - 1) * stride + cols) * size; }

bool fits(const Arg *a, int i, uint64_t bytes, int align, const char *what, std::string *err) {
  if (!a[i].ptr) {
    *err = std::string(what) + " is not bound";
    return false;
  }
  if (bytes > a[i].avail) {
    *err = std::string(what) + " needs " + std::to_string(bytes) + " bytes, its buffer holds " + std::to_string(a[i].avail);
    return false;
  }
  if ((uintptr_t)a[i].ptr % align) {
    *err = std::string(what) + " must be aligned to its " + std::to_string(align) + "-byte elements";
    return false;
  }
  return true;
}

bool overlap(const char *p, uint64_t n, const char *q, uint64_t k) { return p < q + k && q < p + n; }

template <int XT, int RT, bool I8>
int launch_norm(const Pipeline &pl, const Exec &ex, const Arg *a, int nargs, const void *params, uint32_t params_len,
                std::string *err) {
  (void)pl;
  if (params_len != sizeof(NormQ8Params)) {
    *err = "parameter block of " + std::to_string(params_len) + " bytes, expected " + std::to_string(sizeof(NormQ8Params));
    return -1;
  }
  NormQ8Params p;
  memcpy(&p, params, sizeof p);
  const bool has_res = RT != T_NONE;
  if (p.M < 0 || p.D < 1 || p.D > (1 << 20) || p.x_stride < p.D || p.o_stride < p.D ||
      (has_res && (p.r_stride < p.D || p.ro_stride < p.D)) || !(p.eps >= 0.0f)) {
    *err = "bad shape: M " + std::to_string(p.M) + " D " + std::to_string(p.D) + " (1 to 2^20) x_stride " +
           std::to_string(p.x_stride) + " res_stride " + std::to_string(p.r_stride) + ", " + std::to_string(p.ro_stride) +
           " o_stride " + std::to_string(p.o_stride) + " eps " + std::to_string(p.eps);
    return -1;
  }
  if (nargs < 6) {
    *err = "expected buffers x, res, w, out, scale, res_out";
    return -1;
  }
  if (p.M == 0) return 0;
  if (p.M >= 1 << 24) {  // a grid holds less than 2^32 threads
    *err = "over 2^24 - 1 rows";
    return -1;
  }
  const int nb = (p.D + FB - 1) / FB;
  const uint64_t xb = extent(p.M, p.x_stride, p.D, esize(XT)), ob = extent(p.M, p.o_stride, p.D, 1);
  const uint64_t rb = extent(p.M, p.r_stride, p.D, esize(RT)), wb = extent(p.M, p.ro_stride, p.D, esize(RT));
  const uint64_t sb = (uint64_t)p.M * (I8 ? 1 : nb) * 4;
  if (!fits(a, 0, xb, esize(XT), "x", err) || (has_res && !fits(a, 1, rb, esize(RT), "res", err)) ||
      (a[2].ptr && !fits(a, 2, (uint64_t)p.D * 4, 4, "w", err)) || !fits(a, 3, ob, 1, "out", err) ||
      !fits(a, 4, sb, 4, "scale", err) || (has_res && !fits(a, 5, wb, esize(RT), "res_out", err)))
    return -1;
  // Rows are worked on in any order and a value is read before its own place is written: the sum may take its residual's
  // (or x's) own place, nothing else may share memory with an output.
  struct Range { const char *p; uint64_t n; int stride, size; const char *name; };
  const Range in[] = {{a[0].ptr, xb, p.x_stride, esize(XT), "x"},
                      {has_res ? a[1].ptr : nullptr, rb, p.r_stride, esize(RT), "res"},
                      {a[2].ptr, (uint64_t)p.D * 4, 0, 4, "w"}};
  const Range to[] = {{a[3].ptr, ob, 0, 1, "out"}, {a[4].ptr, sb, 0, 4, "scale"},
                      {has_res ? a[5].ptr : nullptr, wb, p.ro_stride, esize(RT), "res_out"}};
  for (int i = 0; i < 3; i++) {
    if (!to[i].p) continue;
    for (const Range &q : in)
      if (q.p && overlap(to[i].p, to[i].n, q.p, q.n) &&
          !(i == 2 && to[i].p == q.p && to[i].stride == q.stride && to[i].size == q.size)) {
        *err = std::string(to[i].name) + " shares memory with " + q.name;
        return -1;
      }
    for (int k = 0; k < i; k++)
      if (overlap(to[i].p, to[i].n, to[k].p, to[k].n)) {
        *err = std::string(to[i].name) + " shares memory with " + to[k].name;
        return -1;
      }
  }
  const NormArgs g{a[0].ptr, has_res ? a[1].ptr : nullptr, (const float *)a[2].ptr, (unsigned char *)a[3].ptr,
                   (float *)a[4].ptr, has_res ? a[5].ptr : nullptr};
  // Lanes a row. Short rows share a workgroup: bf16 rows and residual, 16896 of 256 columns 7.8 us with 32 lanes (64: 10.6,
  // 256: 22.3), of 1024 columns 20 with 64 (256: 29), of 2048 columns 35 with 64 (256: 38), of 4096 columns 91 with 256 (64:
  // 98; 300 rows 6.0, 64: 12.7).
  auto go = [&](auto lpr) {
    constexpr int LPR = decltype(lpr)::value, ROWS = 256 / LPR;
    hipLaunchKernelGGL((rms_norm_q8_kernel<XT, RT, I8, LPR>), dim3((unsigned)((p.M + ROWS - 1) / ROWS)), dim3(256),
                       I8 ? 0 : ROWS * nb * 4, ex.stream, g, p);
  };
  if (p.D <= 32 * PL) go(std::integral_constant<int, 32>{});
  else if (p.D <= 256 * PL) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 256>{});
  return 0;
}

template <int XT>
int launch_swiglu(const Pipeline &pl, const Exec &ex, const Arg *a, int nargs, const void *params, uint32_t params_len,
                  std::string *err) {
  (void)pl;
  if (params_len != sizeof(SwigluF8Params)) {
    *err = "parameter block of " + std::to_string(params_len) + " bytes, expected " + std::to_string(sizeof(SwigluF8Params));
    return -1;
  }
  SwigluF8Params p;
  memcpy(&p, params, sizeof p);
  if (p.M < 0 || p.D < 1 || p.D > (1 << 20) || p.x_stride < 2 * p.D || p.o_stride < p.D) {
    *err = "bad shape: M " + std::to_string(p.M) + " D " + std::to_string(p.D) + " (1 to 2^20) x_stride " +
           std::to_string(p.x_stride) + " o_stride " + std::to_string(p.o_stride);
    return -1;
  }
  if (nargs < 3) {
    *err = "expected buffers x, out, scale";
    return -1;
  }
  if (p.M == 0) return 0;
  const int nb = (p.D + FB - 1) / FB;
  const uint64_t xb = extent(p.M, p.x_stride, 2 * p.D, esize(XT)), ob = extent(p.M, p.o_stride, p.D, 1);
  const uint64_t blocks = (uint64_t)p.M * nb, sb = blocks * 4;
  if (!fits(a, 0, xb, esize(XT), "x", err) || !fits(a, 1, ob, 1, "out", err) || !fits(a, 2, sb, 4, "scale", err)) return -1;
  if (overlap(a[0].ptr, xb, a[1].ptr, ob) || overlap(a[0].ptr, xb, a[2].ptr, sb) || overlap(a[1].ptr, ob, a[2].ptr, sb)) {
    *err = "x, out and scale share memory";
    return -1;
  }
  if (blocks >= (1ull << 28)) {  // 16 threads each, and a grid holds less than 2^32
    *err = "over 2^28 - 1 blocks of 128 columns";
    return -1;
  }
  Divide d{(unsigned)nb, 0, 0};
  while (nb > 16 << d.shift) d.shift++;
  if (nb > 1) d.magic = (unsigned)(((1ull << (32 + d.shift)) + nb - 1) / nb);
  hipLaunchKernelGGL((swiglu_f8_kernel<XT>), dim3((unsigned)((blocks + 15) / 16)), dim3(256), 0, ex.stream, a[0].ptr,
                     (unsigned char *)a[1].ptr, (float *)a[2].ptr, p, d);
  return 0;
}

template <int XT, int RT>
LaunchFn pick_out(bool i8) {
  return i8 ? launch_norm<XT, RT, true> : launch_norm<XT, RT, false>;
}
template <int XT>
LaunchFn pick_res(int rt, bool i8) {
  return rt == T_NONE   ? pick_out<XT, T_NONE>(i8)
         : rt == T_BF16 ? pick_out<XT, T_BF16>(i8)
         : rt == T_F16  ? pick_out<XT, T_F16>(i8)
                        : pick_out<XT, T_F32>(i8);
}

int type_of(const std::string &s) {
  if (s == "bfloat" || s == "bf16") return T_BF16;
  if (s == "half" || s == "f16") return T_F16;
  if (s == "float" || s == "f32") return T_F32;
  if (s == "none") return T_NONE;
  return -1;
}

}  // namespace

// Macros: IN_T (half | bfloat | float), and for rms_norm_q8 RES_T (the residual's type, none without one) and OUT_T (f8 |
// i8).
bool make_rows_q8(const std::string &fn, const Macros &m, Pipeline *pl, std::string *err) {
  const bool norm = fn == "rms_norm_q8";
  for (auto &kv : m)
    if (kv.first != "IN_T" && !(norm && (kv.first == "RES_T" || kv.first == "OUT_T"))) {
      *err = "unknown macro " + kv.first;
      return false;
    }
  const int xt = type_of(macro_str(m, "IN_T", "bfloat")), rt = type_of(macro_str(m, "RES_T", "none"));
  const std::string ot = macro_str(m, "OUT_T", "f8");
  if (xt <= 0 || rt < 0 || (ot != "f8" && ot != "i8")) {
    *err = "IN_T must be half|bfloat|float, RES_T that or none, OUT_T f8|i8";
    return false;
  }
  const bool i8 = ot == "i8";
  if (norm)
    pl->launch = xt == T_BF16 ? pick_res<T_BF16>(rt, i8) : xt == T_F16 ? pick_res<T_F16>(rt, i8) : pick_res<T_F32>(rt, i8);
  else
    pl->launch = xt == T_BF16 ? launch_swiglu<T_BF16> : xt == T_F16 ? launch_swiglu<T_F16> : launch_swiglu<T_F32>;
  pl->threads = 256;
  return true;
}

}  // namespace h3
