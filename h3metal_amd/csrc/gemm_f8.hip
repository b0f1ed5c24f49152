// Matrix product of e4m3 operands with a float scale for each block of 128, for gfx950 (weight format f8):
//   v[m][n] = sum over blocks b of K of sa[m][b] * sw[n / 128][b] * (sum over k in b of A[m][k] * W[n][k])
// A [M][K] and W [N][K] e4m3, row-major in k, sa a scale for each row and block of 128 columns, sw one for each 128 x 128
// block of W (the last blocks of K and of N may be short). The epilogues are gemm.hip's: C[m][n] = OUT_T(v + bias[n]), or
// X[m][n] += gate[rtype[m]][n] * (v + bias[n]) with X float.
// Products are exact and a block's 128 are summed by the matrix unit in float; each block's sum enters the float
// accumulator in one fused step with the product of its two scales.
//
// One wave per 32 x 32 tile, operands straight from memory.
#include "gemm_common.h"

#include <cstring>

namespace h3 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int KB = 128;  // K of a block

__device__ __forceinline__ f32x16 mma_f8(i32x8 a, i32x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}

__global__ __launch_bounds__(64) void gemm_f8_kernel(GemmArgs g, GemmParams p, int ntm, int ot, int epi) {
  const int lane = threadIdx.x, l32 = lane & 31, hl = lane >> 5;
  const int nt = blockIdx.x / ntm, mt = blockIdx.x - nt * ntm;
  const int m = mt * 32 + l32, n0 = nt * 32;
  const int nb = (p.K + KB - 1) / KB;
  const int mc = min(m, p.M - 1), nc = min(n0 + l32, p.N - 1);
  const char *ar = g.a + (size_t)mc * p.a_stride, *wr = g.w + (size_t)nc * p.w_stride;
  const float *sa = g.sa + (size_t)mc * p.groups, *sw = g.sw + (size_t)(n0 / KB) * p.groups;
  auto piece = [&](const char *r, int k) __attribute__((always_inline)) {  // 16 codes from k, zero past K
    i32x4 z = {0, 0, 0, 0};
    return k < p.K ? *(const i32x4 *)(r + k) : z;
  };
  f32x16 acc = {};
  for (int b = 0; b < nb; b++) {
    f32x16 t = {};
#pragma unroll
    for (int c = 0; c < 2; c++) {
      const int k = b * KB + c * 64 + hl * 32;
      const i32x4 a0 = piece(ar, k), a1 = piece(ar, k + 16), w0 = piece(wr, k), w1 = piece(wr, k + 16);
      t = mma_f8(__builtin_shufflevector(w0, w1, 0, 1, 2, 3, 4, 5, 6, 7),
                 __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7), t);
    }
    const float s = sa[b] * sw[b];
#pragma unroll
    for (int e = 0; e < 16; e++) acc[e] = __builtin_fmaf(t[e], s, acc[e]);
  }
  if (m >= p.M) return;
#pragma unroll
  for (int e = 0; e < 16; e++) {
    const int n = n0 + 8 * (e >> 2) + 4 * hl + (e & 3);
    if (n >= p.N) continue;
    float v = acc[e];
    if (g.bias) v += g.bias[n];
    const size_t at = (size_t)m * p.c_stride + n;
    if (epi) {
      const float *gr = g.gate + (size_t)min((int)g.rtype[m], g.ntypes - 1) * p.g_stride;
      ((float *)g.out)[at] += gr[n] * v;
    } else if (ot == T_F32) {
      ((float *)g.out)[at] = v;
    } else {
      ((unsigned short *)g.out)[at] = ot == T_BF16 ? __builtin_bit_cast(unsigned short, (__bf16)v)
                                                   : __builtin_bit_cast(unsigned short, (_Float16)v);
    }
  }
}

int launch_f8(const Pipeline &pl, const Exec &ex, const Arg *a, int nargs, const void *params, uint32_t params_len,
              std::string *err) {
  const int epi = pl.ival[1], ot = pl.ival[2], has_bias = pl.ival[3];
  if (params_len != sizeof(GemmParams)) {
    *err = "parameter block of " + std::to_string(params_len) + " bytes, expected " + std::to_string(sizeof(GemmParams));
    return -1;
  }
  GemmParams p;
  memcpy(&p, params, sizeof p);
  constexpr int MAX_STRIDE = 1 << 22;  // 256 rows of a tile then lie within 2^30 bytes
  const int nb = p.K > 0 ? (p.K - 1) / KB + 1 : 0;
  if (p.M < 0 || p.N < 1 || p.K < 16 || p.K % 16 || p.a_stride < p.K || p.w_stride < p.K || p.c_stride < p.N ||
      p.a_stride % 16 || p.w_stride % 16 || p.a_stride > MAX_STRIDE || p.w_stride > MAX_STRIDE || p.groups < nb) {
    *err = "bad shape: M " + std::to_string(p.M) + " N " + std::to_string(p.N) + " K " + std::to_string(p.K) +
           " (a multiple of 16) a_stride " + std::to_string(p.a_stride) + " w_stride " + std::to_string(p.w_stride) +
           " (multiples of 16 up to 2^22) c_stride " + std::to_string(p.c_stride) + " scales a row " +
           std::to_string(p.groups);
    return -1;
  }
  if (nargs < (epi ? 8 : 5)) {
    *err = epi ? "expected buffers a, w, sw, sa, x, bias, rtype, gate" : "expected buffers a, w, sw, sa, out";
    return -1;
  }
  auto need = [&](int i, uint64_t bytes, int align, const char *what) {
    if (i >= nargs || !a[i].ptr) {
      *err = std::string(what) + " is not bound";
      return false;
    }
    if (bytes > a[i].avail) {
      *err = std::string(what) + " needs " + std::to_string(bytes) + " bytes, its buffer holds " + std::to_string(a[i].avail);
      return false;
    }
    if ((uintptr_t)a[i].ptr % align) {
      *err = std::string(what) + " must be " + std::to_string(align) + "-byte aligned";
      return false;
    }
    return true;
  };
  if (p.M == 0) return 0;
  const uint64_t M = p.M, N = p.N, NB = (N + KB - 1) / KB;
  const int osz = ot == T_F32 ? 4 : 2;
  if (!need(0, (M - 1) * p.a_stride + p.K, 16, "a") || !need(1, (N - 1) * p.w_stride + p.K, 16, "w") ||
      !need(2, ((NB - 1) * p.groups + nb) * 4, 4, "sw") || !need(3, ((M - 1) * p.groups + nb) * 4, 4, "sa") ||
      !need(4, ((M - 1) * p.c_stride + N) * osz, osz, "out") || (has_bias && !need(5, N * 4, 4, "bias")))
    return -1;
  int ntypes = 1;
  if (epi) {
    if (!need(6, M, 1, "rtype") || !need(7, N * 4, 4, "gate")) return -1;
    if (p.g_stride < p.N) {
      *err = "g_stride " + std::to_string(p.g_stride) + " smaller than N";
      return -1;
    }
    ntypes = (int)std::min<uint64_t>(256, (a[7].avail / 4 - N) / p.g_stride + 1);
  }
  const GemmArgs g{a[0].ptr, a[1].ptr, (const float *)a[2].ptr, (const float *)a[3].ptr, a[4].ptr,
                   has_bias ? (const float *)a[5].ptr : nullptr, epi ? (const unsigned char *)a[6].ptr : nullptr,
                   epi ? (const float *)a[7].ptr : nullptr, ntypes, false};
  const int ntm = (p.M + 31) / 32, ntn = (p.N + 31) / 32;
  if ((uint64_t)ntm * ntn * 64 >= (1ull << 32)) {
    *err = "too many tiles";
    return -1;
  }
  hipLaunchKernelGGL(gemm_f8_kernel, dim3((unsigned)(ntm * ntn)), dim3(64), 0, ex.stream, g, p, ntm, ot, epi);
  return 0;
}

}  // namespace

bool make_gemm_f8(int epi, int out_t, bool bias, int tile, Pipeline *pl, std::string *err) {
  if (tile != 0) {
    *err = "TILE must be 0 with format f8";
    return false;
  }
  pl->launch = launch_f8;
  pl->threads = 64;
  pl->ival[0] = tile;
  pl->ival[1] = epi;
  pl->ival[2] = out_t;
  pl->ival[3] = bias;
  return true;
}

}  // namespace h3
