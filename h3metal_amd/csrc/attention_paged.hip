// Attention of a batch's new tokens over a paged cache for gfx950: query row i of sequence b (n_b new rows, L_b keys) sees
// the keys j < L_b, with a causal mask those up to L_b - n_b + i;
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j, 0 where no key is visible
// Query head h reads key/value head h / (H / KVH). A key whose page number lies outside the cache has the score NaN.
#include "paged.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace h3 {
namespace {

// One wave per query row and head: a lane scores one of 64 keys, then every lane sums its channels of the values.
template <int D, int T>
__global__ __launch_bounds__(256) void attention_paged_simple(const char *q, const char *kc, const char *vc, char *out,
                                                              Batch bt, PagedAttnParams p, int causal) {
  using E = typename PElem<T>::type;
  const int lane = threadIdx.x & 63, m = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (h >= p.H) return;
  int b = 0;
  for (int k = 0; k < bt.B; k += 64) b += __popcll(__ballot(k + lane < bt.B && bt.q_start[k + lane + 1] <= m));
  if (b >= bt.B || bt.q_start[b] > m) return;
  const long long most = (long long)bt.width << bt.lg, L = min(max((long long)bt.kv_len[b], 0ll), most);
  const long long end = causal ? min(L, (long long)bt.kv_len[b] - bt.q_start[b + 1] + m + 1) : L;
  const int kvh = h / (p.H / p.KVH);
  const E *qr = (const E *)q + (size_t)m * p.q_stride + h * D;
  float top = -INFINITY, sum = 0.0f, o[2] = {0.0f, 0.0f};
  for (long long j0 = 0; j0 < end; j0 += 64) {
    const long long j = j0 + lane;
    float s = -INFINITY;
    long long row = -1;
    if (j < end) {
      const int pg = bt.table[(long long)b * bt.width + (j >> bt.lg)];
      s = NAN;
      if (pg >= 0 && pg < bt.pages) {
        row = (((long long)pg * p.KVH + kvh) << bt.lg) + (j & ((1 << bt.lg) - 1));
        s = 0.0f;
        for (int d = 0; d < D; d++) s = fmaf((float)qr[d], (float)((const E *)kc)[row * D + d], s);
        s *= p.scale;
      }
    }
    float mx = s;
    for (int i = 32; i; i /= 2) mx = fmaxf(mx, __shfl_xor(mx, i));
    mx = fmaxf(mx, top);
    const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - mx);
    const float w = j < end ? (mx == -INFINITY ? s - s : __builtin_amdgcn_exp2f(s - mx)) : 0.0f;
    top = mx;
    sum = sum * f + w;
    o[0] *= f;
    o[1] *= f;
    for (int k = 0; k < 64 && j0 + k < end; k++) {
      const long long r = __shfl(row, k);
      const float wk = __shfl(w, k);
      for (int e = 0; e < 2; e++)
        if (e * 64 + lane < D) o[e] += wk * (r < 0 ? 0.0f : (float)((const E *)vc)[r * D + e * 64 + lane]);
    }
  }
  for (int i = 32; i; i /= 2) sum += __shfl_xor(sum, i);
  const float inv = end > 0 ? 1.0f / sum : 0.0f;
  for (int e = 0; e < 2; e++)
    if (e * 64 + lane < D) ((E *)out)[(size_t)m * p.o_stride + h * D + e * 64 + lane] = (E)(o[e] * inv);
}

template <int D, int T>
int launch(const Pipeline &pl, const Exec &ex, const Arg *a, int nargs, const void *params, uint32_t params_len,
           std::string *err) {
  if (params_len != sizeof(PagedAttnParams)) {
    *err = "parameter block of " + std::to_string(params_len) + " bytes, expected " + std::to_string(sizeof(PagedAttnParams));
    return -1;
  }
  PagedAttnParams p;
  memcpy(&p, params, sizeof p);
  const int lg = log2_page(p.page);
  if (p.M < 0 || p.M >= 1 << 24 || p.B < 0 || p.B >= 1 << 24 || p.H < 1 || p.H > 4096 || p.KVH < 1 || p.H % p.KVH ||
      p.q_stride < p.H * D || p.o_stride < p.H * D) {
    *err = "bad shape: M " + std::to_string(p.M) + " B " + std::to_string(p.B) + " (below 2^24) H " + std::to_string(p.H) +
           " (up to 4096, a multiple of KVH) KVH " + std::to_string(p.KVH) + " q_stride " + std::to_string(p.q_stride) +
           " o_stride " + std::to_string(p.o_stride);
    return -1;
  }
  if (lg < 0 || p.pages < 0 || p.width < 0) {
    *err = "bad cache: " + std::to_string(p.pages) + " pages of " + std::to_string(p.page) +
           " rows (a power of two from 16 to 256), " + std::to_string(p.width) + " in a row of the table";
    return -1;
  }
  if (!(p.scale > 0.0f) || !std::isfinite(p.scale)) {
    *err = "softmax scale must be positive and finite";
    return -1;
  }
  if (nargs < 7) {
    *err = "expected buffers q, kc, vc, out, table, q_start, kv_len";
    return -1;
  }
  if (p.M == 0 || p.B == 0) return 0;
  const uint64_t cache = (uint64_t)p.pages * p.KVH * p.page * D * 2;
  const uint64_t need[7] = {((uint64_t)(p.M - 1) * p.q_stride + (uint64_t)p.H * D) * 2, cache, cache,
                            ((uint64_t)(p.M - 1) * p.o_stride + (uint64_t)p.H * D) * 2, (uint64_t)p.B * p.width * 4,
                            ((uint64_t)p.B + 1) * 4, (uint64_t)p.B * 4};
  static const char *what[7] = {"q", "kc", "vc", "out", "table", "q_start", "kv_len"};
  const int align[7] = {16, 16, 16, 8, 4, 4, 4};
  for (int i = 0; i < 7; i++)
    if (need[i] && !paged_fits(a, i, need[i], align[i], what[i], err)) return -1;
  if (p.q_stride % 8 || p.o_stride % 4) {
    *err = "q_stride must be a multiple of 8 elements, o_stride of 4";
    return -1;
  }
  for (int i = 0; i < 7; i++)
    if (i != 3 && paged_overlap(a[3], need[3], a[i], need[i])) {
      *err = std::string("out shares memory with ") + what[i];
      return -1;
    }
  const Batch bt{(const int *)a[4].ptr, (const int *)a[5].ptr, (const int *)a[6].ptr, p.B, p.width, p.pages, lg};
  hipLaunchKernelGGL((attention_paged_simple<D, T>), dim3((unsigned)p.M, (unsigned)((p.H + 3) / 4)), dim3(256), 0, ex.stream,
                     a[0].ptr, a[1].ptr, a[2].ptr, a[3].ptr, bt, p, pl.ival[0]);
  return 0;
}

template <int D>
LaunchFn pick(int t) {
  return t == P_BF16 ? launch<D, P_BF16> : launch<D, P_F16>;
}

}  // namespace

// Macros: HD (64, 96 or 128), IN_T (half | bfloat: queries, cache and output), CAUSAL.
bool make_attention_paged(const Macros &m, Pipeline *pl, std::string *err) {
  int hd, causal;
  if (!macro_int(m, "HD", 128, &hd, err) || !macro_int(m, "CAUSAL", 1, &causal, err)) return false;
  for (auto &kv : m)
    if (kv.first != "HD" && kv.first != "CAUSAL" && kv.first != "IN_T") {
      *err = "unknown macro " + kv.first;
      return false;
    }
  const int t = paged_type(macro_str(m, "IN_T", "bfloat"));
  if (t != P_BF16 && t != P_F16) {
    *err = "IN_T must be half|bfloat";
    return false;
  }
  if (hd != 64 && hd != 96 && hd != 128) {
    *err = "HD " + std::to_string(hd) + " not supported (64, 96 or 128)";
    return false;
  }
  pl->launch = hd == 128 ? pick<128>(t) : hd == 96 ? pick<96>(t) : pick<64>(t);
  pl->ival[0] = causal != 0;
  pl->threads = 256;
  return true;
}

}  // namespace h3
