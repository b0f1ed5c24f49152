// Attention of a batch's new tokens over a paged cache for gfx950: query row i of sequence b (n_b new rows, L_b keys) sees
// the keys j < L_b, with a causal mask those up to L_b - n_b + i;
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j, 0 where no key is visible
// Query head h reads key/value head h / (H / KVH). A key whose page number lies outside the cache has the score NaN.
//
// A tile's 32 rows are (token, head) pairs that share a key/value head, so that a single token of grouped heads reads its
// keys once. The work is cut as paged_plan.h says; lengths are known on the device only, so every workgroup finds its slice by
// itself. Within a workgroup the waves split the keys: wave w takes the 32-key blocks w, w + NW, ... of its part of a tile,
// with a running maximum, sum and output of its own, staged through LDS of its own by LDS-direct loads that its own vmcnt
// orders, with no barrier; the waves' states meet in LDS at the end. Scores are S^T = K Q^T and outputs O^T = V^T P^T on the
// 32 x 32 MFMA, in attention_small.hip's layouts (a lane holds one query's keys, so the softmax is per lane; V's operands are
// transposing LDS reads). The loads of a block's two 16-key halves go through descriptors that end at the sequence's last
// key: what a page holds behind it reads as zero. Two workgroups a compute unit have up to 128 KB of loads under way, and single
// tokens are bound by HBM: 64 sequences with 275 181 keys (32 + 8 heads of 128) 214 us, 5.3 TB/s; one of 131 072 104 us.
// A few short tiles are bound by the chain of a wave's blocks (1.1 us each, alone): 8 waves instead of 4, 512 keys 13 -> 10 us
// when they came, 8.8 now.
#include "attention_common.h"
#include "paged_attn.h"

#include <algorithm>
#include <cmath>
#include <cstring>

namespace h3 {
namespace {

constexpr int RT = plan::SHORT_ROWS;
constexpr int KB = 32;             // keys of a block
constexpr float SLACK_P = 8.0f;    // log2 units the running maximum may lag behind a score

// -- tiles of 32 rows -------------------------------------------------------------------------------------------------

template <int DG, int NW>
struct Rows {
  static constexpr int D = DG == 96 ? 128 : DG;        // channels of an LDS row
  static constexpr int RB = D * 2, RBG = DG * 2;       // bytes of a row: in LDS, in memory
  static constexpr int NP = RB / 16;                   // 16-byte pieces of a row
  static constexpr int NCH = DG / 16;                  // score MFMAs per 32 x 32 tile
  static constexpr int NDB = DG / 32;                  // 32-channel blocks of O
  static constexpr int BYTES = KB * RB;                // a block of K or V
  static constexpr int NDMA = BYTES / 1024;            // 1 KB loads of it
  static constexpr int ORS = (DG + 4) * 4;             // bytes of a row of a wave's state
  static constexpr int MERGE = NW * RT * (ORS + 8);    // the waves' states: O, then (m, l)
  static constexpr int LDS = NW * 2 * BYTES > MERGE ? NW * 2 * BYTES : MERGE;
};

template <int DG, int T, int NW, bool CAUSAL, bool EACH>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2)))
void attention_rows_kernel(AttnArgs a, Batch bt, PagedAttnParams p, plan::Shape sh, Heads hd, int least) {
  using C = Rows<DG, NW>;
  constexpr int NDB = C::NDB, NCH = C::NCH;
  using VT8 = typename Vec8<T>::type;
  using VE = typename Vec8<T>::elem;
  using VP2 = typename Vec8<T>::pair;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  // a whole tile, or a slice of the batch's weight
  Tile tile;
  int sl = 0;
  plan::Cut cut{};
  i64 x0 = 0, x1 = 1;
  bool more;
  std::conditional_t<EACH, Tiles, Order> order(sh, bt);
  if constexpr (EACH) {
    const int n = min(order.all, (int)gridDim.x);
    if ((int)blockIdx.x >= n) return;
    more = order.tile(n - 1 - slice_of(blockIdx.x, n), &tile);  // with a causal mask the longest tiles go first
  } else {
    cut = plan::cut(order.all, order.tiles, gridDim.x, least);
    if (order.all <= 0 || (int)blockIdx.x >= cut.n) {
      if (tid == 0) left_of(a, blockIdx.x)->R = 0;
      return;
    }
    sl = slice_of(blockIdx.x, cut.n);
    x0 = plan::slice_start(cut, sl);
    x1 = plan::slice_start(cut, sl + 1);
    more = tile_at(order, x0, &tile);
  }

  // this lane's 16 bytes of each 1 KB load: row and swizzled piece (attention_common.h: kswz, voff); pieces past a row in
  // memory (head dim 96) are sent out of the descriptor's range
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem + w * 2 * C::BYTES;
  const char *Ks = smem + w * 2 * C::BYTES, *Vs = Ks + C::BYTES;
  unsigned kgo[C::NDMA], vgo[C::NDMA];
#pragma unroll
  for (int r = 0; r < C::NDMA; r++) {
    constexpr int R = 256 / C::RB > 0 ? 256 / C::RB : 1;
    const int o = r * 1024 + 16 * lane, row = o / C::RB, in = o % C::RB;
    const int kp = (in / 16) ^ kswz<C::RB, C::NP>(row), vp = 2 * ((in >> 5) ^ (2 * ((row & 3) / R))) + ((in >> 4) & 1);
    kgo[r] = kp * 16 < C::RBG ? (row & 15) * C::RBG + kp * 16 : 0x80000000u;
    vgo[r] = vp * 16 < C::RBG ? (row & 15) * C::RBG + vp * 16 : 0x80000000u;
  }
  const int krow = 16 * (l32 >> 4) + 8 * ((l32 >> 2) & 1) + 4 * ((l32 >> 3) & 1) + (l32 & 3);
  const int l16 = lane & 15, tr_row = l16 >> 2, tr_col = (l16 & 3) * 8;

  bool unfinished = false;
  auto next = [&]() {
    if constexpr (EACH) return false;
    else return next_tile(order, &tile) && tile.p < x1;
  };
  if (!EACH) more = more && tile.p < x1;
  for (; more; more = next()) {
    const plan::Seq &q = tile.q;
    const int nblk = plan::tile_blocks(sh, q, tile.t, KB);
    int blk0 = 0, blk1 = nblk;
    bool begun = false, whole = true;
    if constexpr (!EACH) {
      blk0 = plan::block_at(x0, tile.p, tile.w, nblk);
      blk1 = plan::block_at(x1, tile.p, tile.w, nblk);
      begun = tile.p < x0;
      whole = !begun && tile.p + tile.w <= x1;
    }
    const int kvh = tile.v / hd.HS, g0 = (tile.v - kvh * hd.HS) * hd.GP;
    const int m0 = q.lo + tile.t * sh.TT, R = min(sh.TT, q.hi - m0) * hd.GP;
    const int L = (int)q.L;
    const i64 first_last = CAUSAL ? plan::clamp(q.off + m0, -M_MOST, q.L - 1) : q.L - 1;  // of the tile's first token
    float *st = a.ws + (size_t)plan::state_of(sl, begun) * (RT * (DG + 2));
    if (!EACH && !whole && !begun) {
      const int end = last_slice(cut, sl, tile.p + tile.w);
      // (rows of a causal tile that see no key begin before the sequence; without keys none sees any)
      if (tid == 0)
        *left_of(a, sl) = Left{R, m0, kvh * hd.G + g0, hd.GP, min(hd.GP, hd.G - g0),
                               q.L > 0 ? CAUSAL ? (int)first_last : 0 : -M_MOST, end, 0};
      unfinished = true;
    }
    if (!EACH && blk0 == blk1) {  // a part without blocks (a whole tile has one)
      if (tid < R) *(float2 *)(st + RT * DG + 2 * tid) = make_float2(-INFINITY, NO_PART);
      continue;
    }
    // this lane's query row: its token, head and last visible key
    const int ti = (int)((unsigned)l32 / (unsigned)hd.GP), gi = l32 - ti * hd.GP;
    const bool ok = l32 < R && g0 + gi < hd.G;
    const int last = !ok ? -1 : CAUSAL ? (int)plan::clamp(q.off + m0 + ti, -1, q.L - 1) : L - 1;
    i32x4 qreg[NCH];
    {
      const char *qrow = a.q + ((size_t)(m0 + (ok ? ti : 0)) * p.q_stride + (size_t)(kvh * hd.G + (ok ? g0 + gi : 0)) * DG) * 2;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        const i32x4 v = *(const i32x4 *)(qrow + (2 * c + hl) * 16);
        qreg[c] = ok ? v : i32x4{0, 0, 0, 0};
      }
    }

    // Page numbers of this wave's next 32 blocks: lane 2 i + h holds that of half h of the i-th; -1: outside the cache.
    int ids = 0;
    auto fetch_ids = [&](int blk) __attribute__((always_inline)) {
      const i64 key = (i64)(blk + (lane >> 1) * NW) * KB + 16 * (lane & 1), pi = key >> bt.lg;
      ids = 0;
      if (key < L) {
        ids = bt.table[(size_t)tile.b * bt.width + pi];
        if (ids < 0 || ids >= bt.pages) ids = -1;
      }
    };
    auto page_of = [&](int it, int h) __attribute__((always_inline)) {
      return __builtin_amdgcn_readlane(ids, 2 * (it & 31) + h);
    };
    auto half_rsrc = [&](const char *base, int pg, i64 key) __attribute__((always_inline)) {
      const size_t row = ((((size_t)max(pg, 0) * p.KVH + kvh) << bt.lg) + (size_t)(key & ((1 << bt.lg) - 1)));
      const int n = pg < 0 ? 0 : (int)plan::clamp(L - key, 0, 16);
      return __builtin_amdgcn_make_buffer_rsrc((void *)(base + row * C::RBG), (short)0, n * C::RBG, 0x00020000);
    };
    auto load = [&](const char *base, unsigned lds, const unsigned (&go)[C::NDMA], int blk, int pg0, int pg1)
        __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const __amdgpu_buffer_rsrc_t r = half_rsrc(base, h ? pg1 : pg0, (i64)blk * KB + 16 * h);
#pragma unroll
        for (int i = 0; i < C::NDMA / 2; i++) dma16(lds + (h * (C::NDMA / 2) + i) * 1024, go[h * (C::NDMA / 2) + i], r);
      }
    };

    f32x16 o[NDB];
    float m = -INFINITY, l = 0.0f;
    bool odd = false;
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
      for (int i = 0; i < 16; i++) o[db][i] = 0.0f;

    int blk = blk0 + w, it = 0;
    if (blk < blk1) {
      fetch_ids(blk);
      int pg0 = page_of(0, 0), pg1 = page_of(0, 1);
      load(a.kc, lds0, kgo, blk, pg0, pg1);
      load(a.vc, lds0 + C::BYTES, vgo, blk, pg0, pg1);
      for (;; blk += NW) {
        const bool next = blk + NW < blk1;
        const bool lost0 = pg0 < 0, lost1 = pg1 < 0;
        if (next) {
          if ((++it & 31) == 0) fetch_ids(blk + NW);
          pg0 = page_of(it, 0);
          pg1 = page_of(it, 1);
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::NDMA) : "memory");  // the block's K has landed (V may be in flight)
        i32x4 ka[NCH];
#pragma unroll
        for (int c = 0; c < NCH; c++)
          ka[c] = *(const i32x4 *)(Ks + krow * C::RB + (((2 * c + hl) ^ kswz<C::RB, C::NP>(krow)) * 16));
        f32x16 x;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; c++) x = mma_qk<T>(ka[c], qreg[c], x);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the K slot's reads are done
        if (next) load(a.kc, lds0, kgo, blk + NW, pg0, pg1);
        if (__builtin_expect(lost0 || lost1, 0)) {
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (i < 8 ? lost0 : lost1) x[i] = NAN;
        }
        const bool edge = (i64)blk * KB + KB - 1 > first_last;  // some row does not see some key
        if (edge) {
          // element i of lane half hl holds key KB blk + 16 (i / 8) + 8 hl + i % 8
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (blk * KB + 16 * (i >> 3) + 8 * hl + (i & 7) > last) x[i] = -INFINITY;
        }
        float am[2] = {x[0], x[1]};
#pragma unroll
        for (int i = 2; i < 16; i++) am[i & 1] = fmaxf(am[i & 1], x[i]);
        const float amax = fmaxf(am[0], am[1]);
        // lazy running maximum (wave-uniform branch); partner lanes (the same query) always update together
        if (__any(amax * p.scale > m + SLACK_P)) {
          const float ap = fmaxf(amax, __shfl_xor(amax, 32));
          const float mn = fmaxf(m, ap * p.scale);
          const float f = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
          m = mn;
          l *= f;
#pragma unroll
          for (int db = 0; db < NDB; db++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[db][i] *= f;
        }
        const float nm = m == -INFINITY ? 0.0f : -m;
        float ls[2] = {0.0f, 0.0f};  // of the rounded weights, which the product with V takes
        i32x4 pb[2];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(x[i], p.scale, nm));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(x[i + 1], p.scale, nm));
          const VP2 pr = {(VE)p0, (VE)p1};
          pb[i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, pr);
          ls[(i >> 1) & 1] = sum2<T>(pr, ls[(i >> 1) & 1]);
        }
        l += ls[0] + ls[1];
        if (next) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::NDMA) : "memory");  // the block's V has landed
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int s2 = 0; s2 < 2; s2++) {
          const int k0 = 16 * s2 + 8 * hl + tr_row;
          i16x8 va[NDB];
#pragma unroll
          for (int db = 0; db < NDB; db++) {
            const int pc = (db * 32 + (l32 & 16)) / 8;
            const i16x4 lo = lds_tr16(Vs + voff<C::D>(k0, pc) + tr_col);
            const i16x4 hi = lds_tr16(Vs + voff<C::D>(k0 + 4, pc) + tr_col);
            va[db] = i16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          }
          if (CAUSAL && edge) {
            // A weight of 0 does not keep a value that is infinite or NaN out of a sum: such values are taken as 0 here, and
            // the rows that see them get them at the end.
            bool some = false;
#pragma unroll
            for (int db = 0; db < NDB; db++) {
              const i32x4 d = __builtin_bit_cast(i32x4, va[db]);
#pragma unroll
              for (int i = 0; i < 4; i++) some |= odd16<T>((unsigned)d[i]) | odd16<T>((unsigned)d[i] << 16);
            }
            if (__builtin_expect(__any(some), 0)) {
              odd = true;
#pragma unroll
              for (int db = 0; db < NDB; db++)
#pragma unroll
                for (int e = 0; e < 8; e++)
                  if (odd16<T>((unsigned)va[db][e] << 16)) va[db][e] = 0;
            }
          }
#pragma unroll
          for (int db = 0; db < NDB; db++) o[db] = mma_pv<T>(va[db], __builtin_bit_cast(VT8, pb[s2]), o[db]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the V slot's reads are done
        if (!next) break;
        load(a.vc, lds0 + C::BYTES, vgo, blk + NW, pg0, pg1);
      }
    }

    // the waves' states meet: each leaves O, m and l, then a thread takes 8 channels of a row
    const float lt = l + __shfl_xor(l, 32);
    __syncthreads();
    char *orow = smem + (w * RT + l32) * C::ORS;
#pragma unroll
    for (int db = 0; db < NDB; db++)
#pragma unroll
      for (int g = 0; g < 4; g++)
        store4<T_F32>(orow + (db * 32 + 8 * g + 4 * hl) * 4, o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2],
                      o[db][4 * g + 3]);
    float *ml = (float *)(smem + NW * RT * C::ORS);
    if (hl == 0) *(float2 *)(ml + (w * RT + l32) * 2) = make_float2(m, lt);
    if (CAUSAL) odd = __syncthreads_or(odd);
    else __syncthreads();
    constexpr int PPR = DG / 8;
    for (int c = tid; c < R * PPR; c += NW * 64) {
      const int r = c / PPR, d0 = 8 * (c - r * PPR);
      const int rt = (int)((unsigned)r / (unsigned)hd.GP), rg = r - rt * hd.GP;
      if (g0 + rg >= hd.G) continue;
      float2 s[NW];
      float mx = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int k = 0; k < NW; k++) {
        s[k] = *(const float2 *)(ml + (k * RT + r) * 2);
        mx = fmaxf(mx, s[k].x);
      }
      float v[8] = {};
#pragma unroll
      for (int k = 0; k < NW; k++) {
        // a sum of 0: nothing was seen (a sum of NaN counts, whatever its maximum)
        const float wt = s[k].y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(s[k].x - mx);
        sum += wt * s[k].y;
        const char *pr = smem + (k * RT + r) * C::ORS + d0 * 4;
        const f32x4 lo = *(const f32x4 *)pr, hi = *(const f32x4 *)(pr + 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          v[e] += wt * lo[e];
          v[4 + e] += wt * hi[e];
        }
      }
      if (CAUSAL && __builtin_expect(odd, 0)) {  // the values left out above, from the first key that some row does not see
        const i64 seen = plan::clamp(q.off + m0 + rt + 1, 0, min(q.L, (i64)blk1 * KB));
        for (i64 key = max((i64)blk0 * KB, max(first_last + 1, (i64)0) / KB * KB); key < seen; key++) {
          const int pg = bt.table[(size_t)tile.b * bt.width + (key >> bt.lg)];
          if (pg < 0 || pg >= bt.pages) continue;
          const size_t row = (((size_t)pg * p.KVH + kvh) << bt.lg) + (size_t)(key & ((1 << bt.lg) - 1));
          const i32x4 vv = *(const i32x4 *)(a.vc + row * C::RBG + d0 * 2);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const unsigned u = (unsigned)vv[e / 2] << (e & 1 ? 0 : 16);
            if (odd16<T>(u)) v[e] += (u & (T == T_BF16 ? 0x007F0000u : 0x03FF0000u)) ? NAN : (int)u < 0 ? -INFINITY : INFINITY;
          }
        }
      }
      if (EACH || whole) {
        // no sum although a key is visible: all scores are -infinity, and 0 / 0
        const bool any = CAUSAL ? q.L > 0 && q.off + m0 + rt >= 0 : q.L > 0;
        const float inv = sum != 0.0f ? 1.0f / sum : any ? NAN : 0.0f;
        char *dst = a.out + ((size_t)(m0 + rt) * p.o_stride + (size_t)(kvh * hd.G + g0 + rg) * DG + d0) * 2;
        store4<T>(dst, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
        store4<T>(dst + 8, v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
      } else {
        store4<T_F32>((char *)(st + r * DG + d0), v[0], v[1], v[2], v[3]);
        store4<T_F32>((char *)(st + r * DG + d0 + 4), v[4], v[5], v[6], v[7]);
        if (d0 == 0) *(float2 *)(st + RT * DG + 2 * r) = make_float2(mx, sum);
      }
    }
    __syncthreads();  // before the next tile's loads
  }
  if (!EACH && !unfinished && tid == 0) left_of(a, sl)->R = 0;
}

}  // namespace

// Two states for each slice of the tiles of 256 rows, one a compute unit.
size_t attention_paged_workspace_max(int cus) {
  return (size_t)std::max(cus, 1) * (2 * CHUNK_ROWS * (128 + 2) * sizeof(float) + sizeof(Left));
}

namespace {

template <int DG, int T, bool CAUSAL, int NW, bool EACH>
int run_rows(const Exec &ex, const AttnArgs &a, const Batch &bt, const PagedAttnParams &p, const plan::Shape &sh,
             const Heads &hd, unsigned grid, int least, std::string *err) {
  using C = Rows<DG, NW>;
  auto kern = attention_rows_kernel<DG, T, NW, CAUSAL, EACH>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    if (e != hipSuccess) {
      *err = std::string("hipFuncSetAttribute: ") + hipGetErrorString(e);
      return -1;
    }
    attr_set = true;
  }
  hipLaunchKernelGGL(kern, dim3(grid), dim3(NW * 64), C::LDS, ex.stream, a, bt, p, sh, hd, least);
  return 0;
}

template <int DG, int T, bool CAUSAL>
int run(int rows, const Exec &ex, const AttnArgs &a, const Batch &bt, const PagedAttnParams &p, std::string *err) {
  const plan::Choice c = plan::choose(plan::Call{p.M, p.B, p.H, p.KVH, p.max_q, p.max_kv}, DG, CAUSAL, rows,
                                      std::max(1, cu_count()), ex.ws_bytes);
  if (c.rows == CHUNK_ROWS) return launch_attention_chunk(DG, T, CAUSAL, ex, a, bt, p, c, err);
  const Heads hd = plan::heads_of(p.H, p.KVH, RT);
  const int least = 256;  // weight of a slice
  const plan::Shape sh{p.M, p.B, RT / hd.GP, p.KVH * hd.HS, CAUSAL, 128, (i64)bt.width << bt.lg};
  AttnArgs g = a;
  g.ws = (float *)ex.ws;
  g.left = (char *)ex.ws + (size_t)c.most * 2 * RT * (DG + 2) * sizeof(float);
  if (c.each && c.waves == 8) return run_rows<DG, T, CAUSAL, 8, true>(ex, g, bt, p, sh, hd, (unsigned)c.tiles, least, err);
  if (c.each) return run_rows<DG, T, CAUSAL, 4, true>(ex, g, bt, p, sh, hd, (unsigned)c.tiles, least, err);
  if (run_rows<DG, T, CAUSAL, 4, false>(ex, g, bt, p, sh, hd, (unsigned)c.most, least, err)) return -1;
  if (c.most > 1)
    hipLaunchKernelGGL((attention_join_kernel<DG, T, RT, 1>), dim3((unsigned)(c.most - 1), RT / 4), dim3(256), 0, ex.stream, g,
                       p.o_stride);
  return 0;
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
  if (lg < 0 || p.pages < 0 || p.width < 0 || (i64)p.width << lg > 0x7fffffffll) {
    *err = "bad cache: " + std::to_string(p.pages) + " pages of " + std::to_string(p.page) +
           " rows (a power of two from 16 to 256), " + std::to_string(p.width) +
           " in a row of the table (below 2^31 rows in all)";
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
  const AttnArgs g{a[0].ptr, a[1].ptr, a[2].ptr, a[3].ptr, nullptr, nullptr, nullptr};
  const Batch bt{(const int *)a[4].ptr, (const int *)a[5].ptr, (const int *)a[6].ptr, p.B, p.width, p.pages, lg};
  return pl.ival[0] ? run<D, T, true>(pl.ival[1], ex, g, bt, p, err) : run<D, T, false>(pl.ival[1], ex, g, bt, p, err);
}

template <int D>
LaunchFn pick(int t) {
  return t == P_BF16 ? launch<D, T_BF16> : launch<D, T_F16>;
}

}  // namespace

// Macros: HD (64, 96 or 128), IN_T (half | bfloat: queries, cache and output), CAUSAL, and ROWS, which names the rows of a
// tile, 32 or 256; 0 (the default) chooses them by the size.
bool make_attention_paged(const Macros &m, Pipeline *pl, std::string *err) {
  int hd, causal, rows;
  if (!macro_int(m, "HD", 128, &hd, err) || !macro_int(m, "CAUSAL", 1, &causal, err) || !macro_int(m, "ROWS", 0, &rows, err))
    return false;
  for (auto &kv : m)
    if (kv.first != "HD" && kv.first != "CAUSAL" && kv.first != "IN_T" && kv.first != "ROWS") {
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
  if (rows != 0 && rows != RT && rows != CHUNK_ROWS) {
    *err = "ROWS must be 0, 32 or 256";
    return false;
  }
  pl->launch = hd == 128 ? pick<128>(t) : hd == 96 ? pick<96>(t) : pick<64>(t);
  pl->ival[0] = causal != 0;
  pl->ival[1] = rows;
  pl->threads = 256;
  return true;
}

}  // namespace h3
