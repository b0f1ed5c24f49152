// The paged attention of long chunks for gfx950 (head dim 128): tiles of 256 (token, head) rows. Semantics and the cut of the
// work: attention_paged.hip.
//
// 4 waves per workgroup, one per SIMD, 64 rows each (two 32-row MFMA tiles that share every K and V operand), so that a tile
// reads its keys 8 times less often than 32-row tiles do. The pipeline is attention_wave.hip's: a wave runs the softmax of
// key block j between the matrix instructions of P V of block j - 1 and of the scores of block j + 1, sub-tile by sub-tile; the
// exponentials take the running maximum of the blocks before, and a block whose row sums outgrow the limit (or the first
// one) is computed again with its own; K and V come by LDS-direct loads two blocks ahead into rings of 4 blocks of 64 keys, one
// barrier a block. What is different here:
//  * A block's four 16-key groups lie on pages of their own. Their addresses are made 64 groups (16 blocks) at a time, one a
//    lane, from page numbers loaded 16 blocks before, and read lane by lane into the descriptors of the loads.
//  * Rows see keys up to one of their own: the blocks that some row does not see whole run in a loop of their own, which masks.
//  * V of those blocks is searched in LDS for infinities and NaN, which a weight of 0 would not keep out of a sum: they are taken
//    as 0, and the rows that see them get them at the end.
#include "paged_attn.h"

#include <algorithm>

namespace h3 {
namespace {

// P V MFMA with the accumulator in AGPRs, as assembly: the score MFMAs are built with VGPR results, and only O and Q live in the
// accumulation registers. A VALU access of O after it is preceded by o_fence; P is written a barrier earlier (the build
// checks both: isa_check.py).
template <int VT>
__device__ __forceinline__ void mma_pv_acc(f32x16 &acc, i16x8 a, typename Vec8<VT>::type b) {
  if constexpr (VT == T_BF16) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
  else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}
__device__ __forceinline__ void o_fence(f32x16 (&o)[2][4]) {  // a 16-pass result needs 18 wait states
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 4"
               : "+a"(o[0][0]), "+a"(o[0][1]), "+a"(o[0][2]), "+a"(o[0][3]), "+a"(o[1][0]), "+a"(o[1][1]),
                 "+a"(o[1][2]), "+a"(o[1][3]));
}

constexpr int NWC = 4;                    // waves per workgroup
constexpr int NU = 2;                     // 32-row tiles per wave
constexpr int RTC = NWC * 32 * NU;        // rows of a tile
static_assert(RTC == CHUNK_ROWS, "rows of a tile");
constexpr int D = 128, RB = D * 2;        // channels, bytes of a row
constexpr int NCH = RB / 32;              // score MFMAs per 32 x 32 tile
constexpr int NR = 4;                     // blocks of a ring
constexpr int KBYTES = BK * RB;           // a block of K or V
constexpr int VOFF = NR * KBYTES;
constexpr int LDSC = 2 * NR * KBYTES;
constexpr int GPB = BK / 16;              // 16-key groups of a block, one 1 KB load of a wave each
static_assert(KBYTES == GPB * NWC * 1024, "a wave loads 4 rows of each group");

// accepted growth of a row sum per key block: bf16 P (float's exponent range) and f16 P (largest finite 65504)
template <int VT>
constexpr float sum_limit() { return VT == T_F16 ? 0x1p15f : 0x1p30f; }

template <int VT>
__device__ __forceinline__ bool odd_high(unsigned v) {  // the 16-bit value in the high half is infinite or NaN
  constexpr unsigned E = VT == T_BF16 ? 0x7F800000u : 0x7C000000u;
  return (v & E) == E;
}

template <int VT, bool CAUSAL>
__global__ __launch_bounds__(NWC * 64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void attention_chunk_kernel(AttnArgs a, Batch bt, PagedAttnParams p, plan::Shape sh, Heads hd, int least) {
  using VT8 = typename Vec8<VT>::type;
  using VE = typename Vec8<VT>::elem;
  using VP2 = typename Vec8<VT>::pair;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;
  const int tid = threadIdx.x, lane = tid & 63, hl = lane >> 5, l32 = lane & 31;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  const Order order(sh, bt);
  plan::Cut cut{1, (int)(order.all < (i64)gridDim.x ? order.all : (i64)gridDim.x), 0};
  if (!sh.each) cut = plan::cut(order.all, order.tiles, gridDim.x, least);
  if (order.all <= 0 || (int)blockIdx.x >= cut.n) {
    if (!sh.each && tid == 0) left_of(a, blockIdx.x)->R = 0;
    return;
  }
  int sl = slice_of(blockIdx.x, cut.n);
  if (sh.each) sl = cut.n - 1 - sl;  // with a causal mask the longest tiles go first
  const i64 x0 = plan::slice_start(cut, sl), x1 = plan::slice_start(cut, sl + 1);

  // this lane's 16 bytes of each 1 KB load, within a group of 16 rows: row and swizzled piece (attention_common.h: kswz, voff)
  const int lrow = w * 4 + (lane >> 4);
  const unsigned kgo = lrow * RB + ((lane & 15) ^ lrow) * 16;
  const unsigned vgo = lrow * RB + (2 * (((lane & 15) >> 1) ^ (2 * (lrow & 3))) + (lane & 1)) * 16;
  const int krow = 16 * (l32 >> 4) + 8 * ((l32 >> 2) & 1) + 4 * ((l32 >> 3) & 1) + (l32 & 3);
  const int l16 = lane & 15, tr_row = l16 >> 2, tr_col = (l16 & 3) * 8;
  unsigned vbase[D / 32], kbase[NCH];
#pragma unroll
  for (int db = 0; db < D / 32; db++) vbase[db] = voff<D>(8 * hl + tr_row, (db * 32 + (l32 & 16)) / 8) + tr_col;
#pragma unroll
  for (int c = 0; c < NCH; c++) kbase[c] = krow * RB + (((2 * c + hl) ^ kswz<RB, RB / 16>(krow)) * 16);

  Tile tile;
  bool unfinished = false;
  bool more = tile_at(order, x0, &tile);
  for (; more && tile.p < x1; more = next_tile(order, &tile)) {
    const plan::Seq &q = tile.q;
    const int all = plan::tile_blocks(sh, q, tile.t, BK);
    int blk0 = 0, blk1 = all;
    bool begun = false, whole = true;
    if (!sh.each) {
      blk0 = plan::block_at(x0, tile.p, tile.w, all);
      blk1 = plan::block_at(x1, tile.p, tile.w, all);
      begun = tile.p < x0;
      whole = !begun && tile.p + tile.w <= x1;
    }
    blk0 = __builtin_amdgcn_readfirstlane(blk0);
    const int nblk = __builtin_amdgcn_readfirstlane(blk1 - blk0);
    const int kvh = tile.v / hd.HS, g0 = (tile.v - kvh * hd.HS) * hd.GP;
    const int m0 = q.lo + tile.t * sh.TT, R = min(sh.TT, q.hi - m0) * hd.GP;
    const int L = (int)q.L;
    const i64 first_last = CAUSAL ? plan::clamp(q.off + m0, -M_MOST, q.L - 1) : q.L - 1;  // last key of the tile's first token
    float *st = a.ws + (size_t)plan::state_of(sl, begun) * (RTC * (D + 2));
    if (!whole && !begun) {
      const int end = last_slice(cut, sl, tile.p + tile.w);
      if (tid == 0)
        *left_of(a, sl) = Left{R, m0, kvh * hd.G + g0, hd.GP, min(hd.GP, hd.G - g0),
                               q.L > 0 ? CAUSAL ? (int)first_last : 0 : -M_MOST, end, 0};
      unfinished = true;
    }
    if (blk0 == blk1) {  // a part without blocks (a whole tile has one)
      if (tid < R) *(float2 *)(st + RTC * D + 2 * tid) = make_float2(-INFINITY, 0.0f);
      continue;
    }
    // blocks (from blk0 on) that every row sees whole
    const int clear = __builtin_amdgcn_readfirstlane((int)plan::clamp(max(first_last + 1, (i64)0) / BK - blk0, 0, nblk));

    // Q operands (B of S^T = K Q^T) and the last visible key of this lane's rows
    i32x4 qreg[NU][NCH];
    int last[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) {
      const int r = w * (32 * NU) + 32 * u + l32;
      const int ti = (int)((unsigned)r / (unsigned)hd.GP), gi = r - ti * hd.GP;
      const bool ok = r < R && g0 + gi < hd.G;
      last[u] = !ok ? -1 : CAUSAL ? (int)plan::clamp(q.off + m0 + ti, -1, q.L - 1) : L - 1;
      const char *qrow = a.q + ((size_t)(m0 + (ok ? ti : 0)) * p.q_stride + (size_t)(kvh * hd.G + (ok ? g0 + gi : 0)) * D) * 2;
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        i32x4 v = *(const i32x4 *)(qrow + (2 * c + hl) * 16);
        qreg[u][c] = ok ? v : i32x4{0, 0, 0, 0};
        asm volatile("" : "+a"(qreg[u][c]));  // from here on Q lives in AGPRs only
      }
    }

    // -- staging. 64 groups of 16 keys (16 blocks from a multiple of 16 on, counted from blk0), one a lane: the offset of their rows
    // in either cache and the rows that are there; those of K (blocks up to j + 3) and those of V (up to j + 1)
    unsigned koff_lo, koff_hi, krows, voff_lo, voff_hi, vrows;
    i64 lost = 0x7fffffffffffffffll;  // the first key whose page number lies outside the cache
    auto group_key = [&](int win) __attribute__((always_inline)) { return ((i64)blk0 * GPB + win * 64 + lane) * 16; };
    auto fetch = [&](int win) __attribute__((always_inline)) {
      const i64 key = group_key(win);
      return key < L && key < (i64)blk1 * BK ? bt.table[(size_t)tile.b * bt.width + (key >> bt.lg)] : 0;
    };
    auto addresses = [&](int id, int win) __attribute__((always_inline)) {
      const i64 key = group_key(win);
      const bool there = key < L && key < (i64)blk1 * BK, in = id >= 0 && id < bt.pages;
      const unsigned long long bad = __ballot(there && !in);
      if (__builtin_expect(bad != 0, 0)) lost = min(lost, ((i64)blk0 * GPB + win * 64 + __builtin_ctzll(bad)) * 16);
      const unsigned long long off =
          ((((unsigned long long)(there && in ? id : 0) * p.KVH + kvh) << bt.lg) + (key & ((1 << bt.lg) - 1))) * RB;
      koff_lo = (unsigned)off;
      koff_hi = (unsigned)(off >> 32);
      krows = there && in ? (unsigned)plan::clamp(L - key, 0, 16) : 0;
    };
    int ahead;  // page numbers of the window behind K's
    auto windows = [&](int j) __attribute__((always_inline)) {  // before the loads of step j
      if (((j + 1) & 15) == 0) {
        voff_lo = koff_lo;
        voff_hi = koff_hi;
        vrows = krows;
      }
      if (((j + 3) & 15) == 0) {
        addresses(ahead, (j + 3) >> 4);
        ahead = fetch(((j + 3) >> 4) + 1);
      }
    };
    auto rsrc = [&](const char *base, unsigned lo, unsigned hi, unsigned rows, int at) __attribute__((always_inline)) {
      const unsigned long long off = (unsigned)__builtin_amdgcn_readlane((int)lo, at) |
                                     (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)hi, at) << 32;
      return __builtin_amdgcn_make_buffer_rsrc((void *)(base + off), (short)0,
                                               __builtin_amdgcn_readlane((int)rows, at) * RB, 0x00020000);
    };
    // load i < 4: group i of K of block kb; from 4 on: of V of block vb
    auto stage_one = [&](int i, int kb, int vb) __attribute__((always_inline)) {
      if (i < GPB) {
        dma16(lds0 + (kb & (NR - 1)) * KBYTES + (i * NWC + w) * 1024, kgo,
              rsrc(a.kc, koff_lo, koff_hi, krows, (kb & 15) * GPB + i));
      } else {
        const int r = i - GPB;
        dma16(lds0 + VOFF + (vb & (NR - 1)) * KBYTES + (r * NWC + w) * 1024, vgo,
              rsrc(a.vc, voff_lo, voff_hi, vrows, (vb & 15) * GPB + r));
      }
    };

    f32x16 o[NU][D / 32];
    float m[NU], l[NU], nmv[NU], la[NU][4];  // maximum, sum, -maximum (0 at -inf), running partial sums
#pragma unroll
    for (int u = 0; u < NU; u++) {
#pragma unroll
      for (int db = 0; db < D / 32; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[u][db][i] = 0.0f;
      m[u] = -INFINITY;
      l[u] = nmv[u] = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; c++) la[u][c] = 0.0f;
    }
    f32x16 s[2][NU];     // scores [key tile t][row tile u]
    i32x4 pb[2][NU][2];  // weights [t][u][16-key step]
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int u = 0; u < NU; u++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[t][u][i] = 0.0f;
        pb[t][u][0] = pb[t][u][1] = i32x4{0, 0, 0, 0};
      }
    bool odd = false;

    struct Ops {  // operands of one key tile of a step: V of block j - 1 (index 4 * s2 + db), K of block j + 1
      i16x8 va[8];
      i32x4 ka[NCH];
    };
    auto vread = [&](int j, int t, int k) __attribute__((always_inline)) {
      const char *Vs = smem + VOFF + (j & (NR - 1)) * KBYTES + (32 * t + 16 * (k >> 2)) * RB + vbase[k & 3];
      const i16x4 lo = lds_tr16(Vs);
      const i16x4 hi = lds_tr16(Vs + 4 * RB);
      return i16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto kread = [&](int j, int t, int c) __attribute__((always_inline)) {
      return *(const i32x4 *)(smem + (j & (NR - 1)) * KBYTES + 32 * t * RB + kbase[c]);
    };
    // keys that this lane's row u does not see: element i holds key BK (blk0 + j) + 32 t + 16 (i / 8) + 8 hl + i % 8
    auto beyond = [&](int j, int u) __attribute__((always_inline)) { return last[u] - 8 * hl - (blk0 + j) * BK; };
    // this wave's own loads of V of block j, landed: infinities and NaN out
    auto clean = [&](int j) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < GPB; r++) {
        i32x4 *at = (i32x4 *)(smem + VOFF + (j & (NR - 1)) * KBYTES + (r * NWC + w) * 1024 + 16 * lane);
        i32x4 v = *at;
        bool some = false;
#pragma unroll
        for (int e = 0; e < 4; e++) some |= odd_high<VT>((unsigned)v[e]) | odd_high<VT>((unsigned)v[e] << 16);
        if (__builtin_expect(__any(some), 0)) {
          odd = true;
#pragma unroll
          for (int e = 0; e < 4; e++) {
            unsigned d = (unsigned)v[e];
            if (odd_high<VT>(d)) d &= 0xFFFFu;
            if (odd_high<VT>(d << 16)) d &= 0xFFFF0000u;
            v[e] = (int)d;
          }
          *at = v;
        }
      }
    };

    // One (key tile t, row tile u) of step j, in issue order: P V of block j - 1 and scores of block j + 1 spread between runs of
    // independent VALU work on block j. With `refresh` each operand is replaced by the next tile's (jn, tn) after its last use.
    auto sub_tile = [&](Ops &op, int j, int t, int u, bool has_pv, bool has_next, bool mask, bool refresh, int jn, int tn,
                        int nst) __attribute__((always_inline)) {
      const float nm = nmv[u];
      const int see = mask ? beyond(j, u) : 0;
      float xv[16];
      int npv = 0, ns = 0;
      auto pv = [&]() __attribute__((always_inline)) {
        const int k = npv++;
        if (has_pv) mma_pv_acc<VT>(o[u][k & 3], op.va[k], __builtin_bit_cast(VT8, pb[t][u][k >> 2]));
        if (refresh) op.va[k] = vread(jn - 1, tn, k);
        if (k < nst) stage_one(k, j + 3, j + 1);
      };
      auto sm = [&]() __attribute__((always_inline)) {
        const int c = ns++;
        f32x16 zero;
#pragma unroll
        for (int i = 0; i < 16; i++) zero[i] = 0.0f;
        if (has_next) s[t][u] = mma_qk<VT>(op.ka[c], qreg[u][c], c == 0 ? zero : s[t][u]);
        if (refresh) op.ka[c] = kread(jn + 1, tn, c);
      };
      auto cv = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int i = 4 * g + e;
          xv[i] = s[t][u][i];
          if (mask && 32 * t + 16 * (i >> 3) + (i & 7) > see) xv[i] = -INFINITY;
        }
      };
      auto fm = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) xv[4 * g + e] = fmaf(xv[4 * g + e], p.scale, nm);
      };
      auto ex = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; e++) xv[4 * g + e] = __builtin_amdgcn_exp2f(xv[4 * g + e]);
      };
      auto pk = [&](int g) __attribute__((always_inline)) {  // round to the value type, sum the rounded weights
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int i = 4 * g + e;
          const VP2 pp = {(VE)xv[i], (VE)xv[i + 1]};
          pb[t][u][i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, pp);
          la[u][(g & 1) * 2 + (e >> 1)] = sum2<VT>(pp, la[u][(g & 1) * 2 + (e >> 1)]);
        }
      };
#define SB __builtin_amdgcn_sched_barrier(0)
      pv(); cv(0); cv(1); SB; pv(); fm(0); SB; pv(); fm(1); SB; pv(); cv(2); cv(3); ex(0); SB; pv(); fm(2); SB;
      pv(); ex(1); SB; pv(); fm(3); SB; pv(); ex(2); SB; sm(); pk(0); SB; sm(); ex(3); SB; sm(); pk(1); SB;
      sm(); SB; sm(); pk(2); SB; sm(); SB; sm(); pk(3); SB; sm(); SB;
#undef SB
    };

    // Step j: P V of block j - 1, softmax of block j, scores of block j + 1. The barrier sits before the last sub-tile: the loads
    // behind it (K of block j + 3, V of block j + 1) land during the next step, and the last sub-tile reads the next step's
    // first operands. Ring slots: K(j + 3) replaces K(j - 1), V(j + 1) V(j - 3).
    auto step = [&](Ops &op, int j, bool has_pv, bool has_next, bool mask) __attribute__((always_inline)) {
      float tot[NU];
      bool bad = false;
      windows(j);
#pragma unroll
      for (int idx = 0; idx < 2 * NU - 1; idx++) {
        const int t = idx / NU, u = idx % NU;
        sub_tile(op, j, t, u, has_pv, has_next, mask, u == NU - 1, t == 0 ? j : j + 1, t == 0 ? 1 : 0, 0);
        if (t == 1) {
          tot[u] = (la[u][0] + la[u][1]) + (la[u][2] + la[u][3]);
          bad = bad | !(tot[u] - l[u] <= sum_limit<VT>());
        }
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the previous step
      if (CAUSAL && mask) clean(j);
      __syncthreads();
      sub_tile(op, j, 1, NU - 1, has_pv, has_next, mask, true, j + 1, 0, 2 * GPB);
      tot[NU - 1] = (la[NU - 1][0] + la[NU - 1][1]) + (la[NU - 1][2] + la[NU - 1][3]);
      bad = bad | !(tot[NU - 1] - l[NU - 1] <= sum_limit<VT>());
      // rare: a score far above the running maximum, or the first block: block j's weights again with the exact maximum (its K is
      // still in its ring slot). A row that sees no key of the first block sees none of the later ones either.
      if (__builtin_expect(j == 0 || __builtin_amdgcn_ballot_w64(bad) != 0, 0)) {
        o_fence(o);  // P V MFMAs of this step may still be writing O
#pragma unroll
        for (int u = 0; u < NU; u++) {
          f32x16 xs[2];
          float bmax = -INFINITY;
#pragma unroll
          for (int t = 0; t < 2; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) xs[t][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; c++) xs[t] = mma_qk<VT>(kread(j, t, c), qreg[u][c], xs[t]);
            if (mask) {
              const int see = beyond(j, u);
#pragma unroll
              for (int i = 0; i < 16; i++)
                if (32 * t + 16 * (i >> 3) + (i & 7) > see) xs[t][i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) bmax = fmaxf(bmax, xs[t][i]);
          }
          const float mn = fmaxf(m[u], fmaxf(bmax, __shfl_xor(bmax, 32)) * p.scale);
          const float f = (m[u] == -INFINITY || mn == -INFINITY) ? 1.0f : __builtin_amdgcn_exp2f(m[u] - mn);
          m[u] = mn;
          l[u] *= f;
#pragma unroll
          for (int db = 0; db < D / 32; db++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[u][db][i] *= f;
          const float nm = mn == -INFINITY ? 0.0f : -mn;
          nmv[u] = nm;
          float add[2] = {0.0f, 0.0f};
#pragma unroll
          for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const VP2 pp = {(VE)__builtin_amdgcn_exp2f(fmaf(xs[t][i], p.scale, nm)),
                              (VE)__builtin_amdgcn_exp2f(fmaf(xs[t][i + 1], p.scale, nm))};
              pb[t][u][i >> 3][(i & 7) >> 1] = __builtin_bit_cast(int, pp);
              add[t] = sum2<VT>(pp, add[t]);
            }
          tot[u] = l[u] + (add[0] + add[1]);
          la[u][0] = tot[u];
          la[u][1] = la[u][2] = la[u][3] = 0.0f;
        }
        asm volatile("s_nop 2" ::: "memory");  // VALU writes of O before the next MFMA reads it
      }
#pragma unroll
      for (int u = 0; u < NU; u++) l[u] = tot[u];
    };

    ahead = fetch(0);
    addresses(ahead, 0);
    voff_lo = koff_lo;
    voff_hi = koff_hi;
    vrows = krows;
    ahead = fetch(1);
#pragma unroll
    for (int b = 0; b < 3; b++)
#pragma unroll
      for (int i = 0; i < GPB; i++) stage_one(i, b, 0);
#pragma unroll
    for (int i = 0; i < GPB; i++) stage_one(GPB + i, 0, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (CAUSAL && clear == 0) clean(0);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int u = 0; u < NU; u++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[t][u][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; c++) s[t][u] = mma_qk<VT>(kread(0, t, c), qreg[u][c], s[t][u]);
      }
    Ops op;
#pragma unroll
    for (int k = 0; k < 8; k++) op.va[k] = vread(-1, 0, k);  // (not used: there is no P V yet)
#pragma unroll
    for (int c = 0; c < NCH; c++) op.ka[c] = kread(1, 0, c);
    if (nblk == 1) {
      step(op, 0, false, false, true);
    } else {
      step(op, 0, false, true, true);
      int j = 1;
      for (; j < min(clear, nblk - 1); j++) step(op, j, true, true, false);
      for (; j < nblk - 1; j++) step(op, j, true, true, true);
      step(op, nblk - 1, true, false, true);
    }
    // P V of the last block (its tile-0 V operands were read by the last step)
#pragma unroll
    for (int t = 0; t < 2; t++) {
      if (t == 1) {
#pragma unroll
        for (int k = 0; k < 8; k++) op.va[k] = vread(nblk - 1, 1, k);
      }
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int k = 0; k < 8; k++) mma_pv_acc<VT>(o[u][k & 3], op.va[k], __builtin_bit_cast(VT8, pb[t][u][k >> 2]));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads past the last block land before the slots are used again
    o_fence(o);

#pragma unroll
    for (int u = 0; u < NU; u++) {
      const int r = w * (32 * NU) + 32 * u + l32;
      const int ti = (int)((unsigned)r / (unsigned)hd.GP), gi = r - ti * hd.GP;
      float sum = l[u] + __shfl_xor(l[u], 32);
      if (last[u] >= lost) sum = NAN;
      if (r >= R || g0 + gi >= hd.G) continue;
      if (whole) {
        // no sum although a key is visible: all scores are -infinity, and 0 / 0
        const float inv = sum != 0.0f ? 1.0f / sum : last[u] >= 0 ? NAN : 0.0f;
        char *dst = a.out + ((size_t)(m0 + ti) * p.o_stride + (size_t)(kvh * hd.G + g0 + gi) * D) * 2;
#pragma unroll
        for (int db = 0; db < D / 32; db++)
#pragma unroll
          for (int g = 0; g < 4; g++)
            store4<VT>(dst + (db * 32 + 8 * g + 4 * hl) * 2, o[u][db][4 * g] * inv, o[u][db][4 * g + 1] * inv,
                       o[u][db][4 * g + 2] * inv, o[u][db][4 * g + 3] * inv);
      } else {
#pragma unroll
        for (int db = 0; db < D / 32; db++)
#pragma unroll
          for (int g = 0; g < 4; g++)
            store4<T_F32>((char *)(st + r * D + db * 32 + 8 * g + 4 * hl), o[u][db][4 * g], o[u][db][4 * g + 1],
                          o[u][db][4 * g + 2], o[u][db][4 * g + 3]);
        if (hl == 0) *(float2 *)(st + RTC * D + 2 * r) = make_float2(m[u], sum);
      }
    }
    if (CAUSAL) odd = __syncthreads_or(odd);
    else __syncthreads();
    if (CAUSAL && __builtin_expect(odd, 0)) {  // the values left out above, for the rows that see them
      __threadfence_block();
      for (int c = tid; c < R * (D / 8); c += NWC * 64) {
        const int r = c / (D / 8), d0 = 8 * (c - r * (D / 8));
        const int ti = (int)((unsigned)r / (unsigned)hd.GP), gi = r - ti * hd.GP;
        if (g0 + gi >= hd.G) continue;
        const i64 seen = plan::clamp(q.off + m0 + ti + 1, 0, min(q.L, (i64)blk1 * BK));
        float v[8] = {};
        bool some = false;
        for (i64 key = (i64)(blk0 + clear) * BK; key < seen; key++) {
          const int pg = bt.table[(size_t)tile.b * bt.width + (key >> bt.lg)];
          if (pg < 0 || pg >= bt.pages) continue;
          const size_t row = (((size_t)pg * p.KVH + kvh) << bt.lg) + (size_t)(key & ((1 << bt.lg) - 1));
          const i32x4 vv = *(const i32x4 *)(a.vc + row * RB + d0 * 2);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const unsigned x = (unsigned)vv[e / 2] << (e & 1 ? 0 : 16);
            if (odd_high<VT>(x)) {
              v[e] += x & (VT == T_BF16 ? 0x007F0000u : 0x03FF0000u) ? NAN : (int)x < 0 ? -INFINITY : INFINITY;
              some = true;
            }
          }
        }
        if (!some) continue;
        if (whole) {
          VE *dst = (VE *)a.out + (size_t)(m0 + ti) * p.o_stride + (size_t)(kvh * hd.G + g0 + gi) * D + d0;
#pragma unroll
          for (int e = 0; e < 8; e++) dst[e] = (VE)((float)dst[e] + v[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) st[r * D + d0 + e] += v[e];
        }
      }
    }
  }
  if (!sh.each && !unfinished && tid == 0) left_of(a, sl)->R = 0;
}

template <int VT, bool CAUSAL>
int run(const Exec &ex, const AttnArgs &a, const Batch &bt, const PagedAttnParams &p, std::string *err) {
  auto kern = attention_chunk_kernel<VT, CAUSAL>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, LDSC);
    if (e != hipSuccess) {
      *err = std::string("hipFuncSetAttribute: ") + hipGetErrorString(e);
      return -1;
    }
    attr_set = true;
  }
  const int G = p.H / p.KVH, HS = (G + RTC - 1) / RTC, GP = (G + HS - 1) / HS, TT = RTC / GP;
  const Heads hd{G, HS, GP};
  const int cus = std::max(1, cu_count());
  const i64 tiles = (i64)p.KVH * HS * std::min<i64>(p.M, ((i64)p.M + (i64)p.B * (TT - 1)) / TT);
  const size_t state = (size_t)2 * RTC * (D + 2) * sizeof(float) + sizeof(Left);  // of a slice
  const int least = 512, most = std::max(1, (int)std::min<i64>(cus, (i64)(ex.ws_bytes / state)));
  const bool each = tiles <= 1 << 22 && tiles >= 3 * most;
  const plan::Shape sh{p.M, p.B, TT, p.KVH * HS, CAUSAL, each, 256, (i64)bt.width << bt.lg};
  AttnArgs g = a;
  g.ws = (float *)ex.ws;
  g.left = (char *)ex.ws + most * (state - sizeof(Left));
  hipLaunchKernelGGL(kern, dim3((unsigned)(each ? tiles : most)), dim3(NWC * 64), LDSC, ex.stream, g, bt, p, sh, hd, least);
  if (!each && most > 1)
    hipLaunchKernelGGL((attention_join_kernel<D, VT, RTC, 4>), dim3((unsigned)(most - 1), RTC / 16), dim3(256), 0, ex.stream, g,
                       p.o_stride);
  return 0;
}

}  // namespace

int launch_attention_chunk(int t, bool causal, const Exec &ex, const AttnArgs &a, const Batch &bt, const PagedAttnParams &p,
                           std::string *err) {
  if (t == T_BF16) return causal ? run<T_BF16, true>(ex, a, bt, p, err) : run<T_BF16, false>(ex, a, bt, p, err);
  return causal ? run<T_F16, true>(ex, a, bt, p, err) : run<T_F16, false>(ex, a, bt, p, err);
}

}  // namespace h3
