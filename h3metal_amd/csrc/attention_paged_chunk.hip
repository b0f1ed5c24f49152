// The paged attention of long chunks for gfx950: tiles of 256 (token, head) rows. Semantics and the cut of the work:
// attention_paged.hip.
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
//    as 0, and the rows that see them get them at the end. So is what a page holds behind the sequence's end.
// LDS rows of head dim 96 are as wide as those of 128 (what is behind its channels is never read); a step has as many slots for
// instructions and loads at every head dim, some of them empty.
// A prompt of 8192 tokens (32 + 8 heads) takes 500 us, 1.1 PFLOP/s, a large library product's rate on the same card; a step of
// 64 keys 2.1 us, of which its 64 matrix instructions would take 0.9: the softmax's instructions beside them bound it. A tile
// starts and ends in about 15 us, so code is kept in two copies only and everything of a start is asked for at once. A
// prompt of 4096 tokens takes 135 us at head dim 128 (1.02 PFLOP/s), 121 at 96 (0.85) and 93 at 64 (0.74), where as many
// exponentials stand beside half the matrix instructions. The kernel that takes whole tiles uses no scratch memory; the one that
// takes slices keeps the order of tiles beside them and spills at head dim 128 (61 vector registers with a causal mask, 46
// without; scalars at every head dim), in a tile's start and end and the rare path, not in the steps themselves.
#include "paged_attn.h"

#include <algorithm>
#include <cfloat>

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
template <int NDB>
__device__ __forceinline__ void o_fence(f32x16 (&o)[2][NDB]) {  // a 16-pass result needs 18 wait states
  if constexpr (NDB == 4)
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 4"
                 : "+a"(o[0][0]), "+a"(o[0][1]), "+a"(o[0][2]), "+a"(o[0][3]), "+a"(o[1][0]), "+a"(o[1][1]),
                   "+a"(o[1][2]), "+a"(o[1][3]));
  else if constexpr (NDB == 3)
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 4"
                 : "+a"(o[0][0]), "+a"(o[0][1]), "+a"(o[0][2]), "+a"(o[1][0]), "+a"(o[1][1]), "+a"(o[1][2]));
  else
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 4" : "+a"(o[0][0]), "+a"(o[0][1]), "+a"(o[1][0]), "+a"(o[1][1]));
}

constexpr int NWC = 4;                    // waves per workgroup
constexpr int NU = 2;                     // 32-row tiles per wave
constexpr int RTC = NWC * 32 * NU;        // rows of a tile
static_assert(RTC == CHUNK_ROWS, "rows of a tile");
constexpr int NR = 4;                     // blocks of a ring
constexpr int GPB = BK / 16;              // 16-key groups of a block

template <int DG>
struct Chunk {
  static constexpr int D = DG == 96 ? 128 : DG;              // channels of an LDS row
  static constexpr int RB = D * 2, RBG = DG * 2;             // bytes of a row: in LDS, in memory
  static constexpr int NCH = DG / 16, NDB = DG / 32;         // score MFMAs per 32 x 32 tile, 32-channel blocks of O
  static constexpr int KBYTES = BK * RB, VOFF = NR * KBYTES;  // a block of K or V; the V ring
  static constexpr int LPB = KBYTES / (NWC * 1024);          // 1 KB loads of a wave and block
  static constexpr int S16 = DG * 2 + 8, S32 = DG * 4 + 16;  // bytes between output rows in LDS
  static constexpr int LDS = RTC * S32 > 2 * VOFF ? RTC * S32 : 2 * VOFF;  // rings, then outputs
  static_assert(LPB == 4 || LPB == 2, "a load holds 4 or 8 rows of a group");
};

// accepted growth of a row sum per key block: bf16 P (float's exponent range) and f16 P (largest finite 65504)
template <int VT>
constexpr float sum_limit() { return VT == T_F16 ? 0x1p15f : 0x1p30f; }

struct __attribute__((packed, aligned(8))) Piece {  // 16 bytes of an output row, whose rows are aligned to 8
  float v[4];
};

template <int D, int VT, bool CAUSAL, bool EACH>
__global__ __launch_bounds__(NWC * 64) __attribute__((amdgpu_waves_per_eu(1, 1)))
void attention_chunk_kernel(AttnArgs a, Batch bt, PagedAttnParams p, plan::Shape sh, Heads hd, int least) {
  using C = Chunk<D>;
  constexpr int RB = C::RB, NCH = C::NCH, NDB = C::NDB, KBYTES = C::KBYTES, VOFF = C::VOFF, LPB = C::LPB;
  using VT8 = typename Vec8<VT>::type;
  using VE = typename Vec8<VT>::elem;
  using VP2 = typename Vec8<VT>::pair;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char *)smem;
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

  // this lane's 16 bytes of each 1 KB load, within a group of 16 rows: row and swizzled piece (attention_common.h: kswz, voff);
  // what lies past a row in memory (head dim 96) is never read and takes another piece of it
  constexpr int NP = RB / 16, R1 = 64 / NP, RW = 256 / RB;  // pieces of a row, rows of a load, of 256 bytes
  const int lrow = (w * R1 + lane / NP) & 15, lpc = lane % NP;
  const int kp = lpc ^ kswz<RB, NP>(lrow), vp = 2 * ((lpc >> 1) ^ (2 * ((lrow & 3) / RW))) + (lpc & 1);
  const unsigned kgo = lrow * C::RBG + (kp * 16 < C::RBG ? kp : kp - NP / 2) * 16;
  const unsigned vgo = lrow * C::RBG + (vp * 16 < C::RBG ? vp : vp - NP / 2) * 16;
  auto group_of = [&](int r) __attribute__((always_inline)) { return (r * NWC + w) * R1 / 16; };  // of load r of a block
  const int krow = 16 * (l32 >> 4) + 8 * ((l32 >> 2) & 1) + 4 * ((l32 >> 3) & 1) + (l32 & 3);
  const int l16 = lane & 15, tr_row = l16 >> 2, tr_col = (l16 & 3) * 8;
  unsigned vbase[NDB], kbase[NCH];
#pragma unroll
  for (int db = 0; db < NDB; db++) vbase[db] = voff<C::D>(8 * hl + tr_row, (db * 32 + (l32 & 16)) / 8) + tr_col;
#pragma unroll
  for (int c = 0; c < NCH; c++) kbase[c] = krow * RB + (((2 * c + hl) ^ kswz<RB, RB / 16>(krow)) * 16);

  const float per_token = 1.0f / (float)hd.GP;
  auto row_token = [&](int r) __attribute__((always_inline)) { return (int)(((float)r + 0.5f) * per_token); };  // r / GP

  bool unfinished = false;
  auto next = [&]() {
    if constexpr (EACH) return false;
    else return next_tile(order, &tile) && tile.p < x1;
  };
  if (!EACH) more = more && tile.p < x1;
  for (; more; more = next()) {
    const plan::Seq &q = tile.q;
    const int all = plan::tile_blocks(sh, q, tile.t, BK);
    int blk0 = 0, blk1 = all;
    bool begun = false, whole = true;
    if constexpr (!EACH) {
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
    if (!EACH && !whole && !begun) {
      const int end = last_slice(cut, sl, tile.p + tile.w);
      if (tid == 0)
        *left_of(a, sl) = Left{R, m0, kvh * hd.G + g0, hd.GP, min(hd.GP, hd.G - g0),
                               q.L > 0 ? CAUSAL ? (int)first_last : 0 : -M_MOST, end, 0};
      unfinished = true;
    }
    if (!EACH && blk0 == blk1) {  // a part without blocks (a whole tile has one)
      if (tid < R) *(float2 *)(st + RTC * D + 2 * tid) = make_float2(-INFINITY, NO_PART);
      continue;
    }
    // blocks (from blk0 on) that every row sees whole
    const int clear = __builtin_amdgcn_readfirstlane((int)plan::clamp(max(first_last + 1, (i64)0) / BK - blk0, 0, nblk));

    // Q operands (B of S^T = K Q^T), and the last visible key of this lane's rows
    i32x4 qreg[NU][NCH];
    int last[NU];
    const char *qrow[NU];
    bool ok[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) {
      const int r = w * (32 * NU) + 32 * u + l32;
      const int ti = row_token(r), gi = r - ti * hd.GP;
      ok[u] = r < R && g0 + gi < hd.G;
      // (a lane without a row looks at every key with a query of zeros, so that it never asks for a block to be done again)
      last[u] = ok[u] && CAUSAL ? (int)plan::clamp(q.off + m0 + ti, -1, q.L - 1) : L - 1;
      qrow[u] = a.q + ((size_t)(m0 + (ok[u] ? ti : 0)) * p.q_stride + (size_t)(kvh * hd.G + (ok[u] ? g0 + gi : 0)) * D) * 2;
    }

    // -- staging. The addresses of 64 groups of 16 keys (16 blocks from a multiple of 16 on, counted from blk0), one a lane: those
    // of K (blocks up to j + 3), those of V beside them, and those of V still in use (up to j + 1). Groups past the sequence and
    // those whose page number lies outside the cache take other memory, which their rows' masks or `lost` keep out.
    unsigned k_lo, k_hi, v_lo, v_hi, vnext_lo, vnext_hi;
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
          ((((unsigned long long)id * p.KVH + kvh) << bt.lg) + (key & ((1 << bt.lg) - 1))) * C::RBG;
      const unsigned long long ka = (unsigned long long)(there && in ? a.kc + off : a.spare);
      const unsigned long long va = (unsigned long long)(there && in ? a.vc + off : a.spare);
      k_lo = (unsigned)ka;
      k_hi = (unsigned)(ka >> 32);
      vnext_lo = (unsigned)va;
      vnext_hi = (unsigned)(va >> 32);
    };
    int ahead;  // page numbers of the window behind K's
    auto windows = [&](int j) __attribute__((always_inline)) {  // before the loads of step j
      if (((j + 1) & 15) == 0) {
        v_lo = vnext_lo;
        v_hi = vnext_hi;
      }
      if (((j + 3) & 15) == 0) {
        addresses(ahead, (j + 3) >> 4);
        ahead = fetch(((j + 3) >> 4) + 1);
      }
    };
    auto stage = [&](unsigned lds, int add, unsigned go, unsigned lo, unsigned hi, int at) __attribute__((always_inline)) {
      const unsigned long long base = (unsigned)__builtin_amdgcn_readlane((int)lo, at) |
                                      (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)hi, at) << 32;
      // a lane value takes 5 wait states to reach a memory access as a scalar
      asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %2, %3" ::"s"(lds), "i"(add), "v"(go), "s"(base)
                   : "memory", "m0", "scc");
    };
    const unsigned lds_w = lds0 + w * 1024;
    // load i < LPB: of K of block kb; from there on: of V of block vb
    auto stage_one = [&](auto ic, int kb, int vb) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, r = i % LPB;
      if constexpr (i < LPB)
        stage(lds_w + (kb & (NR - 1)) * KBYTES, r * NWC * 1024, kgo, k_lo, k_hi, (kb & 15) * GPB + group_of(r));
      else if constexpr (i < 2 * LPB)
        stage(lds_w + (vb & (NR - 1)) * KBYTES, VOFF + r * NWC * 1024, vgo, v_lo, v_hi, (vb & 15) * GPB + group_of(r));
    };

    auto stage_k = [&](int k, int kb, int vb) __attribute__((always_inline)) {  // (k is known where this is inlined)
      switch (k) {
        case 0: stage_one(std::integral_constant<int, 0>{}, kb, vb); break;
        case 1: stage_one(std::integral_constant<int, 1>{}, kb, vb); break;
        case 2: stage_one(std::integral_constant<int, 2>{}, kb, vb); break;
        case 3: stage_one(std::integral_constant<int, 3>{}, kb, vb); break;
        case 4: stage_one(std::integral_constant<int, 4>{}, kb, vb); break;
        case 5: stage_one(std::integral_constant<int, 5>{}, kb, vb); break;
        case 6: stage_one(std::integral_constant<int, 6>{}, kb, vb); break;
        default: stage_one(std::integral_constant<int, 7>{}, kb, vb);
      }
    };

    f32x16 o[NU][NDB];
    float m[NU], l[NU], nmv[NU], la[NU][4];  // maximum, sum, -maximum (FLT_MAX at -inf), running partial sums
#pragma unroll
    for (int u = 0; u < NU; u++) {
#pragma unroll
      for (int db = 0; db < NDB; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[u][db][i] = 0.0f;
      m[u] = -INFINITY;
      l[u] = 0.0f;
      nmv[u] = FLT_MAX;
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

    struct Ops {  // operands of one key tile of a step: V of block j - 1 (index NDB * s2 + db), K of block j + 1
      i16x8 va[2 * NDB];
      i32x4 ka[NCH];
    };
    auto vread = [&](int j, int t, int k) __attribute__((always_inline)) {
      const char *Vs = smem + VOFF + (j & (NR - 1)) * KBYTES + (32 * t + 16 * (k / NDB)) * RB + vbase[k % NDB];
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
      for (int r = 0; r < LPB; r++) {
        i32x4 *at = (i32x4 *)(smem + VOFF + (j & (NR - 1)) * KBYTES + (r * NWC + w) * 1024 + 16 * lane);
        i32x4 v = *at;
        bool some = false;
#pragma unroll
        for (int e = 0; e < 4; e++) some |= odd16<VT>((unsigned)v[e]) | odd16<VT>((unsigned)v[e] << 16);
        if (__builtin_expect(__any(some), 0)) {
          odd = odd || (some && ((i64)blk0 + j) * BK + 16 * group_of(r) + lrow < L);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            unsigned d = (unsigned)v[e];
            if (odd16<VT>(d)) d &= 0xFFFFu;
            if (odd16<VT>(d << 16)) d &= 0xFFFF0000u;
            v[e] = (int)d;
          }
          *at = v;
        }
      }
    };

    // One (key tile t, row tile u) of step j, in issue order: P V of block j - 1 and scores of block j + 1 spread between runs of
    // independent VALU work on block j. With `refresh` each operand is replaced by the next tile's (jn, tn) after its last use.
    auto sub_tile = [&](Ops &op, int j, int t, int u, bool mask, bool refresh, int jn, int tn, int nst)
        __attribute__((always_inline)) {
      const float nm = nmv[u];
      const int see = mask ? beyond(j, u) : 0;
      float xv[16];
      int npv = 0, ns = 0, pslot = 0, sslot = 0;
      // 8 slots for either product's instructions, some of them empty at smaller head dims
      auto taken = [](int slot) { return D == 128 || (D == 96 ? (slot & 3) != 3 : (slot & 1) == 0); };
      auto pv = [&]() __attribute__((always_inline)) {
        const int slot = pslot++;
        if (taken(slot)) {
          const int k = npv++;
          mma_pv_acc<VT>(o[u][k % NDB], op.va[k], __builtin_bit_cast(VT8, pb[t][u][k / NDB]));
          if (refresh) op.va[k] = vread(jn - 1, tn, k);
        }
        if (nst) stage_k(slot, j + 3, j + 1);
      };
      auto sm = [&]() __attribute__((always_inline)) {
        if (!taken(sslot++)) return;
        const int c = ns++;
        f32x16 zero;
#pragma unroll
        for (int i = 0; i < 16; i++) zero[i] = 0.0f;
        s[t][u] = mma_qk<VT>(op.ka[c], qreg[u][c], c == 0 ? zero : s[t][u]);
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

    // Row tile u's weights of block j with the block's own maximum, its sum so far in la[u][0]; returns the factor of what was
    // summed before. A row whose scores are all -infinity so far, or that sees no key, keeps the weights 0: its offset of FLT_MAX
    // takes -infinity to 0 and any finite score to an infinite weight, so that the first block with one comes here.
    auto exact = [&](int j, int u, bool mask) __attribute__((always_inline)) {
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
      const float nm = mn == -INFINITY ? FLT_MAX : -mn;
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
      la[u][0] = l[u] * f + (add[0] + add[1]);
      la[u][1] = la[u][2] = la[u][3] = 0.0f;
      return f;
    };

    // Step j from 1 on: P V of block j - 1, softmax of block j, scores of block j + 1 (behind the last one: of the spare rows
    // that its loads took; nothing reads them).
    // The barrier sits before the last sub-tile: the loads behind it (K of block j + 3, V of block j + 1) land during the next
    // step, and the last sub-tile reads the next step's first operands. Ring slots: K(j + 3) replaces K(j - 1), V(j + 1) V(j - 3).
    // The masking steps and the others are the only two copies of this code: a tile of few blocks is bound by fetching it.
    static_assert(NU == 2, "two row tiles");
    auto step = [&](Ops &op, int j, bool mask) __attribute__((always_inline)) {
      float tot[NU];
      bool bad = false;
      auto sums = [&](int u) __attribute__((always_inline)) {
        tot[u] = (la[u][0] + la[u][1]) + (la[u][2] + la[u][3]);
        bad = bad | !(tot[u] - l[u] <= sum_limit<VT>());
      };
      windows(j);
      sub_tile(op, j, 0, 0, mask, false, j, 1, 0);
      sub_tile(op, j, 0, 1, mask, true, j, 1, 0);
      sub_tile(op, j, 1, 0, mask, false, j + 1, 0, 0);
      sums(0);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the previous step
      if (mask) clean(j);
      __syncthreads();
      sub_tile(op, j, 1, 1, mask, true, j + 1, 0, 1);
      sums(1);
      // rare: a score far above the running maximum: block j's weights again with the exact one (its K is still in its slot)
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad) != 0, 0)) {
        o_fence(o);  // P V MFMAs of this step may still be writing O
#pragma unroll
        for (int u = 0; u < NU; u++) {
          const float f = exact(j, u, mask);
#pragma unroll
          for (int db = 0; db < NDB; db++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[u][db][i] *= f;
          tot[u] = la[u][0];
        }
        o_fence(o);  // VALU writes of O before the next MFMA reads it
      }
#pragma unroll
      for (int u = 0; u < NU; u++) l[u] = tot[u];
    };

    // the first loads: page numbers, Q operands (B of S^T = K Q^T) under way while K and V of the first blocks are asked for
    const int id0 = fetch(0);
    ahead = fetch(1);
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int c = 0; c < NCH; c++) qreg[u][c] = *(const i32x4 *)(qrow[u] + (2 * c + hl) * 16);
    __builtin_amdgcn_sched_barrier(0);
    addresses(id0, 0);
    v_lo = vnext_lo;
    v_hi = vnext_hi;
#pragma unroll
    for (int b = 0; b < 3; b++)
#pragma unroll
      for (int i = 0; i < LPB; i++) stage_k(i, b, 0);
#pragma unroll
    for (int i = 0; i < LPB; i++) stage_k(LPB + i, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int c = 0; c < NCH; c++) {
        qreg[u][c] = ok[u] ? qreg[u][c] : i32x4{0, 0, 0, 0};
        asm volatile("" : "+a"(qreg[u][c]));  // from here on Q lives in AGPRs only
      }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (clear == 0) clean(0);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * LPB; i++) stage_k(i, 3, 1);
#pragma unroll
    for (int u = 0; u < NU; u++) {
      exact(0, u, true);
      l[u] = la[u][0];
    }
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int u = 0; u < NU; u++) {
#pragma unroll
        for (int i = 0; i < 16; i++) s[t][u][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < NCH; c++) s[t][u] = mma_qk<VT>(kread(1, t, c), qreg[u][c], s[t][u]);
      }
    Ops op;
#pragma unroll
    for (int k = 0; k < 2 * NDB; k++) op.va[k] = vread(0, 0, k);
#pragma unroll
    for (int c = 0; c < NCH; c++) op.ka[c] = kread(2, 0, c);
    // from here on O lives in AGPRs only
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
      for (int db = 0; db < NDB; db++) asm volatile("" : "+a"(o[u][db]));
    int j = 1;
    for (; j < clear; j++) step(op, j, false);
    for (; j < nblk; j++) step(op, j, true);
    // P V of the last block (its tile-0 V operands were read by the last step)
#pragma unroll
    for (int t = 0; t < 2; t++) {
      if (t == 1) {
#pragma unroll
        for (int k = 0; k < 2 * NDB; k++) op.va[k] = vread(nblk - 1, 1, k);
      }
#pragma unroll
      for (int u = 0; u < NU; u++)
#pragma unroll
        for (int k = 0; k < 2 * NDB; k++)
          mma_pv_acc<VT>(o[u][k % NDB], op.va[k], __builtin_bit_cast(VT8, pb[t][u][k / NDB]));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // loads past the last block land before the slots are used again
    o_fence(o);

    // Outputs go through LDS (each wave its own rows, a few bytes apart, so that neither side meets bank conflicts): a lane holds
    // 4 channels of a row here and there, and stores 16 bytes of whole rows.
    __syncthreads();
    constexpr int S16 = C::S16, S32 = C::S32;
    const unsigned mine = w * (32 * NU) * S32;
    float sum[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) {
      sum[u] = l[u] + __shfl_xor(l[u], 32);
      if (last[u] >= lost) sum[u] = NAN;
    }
    if (EACH || whole) {
      constexpr int LR = D == 64 ? 8 : 16, RI = 64 / LR;  // lanes a row (12 of 16 at head dim 96), rows at a time
      const int piece = lane % LR;
      unsigned to = mine + l32 * S16 + 8 * hl, from = mine + lane / LR * S16 + min(piece, D / 8 - 1) * 16;
      asm volatile("" : "+v"(to), "+v"(from));  // (the addresses of all pieces would be kept over the tiles' loop otherwise)
#pragma unroll
      for (int u = 0; u < NU; u++) {
        // no sum although a key is visible: all scores are -infinity, and 0 / 0 (the reciprocal is a float's last bit off at
        // most, far below the rounding to 16 bits)
        const float inv = sum[u] != 0.0f ? __builtin_amdgcn_rcpf(sum[u]) : last[u] >= 0 ? NAN : 0.0f;
#pragma unroll
        for (int db = 0; db < NDB; db++)
#pragma unroll
          for (int g = 0; g < 4; g++)
            store4<VT>(smem + to + 32 * u * S16 + (db * 32 + 8 * g) * 2, o[u][db][4 * g] * inv, o[u][db][4 * g + 1] * inv,
                       o[u][db][4 * g + 2] * inv, o[u][db][4 * g + 3] * inv);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      char *base = a.out + ((size_t)m0 * p.o_stride + (size_t)(kvh * hd.G + g0) * D) * 2 + piece * 16;
#pragma unroll 1
      for (int i = 0; i < 32 * NU / RI; i += 4) {
        float2 lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          lo[k] = *(const float2 *)(smem + from + RI * k * S16);
          hi[k] = *(const float2 *)(smem + from + RI * k * S16 + 8);
        }
        from += 4 * RI * S16;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int row = w * (32 * NU) + RI * (i + k) + lane / LR, ti = row_token(row), gi = row - ti * hd.GP;
          if (row < R && g0 + gi < hd.G && piece < D / 8)
            *(Piece *)(base + ((size_t)ti * p.o_stride + gi * D) * 2) = Piece{{lo[k].x, lo[k].y, hi[k].x, hi[k].y}};
        }
      }
    } else {
      constexpr int LR = D == 64 ? 16 : 32, RI = 64 / LR;  // (24 of 32 at head dim 96)
      const int piece = lane % LR;
      unsigned to = mine + l32 * S32 + 16 * hl, from = mine + lane / LR * S32 + min(piece, D / 4 - 1) * 16;
      asm volatile("" : "+v"(to), "+v"(from));
#pragma unroll
      for (int u = 0; u < NU; u++) {
#pragma unroll
        for (int db = 0; db < NDB; db++)
#pragma unroll
          for (int g = 0; g < 4; g++)
            store4<T_F32>(smem + to + 32 * u * S32 + (db * 32 + 8 * g) * 4, o[u][db][4 * g], o[u][db][4 * g + 1],
                          o[u][db][4 * g + 2], o[u][db][4 * g + 3]);
        if (hl == 0) *(float2 *)(st + RTC * D + 2 * (w * (32 * NU) + 32 * u + l32)) = make_float2(m[u], sum[u]);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      float *base = st + (w * (32 * NU) + lane / LR) * D + 4 * piece;
#pragma unroll 1
      for (int i = 0; i < 32 * NU / RI; i += 8) {
        f32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = *(const f32x4 *)(smem + from + RI * k * S32);
        from += 8 * RI * S32;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (piece < D / 4) *(f32x4 *)(base + RI * (i + k) * D) = v[k];
      }
    }
    odd = __syncthreads_or(odd);
    if (__builtin_expect(odd, 0)) {  // the values left out above, for the rows that see them
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every wave's outputs are written before another adds to them
      __syncthreads();
      for (int c = tid; c < R * (D / 8); c += NWC * 64) {
        const int r = c / (D / 8), d0 = 8 * (c - r * (D / 8));
        const int ti = row_token(r), gi = r - ti * hd.GP;
        if (g0 + gi >= hd.G) continue;
        const i64 seen = plan::clamp(CAUSAL ? q.off + m0 + ti + 1 : q.L, 0, min(q.L, (i64)blk1 * BK));
        float v[8] = {};
        bool some = false;
        for (i64 key = (i64)(blk0 + clear) * BK; key < seen; key++) {
          const int pg = bt.table[(size_t)tile.b * bt.width + (key >> bt.lg)];
          if (pg < 0 || pg >= bt.pages) continue;
          const size_t row = (((size_t)pg * p.KVH + kvh) << bt.lg) + (size_t)(key & ((1 << bt.lg) - 1));
          const i32x4 vv = *(const i32x4 *)(a.vc + row * C::RBG + d0 * 2);
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const unsigned x = (unsigned)vv[e / 2] << (e & 1 ? 0 : 16);
            if (odd16<VT>(x)) {
              v[e] += x & (VT == T_BF16 ? 0x007F0000u : 0x03FF0000u) ? NAN : (int)x < 0 ? -INFINITY : INFINITY;
              some = true;
            }
          }
        }
        if (!some) continue;
        if (EACH || whole) {
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
  if (!EACH && !unfinished && tid == 0) left_of(a, sl)->R = 0;
}

template <int D, int VT, bool CAUSAL, bool EACH>
int run(const Exec &ex, const AttnArgs &a, const Batch &bt, const PagedAttnParams &p, const plan::Shape &sh, const Heads &hd,
        unsigned grid, int least, std::string *err) {
  auto kern = attention_chunk_kernel<D, VT, CAUSAL, EACH>;
  static bool attr_set = false;
  if (!attr_set) {
    hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, Chunk<D>::LDS);
    if (e != hipSuccess) {
      *err = std::string("hipFuncSetAttribute: ") + hipGetErrorString(e);
      return -1;
    }
    attr_set = true;
  }
  hipLaunchKernelGGL(kern, dim3(grid), dim3(NWC * 64), Chunk<D>::LDS, ex.stream, a, bt, p, sh, hd, least);
  return 0;
}

template <int D, int VT, bool CAUSAL>
int run(const Exec &ex, const AttnArgs &a, const Batch &bt, const PagedAttnParams &p, const plan::Choice &c, std::string *err) {
  const Heads hd = plan::heads_of(p.H, p.KVH, RTC);
  const int least = 512;  // weight of a slice
  const plan::Shape sh{p.M, p.B, RTC / hd.GP, p.KVH * hd.HS, CAUSAL, 256, (i64)bt.width << bt.lg};
  AttnArgs g = a;
  g.ws = (float *)ex.ws;
  g.left = (char *)ex.ws + (size_t)c.most * 2 * RTC * (D + 2) * sizeof(float);
  g.spare = p.pages ? a.kc : (const char *)ex.ws;  // 16 rows that can be read (no page has fewer)
  if (c.each) return run<D, VT, CAUSAL, true>(ex, g, bt, p, sh, hd, (unsigned)c.tiles, least, err);
  if (run<D, VT, CAUSAL, false>(ex, g, bt, p, sh, hd, (unsigned)c.most, least, err)) return -1;
  if (c.most > 1)
    hipLaunchKernelGGL((attention_join_kernel<D, VT, RTC, 4>), dim3((unsigned)(c.most - 1), RTC / 16), dim3(256), 0, ex.stream,
                       g, p.o_stride);
  return 0;
}

}  // namespace

int launch_attention_chunk(int d, int t, bool causal, const Exec &ex, const AttnArgs &a, const Batch &bt,
                           const PagedAttnParams &p, const plan::Choice &c, std::string *err) {
  auto go = [&](auto dc) {
    constexpr int D = decltype(dc)::value;
    if (t == T_BF16) return causal ? run<D, T_BF16, true>(ex, a, bt, p, c, err) : run<D, T_BF16, false>(ex, a, bt, p, c, err);
    return causal ? run<D, T_F16, true>(ex, a, bt, p, c, err) : run<D, T_F16, false>(ex, a, bt, p, c, err);
  };
  if (d == 64) return go(std::integral_constant<int, 64>{});
  if (d == 96) return go(std::integral_constant<int, 96>{});
  return go(std::integral_constant<int, 128>{});
}

}  // namespace h3
