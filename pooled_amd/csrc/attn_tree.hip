// Attention of a tree of drafted tokens over a cache, on f16 MFMA for gfx950.
//
// Column c of n sees the cache rows [0, base) and those rows base + j whose bit j is set in its mask:
//   o[c, h] = sum_t softmax_t(q[c, h] . k[t] / sqrt(hd)) v[t]
// The G query heads of a kv head and all columns are stacked rows (row = column x G + head), so K and V are read once for all of them.
//
//   * A workgroup is eight wavefronts, two a SIMD (one a SIMD gets half of what the LDS delivers: four waves of up to three blocks took 174 us where this takes 92), over one split of
//     the context and up to 256 stacked rows in blocks of 16, block b with wave b % 8; every 32-row tile of K and V that it stages in LDS serves all of them.  Tiles go global -> LDS
//     directly, three of them in flight in a ring of four; one barrier a tile.  Int8 rows go through registers, two tiles ahead, and are widened on the way to a ring of two.
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: Q fragments stay in registers, K fragments are 16-byte LDS reads, V^T fragments come from the
//     LDS transpose read.  The accumulator of S^T is the operand of P V, so probabilities never leave registers.
//   * The products take f16, and q is rounded to it; what that drops of f16 rows' q goes into products of its own with the same K fragments, so that q counts to 2^-22 of itself.  Up to eight stacked
//     rows in all leave half of their one block free, and its rows 8 .. 15 hold it, at no cost; else it is in fragments beside q's (24 columns at 2011 rows 13.3 -> 14.5 us a call, 63 at 7001 of heads of
//     128 15.2 -> 16.5: the score products once more).  Not where registers have no room, two blocks a wave of heads of 256, nor for more int8 rows, whose own rounding, K's to f16, is as large.
//   * Online softmax in f32 in the exp2 domain: the reference of a row is raised, and O and l rescaled, only where a P comes out above 2^8 (exact enough in f16); l is
//     the sum of the rounded P, so an output is a convex combination of value rows whatever that rounding did.
//   * The mask is looked at only in tiles that reach the drafted rows.  There a row's 32 bits are one word, cut out of its mask at the tile's offset with the rows in front
//     of the draft as ones.  A drafted row that holds what is not finite must reach those columns alone that see it, and 0 x inf is not 0: such elements go into the product as
//     zeros and are added to the outputs of the columns that see them.  Rows of the context, which all columns see, go into it as they are, also those of the draft's first tile.
//   * Splits leave (m, l) and O / l in f32; pa_tree_merge_kernel joins them.  (In f16 they are half the bytes, which is 0 - 4 us of a call, and 2^-12 of an output: 63 splits of 17 columns at
//     20003 int8 rows 25.7 us against 29.7, 16 of 24 at 2011 12.9 against 13.3.)
//
// Measured (24 query and 4 key heads of 256, 65536 rows of f16, 268 MB): 16 columns 52 us = 5.1 TB/s, which is what a large copy reaches; 48 columns 95 us = 813 TFLOP/s (a large matrix
// product: 1330), and 3 % less with every tile read from the L2, so there the SIMDs' work bounds it: a tile of nine blocks, three of them on one SIMD, takes 1.3 us, of which the matrix
// instructions are 0.8 at the 1.9 GHz that the power limit leaves.  The merge adds 9.3 us there (38 MB of partials), 3 - 4 for small drafts, most of it the launch.  Int8: 17 columns at 20003 rows
// 24.4 us and 7.5: the widening through registers, 1.1 us a tile of seven blocks, and 26 MB of partials.  5 columns at 190 rows, 16 and 8 heads of 128: 8.3 us a call in one launch; 7.2 before
// q's second products, and then 7.8 with seven splits and the merge (at 100 rows 5.9 and 8.3).
#include "tree_internal.h"
#include "pf_common.h"
#include "tree_mask.h"

#define TREE_ISSUE 4         // waves that send for tiles
template <int HD, int W> struct TreeShape {
  static constexpr int ROWB = HD * 2;               // bytes of a staged row
  static constexpr int TILE = 32 * ROWB;            // bytes of a staged tile of K or of V
  static constexpr int KS = HD / 32;                // k-steps of the QK product
  static constexpr int DB = HD / 16;                // 16-dim blocks of the output
  static constexpr int CPR = HD / 8;                // 16-byte chunks of a staged row
  static constexpr int RPB = 64 / CPR;              // rows of a 1 KB LDS-direct load
  static constexpr int NLD = 32 / RPB / TREE_ISSUE; // LDS-direct loads of a wave that issues them, a tensor and tile
  static constexpr int PIECES = 32 * HD / 16;       // int8 rows: 16-byte pieces of a tile of K or of V ...
  static constexpr int NP8 = 2 * PIECES / (W * 64); // ... and a thread's share of both
  static_assert(NLD * TREE_ISSUE * RPB == 32, "a tile divides evenly over the waves");
  static_assert(NP8 * W * 64 == 2 * PIECES && PIECES % 64 == 0, "an int8 tile divides evenly over the threads, a wave's pieces are of one tensor");
};

static __device__ inline bool not_finite2(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }   // any of two f16

// An int8 row's values v as f16: v 2^-k, exactly, times scale 2^k, which is given as the f16 nearest to it and the rest.  k brings the scale to [1, 2) where 2^-24 <= scale < 64 (-5 <= k <= 24), so that
// the two parts hold it to 2^-24 of itself and the product is rounded once, to what f16 holds of it, subnormal numbers too (the part of the rest, rounded before, adds 2^-21 of a value, or 2^-25).
// Other scales give what f16 holds of their values too; from 2^21 on they count as infinite.
// v 2^-k is the bit pattern of 2^(10 - k) + (v + 128) 2^-k, whose upper byte is (25 - k) << 2, less 1152 x 2^-k.
struct Widen { _Float16 hi, lo, off; uint32_t top; };
static __device__ inline Widen widen_of(float sc) {
  const int e = min(max(__builtin_amdgcn_frexp_expf(sc) + 24, 1), 30);     // 25 - k: the exponent field of 1024 x 2^-k
  const float s = __builtin_amdgcn_ldexpf(sc, 25 - e);
  Widen w;
  w.hi = (_Float16)s;
  const float rest = s - (float)w.hi;
  w.lo = (_Float16)(__builtin_fabsf(rest) < 64.f ? rest : 0.f);            // (at most 2^-11 of s; where that is infinite there is none)
  w.top = (uint32_t)e << 2;
  const uint16_t off = (uint16_t)(e << 10 | 128);
  __builtin_memcpy(&w.off, &off, 2);
  return w;
}

// What the drafted rows that column `col` sees hold that is not finite, added to E dims of its output (of one block of 32): rows of v head g, dims d ..
template <int E> static __device__ inline void add_not_finite(const TreeParams& p, uint32_t hd, uint32_t col, uint32_t g, uint32_t d, float (&o)[E]) {
  const uint32_t* words = p.mask + (size_t)col * p.mask_stride;
#pragma unroll 1
  for (uint32_t j = 0; j < p.n_cols; j++) {
    if (!(words[j / 32] >> (j % 32) & 1)) continue;
    const size_t row = (size_t)g * ((size_t)p.max_seq + 32) + p.base_pos + j;
#pragma unroll
    for (int e = 0; e < E; e++) {
      float v;
      if (p.v_scale) {                              // (as it was widened: what f16 does not hold is infinite)
        const Widen w = widen_of(p.v_scale[row * (hd / 32) + d / 32]);
        uint16_t bits = (uint16_t)(w.top << 8 | ((uint32_t)((const unsigned char*)p.v_cache)[row * hd + d + e] ^ 0x80u));
        _Float16 x;
        __builtin_memcpy(&x, &bits, 2);
        x -= w.off;
        v = (float)__builtin_elementwise_fma(x, w.hi, x * w.lo);
      } else v = (float)((const _Float16*)p.v_cache)[row * hd + d + e];
      o[e] += __builtin_fabsf(v) < __builtin_inff() ? 0.f : v;
    }
  }
}

template <int N> static __device__ inline void wait_and_meet() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory"); }

// orders a wave's LDS accesses for the compiler (the hardware executes them in order)
static __device__ inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
static __device__ inline void wait_and_meet_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// LDS behind the ring: mask words of WIN tiles, and a flag of each wave
template <int NB> struct TreeLds { static constexpr int WIN = 4 / NB, bytes = WIN * 16 * NB * TREE_W * 4 + TREE_W * 4; };

// sigmoid; the reciprocal is off by 2^-23 of itself, an exact division is a dozen instructions a value
static __device__ inline float gate_of(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// E dims of an output column, four or eight
template <int E> static __device__ inline void store_dims(const TreeParams& p, uint32_t col, uint32_t d, const float (&o)[E]) {
#pragma unroll
  for (int e = 0; e < E; e += 4) {
    if (p.out_f16) *(h4*)((_Float16*)p.out + (size_t)col * p.out_stride + d + e) = (h4){ (_Float16)o[e], (_Float16)o[e + 1], (_Float16)o[e + 2], (_Float16)o[e + 3] };     // (columns of f16 are 8 bytes aligned)
    else *(f4*)((float*)p.out + (size_t)col * p.out_stride + d + e) = (f4){ o[e], o[e + 1], o[e + 2], o[e + 3] };
  }
}

// What f16 drops of q: left out, in rows 8 .. 15 of the one block, or in fragments of its own (see the head of the file)
enum { Q_F16 = 0, Q_SPARE_ROWS = 1, Q_TWICE = 2 };
template <int HD, int NB, bool Q8, int D, int QP>
__global__ __launch_bounds__(TREE_W * 64, TREE_W / 4) void pa_tree_kernel(TreeParams p) {
  static_assert(QP != Q_SPARE_ROWS || NB == 1, "one block of rows");
  constexpr int W = TREE_W, ROWS = 16 * NB * W;
  typedef TreeShape<HD, W> S;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];     // [D][K tile | V tile], mask words [WIN][ROWS], a flag of each wave
  constexpr int RING = D * 2 * S::TILE, WIN = TreeLds<NB>::WIN;
  uint32_t* win_lds = (uint32_t*)(smem + RING);
  uint32_t* bad_lds = win_lds + WIN * ROWS;
  // work items are (kv head, split, group of rows), the group fastest; dispatch id i runs on XCD i % 8, which owns a contiguous range of items, so the groups that
  // read the same rows share an L2
  const uint32_t total = p.n_groups * p.n_kv_heads * p.n_splits, per = (total + 7) / 8;
  const uint32_t item = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (item >= total) return;
  const uint32_t gs = div_by(item, p.n_groups, p.ng_magic), grp = item - gs * p.n_groups;
  const uint32_t g = div_by(gs, p.n_splits, p.ns_magic), sp = gs - g * p.n_splits;
  const uint32_t tid = threadIdx.x, lane = tid & 63, ln = lane & 15, kg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t G = p.group;
  auto col_of = [&](uint32_t x) __attribute__((always_inline)) -> uint32_t { return div_by(x, G, p.g_magic); };
  const uint32_t x0 = grp * p.group_rows, R = min(p.group_rows, p.n_cols * G - x0);     // the group's stacked rows [x0, x0 + R)
  const uint32_t end = p.base_pos + p.n_cols;
  const uint32_t tile0 = sp * p.split_tiles, n_tiles = min(p.split_tiles, (end + 31) / 32 - tile0);
  const uint32_t draft0 = max(p.base_pos / 32, tile0) - tile0;              // the split's first tile that reaches the drafted rows, if it is below n_tiles
  const size_t head_rows = (size_t)p.max_seq + 32;

  // ---- staging: tile i goes to buffer i % D ----
  auto k_slot = [](uint32_t row, uint32_t chunk) __attribute__((always_inline)) { return chunk ^ (row & 15); };      // conflict-free 16-byte fragment reads
  auto v_slot = [](uint32_t row, uint32_t chunk) __attribute__((always_inline)) { return chunk ^ (4 * (row & 3)) ^ (2 * ((row >> 2) & 1)); };   // 2-way for the transpose reads, their best
  auto buf = [&](uint32_t i) __attribute__((always_inline)) { return smem + (i % D) * 2 * S::TILE; };
  // f16 rows: load j of wave w fills the 1 KB block j W + w of a buffer, rows (j W + w) RPB ..; lane l lands at (row l / CPR, slot l % CPR) and fetches the chunk that belongs there
  const unsigned char* kb0 = (const unsigned char*)p.k_cache + (size_t)g * head_rows * S::ROWB;
  const unsigned char* vb0 = (const unsigned char*)p.v_cache + (size_t)g * head_rows * S::ROWB;
  // Only the last waves, which have the fewest rows, send for tiles: a CU takes in 64 bytes a clock, so a tile's loads hold up who issues them for hundreds of clocks, and one wave of each SIMD computes meanwhile.
  constexpr int IS = TREE_ISSUE;
  const bool issuer = wave >= W - IS;
  const uint32_t iw = wave - (W - IS), ld_row = iw * S::RPB + lane / S::CPR, ld_c = lane % S::CPR;
  constexpr int NOFF = IS * S::RPB % 16 ? 16 / (IS * S::RPB) : 1;            // loads after which the swizzle, and with it a lane's offset in a load's rows, comes again
  uint32_t k_off[NOFF], v_off[NOFF];
#pragma unroll
  for (int j = 0; j < NOFF; j++) {
    const uint32_t r = j * IS * S::RPB + ld_row;
    k_off[j] = ld_row * S::ROWB + k_slot(r, ld_c) * 16;
    v_off[j] = ld_row * S::ROWB + v_slot(r, ld_c) * 16;
  }
  auto issue = [&](uint32_t i) __attribute__((always_inline)) {
    const uint32_t tp = (tile0 + i) * 32;
    unsigned char* dst = buf(i);
    if (tp + 32 <= end) {
      const unsigned char *kt = kb0 + (size_t)tp * S::ROWB, *vt = vb0 + (size_t)tp * S::ROWB;
#pragma unroll
      for (int j = 0; j < S::NLD; j++) PF_GLL_S(kt + j * IS * S::RPB * S::ROWB, k_off[j % NOFF], dst + (j * IS + iw) * 1024);
#pragma unroll
      for (int j = 0; j < S::NLD; j++) PF_GLL_S(vt + j * IS * S::RPB * S::ROWB, v_off[j % NOFF], dst + S::TILE + (j * IS + iw) * 1024);
    } else {                                        // rows behind the last one: the cache's zero padding
#pragma unroll 1
      for (int j = 0; j < S::NLD; j++) {
        const uint32_t r = j * IS * S::RPB + ld_row;
        const size_t row = tp + r < end ? tp + r : p.max_seq;
        PF_GLL(kb0 + row * S::ROWB + k_slot(r, ld_c) * 16, dst + (j * IS + iw) * 1024);
        PF_GLL(vb0 + row * S::ROWB + v_slot(r, ld_c) * 16, dst + S::TILE + (j * IS + iw) * 1024);
      }
    }
  };
  // int8 rows: a thread's 16-byte pieces of a tile, K's and then V's, and their scales; two tiles in registers
  u4 raw8[2][S::NP8];
  float sc8[2][S::NP8];
  auto fetch8 = [&](uint32_t i, auto AT) __attribute__((always_inline)) {
    constexpr int at = decltype(AT)::value;
    const uint32_t tp = (tile0 + i) * 32;
    const size_t row0 = (size_t)g * head_rows + tp;
#pragma unroll
    for (int j = 0; j < S::NP8; j++) {
      const uint32_t e = tid + j * W * 64, of_v = (wave * 64 + j * W * 64) / S::PIECES, r = e % S::PIECES / (HD / 16), c = e % (HD / 16);
      const unsigned char* rows = (const unsigned char*)(of_v ? p.v_cache : p.k_cache) + row0 * HD;
      const float* scales = (of_v ? p.v_scale : p.k_scale) + row0 * (HD / 32);
      if (tp + 32 <= end) {                         // (one offset a thread for all tiles)
        raw8[at][j] = *(const u4*)(rows + (e % S::PIECES) * 16);
        sc8[at][j] = scales[e % S::PIECES / 2];
      } else {                                      // rows behind the last one: the cache's zero padding
        const uint32_t rr = tp + r < end ? r : p.max_seq - tp;
        raw8[at][j] = *(const u4*)(rows + (size_t)rr * HD + c * 16);
        sc8[at][j] = scales[(size_t)rr * (HD / 32) + c / 2];
      }
    }
  };
  auto widen = [&](u4 raw, float sc, unsigned char* row, uint32_t s0, uint32_t s1) __attribute__((always_inline)) {
    const Widen w = widen_of(sc);
    const h2 sh = { w.hi, w.hi }, sl = { w.lo, w.lo }, off = { w.off, w.off };
    h2 o[8];
#pragma unroll
    for (int d = 0; d < 4; d++) {
      const uint32_t u = raw[d] ^ 0x80808080u;
      const uint32_t a = __builtin_amdgcn_perm(w.top, u, 0x04010400u), b = __builtin_amdgcn_perm(w.top, u, 0x04030402u);
      h2 xa, xb;
      __builtin_memcpy(&xa, &a, 4);
      __builtin_memcpy(&xb, &b, 4);
      xa -= off;
      xb -= off;
      o[2 * d] = __builtin_elementwise_fma(xa, sh, xa * sl);
      o[2 * d + 1] = __builtin_elementwise_fma(xb, sh, xb * sl);
    }
    *(h8*)(row + s0 * 16) = (h8){ o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1] };
    *(h8*)(row + s1 * 16) = (h8){ o[4][0], o[4][1], o[5][0], o[5][1], o[6][0], o[6][1], o[7][0], o[7][1] };
  };
  auto stage8 = [&](uint32_t i, auto AT) __attribute__((always_inline)) {
    constexpr int at = decltype(AT)::value;
    unsigned char* dst = buf(i);
#pragma unroll
    for (int j = 0; j < S::NP8; j++) {
      const uint32_t e = tid + j * W * 64, of_v = (wave * 64 + j * W * 64) / S::PIECES, r = e % S::PIECES / (HD / 16), c = e % (HD / 16) * 2;
      widen(raw8[at][j], sc8[at][j], dst + of_v * S::TILE + r * S::ROWB, of_v ? v_slot(r, c) : k_slot(r, c), of_v ? v_slot(r, c + 1) : k_slot(r, c + 1));
    }
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  // the rows' words of the mask at WIN tiles from the split's draft tile d on
  auto fill_windows = [&](uint32_t d) __attribute__((always_inline)) {
#pragma unroll 1
    for (uint32_t e = tid; e < WIN * ROWS; e += W * 64) {
      const uint32_t r = e % ROWS, i = draft0 + d + e / ROWS, x = x0 + min(r, R - 1);
      if (i < n_tiles) win_lds[e] = mask_window(p.mask + (size_t)col_of(x) * p.mask_stride, (int)((tile0 + i) * 32 - p.base_pos), p.n_cols);
    }
  };

  // ---- start: the first tile goes out, then what the wave's rows need; the other tiles behind them, since loads return in order ----
  // (block nb of a wave is rows 16 (nb W + wave) ..: the blocks of a group spread over the SIMDs evenly)
  auto row_of = [&](uint32_t nb, uint32_t r) __attribute__((always_inline)) -> uint32_t { return (nb * W + wave) * 16 + r; };
  const uint32_t blocks = R > wave * 16 ? (R - wave * 16 + W * 16 - 1) / (W * 16) : 0;      // the wave's live blocks
  if constexpr (Q8) fetch8(0, I0{}); else if (issuer) issue(0);
  // ---- what follows is one program for the waves of two live blocks, of one, and of none, which pass the same barriers ----
  auto run = [&](auto BLOCKS) __attribute__((always_inline)) {
  constexpr int LIVE = decltype(BLOCKS)::value, NL = LIVE ? LIVE : 1, KD = NL == 1 ? 4 : 3, VD = NL == 1 ? 4 : 3;      // K and V^T fragments (NL products each) fetched ahead
  // Q: whole rows as they lie in memory, through a wave-private part of the ring's last buffer (taken by a tile only behind the first barrier), eight rows at a time, to the fragments: row ln of block nb, dims 32 ks + 8 kg .. + 7
  constexpr bool TWICE = QP == Q_TWICE;
  h8 qf[NL][S::KS], ql[NL][TWICE ? S::KS : 1];
  if constexpr (LIVE == 0) { if (draft0 < n_tiles) fill_windows(0); } else {
    constexpr int LPQ = HD / 4, RPL = 64 / LPQ, QL = 8 / RPL;               // lanes of a row, rows of a load, loads of eight rows
    unsigned char* qs = smem + (D - 1) * 2 * S::TILE + wave * 8 * S::ROWB;
    static_assert(8 * W * S::ROWB <= 2 * S::TILE, "eight rows of each wave fit a buffer");
    f4 qv[2 * NL][QL];
#pragma unroll
    for (int b = 0; b < 2 * NL; b++)
#pragma unroll
      for (int j = 0; j < QL; j++) {
        const uint32_t x = x0 + min(row_of(b / 2, b % 2 * 8 + j * RPL + lane / LPQ), R - 1), col = col_of(x);
        qv[b][j] = *(const f4*)(p.q + (size_t)col * p.q_stride + (size_t)(g * G + x - col * G) * HD + lane % LPQ * 4);
      }
    if (draft0 < n_tiles) fill_windows(0);
#pragma unroll
    for (int b = 0; b < 2 * NL; b++) {
#pragma unroll
      for (int part = 0; part < (TWICE ? 2 : 1); part++) {
#pragma unroll
      for (int j = 0; j < QL; j++) {
        const uint32_t r = j * RPL + lane / LPQ, c = lane % LPQ;
        const bool low = part || (QP == Q_SPARE_ROWS && b == 1);
        f4 v = qv[QP == Q_SPARE_ROWS ? 0 : b][j];
        if (low) {
#pragma unroll
          for (int e = 0; e < 4; e++) v[e] -= (float)(_Float16)v[e];
        }
        *(h4*)(qs + r * S::ROWB + ((c / 2) ^ r) * 16 + c % 2 * 8) = (h4){ (_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3] };
      }
      wave_fence();
#pragma unroll
      for (int ks = 0; ks < S::KS; ks++) {
        const h8 f = *(const h8*)(qs + (ln & 7) * S::ROWB + ((ks * 4 + kg) ^ (ln & 7)) * 16);
        h8& to = part ? ql[b / 2][TWICE ? ks : 0] : qf[b / 2][ks];
        to = b % 2 == 0 || ln >= 8 ? f : to;
      }
      wave_fence();
      }
    }
  }
  if constexpr (Q8) {
    fetch8(min(1u, n_tiles - 1), I1{});
  } else {
#pragma unroll
    for (int i = 1; i < D - 1; i++) if (issuer && (uint32_t)i < n_tiles) issue(i);
  }
  f4 acc[S::DB][NL];
  float m_ref[NL], l_run[NL];
#pragma unroll
  for (int nb = 0; nb < NL; nb++) {
#pragma unroll
    for (int db = 0; db < S::DB; db++) acc[db][nb] = (f4){0.f, 0.f, 0.f, 0.f};
    m_ref[nb] = NEG_INF;
    l_run[nb] = 0.f;
  }
  bool unseen = true;                               // a row of the wave has no reference yet
  bool bad = false;                                 // a drafted row holds what is not finite
  const float c1 = p.scale * 1.4426950408889634f;   // scores -> log2 domain
  const uint32_t k_rd = ln * S::ROWB + (kg ^ ln) * 16;                                                                        // K fragment of k-step ks at k_rd ^ 64 ks
  const uint32_t v_rd = (4 * kg + (ln >> 2)) * S::ROWB + (((ln & 3) >> 1) ^ (4 * (ln >> 2)) ^ (2 * (kg & 1))) * 16 + (ln & 1) * 8;   // V fragment of block db at v_rd ^ 32 db

  f4 s[2][NL];                                      // a tile's scores: a lane holds row ln of each block, positions tp + 16 pb + 4 kg + i
  h8 pf[NL];
  // one tile: scores, softmax, product
  auto turn = [&](uint32_t i) __attribute__((always_inline)) {
    const unsigned char *kb = buf(i), *vb = kb + S::TILE;
    // ---- S^T = K Q^T ----
    {
      constexpr int NF = 2 * S::KS;
      h8 ka[KD];
      f4 sl[2][NL];
      auto at = [&](int f) __attribute__((always_inline)) { return kb + (k_rd ^ (f / 2 % 4 * 64)) + f / 8 * 256 + f % 2 * 16 * S::ROWB; };
#pragma unroll
      for (int f = 0; f < KD; f++) ka[f] = *(const h8*)at(f);
#pragma unroll
      for (int pb = 0; pb < 2; pb++)
#pragma unroll
        for (int nb = 0; nb < NL; nb++) s[pb][nb] = sl[pb][nb] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int f = 0; f < NF; f++) {
        const h8 a = ka[f % KD];
        if (f + KD < NF) ka[f % KD] = *(const h8*)at(f + KD);
#pragma unroll
        for (int nb = 0; nb < NL; nb++) s[f % 2][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[nb][f / 2], s[f % 2][nb], 0, 0, 0);
        if constexpr (TWICE) {
#pragma unroll
          for (int nb = 0; nb < NL; nb++) sl[f % 2][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[nb][f / 2], sl[f % 2][nb], 0, 0, 0);
        }
      }
      __builtin_amdgcn_sched_group_barrier(0x100, KD, 0);
#pragma unroll
      for (int f = 0; f < NF; f++) {
        __builtin_amdgcn_sched_group_barrier(0x008, TWICE ? 2 * NL : NL, 0);
        if (f + KD < NF) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      if constexpr (TWICE) {
#pragma unroll
        for (int j = 0; j < 2 * NL; j++) s[j / NL][j % NL] += sl[j / NL][j % NL];
      }
    }
    // (the first fragments of V^T, with one block on their way during the softmax: with two the registers are full)
    h4 lo[VD], hi[VD];
    auto fetch = [&](int f) __attribute__((always_inline)) {
      const unsigned char* vp = vb + (v_rd ^ (f % 8 * 32)) + f / 8 * 256;
      lo[f % VD] = lds_read_tr16(vp);
      hi[f % VD] = lds_read_tr16(vp + 16 * S::ROWB);
    };
    if constexpr (NL == 1) {
#pragma unroll
      for (int f = 0; f < VD; f++) fetch(f);
    }
    if constexpr (QP == Q_SPARE_ROWS) {
#pragma unroll
      for (int j = 0; j < 8; j++) s[j / 4][0][j % 4] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(s[j / 4][0][j % 4]), 0x128, 0xF, 0xF, false));     // row_ror:8
    }
    if (__builtin_expect(i >= draft0, 0)) {
#pragma unroll
      for (int nb = 0; nb < NL; nb++) {
        const uint32_t win = win_lds[(i - draft0) % WIN * ROWS + row_of(nb, ln)] >> (4 * kg);
#pragma unroll
        for (int pb = 0; pb < 2; pb++)
#pragma unroll
          for (int e = 0; e < 4; e++) s[pb][nb][e] = win >> (16 * pb + e) & 1 ? s[pb][nb][e] : NEG_INF;
      }
    }
    // ---- softmax ----
    // the references of the rows raised to the tile's maxima, O and l rescaled
    auto raise = [&]() __attribute__((always_inline)) {
      bool none = false;
#pragma unroll
      for (int nb = 0; nb < NL; nb++) {
        float mx = s[0][nb][0];
#pragma unroll
        for (int j = 1; j < 8; j++) mx = fmaxf(mx, s[j / 4][nb][j % 4]);
        const auto s16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(s16[0]), __uint_as_float(s16[1]));
        const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        const float m_new = fmaxf(m_ref[nb], fmaxf(__uint_as_float(s32[0]), __uint_as_float(s32[1])) * c1);
        const float alpha = m_new == NEG_INF ? 1.f : __builtin_amdgcn_exp2f(m_ref[nb] - m_new);
        m_ref[nb] = m_new;
        l_run[nb] *= alpha;
        none |= m_new == NEG_INF;
#pragma unroll
        for (int db = 0; db < S::DB; db++) acc[db][nb] *= alpha;
      }
      unseen = __any(none);
    };
    // P of the tile against the references; whether one passes them by more than f16 should hold
    auto probs = [&]() __attribute__((always_inline)) -> bool {
      h2 top = { (_Float16)0.f, (_Float16)0.f };
#pragma unroll
      for (int nb = 0; nb < NL; nb++) {
        const float nmr = m_ref[nb] == NEG_INF ? 0.f : -m_ref[nb];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 4][nb][j % 4], c1, nmr));
          const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j / 4][nb][j % 4 + 1], c1, nmr));
          const h2 pp = { (_Float16)e0, (_Float16)e1 };
          top = __builtin_elementwise_max(top, pp);
          pf[nb][j] = pp[0];
          pf[nb][j + 1] = pp[1];
        }
      }
      const _Float16 lim = (_Float16)256.f;
      return __any(top[0] > lim || top[1] > lim);
    };
    if (__builtin_expect(unseen, 0)) raise();
    if (__builtin_expect(probs(), 0)) { raise(); probs(); }
    // ---- O^T += V^T P^T, contraction slot 8 kg + j: position 4 kg + j, or 16 + 4 kg + j - 4; and l += the P that it uses ----
    const h2 ones = { (_Float16)1.f, (_Float16)1.f };
#pragma unroll
    for (int nb = 0; nb < NL; nb++)
#pragma unroll
      for (int j = 0; j < 8; j += 2) { const h2 pp = { pf[nb][j], pf[nb][j + 1] }; l_run[nb] = __builtin_amdgcn_fdot2(pp, ones, l_run[nb], false); }
    if constexpr (NL > 1) {
#pragma unroll
      for (int f = 0; f < VD; f++) fetch(f);
    }
#pragma unroll
    for (int f = 0; f < S::DB; f++) {
      const h4 l = lo[f % VD], h = hi[f % VD];
      const h8 a = { l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3] };
      if (f + VD < S::DB) fetch(f + VD);
#pragma unroll
      for (int nb = 0; nb < NL; nb++) acc[f][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf[nb], acc[f][nb], 0, 0, 0);
    }
    if constexpr (NL > 1) __builtin_amdgcn_sched_group_barrier(0x100, 2 * VD, 1);
#pragma unroll
    for (int f = 0; f < S::DB; f++) {
      __builtin_amdgcn_sched_group_barrier(0x008, NL, 1);
      if (f + VD < S::DB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
    }
  };
  // A tile that reaches the drafted rows: the next mask words where the ones at hand are through; and what is not finite in V's drafted rows becomes zero in LDS (see the head of the file)
  auto draft_tile = [&](uint32_t i) __attribute__((always_inline)) {
    const uint32_t d = i - draft0;
    if (d && d % WIN == 0) { fill_windows(d); __syncthreads(); }
    const uint32_t at = (wave * 64 + lane) * 16, context = p.base_pos > (tile0 + i) * 32 ? p.base_pos - (tile0 + i) * 32 : 0;     // the tile's rows in front of the draft
    unsigned char* vb = buf(i) + S::TILE + at;
    constexpr int NV = S::TILE / (W * 1024);
    bool any = false;
    u4 v[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
      v[j] = *(const u4*)(vb + j * W * 1024);
      any |= (at + j * W * 1024) / S::ROWB >= context && (not_finite2(v[j][0]) || not_finite2(v[j][1]) || not_finite2(v[j][2]) || not_finite2(v[j][3]));
    }
    any = __any(any);
    if (any) {
#pragma unroll
      for (int j = 0; j < NV; j++) {
        if ((at + j * W * 1024) / S::ROWB < context) continue;
#pragma unroll
        for (int e = 0; e < 4; e++) v[j][e] &= ((v[j][e] & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) | ((v[j][e] & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u);
        *(u4*)(vb + j * W * 1024) = v[j];
      }
    }
    if (lane == 0) bad_lds[wave] = any;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < W; w++) all |= bad_lds[w];
    bad |= all != 0;
  };

  // ---- main loop: behind turn i's barrier tile i is there for every wave, and every wave has done turn i - 1, so that tile i - 1's buffer takes what comes next ----
  if constexpr (Q8) {
    static_assert(!Q8 || D == 2, "int8 rows: a turn's tile and the one that is staged meanwhile");
    // When turn i begins, the registers of the other parity hold tile i + 1, those of its own tile i + 2.  Fetches and stores go on behind the last tile (the last one again, which nobody looks at):
    // under a condition the wait for the older registers would be one for the younger too.
    const uint32_t last = n_tiles - 1;
    stage8(0, I0{});
    fetch8(min(2u, last), I0{});
    auto step = [&](uint32_t i, auto NEXT) __attribute__((always_inline)) {
      wait_and_meet_lds();
      stage8(i + 1, NEXT);
      fetch8(min(i + 3, last), NEXT);
      if (__builtin_expect(i >= draft0, 0)) draft_tile(i);
      if constexpr (LIVE > 0) turn(i);
    };
    uint32_t i = 0;
    for (; i + 1 < n_tiles; i += 2) { step(i, I1{}); step(i + 1, I0{}); }
    if (i < n_tiles) step(i, I1{});
  } else {
    constexpr int LOADS = 2 * S::NLD;               // an issuing wave's loads of a tile
    for (uint32_t i = 0; i < n_tiles; i++) {
      // tiles up to i + D - 2 were issued: tile i is there when D - 2 tiles' loads are left
      if (!issuer) wait_and_meet_lds(); else if (i + D - 2 < n_tiles) wait_and_meet<LOADS * (D - 2)>(); else wait_and_meet<0>();
      if (issuer && i + D - 1 < n_tiles) issue(i + D - 1);
      if (__builtin_expect(i >= draft0, 0)) draft_tile(i);
      if constexpr (LIVE > 0) turn(i);
    }
  }

  // ---- the split's outputs: through LDS, so that a row leaves in whole lines ----
  wait_and_meet_lds();                              // every wave has read the last tile
  if constexpr (LIVE > 0) {
  // partials: O [kv head][split][stacked row][HD], so that what a wave writes is one piece; (m, l) [kv head][stacked row][split]
  const uint32_t rows_all = p.n_cols * G, c = lane % (HD / 8);
  constexpr int RPI = 64 / (HD / 8);                // rows of the wave at once, eight dims a lane
  constexpr int EROWS = RING / W / (HD * 4) < 16 ? 8 : 16;                  // f32 rows that a wave's part of the ring holds
  static_assert(EROWS * HD * 4 * W <= RING, "the rows fit the ring");
  float* os = (float*)(smem + wave * EROWS * HD * 4);
  auto put = [&](int nb, int half, float inv) __attribute__((always_inline)) {
    if (EROWS == 16 || (int)(ln / 8) == half) {
      const uint32_t r = ln % EROWS;
#pragma unroll
      for (int db = 0; db < S::DB; db++) *(f4*)(os + r * HD + ((4 * db + kg) ^ r) * 4) = acc[db][nb] * inv;
    }
    wave_fence();
  };
#pragma unroll
  for (int nb = 0; nb < NL; nb++) {
    l_run[nb] += __shfl_xor(l_run[nb], 16, 64);
    l_run[nb] += __shfl_xor(l_run[nb], 32, 64);
    const float inv = l_run[nb] == 0.f ? 0.f : 1.f / l_run[nb];             // a row that sees nothing: zeros
    const uint32_t r0 = row_of(nb, 0);
    if (p.n_splits > 1) {
      // (the sign of l says that a drafted row of the split holds what is not finite; a row of NaN scores may have found no reference)
      if (kg == 0 && r0 + ln < R)
        p.part_ml[((size_t)g * rows_all + x0 + r0 + ln) * p.n_splits + sp] = make_float2(l_run[nb] != l_run[nb] ? __builtin_inff() : m_ref[nb], bad ? -l_run[nb] : l_run[nb]);
      float* to = p.part_o + (((size_t)g * p.n_splits + sp) * rows_all + x0 + r0) * HD + lane * 4;
#pragma unroll
      for (int half = 0; half < 16 / EROWS; half++) {
        put(nb, half, inv);
#pragma unroll
        for (int it = 0; it < EROWS * HD / 256; it++) {                       // (1 KB of rows at once)
          const uint32_t r = it * 256 / HD + lane / (HD / 4), u = lane % (HD / 4);
          const f4 v = *(const f4*)(os + r * HD + (u ^ r) * 4);
          if (r0 + half * EROWS + r < R) __builtin_nontemporal_store(v, (f4*)(to + (half * EROWS * HD + it * 256)));
        }
        wave_fence();
      }
    } else {
      // all of the block's gates ahead (one after the other they are a trip to memory each: 5 columns at 20 rows, 16 / 2 heads of 256, 9.5 us a call, so 8.8, and 7.7 with a reciprocal for the division)
      f4 gt[16 / RPI][2];
      if (p.gate) {
#pragma unroll
        for (int it = 0; it < 16 / RPI; it++) {
          const uint32_t x = x0 + min(r0 + it * RPI + lane / (HD / 8), R - 1), col = col_of(x), hq = g * G + x - col * G;
          const float* gate = p.gate + (size_t)col * p.gate_stride + hq * HD + 8 * c;
          gt[it][0] = *(const f4*)gate;
          gt[it][1] = *(const f4*)(gate + 4);
        }
      }
#pragma unroll
      for (int half = 0; half < 16 / EROWS; half++) {
        put(nb, half, inv);
#pragma unroll
        for (int it = 0; it < EROWS / RPI; it++) {
          const uint32_t r = it * RPI + lane / (HD / 8), wr = r0 + half * EROWS + r;
          if (wr >= R) continue;
          const f4 a = *(const f4*)(os + r * HD + ((2 * c) ^ r) * 4), b = *(const f4*)(os + r * HD + ((2 * c + 1) ^ r) * 4);
          float o[8] = { a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3] };
          const uint32_t x = x0 + wr, col = col_of(x), hq = g * G + x - col * G;
          if (__builtin_expect(bad, 0)) add_not_finite(p, HD, col, g, 8 * c, o);
          if (p.gate) {
            const f4 ga = gt[half * (EROWS / RPI) + it][0], gb = gt[half * (EROWS / RPI) + it][1];
#pragma unroll
            for (int i = 0; i < 4; i++) { o[i] *= gate_of(ga[i]); o[4 + i] *= gate_of(gb[i]); }
          }
          store_dims(p, col, hq * HD + 8 * c, o);
        }
        wave_fence();
      }
    }
  }
  }
  };
  if (blocks == 1) run(std::integral_constant<int, 1>{});
  else if (blocks == 0) run(std::integral_constant<int, 0>{});
  else if constexpr (NB == 2) run(std::integral_constant<int, 2>{});
}

// Joins the splits of a (column, head): w_s = l_s 2^(m_s - M), out = sum w_s o_s / sum w_s, times sigmoid(gate).  A wavefront takes LPG x 4 dims of a (column, head): LPG lanes of four
// dims, 64 / LPG groups of lanes over the splits in turn, eight splits of a group in one round trip.
template <int HD, int LPG>
__global__ __launch_bounds__(256) void pa_tree_merge_kernel(TreeParams p) {
  constexpr uint32_t NG = 64 / LPG, B = 8, SL = HD / 4 / LPG;
  const uint32_t lane = threadIdx.x & 63, l4 = lane % LPG, grp = lane / LPG;
  const uint32_t wv = blockIdx.x * 4 + (threadIdx.x >> 6), row = wv / SL, rows_all = p.n_cols * p.group, ns = p.n_splits;
  if (row >= p.n_cols * p.n_heads) return;
  const uint32_t g = div_by(row, rows_all, p.rows_magic), x = row - g * rows_all;                 // kv head, stacked row
  const uint32_t col = div_by(x, p.group, p.g_magic), h = g * p.group + x - col * p.group, d = (wv % SL * LPG + l4) * 4;
  const float2* ml = p.part_ml + (size_t)row * ns;
  const float* po = p.part_o + ((size_t)g * ns * rows_all + x) * HD + d;
  const size_t step = (size_t)rows_all * HD;
  float2 m[B];
  f4 v[B];
  auto load = [&](uint32_t s0) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t k = 0; k < B; k++) {
      const uint32_t s = s0 + NG * k, at = min(s, ns - 1);
      m[k] = ml[at];
      u4 o = __builtin_nontemporal_load((const u4*)(po + at * step));
      o &= s < ns ? 0xffffffffu : 0u;               // (a surplus one is zeros: what is there may be infinite, and 0 x inf is not 0)
      __builtin_memcpy(&v[k], &o, 16);
      if (s >= ns) m[k] = make_float2(NEG_INF, 0.f);
    }
  };
  load(grp);
  f4 gt = {0.f, 0.f, 0.f, 0.f};
  if (p.gate) gt = *(const f4*)(p.gate + (size_t)col * p.gate_stride + h * HD + d);
  float M = NEG_INF;
#pragma unroll
  for (uint32_t k = 0; k < B; k++) M = fmaxf(M, m[k].x);
  for (uint32_t s = grp + NG * B; s < ns; s += NG) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (uint32_t o = LPG; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t sign = 0;
  if (M != NEG_INF) {
    for (uint32_t s0 = grp;;) {
#pragma unroll
      for (uint32_t k = 0; k < B; k++) {
        sign |= __float_as_uint(m[k].y);
        const float w = m[k].y == 0.f ? 0.f : __builtin_fabsf(m[k].y) * __builtin_amdgcn_exp2f(m[k].x - M);      // (a split that the row saw nothing of holds zeros)
        L += w;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(w, v[k][i], o[i]);
      }
      s0 += NG * B;
      if (s0 - grp >= ns) break;
      load(s0);
    }
  }
#pragma unroll
  for (uint32_t k = LPG; k < 64; k <<= 1) {
    L += __shfl_xor(L, k, 64);
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] += __shfl_xor(o[i], k, 64);
  }
  sign = __any(sign >> 31);
  if (grp) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] *= inv;
  if (__builtin_expect(sign, 0)) add_not_finite(p, HD, col, g, d, o);
  if (p.gate) {
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] *= gate_of(gt[i]);
  }
  store_dims(p, col, h * HD + d, o);
}

// (the divisions at the head of the kernels, some thirty instructions each, cost 1 - 2 us a call)
static void set_magics(TreeParams& p) {
  const uint64_t gs = (uint64_t)p.n_kv_heads * p.n_splits;
  p.ng_magic = div_magic(gs * p.n_groups + 8, p.n_groups);
  p.ns_magic = div_magic(gs + 8, p.n_splits);
  p.g_magic = div_magic((uint64_t)p.n_cols * p.group, p.group);
  p.rows_magic = div_magic((uint64_t)p.n_cols * p.n_heads, p.n_cols * p.group);
}

template <int HD, int NB, bool Q8, int QP>
static hipError_t launch_tree_k(const TreeParams& p, hipStream_t s, const PaTiming* t) {
  typedef TreeShape<HD, TREE_W> S;
  constexpr int D = Q8 ? 2 : 4;
  constexpr size_t lds = (size_t)D * 2 * S::TILE + TreeLds<NB>::bytes;
  static_assert(lds <= 160 * 1024, "the ring fits a CU");
  if (p.n_groups == 0 || p.group_rows == 0 || p.group_rows > 16u * NB * TREE_W || (uint64_t)(p.n_groups - 1) * p.group_rows >= (uint64_t)p.n_cols * p.group ||
      (uint64_t)p.n_groups * p.group_rows < (uint64_t)p.n_cols * p.group || p.n_splits == 0 ||
      (uint64_t)(p.n_splits - 1) * p.split_tiles * 32 >= (uint64_t)p.base_pos + p.n_cols || (uint64_t)p.n_splits * p.split_tiles * 32 < (uint64_t)p.base_pos + p.n_cols) return hipErrorInvalidValue;
  if (QP == Q_SPARE_ROWS && (uint64_t)p.n_cols * p.group > 8) return hipErrorInvalidValue;
  const uint64_t total = (uint64_t)p.n_groups * p.n_kv_heads * p.n_splits;
  if (total > 0x7fffff00ull) return hipErrorInvalidValue;
  static PaPerDevice lds_set;
  const hipError_t e = pa_lds_limit(lds_set, (const void*)pa_tree_kernel<HD, NB, Q8, D, QP>, lds);
  if (e != hipSuccess) return e;
  TreeParams pk = p;
  set_magics(pk);
  PA_LAUNCH((pa_tree_kernel<HD, NB, Q8, D, QP>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(TREE_W * 64), lds, s, t, pk);
  return hipGetLastError();
}

template <int HD, bool Q8>
static hipError_t launch_tree_hd(const TreeParams& p, const TreePlan& pl, hipStream_t s, const PaTiming* t) {
  switch (pl.nb) {
    case 1: return (uint64_t)p.n_cols * p.group <= 8 ? launch_tree_k<HD, 1, Q8, Q_SPARE_ROWS>(p, s, t) : launch_tree_k<HD, 1, Q8, Q8 ? Q_F16 : Q_TWICE>(p, s, t);
    case 2: if constexpr (HD == 128 || !Q8) return launch_tree_k<HD, 2, Q8, Q8 || HD == 256 ? Q_F16 : Q_TWICE>(p, s, t); else return hipErrorInvalidValue;
    default: return hipErrorInvalidValue;
  }
}

hipError_t pa_launch_tree(const TreeParams& p, const TreePlan& pl, uint32_t hd, hipStream_t s, const PaTiming* t) {
  if (hd == 256) return p.k_scale ? launch_tree_hd<256, true>(p, pl, s, t) : launch_tree_hd<256, false>(p, pl, s, t);
  if (hd == 128) return p.k_scale ? launch_tree_hd<128, true>(p, pl, s, t) : launch_tree_hd<128, false>(p, pl, s, t);
  return hipErrorInvalidValue;
}

// As many lanes a slice as leave groups for all of a row's splits in one round trip: whole rows a wave for few splits, narrow slices for many
template <int HD>
static void launch_merge(const TreeParams& p, hipStream_t s, const PaTiming* t) {
  const uint32_t rows = p.n_cols * p.n_heads;
  auto grid = [&](uint32_t lpg) { return dim3((unsigned)(((uint64_t)rows * (HD / 4 / lpg) + 3) / 4)); };
  if (HD == 256 && p.n_splits <= 8) PA_LAUNCH((pa_tree_merge_kernel<256, 64>), grid(64), dim3(256), 0, s, t, p);
  else if (p.n_splits <= 16) PA_LAUNCH((pa_tree_merge_kernel<HD, 32>), grid(32), dim3(256), 0, s, t, p);
  else if (p.n_splits <= 32) PA_LAUNCH((pa_tree_merge_kernel<HD, 16>), grid(16), dim3(256), 0, s, t, p);
  else if (p.n_splits <= 64) PA_LAUNCH((pa_tree_merge_kernel<HD, 8>), grid(8), dim3(256), 0, s, t, p);
  else PA_LAUNCH((pa_tree_merge_kernel<HD, 4>), grid(4), dim3(256), 0, s, t, p);
}

hipError_t pa_launch_tree_merge(const TreeParams& p_in, uint32_t hd, hipStream_t s, const PaTiming* t) {
  TreeParams p = p_in;
  set_magics(p);
  if (hd == 256) launch_merge<256>(p, s, t);
  else if (hd == 128) launch_merge<128>(p, s, t);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}
