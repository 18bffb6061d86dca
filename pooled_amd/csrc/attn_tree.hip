// Attention of a tree of drafted tokens over a cache, on f16 MFMA for gfx950.
//
// Column c of n sees the cache rows [0, base) and those rows base + j whose bit j is set in its mask:
//   o[c, h] = sum_t softmax_t(q[c, h] . k[t] / sqrt(hd)) v[t]
// The G query heads of a kv head and all columns are stacked rows (row = column x G + head), so K and V are read once for all of them.
//
//   * A workgroup is W wavefronts of 16 NB stacked rows each over one split of the context; every 32-row tile of K and V that it stages in LDS serves
//     all of its waves.  Tiles go global -> LDS directly, D - 1 of them in flight (int8 rows: through registers, widened on the way); one barrier a tile.
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_f16: Q fragments stay in registers, K fragments are 16-byte LDS reads, V^T fragments come from the
//     LDS transpose read.  The accumulator of S^T is the operand of P V, so probabilities never leave registers.
//   * Online softmax in f32 in the exp2 domain: the reference of a row is raised, and O and l rescaled, only where a P comes out above 2^8 (exact enough in f16); l is
//     the sum of the rounded P, so an output is a convex combination of value rows whatever that rounding did.
//   * The mask is looked at only in tiles that reach the drafted rows.  There a row's 32 bits are one word, cut out of its mask at the tile's offset with the rows in front
//     of the draft as ones.  A drafted row that holds what is not finite must reach those columns alone that see it, and 0 x inf is not 0: such elements go into the product as
//     zeros and are added to the outputs of the columns that see them.
//   * Splits leave (m, l) and O / l in f16: a convex combination of f16 values loses 2^-12 of itself by that (mean of a rounding of at most 2^-11), below what the f16 P
//     lose, and the partials are half the bytes; pa_tree_merge_kernel joins them.
#include "tree_internal.h"
#include "pf_common.h"
#include "tree_mask.h"

template <int HD, int W> struct TreeShape {
  static constexpr int ROWB = HD * 2;               // bytes of a staged row
  static constexpr int TILE = 32 * ROWB;            // bytes of a staged tile of K or of V
  static constexpr int KS = HD / 32;                // k-steps of the QK product
  static constexpr int DB = HD / 16;                // 16-dim blocks of the output
  static constexpr int CPR = HD / 8;                // 16-byte chunks of a staged row
  static constexpr int RPB = 64 / CPR;              // rows of a 1 KB LDS-direct load
  static constexpr int NLD = 32 / RPB / W;          // LDS-direct loads of a wave, a tensor and tile
  static constexpr int PIECES = 32 * HD / 16;       // int8 rows: 16-byte pieces of a tile of K or of V ...
  static constexpr int NP8 = 2 * PIECES / (W * 64); // ... and a thread's share of both
  static_assert(NLD * W * RPB == 32, "a tile divides evenly over the waves");
  static_assert(NP8 * W * 64 == 2 * PIECES && PIECES % 64 == 0, "an int8 tile divides evenly over the threads, a wave's pieces are of one tensor");
};

static __device__ inline bool not_finite(_Float16 v) {
  unsigned short b;
  __builtin_memcpy(&b, &v, 2);
  return (b & 0x7C00u) == 0x7C00u;
}

template <int N> static __device__ inline void wait_and_meet() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory"); }

template <int HD, int NB, int W, bool Q8, int D>
__global__ __launch_bounds__(W * 64, W / 4) void pa_tree_kernel(TreeParams p) {
  typedef TreeShape<HD, W> S;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];     // [D][K tile | V tile]
  // work items are (kv head, split, group of rows), the group fastest; dispatch id i runs on XCD i % 8, which owns a contiguous range of items, so the groups that
  // read the same rows share an L2
  const uint32_t total = p.n_groups * p.n_kv_heads * p.n_splits, per = (total + 7) / 8;
  const uint32_t item = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per || item >= total) return;
  const uint32_t grp = item % p.n_groups, gs = item / p.n_groups, sp = gs % p.n_splits, g = gs / p.n_splits;
  const uint32_t tid = threadIdx.x, lane = tid & 63, ln = lane & 15, kg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t G = p.group, nH = p.n_heads;
  const uint32_t x0 = grp * p.group_rows, R = min(p.group_rows, p.n_cols * G - x0);     // the group's stacked rows [x0, x0 + R)
  const uint32_t end = p.base_pos + p.n_cols;
  const uint32_t tile0 = sp * p.split_tiles, n_tiles = min(p.split_tiles, (end + 31) / 32 - tile0);
  const size_t head_rows = (size_t)p.max_seq + 32;

  // ---- staging ----
  auto k_slot = [](uint32_t row, uint32_t chunk) __attribute__((always_inline)) { return chunk ^ (row & 15); };      // conflict-free 16-byte fragment reads
  auto v_slot = [](uint32_t row, uint32_t chunk) __attribute__((always_inline)) { return chunk ^ (4 * (row & 3)) ^ (2 * ((row >> 2) & 1)); };   // 2-way for the transpose reads, their best
  auto kbuf = [&](uint32_t i) __attribute__((always_inline)) { return smem + (i % D) * 2 * S::TILE; };
  // f16 rows: load j of wave w fills the 1 KB block j W + w of a buffer, rows (j W + w) RPB ..; lane l lands at (row l / CPR, slot l % CPR) and fetches the chunk that belongs there
  auto issue = [&](uint32_t i) __attribute__((always_inline)) {
    const uint32_t tp = (tile0 + i) * 32;
    const unsigned char* kb = (const unsigned char*)p.k_cache + (size_t)g * head_rows * S::ROWB;
    const unsigned char* vb = (const unsigned char*)p.v_cache + (size_t)g * head_rows * S::ROWB;
    unsigned char* dst = kbuf(i);
#pragma unroll
    for (int j = 0; j < S::NLD; j++) {
      const uint32_t r = (j * W + wave) * S::RPB + lane / S::CPR, c = lane % S::CPR;
      const uint32_t row = tp + r < end ? tp + r : p.max_seq;                // (rows behind the last one: the cache's zero padding)
      PF_GLL(kb + (size_t)row * S::ROWB + k_slot(r, c) * 16, dst + (j * W + wave) * 1024);
      PF_GLL(vb + (size_t)row * S::ROWB + v_slot(r, c) * 16, dst + S::TILE + (j * W + wave) * 1024);
    }
  };
  // int8 rows: a thread's 16-byte pieces of a tile, K's and then V's, and their scales; two tiles in registers
  u4 raw8[2][S::NP8];
  float sc8[2][S::NP8];
  auto fetch8 = [&](uint32_t i, auto AT) __attribute__((always_inline)) {
    constexpr int at = decltype(AT)::value;
    const uint32_t tp = (tile0 + i) * 32;
#pragma unroll
    for (int j = 0; j < S::NP8; j++) {
      const uint32_t e = tid + j * W * 64, of_v = (wave * 64 + j * W * 64) / S::PIECES, r = e % S::PIECES / (HD / 16), c = e % (HD / 16);
      const size_t row = (size_t)g * head_rows + (tp + r < end ? tp + r : p.max_seq);
      raw8[at][j] = *(const u4*)((const unsigned char*)(of_v ? p.v_cache : p.k_cache) + row * HD + c * 16);
      sc8[at][j] = (of_v ? p.v_scale : p.k_scale)[row * (HD / 32) + c / 2];
    }
  };
  auto widen = [&](u4 raw, float sc, unsigned char* row, uint32_t s0, uint32_t s1) __attribute__((always_inline)) {
    // int8 -> f16 through the bit pattern 0x6400 | (v + 128) = 1152 + v, exactly, then times the f16-rounded scale
    const h2 s2 = { (_Float16)sc, (_Float16)sc }, off = { (_Float16)1152.f, (_Float16)1152.f };
    h2 o[8];
#pragma unroll
    for (int d = 0; d < 4; d++) {
      const uint32_t w = raw[d] ^ 0x80808080u;
      const uint32_t a = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u), b = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
      h2 xa, xb;
      __builtin_memcpy(&xa, &a, 4);
      __builtin_memcpy(&xb, &b, 4);
      o[2 * d] = (xa - off) * s2;
      o[2 * d + 1] = (xb - off) * s2;
    }
    *(h8*)(row + s0 * 16) = (h8){ o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1] };
    *(h8*)(row + s1 * 16) = (h8){ o[4][0], o[4][1], o[5][0], o[5][1], o[6][0], o[6][1], o[7][0], o[7][1] };
  };
  auto stage8 = [&](uint32_t i, auto AT) __attribute__((always_inline)) {
    constexpr int at = decltype(AT)::value;
    unsigned char* dst = kbuf(i);
#pragma unroll
    for (int j = 0; j < S::NP8; j++) {
      const uint32_t e = tid + j * W * 64, of_v = (wave * 64 + j * W * 64) / S::PIECES, r = e % S::PIECES / (HD / 16), c = e % (HD / 16) * 2;
      widen(raw8[at][j], sc8[at][j], dst + of_v * S::TILE + r * S::ROWB, of_v ? v_slot(r, c) : k_slot(r, c), of_v ? v_slot(r, c + 1) : k_slot(r, c + 1));
    }
  };
  typedef std::integral_constant<int, 0> I0;
  typedef std::integral_constant<int, 1> I1;
  if constexpr (Q8) {
    fetch8(0, I0{});
    if (n_tiles > 1) fetch8(1, I1{});
  } else {
#pragma unroll
    for (int i = 0; i < D - 1; i++) if ((uint32_t)i < n_tiles) issue(i);
  }

  // ---- the wave's rows: Q fragments (row ln of block nb, dims 32 ks + 8 kg .. + 7) ----
  const uint32_t wrow0 = wave * 16 * NB;
  const bool live = wrow0 < R;
  h8 qf[NB][S::KS];
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
    const uint32_t x = x0 + min(wrow0 + nb * 16 + ln, R - 1), col = x / G;
    const float* qrow = p.q + (size_t)col * p.q_stride + (size_t)(g * G + x - col * G) * HD + 8 * kg;
#pragma unroll
    for (int ks = 0; ks < S::KS; ks++) {
      const f4 a = *(const f4*)(qrow + 32 * ks), b = *(const f4*)(qrow + 32 * ks + 4);
      qf[nb][ks] = (h8){ (_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3], (_Float16)b[0], (_Float16)b[1], (_Float16)b[2], (_Float16)b[3] };
    }
  }
  f4 acc[S::DB][NB];
  float m_ref[NB], l_run[NB];
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
#pragma unroll
    for (int db = 0; db < S::DB; db++) acc[db][nb] = (f4){0.f, 0.f, 0.f, 0.f};
    m_ref[nb] = NEG_INF;
    l_run[nb] = 0.f;
  }
  bool unseen = true;                               // a row of the wave has no reference yet
  const float c1 = p.scale * 1.4426950408889634f;   // scores -> log2 domain
  const uint32_t k_rd = ln * S::ROWB + (kg ^ ln) * 16;                                                                        // K fragment of k-step ks at k_rd ^ 64 ks
  const uint32_t v_rd = (4 * kg + (ln >> 2)) * S::ROWB + (((ln & 3) >> 1) ^ (4 * (ln >> 2)) ^ (2 * (kg & 1))) * 16 + (ln & 1) * 8;   // V fragment of block db at v_rd ^ 32 db

  auto tile = [&](const unsigned char* kb, const uint32_t tp) __attribute__((always_inline)) {
    const unsigned char* vb = kb + S::TILE;
    f4 s[2][NB];
    h8 pf[NB];
    uint32_t win[NB];
#pragma unroll
    for (int pb = 0; pb < 2; pb++)
#pragma unroll
      for (int nb = 0; nb < NB; nb++) s[pb][nb] = (f4){0.f, 0.f, 0.f, 0.f};
    // ---- S^T = K Q^T; a lane then holds row ln of each block, positions tp + 16 pb + 4 kg + i ----
#pragma unroll
    for (int f = 0; f < 2 * S::KS; f++) {
      const h8 a = *(const h8*)(kb + (k_rd ^ (f / 2 % 4 * 64)) + f / 8 * 256 + f % 2 * 16 * S::ROWB);
#pragma unroll
      for (int nb = 0; nb < NB; nb++) s[f % 2][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[nb][f / 2], s[f % 2][nb], 0, 0, 0);
    }
    const bool draft = tp + 32 > p.base_pos;        // the tile reaches the drafted rows
    if (draft) {
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        const uint32_t x = x0 + min(wrow0 + nb * 16 + ln, R - 1);
        win[nb] = mask_window(p.mask + (size_t)(x / G) * p.mask_stride, (int)(tp - p.base_pos), p.n_cols);
#pragma unroll
        for (int pb = 0; pb < 2; pb++)
#pragma unroll
          for (int i = 0; i < 4; i++) s[pb][nb][i] = win[nb] >> (16 * pb + 4 * kg + i) & 1 ? s[pb][nb][i] : NEG_INF;
      }
    }
    // ---- softmax ----
    auto raise = [&]() __attribute__((always_inline)) {
      bool none = false;
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
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
    auto probs = [&]() __attribute__((always_inline)) -> bool {
      h2 top = { (_Float16)0.f, (_Float16)0.f };
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
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
    const h2 ones = { (_Float16)1.f, (_Float16)1.f };
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int j = 0; j < 8; j += 2) { const h2 pp = { pf[nb][j], pf[nb][j + 1] }; l_run[nb] = __builtin_amdgcn_fdot2(pp, ones, l_run[nb], false); }
    // ---- O^T += V^T P^T, contraction slot 8 kg + j: position 4 kg + j, or 16 + 4 kg + j - 4 ----
    auto pv = [&](auto CLEAN) __attribute__((always_inline)) -> bool {
      bool bad = false;
#pragma unroll
      for (int f = 0; f < S::DB; f++) {
        const unsigned char* vp = vb + (v_rd ^ (f % 8 * 32)) + f / 8 * 256;
        const h4 lo = lds_read_tr16(vp), hi = lds_read_tr16(vp + 16 * S::ROWB);
        h8 a = { lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3] };
        if constexpr (decltype(CLEAN)::value) {
#pragma unroll
          for (int j = 0; j < 8; j++) if (not_finite(a[j])) { a[j] = (_Float16)0.f; bad = true; }
        }
#pragma unroll
        for (int nb = 0; nb < NB; nb++) acc[f][nb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf[nb], acc[f][nb], 0, 0, 0);
      }
      return bad;
    };
    if (!draft) pv(std::false_type{});
    else if (__any(pv(std::true_type{}))) {
      // what is not finite, element by element: to the rows that see it
      for (uint32_t r = 0; r < 32; r++)
#pragma unroll
        for (int db = 0; db < S::DB; db++) {
          const uint32_t d = 16 * db + 4 * kg;
          const h4 v = *(const h4*)(vb + r * S::ROWB + v_slot(r, d / 8) * 16 + d % 8 * 2);
#pragma unroll
          for (int i = 0; i < 4; i++)
            if (not_finite(v[i])) {
#pragma unroll
              for (int nb = 0; nb < NB; nb++) if (win[nb] >> r & 1) acc[db][nb][i] += (float)v[i];
            }
        }
    }
  };

  // ---- main loop: tile i is there behind the barrier, and every wave has done tile i - 1, whose buffer takes the load that goes out next ----
  if constexpr (Q8) {
    static_assert(D == 2, "int8 rows: two buffers");
    auto turn = [&](uint32_t i, auto AT, auto NEXT) __attribute__((always_inline)) {
      // registers NEXT hold tile i + 1, registers AT are free
      if (i + 2 < n_tiles) fetch8(i + 2, AT);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (live) tile(kbuf(i), (tile0 + i) * 32);
      if (i + 1 < n_tiles) stage8(i + 1, NEXT);
    };
    stage8(0, I0{});
    uint32_t i = 0;
    for (; i + 1 < n_tiles; i += 2) { turn(i, I0{}, I1{}); turn(i + 1, I1{}, I0{}); }
    if (i < n_tiles) turn(i, I0{}, I1{});
  } else {
    constexpr int AHEAD = 2 * S::NLD * (D - 2);     // a wave's loads behind tile i's
    for (uint32_t i = 0; i < n_tiles; i++) {
      if (i + D - 2 < n_tiles) wait_and_meet<AHEAD>(); else wait_and_meet<0>();
      if (i + D - 1 < n_tiles) issue(i + D - 1);
      if (live) tile(kbuf(i), (tile0 + i) * 32);
    }
  }
  if (!live) return;

  // ---- the split's outputs ----
#pragma unroll
  for (int nb = 0; nb < NB; nb++) {
    l_run[nb] += __shfl_xor(l_run[nb], 16, 64);
    l_run[nb] += __shfl_xor(l_run[nb], 32, 64);
    const uint32_t r = wrow0 + nb * 16 + ln;
    if (r >= R) continue;
    const uint32_t x = x0 + r, col = x / G, hq = g * G + x - col * G;
    const float inv = l_run[nb] == 0.f ? 0.f : 1.f / l_run[nb];             // a row that sees nothing: zeros
    if (p.n_splits == 1) {
      const float* gate = p.gate ? p.gate + (size_t)col * p.gate_stride + (size_t)hq * HD : nullptr;
#pragma unroll
      for (int db = 0; db < S::DB; db++) {
        const uint32_t d = 16 * db + 4 * kg;
        f4 o = acc[db][nb] * inv;
        if (gate) {
          const f4 gt = *(const f4*)(gate + d);
#pragma unroll
          for (int i = 0; i < 4; i++) o[i] *= 1.f / (1.f + __expf(-gt[i]));
        }
        if (p.out_f16) *(h4*)((_Float16*)p.out + (size_t)col * p.out_stride + (size_t)hq * HD + d) = (h4){ (_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3] };
        else *(f4*)((float*)p.out + (size_t)col * p.out_stride + (size_t)hq * HD + d) = o;
      }
    } else {
      const size_t slot = ((size_t)col * nH + hq) * p.n_splits + sp;
#pragma unroll
      for (int db = 0; db < S::DB; db++) {
        const f4 o = acc[db][nb] * inv;
        *(h4*)((_Float16*)p.part_o + slot * HD + 16 * db + 4 * kg) = (h4){ (_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3] };
      }
      if (kg == 0) p.part_ml[slot] = make_float2(m_ref[nb], l_run[nb]);
    }
  }
}

// Joins the splits of a (column, head): w_s = l_s 2^(m_s - M), out = sum w_s o_s / sum w_s, times sigmoid(gate).  A wavefront takes one (column, head): HD / 8 lanes of
// eight dims, 512 / HD groups of lanes over the splits in turn.
template <int HD>
__global__ __launch_bounds__(256) void pa_tree_merge_kernel(TreeParams p) {
  constexpr uint32_t LPR = HD / 8, NG = 64 / LPR, B = 8;
  const uint32_t lane = threadIdx.x & 63, l8 = lane % LPR, grp = lane / LPR;
  const uint32_t x = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (x >= p.n_cols * p.n_heads) return;
  const uint32_t col = x / p.n_heads, h = x - col * p.n_heads, ns = p.n_splits;
  const float2* ml = p.part_ml + (size_t)x * ns;
  const h8* po = (const h8*)((const _Float16*)p.part_o + (size_t)x * ns * HD) + l8;
  float M = NEG_INF;
  for (uint32_t s = lane; s < ns; s += 64) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  float L = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (M != NEG_INF) {
    for (uint32_t s0 = grp; s0 < ns; s0 += NG * B) {
      float2 m[B];
      h8 v[B];
#pragma unroll
      for (uint32_t k = 0; k < B; k++) { const uint32_t s = min(s0 + NG * k, ns - 1); m[k] = ml[s]; v[k] = po[(size_t)s * LPR]; }
#pragma unroll
      for (uint32_t k = 0; k < B; k++) {
        const float w = s0 + NG * k < ns ? m[k].y * __builtin_amdgcn_exp2f(m[k].x - M) : 0.f;
        if (w != 0.f) {                             // (a split that the row saw nothing of holds zeros)
          L += w;
#pragma unroll
          for (int i = 0; i < 8; i++) o[i] += w * (float)v[k][i];
        }
      }
    }
  }
#pragma unroll
  for (uint32_t k = LPR; k < 64; k <<= 1) {
    L += __shfl_xor(L, k, 64);
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] += __shfl_xor(o[i], k, 64);
  }
  if (grp) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const uint32_t d = h * HD + 8 * l8;
  if (p.gate) {
    const float* gate = p.gate + (size_t)col * p.gate_stride + d;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] *= inv / (1.f + __expf(-gate[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] *= inv;
  }
  if (p.out_f16) {
    _Float16* out = (_Float16*)p.out + (size_t)col * p.out_stride + d;
    *(h4*)out = (h4){ (_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3] };
    *(h4*)(out + 4) = (h4){ (_Float16)o[4], (_Float16)o[5], (_Float16)o[6], (_Float16)o[7] };
  } else {
    float* out = (float*)p.out + (size_t)col * p.out_stride + d;
    *(f4*)out = (f4){ o[0], o[1], o[2], o[3] };
    *(f4*)(out + 4) = (f4){ o[4], o[5], o[6], o[7] };
  }
}

template <int HD, int NB, int W, bool Q8>
static hipError_t launch_tree_k(const TreeParams& p, hipStream_t s, const PaTiming* t) {
  typedef TreeShape<HD, W> S;
  constexpr int D = Q8 ? 2 : 4;
  constexpr size_t lds = (size_t)D * 2 * S::TILE;
  static_assert(lds <= 160 * 1024, "the ring fits a CU");
  if (p.n_groups == 0 || p.group_rows == 0 || p.group_rows > 16u * NB * W || (uint64_t)(p.n_groups - 1) * p.group_rows >= (uint64_t)p.n_cols * p.group ||
      (uint64_t)p.n_groups * p.group_rows < (uint64_t)p.n_cols * p.group || p.n_splits == 0 ||
      (uint64_t)(p.n_splits - 1) * p.split_tiles * 32 >= (uint64_t)p.base_pos + p.n_cols || (uint64_t)p.n_splits * p.split_tiles * 32 < (uint64_t)p.base_pos + p.n_cols) return hipErrorInvalidValue;
  const uint64_t total = (uint64_t)p.n_groups * p.n_kv_heads * p.n_splits;
  if (total > 0x7fffff00ull) return hipErrorInvalidValue;
  static PaPerDevice lds_set;
  const hipError_t e = pa_lds_limit(lds_set, (const void*)pa_tree_kernel<HD, NB, W, Q8, D>, lds);
  if (e != hipSuccess) return e;
  PA_LAUNCH((pa_tree_kernel<HD, NB, W, Q8, D>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(W * 64), lds, s, t, p);
  return hipGetLastError();
}

template <int HD, bool Q8>
static hipError_t launch_tree_hd(const TreeParams& p, const TreePlan& pl, hipStream_t s, const PaTiming* t) {
  if (pl.waves != 8) return hipErrorInvalidValue;
  switch (pl.nb) {
    case 1: return launch_tree_k<HD, 1, 8, Q8>(p, s, t);
    case 2: return launch_tree_k<HD, 2, 8, Q8>(p, s, t);
    default: return hipErrorInvalidValue;
  }
}

hipError_t pa_launch_tree(const TreeParams& p, const TreePlan& pl, uint32_t hd, hipStream_t s, const PaTiming* t) {
  if (hd == 256) return p.k_scale ? launch_tree_hd<256, true>(p, pl, s, t) : launch_tree_hd<256, false>(p, pl, s, t);
  if (hd == 128) return p.k_scale ? launch_tree_hd<128, true>(p, pl, s, t) : launch_tree_hd<128, false>(p, pl, s, t);
  return hipErrorInvalidValue;
}

hipError_t pa_launch_tree_merge(const TreeParams& p, uint32_t hd, hipStream_t s, const PaTiming* t) {
  const dim3 grid((p.n_cols * p.n_heads + 3) / 4);
  if (hd == 256) PA_LAUNCH(pa_tree_merge_kernel<256>, grid, dim3(256), 0, s, t, p);
  else if (hd == 128) PA_LAUNCH(pa_tree_merge_kernel<128>, grid, dim3(256), 0, s, t, p);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}
