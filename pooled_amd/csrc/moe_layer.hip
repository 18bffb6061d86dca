// A mixture-of-experts layer over a few tokens on gfx950: rmsnorm, router, top-k, the chosen experts and the shared one, weighted sum, residual.
//
//   xn = rmsnorm(x) w;  l = router xn;  chosen = the top_k largest l;  h_e = silu(gate_e xn) * (up_e xn);  y = x + sum w_e down_e h_e
//
// With a few tokens the work is the stream of the chosen experts' weights: one token of 8 experts of 512 x 2048 and a shared one reads 16 MB of Q4_0
// planes and 2 MB of router and computes 58 MFLOP.  Three launches, because each needs all of the one before: logits, h, y.
//   1. router: a wavefront a row (expert) and token, over the raw x; the norm's factor is taken out of the sum, so sum of squares and dot run together.
//      One more wavefront a token writes xn.
//   2. gate and up: a workgroup 16 rows of an expert.  With a few tokens it finds which expert that is by itself, from the token's logits (a maximum over the 64 lanes per place),
//      while xn is on its way; with more of them the choice is a launch of its own, and for f32 weights a workgroup serves up to four tokens that share an expert.
//   3. down: the experts of a token lie behind one another as ONE input of slots x ffn values, so a wavefront's row is one dot product over it.
// A lane owns whole 32-value blocks of the input (one 16-byte load of Q4_0), for all rows of its wavefront; activations are kept in the order
// in which lanes load them, so that every load is 1 KB of consecutive bytes.  Arithmetic is f32, every sum in an order that depends on the layer's sizes alone:
// no atomics, and a token's bits do not depend on the other tokens of the call.
//
// Measured with 256 experts of 512 x 2048, 8 chosen and one shared (router, choice, gate and up, down, in us): 1 token of Q4_0 4.5 + 7 + 5, each a launch's latency and a trip or two to
// memory; 5 of Q8_0 5 + 22 + 14 for 131 MB of distinct weights, gate and up at 4 TB/s (a large copy runs at 4.9); 16 of Q4_0 7.5 + 5 + 32 + 22 for 182 MB, gate and up at
// 3.8 TB/s.  f32, 27 tokens, 61 experts of 352 x 1056, 5 chosen: 5 + 5 + 41 + 26 for 245 MB.
#include "blocks_internal.h"
#include "glue_math.h"
#include <algorithm>

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

template <int CTRL> static __device__ inline uint32_t dpp_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false); }
static __device__ inline uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp_u32<0xB1>(v));
  v = max(v, dpp_u32<0x4E>(v));
  v = max(v, dpp_u32<0x141>(v));
  v = max(v, dpp_u32<0x140>(v));
  return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
             max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

// ---- weights: what a lane holds of a row at a time -----------------------------------------------
// Q8_0 and Q4_0: a block of 32 values with its scale; F32: two times four values, 64 lanes apart.  X: the float4 of activation that go with it.
// Dequantisation is what bounds a pass of several tokens, so it is kept to 1.1 (Q4_0) and 1 (Q8_0: the conversion of a signed byte in place) instructions a weight beside the multiply-add.
// Q4_0: the bits of an unsigned weight u in the low bits of an f16 ARE the number u 2^-24 (subnormal), and the mixed-precision multiply-add takes an f16 as it is.  A word gives its eight
// nibbles as four masked pairs, every other one 16 times too large in place: the activations that meet those (elements 16 to 31 of a block) are kept divided by 16.  The offset of 8 comes
// off each pair by a packed f16 addition, which is exact there, before the activation is met: taken off the sum instead, as 8 times the block's sum of activations, it needs half an instruction
// a weight less (16 tokens: gate and up 28 us instead of 32, down 20 instead of 22), but an activation much larger than its neighbours that meets a weight of zero then costs them their bits.
template <int KIND> struct Piece { static constexpr int F4 = 8; static constexpr uint32_t STEP = 64; u4 w[KIND == PA_W_Q8_0 ? 2 : 1]; uint16_t sc; };
template <> struct Piece<PA_W_F32> { static constexpr int F4 = 2; static constexpr uint32_t STEP = 128; f4 w[2]; };
template <int KIND> struct Act { f4 x[Piece<KIND>::F4]; uint32_t have; };   // have: how many of the lane's loads lie in the row
template <int KIND> static __device__ inline uint32_t pieces(uint32_t values) { return KIND == PA_W_F32 ? values / 4 : values / 32; }

static __device__ inline float f16_bits_f32(uint16_t b) { _Float16 h; __builtin_memcpy(&h, &b, 2); return (float)h; }
static __device__ inline h2v halves(uint32_t w) { h2v v; __builtin_memcpy(&v, &w, 4); return v; }

// acc + f * (piece . x)
template <int KIND>
static __device__ inline float dot_piece(const Piece<KIND>& r, const Act<KIND>& act, float f, float acc) {
  const auto& x = act.x;
  float a = 0.f, b = 0.f;
  if constexpr (KIND == PA_W_F32) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if (i >= (int)act.have) break;
      a = __builtin_fmaf(r.w[i][0], x[i][0], a); b = __builtin_fmaf(r.w[i][1], x[i][1], b);
      a = __builtin_fmaf(r.w[i][2], x[i][2], a); b = __builtin_fmaf(r.w[i][3], x[i][3], b);
    }
    return __builtin_fmaf(a + b, f, acc);
  } else if constexpr (KIND == PA_W_Q8_0) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t word = r.w[i >> 2][i & 3];
      a = __builtin_fmaf((float)(int8_t)word, x[i][0], a); b = __builtin_fmaf((float)(int8_t)(word >> 8), x[i][1], b);
      a = __builtin_fmaf((float)(int8_t)(word >> 16), x[i][2], a); b = __builtin_fmaf((float)(int8_t)(word >> 24), x[i][3], b);
    }
    return __builtin_fmaf(a + b, f * f16_bits_f32(r.sc), acc);
  } else {
    // byte j of the block = elements j (low nibble) and j + 16 (high)
    const h2v low = halves(0x80088008u), high = halves(0x80808080u);   // -8 2^-24, -8 x 16 2^-24
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t w0 = r.w[0][k], w1 = w0 >> 8;
      const h2v p0 = halves(w0 & 0x000F000Fu) + low, p1 = halves(w0 & 0x00F000F0u) + high, p2 = halves(w1 & 0x000F000Fu) + low, p3 = halves(w1 & 0x00F000F0u) + high;
      a = __builtin_fmaf((float)p0[0], x[k][0], a); b = __builtin_fmaf((float)p1[0], x[k + 4][0], b);
      a = __builtin_fmaf((float)p0[1], x[k][2], a); b = __builtin_fmaf((float)p1[1], x[k + 4][2], b);
      a = __builtin_fmaf((float)p2[0], x[k][1], a); b = __builtin_fmaf((float)p3[0], x[k + 4][1], b);
      a = __builtin_fmaf((float)p2[1], x[k][3], a); b = __builtin_fmaf((float)p3[1], x[k + 4][3], b);
    }
    return __builtin_fmaf(a + b, f * f16_bits_f32(r.sc) * 16777216.0f, acc);
  }
}

// Activations in reading order: for quantised weights groups of 64 blocks, in a group eight times 64 lanes x 4 values; for f32 weights as they are.
#define GROUP_FLOATS MOE_GROUP_FLOATS
// value e of an activation, written where its reader looks for it
template <int KIND>
static __device__ inline uint32_t act_at(uint32_t e) {
  if constexpr (KIND == PA_W_F32) return e;
  const uint32_t b = e / 32;
  return (b / 64) * GROUP_FLOATS + (((e % 32) / 4) * 64 + b % 64) * 4 + e % 4;
}
template <int KIND> static __device__ inline float stored(uint32_t e, float v) { return KIND == PA_W_Q4_0 && (e & 16) ? v * 0.0625f : v; }

// piece q of an activation and of a row (f32: the four from q on); past the end (q >= n) the last one again, which nothing uses
template <int KIND>
static __device__ inline void load_act(Act<KIND>& d, const float* act, uint32_t q, uint32_t n) {
  if constexpr (KIND == PA_W_F32) {
#pragma unroll
    for (int i = 0; i < 2; i++) d.x[i] = ((const f4*)act)[min(q + 64 * i, n - 1)];
    d.have = (q < n) + (q + 64 < n);
  } else {
    const uint32_t c = min(q, n - 1);
    const float* g = act + (c / 64) * GROUP_FLOATS;
#pragma unroll
    for (int i = 0; i < 8; i++) d.x[i] = ((const f4*)g)[i * 64 + c % 64];
  }
}
template <int KIND>
static __device__ inline void load_piece(Piece<KIND>& r, const unsigned char* plane, const uint16_t* scales, size_t row, uint32_t q, uint32_t n) {
  if constexpr (KIND == PA_W_F32) {
#pragma unroll
    for (int i = 0; i < 2; i++) r.w[i] = ((const f4*)plane)[row * n + min(q + 64 * i, n - 1)];
  } else {
    const size_t at = row * n + min(q, n - 1);
    if constexpr (KIND == PA_W_Q8_0) { const u4* s = (const u4*)(plane + at * 32); r.w[0] = s[0]; r.w[1] = s[1]; }
    else r.w[0] = *(const u4*)(plane + at * 16);
    r.sc = scales[at];
  }
}

// ---- 1: router logits and normed activations -----------------------------------------------------
template <int KIND>
__global__ __launch_bounds__(256)
void pa_moe_router_kernel(const float* a_x, const float* a_router, const float* a_norm, uint32_t dim, uint32_t x_stride, uint32_t rows, MoeParams p) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y, n4 = dim / 4;
  const uint32_t at = blockIdx.x * 4 + wave;                       // 0: xn, the longest way, first; otherwise logit at - 1
  const f4* x = (const f4*)(a_x + (size_t)t * x_stride);
  const f4* nw = (const f4*)a_norm;
  if (at > rows) return;
  const f4* r = (const f4*)(a_router + (size_t)(at ? at - 1 : 0) * dim);
  float ss = 0.f, a = 0.f, b = 0.f;
  for (uint32_t i0 = 0; i0 < n4; i0 += 512) {
    f4 xv[8], rv[8], wv[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t q = min(i0 + i * 64 + lane, n4 - 1);
      xv[i] = x[q]; rv[i] = r[q];
      wv[i] = nw ? nw[q] : f4{1.f, 1.f, 1.f, 1.f};
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
      if (i0 + i * 64 + lane < n4) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          ss = __builtin_fmaf(xv[i][j], xv[i][j], ss);
          float& s = j & 1 ? b : a;
          s = __builtin_fmaf(xv[i][j] * wv[i][j], rv[i][j], s);
        }
      }
    }
  }
  ss = wave_sum_f32(ss);
  const float mean = ss / (float)dim + p.eps;
  const float inv = nw ? 1.0f / sqrtf(mean) : 1.f;
  // a token whose squares leave f32's range (from 2^50 a value on; or tiny, without eps): sums and factor again, in 64 bits
  const bool far = nw && !(mean >= 0x1p-80f && mean < 0x1p100f);
  double far_inv = 1.0;
  if (at) a = wave_sum_f32(a + b) * inv;
  if (far) {
    double squares = 0.0, dot = 0.0;
    for (uint32_t q = lane; q < n4; q += 64) {
      const f4 xv = x[q], rv = r[q], wv = nw[q];
#pragma unroll
      for (int j = 0; j < 4; j++) { squares += (double)xv[j] * (double)xv[j]; dot += (double)xv[j] * (double)wv[j] * (double)rv[j]; }
    }
    far_inv = 1.0 / sqrt(wave_sum_f64(squares) / (double)dim + (double)p.eps);
    a = (float)(wave_sum_f64(dot) * far_inv);
  }
  if (at) {
    if (lane == 0) p.logits[(size_t)t * p.logit_stride + at - 1] = a;
    return;
  }
  float* xn = p.xn + (size_t)t * p.xn_floats;
  for (uint32_t q0 = 0; q0 < n4; q0 += 64) {
    const uint32_t q = q0 + lane;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    if (q < n4) {
      v = x[q];
      if (far) {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (float)((double)v[j] * far_inv) * nw[q][j];
      } else if (nw) {
        v = (v * inv) * nw[q];
      }
    }
    if (q < n4) {
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = stored<KIND>(4 * q, v[j]);
      *(f4*)(xn + act_at<KIND>(4 * q)) = v;
    }
  }
}

// ---- the choice ----------------------------------------------------------------------------------
// Logits as unsigned keys in their order: -0 is +0, a NaN is below -infinity, 0 is no candidate.  Expert lane + 64 i is key i of the lane.
template <int NE>
struct Choice {
  uint32_t key[NE];
  __device__ void load(const float* logits, uint32_t n, uint32_t lane) {
#pragma unroll
    for (int i = 0; i < NE; i++) {
      const uint32_t e = lane + 64 * i;
      const float l = logits[min(e, n - 1)] + 0.f;
      const uint32_t u = __float_as_uint(l);
      const uint32_t k = l != l ? 1u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
      key[i] = e < n ? k : 0u;
    }
  }
  static __device__ float logit(uint32_t k) { return k == 1u ? __uint_as_float(0x7FC00000u) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
  // the expert of the largest key m, the lowest among equals; taken out
  __device__ uint32_t next(uint32_t lane, uint32_t& m) {
    m = key[0];
    uint32_t i0 = 0;                                               // of the lane's largest key, the first
#pragma unroll
    for (int i = 1; i < NE; i++) { i0 = key[i] > m ? (uint32_t)i : i0; m = max(m, key[i]); }
    const uint32_t mine = m;
    m = wave_max_u32(m);
    const uint64_t who = __ballot(mine == m);
    uint32_t e = 64 * (uint32_t)__builtin_amdgcn_readlane((int)i0, __builtin_ctzll(who)) + (uint32_t)__builtin_ctzll(who);
    if (who & (who - 1)) {                                         // equal keys in several lanes
      bool found = false;
#pragma unroll
      for (int i = 0; i < NE; i++) {
        const uint64_t at = __ballot(key[i] == m);
        if (!found && at) { found = true; e = 64 * i + (uint32_t)__builtin_ctzll(at); }
      }
    }
#pragma unroll
    for (int i = 0; i < NE; i++) if (e == lane + 64 * i) key[i] = 0u;
    return e;
  }
};

// one wavefront: all of a token's experts and their weights
template <int NE>
static __device__ inline void write_choice(const MoeParams& p, const float* l, uint32_t n_experts, uint32_t top_k, uint32_t t, uint32_t lane) {
  Choice<NE> c;
  c.load(l, n_experts, lane);
  float v[NE];
#pragma unroll
  for (int i = 0; i < NE; i++) v[i] = Choice<NE>::logit(c.key[i]);
  uint32_t mine = 0, mine_key = 0, m;                              // lane r: the expert of place r
  for (uint32_t r = 0; r < top_k; r++) { const uint32_t e = c.next(lane, m); if (lane == r) { mine = e; mine_key = m; } }
  const float top = readlane_f32(Choice<NE>::logit(mine_key), 0);  // the largest logit (a NaN only where all are)
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < NE; i++) if (lane + 64 * i < n_experts) all += expf(v[i] - top);
  all = wave_sum_f32(all);
  const float w = lane < top_k ? expf(Choice<NE>::logit(mine_key) - top) : 0.f;
  float sum = all;
  if (p.norm_topk) { sum = wave_sum_f32(w); if (all != all) sum = all; }
  if (lane < top_k) {
    p.sel[(size_t)t * p.slots + lane] = mine;
    p.sel_w[(size_t)t * p.slots + lane] = w / sum;
    if (p.ids) p.ids[(size_t)t * top_k + lane] = mine;
    if (p.weights) p.weights[(size_t)t * top_k + lane] = w / sum;
  } else if (lane < p.slots) {
    p.sel[(size_t)t * p.slots + lane] = n_experts;
    p.sel_w[(size_t)t * p.slots + lane] = 1.0f / (1.0f + expf(-l[n_experts]));
  }
}

// the choice in a launch of its own, a wavefront a token
template <int NE>
__global__ __launch_bounds__(64)
void pa_moe_choice_kernel(const float* a_logits, uint32_t logit_stride, uint32_t n_experts, uint32_t top_k, MoeParams p) {
  write_choice<NE>(p, a_logits + (size_t)blockIdx.x * logit_stride, n_experts, top_k, blockIdx.x, threadIdx.x);
}

// ---- 2: gate and up ------------------------------------------------------------------------------
// A workgroup: 16 rows of h (half a block of the next kernel's input) of one expert, for up to GROUP tokens that chose it.  Pairs (token, place) are grouped in
// windows of whole tokens, at most MOE_WINDOW pairs: of those with the same expert, every GROUP-th leads, and its workgroups read the weights once for itself and those behind it.
#define MOE_WINDOW 256
template <int KIND, int NE, int RW, int GROUP, bool CHOSEN>
__global__ __launch_bounds__(1024 / RW)
void pa_moe_gate_up_kernel(const float* a_logits, const uint32_t* a_sel, const float* a_xn, uint32_t logit_stride, uint32_t xn_floats, uint32_t n_experts, uint32_t top_k, uint32_t slots,
                           uint32_t dim, MoeParams p) {
  constexpr uint32_t STEP = Piece<KIND>::STEP;
  __shared__ float hs[GROUP][16];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t np = pieces<KIND>(dim), first = blockIdx.x * 16, pair = blockIdx.y;
  uint32_t e = n_experts, count = 1, member[GROUP];
  member[0] = pair;
  Act<KIND> x[2];
  load_act<KIND>(x[0], a_xn + (size_t)(pair / slots) * xn_floats, lane, np);
  if constexpr (!CHOSEN) {
    const uint32_t place = pair % slots;
    if (place < top_k) {
      Choice<NE> c;
      c.load(a_logits + (size_t)(pair / slots) * logit_stride, n_experts, lane);
      uint32_t m;
      for (uint32_t r = 0; r <= place; r++) e = c.next(lane, m);
    }
  } else if constexpr (GROUP == 1) {
    e = a_sel[pair];
  } else {
    // the window's choices, 64 a register
    const uint32_t tokens = MOE_WINDOW / slots, w0 = pair / slots / tokens * tokens * slots, w1 = min(w0 + tokens * slots, p.n * slots), me = pair - w0;
    uint32_t all[MOE_WINDOW / 64], at = 0;
#pragma unroll
    for (int k = 0; k < MOE_WINDOW / 64; k++) all[k] = a_sel[min(w0 + 64 * k + lane, w1 - 1)];
#pragma unroll
    for (int k = 0; k < MOE_WINDOW / 64; k++) if (me / 64 == k) at = all[k];
    e = (uint32_t)__builtin_amdgcn_readlane((int)at, (int)(me & 63));
    uint64_t after[MOE_WINDOW / 64];
    uint32_t rank = 0;
#pragma unroll
    for (int k = 0; k < MOE_WINDOW / 64; k++) {
      const uint64_t same = __ballot(all[k] == e && w0 + 64 * k + lane < w1);
      const uint64_t upto = me >= 64u * k + 63 ? ~0ull : me < 64u * k ? 0ull : (2ull << (me & 63)) - 1;
      rank += (uint32_t)__popcll(same & upto);
      after[k] = same & ~upto;
    }
    if ((rank - 1) % GROUP) return;                                // rank counts the pair itself
#pragma unroll
    for (int j = 1; j < GROUP; j++) {
      member[j] = pair;
      bool found = false;
#pragma unroll
      for (int k = 0; k < MOE_WINDOW / 64; k++) {
        if (!found && after[k]) { member[j] = w0 + 64 * k + (uint32_t)__builtin_ctzll(after[k]); after[k] &= after[k] - 1; found = true; count = j + 1; }
      }
    }
  }
  e = (uint32_t)__builtin_amdgcn_readfirstlane((int)e);
  const size_t row = (size_t)e * p.ffn + first + wave * RW;
  float g[GROUP][RW], u[GROUP][RW];
#pragma unroll
  for (int j = 0; j < GROUP; j++) {
#pragma unroll
    for (int r = 0; r < RW; r++) g[j][r] = u[j][r] = 0.f;
  }
  for (uint32_t q0 = 0; q0 < np; q0 += STEP) {
    const uint32_t q = q0 + lane;
    Piece<KIND> wg[RW], wu[RW];
#pragma unroll
    for (int r = 0; r < RW; r++) {
      load_piece<KIND>(wg[r], p.gate, p.gate_s, row + r, q, np);
      load_piece<KIND>(wu[r], p.up, p.up_s, row + r, q, np);
    }
    if (q0) load_act<KIND>(x[0], a_xn + (size_t)(pair / slots) * xn_floats, q, np);
#pragma unroll
    for (int j = 0; j < GROUP; j++) {
      if (j < (int)count) {
        if (j + 1 < GROUP && j + 1 < (int)count) load_act<KIND>(x[(j + 1) & 1], a_xn + (size_t)(member[j + 1 < GROUP ? j + 1 : 0] / slots) * xn_floats, q, np);
        if (KIND == PA_W_F32 || q < np) {
#pragma unroll
          for (int r = 0; r < RW; r++) { g[j][r] = dot_piece<KIND>(wg[r], x[j & 1], 1.f, g[j][r]); u[j][r] = dot_piece<KIND>(wu[r], x[j & 1], 1.f, u[j][r]); }
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < GROUP; j++) {
    if (j < (int)count) {
#pragma unroll
      for (int r = 0; r < RW; r++) {
        const float a = wave_sum_f32(g[j][r]), b = wave_sum_f32(u[j][r]);
        if (lane == 0) hs[j][wave * RW + r] = a / (1.0f + expf(-a)) * b;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x < count * 16) {
    uint32_t m = member[0];
#pragma unroll
    for (int j = 1; j < GROUP; j++) if (threadIdx.x / 16 == j) m = member[j];
    float* h = p.h + (size_t)(m / slots) * p.h_floats;
    const uint32_t v = (m % slots) * p.ffn + first + threadIdx.x % 16;
    const float y = hs[threadIdx.x / 16][threadIdx.x % 16];
    h[act_at<KIND>(v)] = stored<KIND>(v, y);
  }
  if (!CHOSEN && blockIdx.x == 0 && pair % slots == 0 && wave == 0) write_choice<NE>(p, a_logits + (size_t)(pair / slots) * logit_stride, n_experts, top_k, pair / slots, lane);
}

// ---- 3: down, weighted sum, residual -------------------------------------------------------------
// RW rows of y a wavefront; the next pieces are requested while the present ones are used
template <int KIND, int RW, bool AHEAD>
__global__ __launch_bounds__(256)
void pa_moe_down_kernel(const uint32_t* a_sel, const float* a_sel_w, const float* a_h, uint32_t h_floats, uint32_t slots, uint32_t ffn, uint32_t dim, MoeParams p) {
  constexpr uint32_t STEP = Piece<KIND>::STEP;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y;
  const uint32_t np = pieces<KIND>(ffn), all = slots * np, row0 = (blockIdx.x * 4 + wave) * RW;
  const float* act = a_h + (size_t)t * h_floats;
  const uint32_t* sel = a_sel + (size_t)t * slots;
  const float* sel_w = a_sel_w + (size_t)t * slots;
  float a[RW];
#pragma unroll
  for (int r = 0; r < RW; r++) a[r] = 0.f;
  // a lane's place and piece in it, 64 further each time
  const uint32_t my_sel = sel[min(lane, slots - 1)], step_place = 64 / np, step_piece = 64 % np;
  const float my_w = sel_w[min(lane, slots - 1)];
  uint32_t place = lane / np, piece = lane % np;
  constexpr int LOADS = KIND == PA_W_F32 ? 2 : 1;
  struct Batch { Act<KIND> x; Piece<KIND> w[RW]; float f[LOADS]; };
  auto request = [&](Batch& d, uint32_t q0) __attribute__((always_inline)) {
    load_act<KIND>(d.x, act, q0 + lane, all);
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
      const bool in = q0 + 64 * i + lane < all;
      const uint32_t pl = in ? place : slots - 1, pc = in ? piece : np - 1;
      const size_t e = (uint32_t)__shfl((int)my_sel, (int)pl);
      d.f[i] = __shfl(my_w, (int)pl);
      place += step_place; piece += step_piece;
      if (piece >= np) { piece -= np; place++; }
#pragma unroll
      for (int r = 0; r < RW; r++) {
        const size_t row = e * dim + min(row0 + r, dim - 1);
        if constexpr (KIND == PA_W_F32) d.w[r].w[i] = ((const f4*)p.down)[row * np + pc];
        else load_piece<KIND>(d.w[r], p.down, p.down_s, row, pc, np);
      }
    }
  };
  auto use = [&](Batch& d, uint32_t q0) __attribute__((always_inline)) {
    if constexpr (KIND == PA_W_F32) {
      // a piece's float4 may belong to two experts: their weights go into the activations
#pragma unroll
      for (int i = 0; i < LOADS; i++) d.x.x[i] *= d.f[i];
#pragma unroll
      for (int r = 0; r < RW; r++) a[r] = dot_piece<KIND>(d.w[r], d.x, 1.f, a[r]);
    } else if (q0 + lane < all) {
#pragma unroll
      for (int r = 0; r < RW; r++) a[r] = dot_piece<KIND>(d.w[r], d.x, d.f[0], a[r]);
    }
  };
  if constexpr (AHEAD) {
    Batch b0, b1;
    request(b0, 0);
    for (uint32_t q0 = 0; q0 < all; q0 += 2 * STEP) {
      if (q0 + STEP < all) request(b1, q0 + STEP);
      use(b0, q0);
      if (q0 + STEP < all) {
        if (q0 + 2 * STEP < all) request(b0, q0 + 2 * STEP);
        use(b1, q0 + STEP);
      }
    }
  } else {
    for (uint32_t q0 = 0; q0 < all; q0 += STEP) { Batch b; request(b, q0); use(b, q0); }
  }
#pragma unroll
  for (int r = 0; r < RW; r++) {
    const float s = wave_sum_f32(a[r]);
    if (lane == 0 && row0 + r < dim) p.y[(size_t)t * p.y_stride + row0 + r] = p.x[(size_t)t * p.x_stride + row0 + r] + s;
  }
}

template <int KIND, int NE>
static void launch_experts(const MoeParams& p, hipStream_t s) {
  // Tokens that share an expert read its weights together where the bytes are what bounds: f32 (27 tokens, 61 experts, 5 chosen: 80 us without groups, 41 with).  Quantised
  // weights are bound by their instructions too, which a group does not save (16 tokens of Q4_0, 256 experts, 8 chosen: 32 us without, 42 with; 6: 15.5 and 19.3).
  constexpr int GROUP = KIND == PA_W_F32 ? 4 : 1;
  // Up to so many tokens every workgroup makes its choice itself; more have it made once, in a launch of its own.  Both in us, that launch included, for 4, 8 and 12 tokens (256 experts, 8
  // chosen; f32: 61 and 5): Q4_0 14.4 and 15.9, 24.5 and 22.9, 35.1 and 30.2; Q8_0 19.0 and 23.6, 34.4 and 37.2, 47.4 and 50.0; f32 14.3 and 17.9, 21.8 and 25.8, 30.0 and 32.4, and 56 and 46 for 27.
  constexpr uint32_t INLINE = KIND == PA_W_Q4_0 ? 4 : 12;
  const dim3 grid(p.ffn / 16, p.n * p.slots);
  if (p.n <= INLINE) {
    hipLaunchKernelGGL((pa_moe_gate_up_kernel<KIND, NE, 2, 1, false>), grid, dim3(512), 0, s, p.logits, p.sel, p.xn, p.logit_stride, p.xn_floats, p.n_experts, p.top_k, p.slots, p.dim, p);
  } else {
    hipLaunchKernelGGL(pa_moe_choice_kernel<NE>, dim3(p.n), dim3(64), 0, s, p.logits, p.logit_stride, p.n_experts, p.top_k, p);
    hipLaunchKernelGGL((pa_moe_gate_up_kernel<KIND, NE, 4, GROUP, true>), grid, dim3(256), 0, s, p.logits, p.sel, p.xn, p.logit_stride, p.xn_floats, p.n_experts, p.top_k, p.slots, p.dim, p);
  }
}
template <int KIND>
static hipError_t launch_kind(const MoeParams& p, int n_cu, hipStream_t s) {
  const uint32_t rows = p.n_experts + (p.slots > p.top_k ? 1 : 0);
  hipLaunchKernelGGL(pa_moe_router_kernel<KIND>, dim3((rows + 1 + 3) / 4, p.n), dim3(256), 0, s, p.x, p.router, p.norm_w, p.dim, p.x_stride, rows, p);
  if (p.n_experts <= 256) launch_experts<KIND, 4>(p, s); else launch_experts<KIND, 16>(p, s);
  // Rows a wavefront: quantised weights share the activations' loads over as many rows as still give every SIMD of the chip three wavefronts
  // (16 tokens of Q4_0, 2048 rows: 22.0 us with 8 rows, 26.9 with 4; 6 tokens: 12.5 and 11.6; 5 of Q8_0: 19.0 and 15.1; one token, with 2 and the next loads ahead, without them, with 1 and them: Q4_0 5.1, 5.1, 4.8,
  // Q8_0 5.3, 5.4, 5.0, f32 4.2, 5.0, 3.8, a launch's own spread being 0.5);
  // f32 pieces are short (27 tokens: 26.3 us with 2 rows, 28.8 with 4).
  auto down = [&](auto* kernel, uint32_t rw) { hipLaunchKernelGGL(kernel, dim3((p.dim + 4 * rw - 1) / (4 * rw), p.n), dim3(256), 0, s, p.sel, p.sel_w, p.h, p.h_floats, p.slots, p.ffn, p.dim, p); };
  if (p.n == 1) down(pa_moe_down_kernel<KIND, 2, true>, 2);
  else if constexpr (KIND == PA_W_F32) down(pa_moe_down_kernel<KIND, 2, false>, 2);
  else if ((uint64_t)p.n * (p.dim / 8) >= (uint64_t)n_cu * 12) down(pa_moe_down_kernel<KIND, 8, false>, 8);
  else down(pa_moe_down_kernel<KIND, 4, false>, 4);
  return hipGetLastError();
}

hipError_t pa_launch_moe(const MoeParams& p, int n_cu, hipStream_t s) {
  for (uint32_t t = 0; t < p.n; t += p.batch) {                    // at most 512 x 17 grid rows
    MoeParams q = p;
    q.n = std::min(p.n - t, p.batch);
    q.x += (size_t)t * p.x_stride; q.y += (size_t)t * p.y_stride;
    if (q.ids) q.ids += (size_t)t * p.top_k;
    if (q.weights) q.weights += (size_t)t * p.top_k;
    const hipError_t e = p.kind == PA_W_F32 ? launch_kind<PA_W_F32>(q, n_cu, s) : p.kind == PA_W_Q8_0 ? launch_kind<PA_W_Q8_0>(q, n_cu, s) : launch_kind<PA_W_Q4_0>(q, n_cu, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
