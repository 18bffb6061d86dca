// A mixture-of-experts layer over a few tokens on gfx950: rmsnorm, router, top-k, the chosen experts and the shared one, weighted sum, residual.
//
//   xn = rmsnorm(x) w;  l = router xn;  chosen = the top_k largest l;  h_e = silu(gate_e xn) * (up_e xn);  y = x + sum w_e down_e h_e
//
// With a few tokens the work is the stream of the chosen experts' weights: one token of 8 experts of 512 x 2048 and a shared one reads 16 MB of Q4_0
// planes and 2 MB of router and computes 58 MFLOP.  Three launches, because each needs all of the one before: logits, h, y.
//   1. router: a wavefront a row (expert) and token, over the raw x; the norm's factor is taken out of the sum, so sum of squares and dot run together.
//      Further wavefronts write xn, one a token.
//   2. gate and up: a workgroup a (token, place in the choice, slice of rows).  Which expert that is, every wavefront finds for itself from the token's
//      logits (a maximum over the 64 lanes per place), while xn is on its way.
//   3. down: the experts of a token lie behind one another as ONE input of slots x ffn values, so a wavefront's row is one dot product over it.
// A lane owns whole 32-value blocks of the input (one 16-byte load of Q4_0), for all rows of its wavefront; activations are kept in the order
// in which lanes load them, so that every load is 1 KB of consecutive bytes.  Arithmetic is f32, every sum in an order that depends on the layer's sizes alone:
// no atomics, and a token's bits do not depend on the other tokens of the call.
#include "blocks_internal.h"
#include "glue_math.h"

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
// F32: four values, Q8_0 and Q4_0: a block of 32 with its scale.  F4: float4 of activation that go with it.
template <int KIND> struct Piece { static constexpr int F4 = 8, VALUES = 32; u4 w[KIND == PA_W_Q8_0 ? 2 : 1]; uint16_t sc; };
template <> struct Piece<PA_W_F32> { static constexpr int F4 = 1, VALUES = 4; f4 w; };

template <int KIND>
static __device__ inline void load_piece(Piece<KIND>& r, const unsigned char* plane, const uint16_t* scales, size_t at) {
  if constexpr (KIND == PA_W_F32) {
    r.w = *(const f4*)(plane + at * 16);
  } else if constexpr (KIND == PA_W_Q8_0) {
    const u4* s = (const u4*)(plane + at * 32);
    r.w[0] = s[0]; r.w[1] = s[1]; r.sc = scales[at];
  } else {
    r.w[0] = *(const u4*)(plane + at * 16); r.sc = scales[at];
  }
}

static __device__ inline float f16_bits_f32(uint16_t b) { _Float16 h; __builtin_memcpy(&h, &b, 2); return (float)h; }

// acc + f * (piece . x)
template <int KIND>
static __device__ inline float dot_piece(const Piece<KIND>& r, const f4 (&x)[Piece<KIND>::F4], float f, float acc) {
  float a = 0.f;
  if constexpr (KIND == PA_W_F32) {
#pragma unroll
    for (int j = 0; j < 4; j++) a = __builtin_fmaf(r.w[j], x[0][j], a);
    return __builtin_fmaf(a, f, acc);
  } else if constexpr (KIND == PA_W_Q8_0) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int word = (int)r.w[i >> 2][i & 3];
#pragma unroll
      for (int j = 0; j < 4; j++) a = __builtin_fmaf((float)((word << (24 - 8 * j)) >> 24), x[i][j], a);
    }
    return __builtin_fmaf(a, f * f16_bits_f32(r.sc), acc);
  } else {
    // byte j of the block = elements j (low nibble) and j + 16 (high).  Two nibbles of a word under the f16 exponent of 1024 are 1024 + n, less 1032 exactly
    // n - 8; the mixed-precision fma takes the f16 as it is.
    const h2v off = {(_Float16)1032.f, (_Float16)1032.f};
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const uint32_t word = r.w[0][k];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        const uint32_t pr = ((word >> (4 * t)) & 0x000F000Fu) | 0x64006400u;      // nibbles t and t + 4 of the word
        h2v v; __builtin_memcpy(&v, &pr, 4);
        v = v - off;
        const int i = k + 4 * (t & 1), j = t >> 1;                                // element 4 i + j, and two on
        a = __builtin_fmaf((float)v[0], x[i][j], a);
        a = __builtin_fmaf((float)v[1], x[i][j + 2], a);
      }
    }
    return __builtin_fmaf(a, f * f16_bits_f32(r.sc), acc);
  }
}

// where value e of an activation lies in reading order
template <int KIND>
static __device__ inline uint32_t act_at(uint32_t e) {
  if constexpr (KIND == PA_W_F32) return e;
  const uint32_t b = e / 32;
  return ((((b / 64) * 8 + (e % 32) / 4) * 64) + b % 64) * 4 + e % 4;
}
// the float4 of activation of piece q (lane q % 64)
template <int KIND>
static __device__ inline void load_act(f4 (&x)[Piece<KIND>::F4], const float* act, uint32_t q) {
  if constexpr (KIND == PA_W_F32) {
    x[0] = ((const f4*)act)[q];
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = ((const f4*)act)[((q / 64) * 8 + i) * 64 + q % 64];
  }
}

// ---- 1: router logits and normed activations -----------------------------------------------------
template <int KIND>
__global__ __launch_bounds__(256)
void pa_moe_router_kernel(MoeParams p, uint32_t rows) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y, n4 = p.dim / 4;
  const uint32_t row = blockIdx.x * 4 + wave;
  const f4* x = (const f4*)(p.x + (size_t)t * p.x_stride);
  const f4* nw = (const f4*)p.norm_w;
  if (row > rows) return;
  const f4* r = (const f4*)(p.router + (size_t)min(row, rows - 1) * p.dim);
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
  const float inv = nw ? 1.0f / sqrtf(ss / (float)p.dim + p.eps) : 1.f;
  if (row < rows) {
    a = wave_sum_f32(a + b) * inv;
    if (lane == 0) p.logits[(size_t)t * p.logit_stride + row] = a;
    return;
  }
  float* xn = p.xn + (size_t)t * p.xn_floats;                     // row == rows: the token's normed activations
  for (uint32_t q = lane; q < n4; q += 64) {
    const f4 v = nw ? (x[q] * inv) * nw[q] : x[q];
    *(f4*)(xn + act_at<KIND>(4 * q)) = v;
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
  // the largest key, the lowest expert among equals; taken out
  __device__ uint32_t next(uint32_t lane) {
    uint32_t m = key[0];
#pragma unroll
    for (int i = 1; i < NE; i++) m = max(m, key[i]);
    m = wave_max_u32(m);
    uint32_t e = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < NE; i++) {
      const uint64_t who = __ballot(key[i] == m);
      if (!found && who) { found = true; e = 64 * i + (uint32_t)__builtin_ctzll(who); }
    }
#pragma unroll
    for (int i = 0; i < NE; i++) if (e == lane + 64 * i) key[i] = 0u;
    return e;
  }
};

// one wavefront: all of a token's experts and their weights
template <int NE>
static __device__ void write_choice(const MoeParams& p, uint32_t t, uint32_t lane) {
  const float* l = p.logits + (size_t)t * p.logit_stride;
  Choice<NE> c;
  c.load(l, p.n_experts, lane);
  uint32_t mine = 0;                                               // lane r: the expert of place r
  for (uint32_t r = 0; r < p.top_k; r++) { const uint32_t e = c.next(lane); if (lane == r) mine = e; }
  const float top = l[__builtin_amdgcn_readlane((int)mine, 0)];    // the largest logit (a NaN only where all are)
  float all = 0.f;
  for (uint32_t e = lane; e < p.n_experts; e += 64) all += expf(l[e] - top);
  all = wave_sum_f32(all);
  const float w = lane < p.top_k ? expf(l[mine] - top) : 0.f;
  float sum = all;
  if (p.norm_topk) { sum = wave_sum_f32(w); if (all != all) sum = all; }
  if (lane < p.top_k) {
    p.sel[(size_t)t * p.slots + lane] = mine;
    p.sel_w[(size_t)t * p.slots + lane] = w / sum;
    if (p.ids) p.ids[(size_t)t * p.top_k + lane] = mine;
    if (p.weights) p.weights[(size_t)t * p.top_k + lane] = w / sum;
  } else if (lane < p.slots) {
    p.sel[(size_t)t * p.slots + lane] = p.n_experts;
    p.sel_w[(size_t)t * p.slots + lane] = 1.0f / (1.0f + expf(-l[p.n_experts]));
  }
}

// ---- 2: gate and up ------------------------------------------------------------------------------
template <int KIND, int NE, int RW>
__global__ __launch_bounds__(256)
void pa_moe_gate_up_kernel(MoeParams p) {
  constexpr int F4 = Piece<KIND>::F4, V = Piece<KIND>::VALUES;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t t = blockIdx.y / p.slots, place = blockIdx.y % p.slots;
  const uint32_t np = p.dim / V, row0 = (blockIdx.x * 4 + wave) * RW;
  uint32_t e = p.n_experts;
  if (place < p.top_k) {
    Choice<NE> c;
    c.load(p.logits + (size_t)t * p.logit_stride, p.n_experts, lane);
    for (uint32_t r = 0; r <= place; r++) e = c.next(lane);
    e = (uint32_t)__builtin_amdgcn_readfirstlane((int)e);
  }
  const float* act = p.xn + (size_t)t * p.xn_floats;
  float g[RW], u[RW];
#pragma unroll
  for (int r = 0; r < RW; r++) g[r] = u[r] = 0.f;
  for (uint32_t q0 = 0; q0 < np; q0 += 64) {
    const uint32_t q = min(q0 + lane, np - 1);                     // pieces past the end repeat the last one, times zero
    const float f = q0 + lane < np ? 1.f : 0.f;
    f4 x[F4];
    load_act<KIND>(x, act, q);
    Piece<KIND> wg[RW], wu[RW];
#pragma unroll
    for (int r = 0; r < RW; r++) {
      const size_t at = ((size_t)e * p.ffn + min(row0 + r, p.ffn - 1)) * np + q;
      load_piece<KIND>(wg[r], p.gate, p.gate_s, at);
      load_piece<KIND>(wu[r], p.up, p.up_s, at);
    }
    if (f != 0.f) {
#pragma unroll
      for (int r = 0; r < RW; r++) { g[r] = dot_piece<KIND>(wg[r], x, 1.f, g[r]); u[r] = dot_piece<KIND>(wu[r], x, 1.f, u[r]); }
    }
  }
  float* h = p.h + (size_t)t * p.h_floats;
#pragma unroll
  for (int r = 0; r < RW; r++) {
    const float a = wave_sum_f32(g[r]), b = wave_sum_f32(u[r]);
    if (lane == 0 && row0 + r < p.ffn) h[act_at<KIND>(place * p.ffn + row0 + r)] = a / (1.0f + expf(-a)) * b;
  }
  if (blockIdx.x == 0 && place == 0 && wave == 0) write_choice<NE>(p, t, lane);
}

// ---- 3: down, weighted sum, residual -------------------------------------------------------------
template <int KIND, int RW>
__global__ __launch_bounds__(256)
void pa_moe_down_kernel(MoeParams p) {
  constexpr int F4 = Piece<KIND>::F4, V = Piece<KIND>::VALUES;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.y;
  const uint32_t np = p.ffn / V, all = p.slots * np, row0 = (blockIdx.x * 4 + wave) * RW;
  const float* act = p.h + (size_t)t * p.h_floats;
  const uint32_t* sel = p.sel + (size_t)t * p.slots;
  const float* sel_w = p.sel_w + (size_t)t * p.slots;
  float a[RW];
#pragma unroll
  for (int r = 0; r < RW; r++) a[r] = 0.f;
  for (uint32_t q0 = 0; q0 < all; q0 += 64) {
    const uint32_t q = q0 + lane;
    if (q < all) {
      const uint32_t place = q / np, e = sel[place];
      const float f = sel_w[place];
      f4 x[F4];
      load_act<KIND>(x, act, q);
      Piece<KIND> w[RW];
#pragma unroll
      for (int r = 0; r < RW; r++) load_piece<KIND>(w[r], p.down, p.down_s, ((size_t)e * p.dim + min(row0 + r, p.dim - 1)) * np + q % np);
#pragma unroll
      for (int r = 0; r < RW; r++) a[r] = dot_piece<KIND>(w[r], x, f, a[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < RW; r++) {
    const float s = wave_sum_f32(a[r]);
    if (lane == 0 && row0 + r < p.dim) p.y[(size_t)t * p.y_stride + row0 + r] = p.x[(size_t)t * p.x_stride + row0 + r] + s;
  }
}

template <int KIND>
static hipError_t launch_kind(const MoeParams& p, hipStream_t s) {
  const uint32_t rows = p.n_experts + (p.slots > p.top_k ? 1 : 0);
  hipLaunchKernelGGL(pa_moe_router_kernel<KIND>, dim3((rows + 1 + 3) / 4, p.n), dim3(256), 0, s, p, rows);
  constexpr uint32_t RW = 4;
  const dim3 gu((p.ffn + 4 * RW - 1) / (4 * RW), p.n * p.slots);
  if (p.n_experts <= 256) hipLaunchKernelGGL((pa_moe_gate_up_kernel<KIND, 4, RW>), gu, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((pa_moe_gate_up_kernel<KIND, 16, RW>), gu, dim3(256), 0, s, p);
  hipLaunchKernelGGL((pa_moe_down_kernel<KIND, RW>), dim3((p.dim + 4 * RW - 1) / (4 * RW), p.n), dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t pa_launch_moe(const MoeParams& p, int n_cu, hipStream_t s) {
  (void)n_cu;
  // grid rows are tokens x places: at most 65535 of them a launch
  const uint32_t most = 65535u / p.slots;
  for (uint32_t t = 0; t < p.n; t += most) {
    MoeParams q = p;
    q.n = p.n - t < most ? p.n - t : most;
    q.x += (size_t)t * p.x_stride; q.y += (size_t)t * p.y_stride;
    if (q.ids) q.ids += (size_t)t * p.top_k;
    if (q.weights) q.weights += (size_t)t * p.top_k;
    q.xn += (size_t)t * p.xn_floats; q.h += (size_t)t * p.h_floats; q.logits += (size_t)t * p.logit_stride;
    q.sel += (size_t)t * p.slots; q.sel_w += (size_t)t * p.slots;
    const hipError_t e = p.kind == PA_W_F32 ? launch_kind<PA_W_F32>(q, s) : p.kind == PA_W_Q8_0 ? launch_kind<PA_W_Q8_0>(q, s) : launch_kind<PA_W_Q4_0>(q, s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
