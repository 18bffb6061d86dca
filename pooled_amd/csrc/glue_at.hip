// Pre-step of columns that have positions of their own, on one axis or on several, for gfx950.
//
// Pair i of a head's rotated dims, (x[i], x[i + n_rot / 2]), turns by the angle of the position that the column has on the pair's axis; norm, gate and cache rows as in
// glue_kv.hip, whose arithmetic (glue_math.h) this shares: where every axis holds base + c, the results have the bits of that kernel at base + c.
//
// A wavefront takes 512 values of query heads of one column (two heads of 256, four of 128), or one key head with its value head; every load of a wave goes out ahead of what depends on
// one.  Wide chunks are bound by HBM, which the loads of several heads a wave keep busy where one head a wave does not; a draft's columns by the chain position -> (cos, sin) -> rotation.
#include "tree_internal.h"
#include "glue_math.h"

static __device__ inline uint32_t pack_f16x2(float lo, float hi) {
  return (uint32_t)__half_as_ushort(__float2half_rn(lo)) | ((uint32_t)__half_as_ushort(__float2half_rn(hi)) << 16);
}

// a row of hd f32 values in LDS or global memory -> int8 with one scale per 32 values
static __device__ inline void store_row_q8(const float* src, uint32_t hd, uint32_t lane, unsigned char* dst, float* sc_dst) {
  const bool on = 4 * lane < hd;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (on) { x[0] = src[4 * lane]; x[1] = src[4 * lane + 1]; x[2] = src[4 * lane + 2]; x[3] = src[4 * lane + 3]; }
  uint32_t w; float sc;
  quant4_q8(x, w, sc);
  if (on) {
    *(uint32_t*)(dst + 4 * lane) = w;
    if ((lane & 7) == 0) sc_dst[lane >> 3] = sc;
  }
}

// REGS: the pair distance is one that glue_heads_regs serves
template <int HD, bool REGS>
__global__ __launch_bounds__(256) void pa_glue_at_kernel(GlueAtParams p) {
  constexpr int N = 512 / HD, J = HD / 64;          // query heads of a wave; values of a lane and head
  __shared__ float xs_all[4][N * HD];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), task = blockIdx.x * 4 + wave;
  const uint32_t nH = p.n_heads, qd = nH * HD, half = p.n_rot / 2, q_tasks = (nH + N - 1) / N, per_col = q_tasks + p.n_kv_heads;
  const uint32_t col = div_by(task, per_col, p.per_col_magic), u = task - col * per_col;
  if (col >= p.n_cols) return;
  const bool is_q = u < q_tasks, gated = (p.flags & PA_FLAG_GATE) != 0, norm = (p.flags & PA_FLAG_QK_NORM) != 0;
  const uint32_t h0 = is_q ? u * N : u - q_tasks, heads = is_q ? min((uint32_t)N, nH - h0) : 1;
  float* xs = xs_all[wave];
  // the positions first: two loads hang on them
  uint32_t pair[2], pos[2];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    pair[j] = REGS && half == 32 ? lane & 31 : min(lane + 64 * j, half - 1);
    const uint32_t axis = p.n_axes == 1 ? 0u : p.axis_of_pair[pair[j] / 16] >> (pair[j] % 16 * 2) & 3;
    pos[j] = p.pos[(size_t)axis * p.pos_stride + col];
  }
  const float* src = is_q ? p.q_in + (size_t)col * p.q_stride + (size_t)h0 * (gated ? 2 * HD : HD) : p.k_in + (size_t)col * p.k_stride + (size_t)h0 * HD;
  const uint32_t step = is_q && gated ? 2 * HD : HD;
  float x[N][4], gt[N][J], w[4] = {0.f, 0.f, 0.f, 0.f};
  if (is_q) {
#pragma unroll
    for (int n = 0; n < N; n++) {
      const float* s = src + (size_t)min((uint32_t)n, heads - 1) * step;     // (a wave's heads past the last: that one again, not stored)
#pragma unroll
      for (int j = 0; j < 4; j++) x[n][j] = j < J ? __builtin_nontemporal_load(s + lane + 64 * j) : 0.f;
      if (gated)
#pragma unroll
        for (int j = 0; j < J; j++) gt[n][j] = __builtin_nontemporal_load(s + HD + lane + 64 * j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) x[0][j] = j < J ? src[lane + 64 * j] : 0.f;
  }
  float v[J];
  if (!is_q) {
#pragma unroll
    for (int j = 0; j < J; j++) v[j] = p.v_in[(size_t)col * p.v_stride + (size_t)h0 * HD + lane + 64 * j];
  }
  if (norm) {
#pragma unroll
    for (int j = 0; j < J; j++) w[j] = (is_q ? p.qw : p.kw)[lane + 64 * j];
  }
  float2 cs[2];
#pragma unroll
  for (int j = 0; j < 2; j++) {
    if (j && half <= 64) { cs[j] = cs[0]; continue; }                        // (not looked at)
    if (pos[j] < p.tab_rows) cs[j] = p.rope_tab[(size_t)pos[j] * half + pair[j]];
    else rope_cos_sin(pos[j], p.inv_freq[pair[j]], cs[j].x, cs[j].y);
  }
  if (is_q) {
    const size_t at = (size_t)col * qd + h0 * HD + lane;
    if (gated) {
#pragma unroll
      for (int n = 0; n < N; n++)
        if ((uint32_t)n < heads)
#pragma unroll
          for (int j = 0; j < J; j++) p.gate_out[at + n * HD + 64 * j] = gt[n][j];
    }
    if constexpr (REGS) glue_heads_regs<N>(x, w, norm, p.eps, HD, half, cs, lane);
    else {
      glue_heads_wave<N>(x, w, norm, p.eps, HD, half, cs, xs, HD, lane);
#pragma unroll
      for (int n = 0; n < N; n++)
#pragma unroll
        for (int j = 0; j < J; j++) x[n][j] = xs[n * HD + lane + 64 * j];
    }
#pragma unroll
    for (int n = 0; n < N; n++)
      if ((uint32_t)n < heads)
#pragma unroll
        for (int j = 0; j < J; j++) p.q_out[at + n * HD + 64 * j] = x[n][j];
    return;
  }
  float x1[1][4] = { { x[0][0], x[0][1], x[0][2], x[0][3] } };
  if constexpr (REGS) {
    glue_heads_regs<1>(x1, w, norm, p.eps, HD, half, cs, lane);
#pragma unroll
    for (int j = 0; j < J; j++) xs[lane + 64 * j] = x1[0][j];
  } else glue_heads_wave<1>(x1, w, norm, p.eps, HD, half, cs, xs, HD, lane);
#pragma unroll
  for (int j = 0; j < J; j++) xs[HD + lane + 64 * j] = v[j];                 // the value row beside the key row
  wave_lds_fence();
  const size_t row = (size_t)h0 * p.head_rows + p.base_row + col;
  if (p.ks_cache) {
    store_row_q8(xs, HD, lane, (unsigned char*)p.k_cache + row * HD, p.ks_cache + row * (HD / 32));
    store_row_q8(xs + HD, HD, lane, (unsigned char*)p.v_cache + row * HD, p.vs_cache + row * (HD / 32));
  } else {
#pragma unroll
    for (int t = 0; t < HD / 128; t++) {
      const uint32_t i = lane + 64 * t;
      ((uint32_t*)((uint16_t*)p.k_cache + row * HD))[i] = pack_f16x2(xs[2 * i], xs[2 * i + 1]);
      ((uint32_t*)((uint16_t*)p.v_cache + row * HD))[i] = pack_f16x2(xs[HD + 2 * i], xs[HD + 2 * i + 1]);
    }
  }
}

template <int HD> static hipError_t launch_glue_at(const GlueAtParams& p, uint32_t wgs, hipStream_t s) {
  if (glue_regs_serves(p.n_rot / 2)) hipLaunchKernelGGL((pa_glue_at_kernel<HD, true>), dim3(wgs), dim3(256), 0, s, p);
  else hipLaunchKernelGGL((pa_glue_at_kernel<HD, false>), dim3(wgs), dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t pa_launch_glue_at(const GlueAtParams& p_in, hipStream_t s) {
  GlueAtParams p = p_in;
  const uint32_t n = p.head_dim ? 512 / p.head_dim : 1;
  const uint64_t per_col = (uint64_t)(p.n_heads + n - 1) / n + p.n_kv_heads, tasks = per_col * p.n_cols;
  if (!tasks || tasks > 0x7fffff00ull) return hipErrorInvalidValue;
  p.per_col_magic = div_magic(tasks + 4, (uint32_t)per_col);
  if (p.head_dim == 256) return launch_glue_at<256>(p, (uint32_t)((tasks + 3) / 4), s);
  if (p.head_dim == 128) return launch_glue_at<128>(p, (uint32_t)((tasks + 3) / 4), s);
  return hipErrorInvalidValue;
}
