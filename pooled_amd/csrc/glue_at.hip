// Pre-step of columns that have positions of their own, on one axis or on several, for gfx950.
//
// Pair i of a head's rotated dims, (x[i], x[i + n_rot / 2]), turns by the angle of the position that the column has on the pair's axis; norm, gate and cache rows as in
// glue_kv.hip, whose arithmetic (glue_math.h) this shares: where every axis holds base + c, the results have the bits of that kernel at base + c.
//
// A wavefront takes 512 values of query heads of one column (two heads of 256, four of 128), or as many of key heads with their value heads; every load of a wave goes out ahead of what
// depends on one, the positions first.  Rows of a cache are packed through LDS, eight values a lane.
// Bound: wide chunks by HBM: 5003 columns of 24 query and 4 key heads of 256 with gates (553 MB) take 100 us = 5.5 TB/s; with one head a wavefront 124.  1001 columns of 16 and 8 heads
// of 128 (29 MB) 8.6 us, with one key head a wavefront 10.8.  A draft's columns by the chain position -> (cos, sin) -> rotation: 24 columns 2.6 us.  Int8 rows, packed one by one:
// 1001 columns of 16 and 8 heads of 128 13.1 us a call, f16 9.3; 24 of 16 and 2 heads of 256 4.3 and 4.0.
#include "tree_internal.h"
#include "glue_math.h"

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

// a row of hd f32 values in LDS -> int8 with one scale per 32 values
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
  constexpr int N = 512 / HD, J = HD / 64;          // heads of a wave; values of a lane and head
  __shared__ __attribute__((aligned(16))) float xs_all[4][2 * N * HD];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), task = blockIdx.x * 4 + wave;
  const uint32_t nH = p.n_heads, qd = nH * HD, half = p.n_rot / 2, q_tasks = (nH + N - 1) / N, per_col = q_tasks + (p.n_kv_heads + N - 1) / N;
  const uint32_t col = div_by(task, per_col, p.per_col_magic), u = task - col * per_col;
  if (col >= p.n_cols) return;
  const bool is_q = u < q_tasks, gated = (p.flags & PA_FLAG_GATE) != 0, norm = (p.flags & PA_FLAG_QK_NORM) != 0;
  const uint32_t h0 = (is_q ? u : u - q_tasks) * N, heads = min((uint32_t)N, (is_q ? nH : p.n_kv_heads) - h0);
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
  // (second: the gates of query heads, the values of key heads)
  const float* second = is_q ? src + HD : p.v_in + (size_t)col * p.v_stride + (size_t)h0 * HD;
  float x[N][4], y[N][J], w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int n = 0; n < N; n++) {
    const size_t at = (size_t)min((uint32_t)n, heads - 1) * step + lane;     // (a wave's heads past the last: that one again, not stored)
#pragma unroll
    for (int j = 0; j < 4; j++) x[n][j] = j < J ? __builtin_nontemporal_load(src + at + 64 * j) : 0.f;
    if (!is_q || gated)
#pragma unroll
      for (int j = 0; j < J; j++) y[n][j] = __builtin_nontemporal_load(second + at + 64 * j);
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
  if (is_q && gated) {
    const size_t at = (size_t)col * qd + h0 * HD + lane;
#pragma unroll
    for (int n = 0; n < N; n++)
      if ((uint32_t)n < heads)
#pragma unroll
        for (int j = 0; j < J; j++) p.gate_out[at + n * HD + 64 * j] = y[n][j];
  }
  if constexpr (REGS) glue_heads_regs<N>(x, w, norm, p.eps, HD, half, cs, lane);
  else {
    glue_heads_wave<N>(x, w, norm, p.eps, HD, half, cs, xs, HD, lane);
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
      for (int j = 0; j < J; j++) x[n][j] = xs[n * HD + lane + 64 * j];
    wave_lds_fence();
  }
  if (is_q) {
    const size_t at = (size_t)col * qd + h0 * HD + lane;
#pragma unroll
    for (int n = 0; n < N; n++)
      if ((uint32_t)n < heads)
#pragma unroll
        for (int j = 0; j < J; j++) p.q_out[at + n * HD + 64 * j] = x[n][j];
    return;
  }
  // keys and values through LDS: eight values of a row a lane
#pragma unroll
  for (int n = 0; n < N; n++)
#pragma unroll
    for (int j = 0; j < J; j++) { xs[n * HD + lane + 64 * j] = x[n][j]; xs[(N + n) * HD + lane + 64 * j] = y[n][j]; }
  wave_lds_fence();
  const size_t plane = p.head_rows, row0 = (size_t)h0 * plane + p.base_row + col;
  if (p.ks_cache) {
    for (uint32_t n = 0; n < heads; n++) {
      const size_t row = row0 + n * plane;
      store_row_q8(xs + n * HD, HD, lane, (unsigned char*)p.k_cache + row * HD, p.ks_cache + row * (HD / 32));
      store_row_q8(xs + (N + n) * HD, HD, lane, (unsigned char*)p.v_cache + row * HD, p.vs_cache + row * (HD / 32));
    }
  } else {
    const uint32_t n = lane / (HD / 8), d = lane % (HD / 8) * 8;
    if (n < heads) {
      auto pack = [&](const float* s) -> h8 {
        const f4 a = *(const f4*)s, b = *(const f4*)(s + 4);
        return (h8){ (_Float16)a[0], (_Float16)a[1], (_Float16)a[2], (_Float16)a[3], (_Float16)b[0], (_Float16)b[1], (_Float16)b[2], (_Float16)b[3] };
      };
      const size_t at = (row0 + n * plane) * HD + d;
      *(h8*)((_Float16*)p.k_cache + at) = pack(xs + n * HD + d);
      *(h8*)((_Float16*)p.v_cache + at) = pack(xs + (N + n) * HD + d);
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
  const uint64_t per_col = (uint64_t)(p.n_heads + n - 1) / n + (p.n_kv_heads + n - 1) / n, tasks = per_col * p.n_cols;
  if (!tasks || tasks > 0x7fffff00ull) return hipErrorInvalidValue;
  p.per_col_magic = div_magic(tasks + 4, (uint32_t)per_col);
  if (p.head_dim == 256) return launch_glue_at<256>(p, (uint32_t)((tasks + 3) / 4), s);
  if (p.head_dim == 128) return launch_glue_at<128>(p, (uint32_t)((tasks + 3) / 4), s);
  return hipErrorInvalidValue;
}
