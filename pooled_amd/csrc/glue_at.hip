// Pre-step of columns that have positions of their own, on one axis or on several, for gfx950.
//
// Pair i of a head's rotated dims, (x[i], x[i + n_rot / 2]), turns by the angle of the position that the column has on the pair's axis; norm, gate and cache rows as in
// glue_kv.hip, whose arithmetic (glue_math.h) this shares: where every axis holds base + c, the results have the bits of that kernel at base + c.
//
// One wavefront per (head, column), key heads with their value head.
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

__global__ __launch_bounds__(64) void pa_glue_at_kernel(GlueAtParams p) {
  __shared__ float xs[256];
  const uint32_t hh = blockIdx.x, col = blockIdx.y, lane = threadIdx.x;
  const uint32_t nH = p.n_heads, hd = p.head_dim, qd = nH * hd, half = p.n_rot / 2;
  const bool is_q = hh < nH, gated = (p.flags & PA_FLAG_GATE) != 0, norm = (p.flags & PA_FLAG_QK_NORM) != 0;
  const uint32_t h = is_q ? hh : hh - nH;
  const float* src = is_q ? p.q_in + (size_t)col * p.q_stride + (size_t)h * (gated ? 2 * hd : hd) : p.k_in + (size_t)col * p.k_stride + (size_t)h * hd;
  float x[4], w[4] = {0.f, 0.f, 0.f, 0.f};
  float2 cs[2];
#pragma unroll
  for (int j = 0; j < 4; j++) x[j] = lane + 64 * j < hd ? src[lane + 64 * j] : 0.f;
  if (norm) {
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = lane + 64 * j < hd ? (is_q ? p.qw : p.kw)[lane + 64 * j] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < 2; j++) {
    const uint32_t i = min(lane + 64 * j, half - 1), axis = p.axis_of_pair[i / 16] >> (i % 16 * 2) & 3;
    const uint32_t pos = p.pos[(size_t)axis * p.pos_stride + col];
    if (pos < p.tab_rows) cs[j] = p.rope_tab[(size_t)pos * half + i];
    else rope_cos_sin(pos, p.inv_freq[i], cs[j].x, cs[j].y);
  }
  if (is_q && gated)
    for (uint32_t i = lane; i < hd; i += 64) p.gate_out[(size_t)col * qd + h * hd + i] = src[hd + i];
  glue_head_wave(x, w, norm, p.eps, hd, half, cs, xs, lane);
  if (is_q) {
    for (uint32_t i = lane; i < hd; i += 64) p.q_out[(size_t)col * qd + h * hd + i] = xs[i];
    return;
  }
  const float* v = p.v_in + (size_t)col * p.v_stride + (size_t)h * hd;
  const size_t row = (size_t)h * p.head_rows + p.base_row + col;
  if (p.ks_cache) {
    store_row_q8(xs, hd, lane, (unsigned char*)p.k_cache + row * hd, p.ks_cache + row * (hd / 32));
    store_row_q8(v, hd, lane, (unsigned char*)p.v_cache + row * hd, p.vs_cache + row * (hd / 32));
  } else {
    for (uint32_t i = lane; i < hd / 2; i += 64) {
      ((uint32_t*)((uint16_t*)p.k_cache + row * hd))[i] = pack_f16x2(xs[2 * i], xs[2 * i + 1]);
      ((uint32_t*)((uint16_t*)p.v_cache + row * hd))[i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
    }
  }
}

hipError_t pa_launch_glue_at(const GlueAtParams& p, hipStream_t s) {
  if (!p.n_cols || p.n_cols > 65535u) return hipErrorInvalidValue;
  hipLaunchKernelGGL(pa_glue_at_kernel, dim3(p.n_heads + p.n_kv_heads, p.n_cols), dim3(64), 0, s, p);
  return hipGetLastError();
}
