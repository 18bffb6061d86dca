// The gated delta rule token by token, and its pre-step (short causal convolution and gates), on gfx950.
//
// A linear-attention layer of the hybrid models keeps, per v head, a matrix S [head_v][head_k] instead of cache rows.  Token t:
//   S' = exp(g_t) S_{t-1};  u_t = beta_t (v_t - S' k_t);  S_t = S' + u_t k_t^T;  o_t = scale S_t q_t
// Row r of S is a recurrence of its own: u_t[r] and o_t[r] need row r, k_t and q_t alone.  Sixteen lanes hold one row (head_k / 16 values each, in
// registers over all columns of the call), a wavefront four rows, a workgroup sixteen; the two dot products of a token are sums over sixteen lanes,
// four DPP steps each, and nothing is exchanged between wavefronts.  With 32 v heads of 128 x 128 that is 1024 wavefronts, one per SIMD.
//
// One token moves 2 x 4 bytes per state value and computes 6 operations on it: it is bound by the state's stream and, at these sizes (2 MB), by the
// latency of a launch.  A run of columns is bound by the chain dot -> u -> update of each token; the next columns' q, k, v and gates are
// requested four columns ahead, so the chain alone counts.  Everything is f32.  A column's arithmetic does not depend on how many columns a
// call has: a verify block gives every column the bits of the one-token call at its place.
#include "blocks_internal.h"
#include "glue_math.h"

typedef float f4 __attribute__((ext_vector_type(4)));

// sum over the sixteen lanes of a DPP row, the same bits in all of them
static __device__ inline float row16_sum(float v) {
  v += dpp_f32<0xB1>(v);
  v += dpp_f32<0x4E>(v);
  v += dpp_f32<0x141>(v);
  return v + dpp_f32<0x140>(v);
}

// V4: float4 of a row per lane (head_k = 64 V4)
template <int V4>
__global__ __launch_bounds__(256)
void pa_delta_step_kernel(DeltaParams p) {
  constexpr int AHEAD = 4;
  constexpr uint32_t HK = 64 * V4;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15;
  const uint32_t tiles = p.hv / 16;
  const uint32_t h = blockIdx.x / tiles, row = (blockIdx.x % tiles) * 16 + wave * 4 + (lane >> 4), kh = h / p.group;
  float* const srow = p.state + ((size_t)h * p.hv + row) * HK + 4 * j;
  f4 S[V4];
#pragma unroll
  for (int i = 0; i < V4; i++) S[i] = *(const f4*)(srow + 64 * i);
  const float* const kp = p.k + (size_t)kh * HK + 4 * j;
  const float* const qp = p.q + (size_t)kh * HK + 4 * j;
  const float* const vp = p.v + (size_t)h * p.hv + row;
  const bool out = p.out != nullptr;

  f4 kr[AHEAD][V4], qr[AHEAD][V4];
  float vr[AHEAD], gr[AHEAD], br[AHEAD];
  auto request = [&](int s, uint32_t t) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < V4; i++) kr[s][i] = *(const f4*)(kp + (size_t)t * p.k_stride + 64 * i);
    vr[s] = vp[(size_t)t * p.v_stride];
    gr[s] = p.g[(size_t)t * p.gate_stride + h];
    br[s] = p.beta[(size_t)t * p.gate_stride + h];
    if (out) {
#pragma unroll
      for (int i = 0; i < V4; i++) qr[s][i] = *(const f4*)(qp + (size_t)t * p.q_stride + 64 * i);
    }
  };
#pragma unroll
  for (int s = 0; s < AHEAD; s++) if ((uint32_t)s < p.n) request(s, s);

  for (uint32_t t0 = 0; t0 < p.n; t0 += AHEAD) {
#pragma unroll
    for (int s = 0; s < AHEAD; s++) {
      const uint32_t t = t0 + s;
      if (t < p.n) {
        float kk = 0.f, qq = 0.f, inv_k = 1.f, scale_q = p.scale;
        if (p.l2norm) {                                             // off the chain: needs k_t and q_t alone
#pragma unroll
          for (int i = 0; i < V4; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) kk = __builtin_fmaf(kr[s][i][e], kr[s][i][e], kk);
          inv_k = 1.0f / sqrtf(row16_sum(kk) + p.eps);
        }
        const float decay = expf(gr[s]);
        f4 k[V4];
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int i = 0; i < V4; i++) {
          k[i] = kr[s][i] * inv_k;
          S[i] = S[i] * decay;
          a = __builtin_fmaf(S[i][0], k[i][0], a); b = __builtin_fmaf(S[i][1], k[i][1], b);
          a = __builtin_fmaf(S[i][2], k[i][2], a); b = __builtin_fmaf(S[i][3], k[i][3], b);
        }
        const float u = br[s] * (vr[s] - row16_sum(a + b));
#pragma unroll
        for (int i = 0; i < V4; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) S[i][e] = __builtin_fmaf(u, k[i][e], S[i][e]);
        if (out) {
          if (p.l2norm) {
#pragma unroll
            for (int i = 0; i < V4; i++)
#pragma unroll
              for (int e = 0; e < 4; e++) qq = __builtin_fmaf(qr[s][i][e], qr[s][i][e], qq);
            scale_q = p.scale / sqrtf(row16_sum(qq) + p.eps);
          }
          float c = 0.f, d = 0.f;
#pragma unroll
          for (int i = 0; i < V4; i++) {
            c = __builtin_fmaf(S[i][0], qr[s][i][0], c); d = __builtin_fmaf(S[i][1], qr[s][i][1], d);
            c = __builtin_fmaf(S[i][2], qr[s][i][2], c); d = __builtin_fmaf(S[i][3], qr[s][i][3], d);
          }
          const float o = row16_sum(c + d) * scale_q;
          if (j == 0) {
            const size_t at = (size_t)t * p.out_stride + (size_t)h * p.hv + row;
            if (p.out_f16) ((_Float16*)p.out)[at] = (_Float16)o; else ((float*)p.out)[at] = o;
          }
        }
        if (t + 1 == p.commit) {
#pragma unroll
          for (int i = 0; i < V4; i++) *(f4*)(srow + 64 * i) = S[i];
        }
        if (t + AHEAD < p.n) request(s, t + AHEAD);
      }
    }
  }
}

hipError_t pa_launch_delta_step(const DeltaParams& p, hipStream_t s) {
  const dim3 grid(p.nv * (p.hv / 16)), block(256);
  if (p.hk == 64) hipLaunchKernelGGL(pa_delta_step_kernel<1>, grid, block, 0, s, p);
  else hipLaunchKernelGGL(pa_delta_step_kernel<2>, grid, block, 0, s, p);
  return hipGetLastError();
}

// ---- pre-step ------------------------------------------------------------------------------------
// y[c][ch] = silu(bias[ch] + sum_j w[ch][j] line[c + j][ch]), line = the state's W - 1 inputs, then x;  g = -exp(a_log) softplus(a + dt_bias);
// beta = sigmoid(b).  A stream: every input is read once (the W - 1 rows in front of a run of columns twice) and every output written once.  A lane
// owns four channels and walks GLUE_COLS columns with the last W inputs in registers; the workgroups of the last grid column compute the gates.
#define GLUE_COLS 16u

template <int W>
__global__ __launch_bounds__(64)
void pa_delta_glue_kernel(DeltaGlueParams p) {
  const uint32_t c0 = blockIdx.y * GLUE_COLS, c1 = min(c0 + GLUE_COLS, p.n);
  if (blockIdx.x == gridDim.x - 1) {
    const uint32_t n = (c1 - c0) * p.nv;
    for (uint32_t i = threadIdx.x; i < n; i += 64) {
      const uint32_t c = c0 + i / p.nv, h = i % p.nv;
      const float z = p.a[(size_t)c * p.ab_stride + h] + p.dt_bias[h];
      const float soft = fmaxf(z, 0.f) + log1pf(expf(-fabsf(z)));
      p.g[(size_t)c * p.gate_stride + h] = -expf(p.a_log[h]) * (z != z ? z : soft);
      p.beta[(size_t)c * p.gate_stride + h] = 1.0f / (1.0f + expf(-p.b[(size_t)c * p.ab_stride + h]));
    }
    return;
  }
  const uint32_t ch = (blockIdx.x * 64 + threadIdx.x) * 4;
  if (ch >= p.channels) return;
  f4 w[W], line[W];
  {
    float raw[4 * W];
#pragma unroll
    for (int i = 0; i < W; i++) *(f4*)(raw + 4 * i) = *(const f4*)(p.w + (size_t)ch * W + 4 * i);
#pragma unroll
    for (int i = 0; i < W; i++) w[i] = f4{raw[i], raw[W + i], raw[2 * W + i], raw[3 * W + i]};
  }
  const f4 bias = p.bias ? *(const f4*)(p.bias + ch) : f4{0.f, 0.f, 0.f, 0.f};
  // the W - 1 inputs in front of column c0
#pragma unroll
  for (int i = 0; i < W - 1; i++)
    line[i] = c0 == 0 ? *(const f4*)(p.conv + (size_t)i * p.channels + ch) : *(const f4*)(p.x + (size_t)(c0 + i - (W - 1)) * p.x_stride + ch);
  if constexpr (W > 1) {
    if (c0 == 0 && p.commit) {                        // the state after the committed columns; its old rows are in registers, and no other lane reads them
      f4 keep[W];
#pragma unroll
      for (int i = 0; i < W - 1; i++) {
        const uint32_t at = p.commit + i;             // row of [state; x]
        keep[i] = line[0];
        if (at < W - 1) {
#pragma unroll
          for (int m = 1; m < W - 1; m++) if (at == (uint32_t)m) keep[i] = line[m];
        } else {
          keep[i] = *(const f4*)(p.x + (size_t)(at - (W - 1)) * p.x_stride + ch);
        }
      }
#pragma unroll
      for (int i = 0; i < W - 1; i++) *(f4*)(p.conv + (size_t)i * p.channels + ch) = keep[i];
    }
  }
  f4 x[GLUE_COLS];
#pragma unroll
  for (uint32_t i = 0; i < GLUE_COLS; i++) if (c0 + i < c1) x[i] = *(const f4*)(p.x + (size_t)(c0 + i) * p.x_stride + ch);
#pragma unroll
  for (uint32_t i = 0; i < GLUE_COLS; i++) {
    if (c0 + i >= c1) break;
    line[W - 1] = x[i];
    f4 y = bias;
#pragma unroll
    for (int m = 0; m < W; m++)
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = __builtin_fmaf(line[m][e], w[m][e], y[e]);
#pragma unroll
    for (int m = 0; m < W - 1; m++) line[m] = line[m + 1];
    f4 o;
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = y[e] / (1.0f + expf(-y[e]));
    *(f4*)(p.out + (size_t)(c0 + i) * p.out_stride + ch) = o;
  }
}

hipError_t pa_launch_delta_glue(const DeltaGlueParams& p, hipStream_t s) {
  const dim3 grid((p.channels / 4 + 63) / 64 + 1, (p.n + GLUE_COLS - 1) / GLUE_COLS), block(64);
  switch (p.width) {
    case 1: hipLaunchKernelGGL(pa_delta_glue_kernel<1>, grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL(pa_delta_glue_kernel<2>, grid, block, 0, s, p); break;
    case 3: hipLaunchKernelGGL(pa_delta_glue_kernel<3>, grid, block, 0, s, p); break;
    case 4: hipLaunchKernelGGL(pa_delta_glue_kernel<4>, grid, block, 0, s, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

// zeros by a kernel: a memset node in a captured graph is not relied on
__global__ __launch_bounds__(256)
void pa_fill_zero_kernel(float* p, size_t n) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0.f;
}
hipError_t pa_launch_fill_zero(float* p, size_t n, hipStream_t s) {
  if (!n) return hipSuccess;
  const size_t blocks = (n + 255) / 256;
  hipLaunchKernelGGL(pa_fill_zero_kernel, dim3((uint32_t)(blocks < 1024 ? blocks : 1024)), dim3(256), 0, s, p, n);
  return hipGetLastError();
}
