// The gated delta rule token by token, and its pre-step (short causal convolution and gates), on gfx950.
//
// A linear-attention layer of the hybrid models keeps, per v head, a matrix S [head_v][head_k] instead of cache rows.  Token t:
//   S' = exp(g_t) S_{t-1};  u_t = beta_t (v_t - S' k_t);  S_t = S' + u_t k_t^T;  o_t = scale S_t q_t
// Row r of S is a recurrence of its own: u_t[r] and o_t[r] need row r, k_t and q_t alone.  Sixteen lanes hold one row (head_k / 16 values each, in
// registers over all columns of the call), a wavefront four rows, a workgroup sixteen; the two dot products of a token are sums over sixteen lanes,
// four DPP steps each, and nothing is exchanged between wavefronts.  With 32 v heads of 128 x 128 that is 1024 wavefronts, one per SIMD.
//
// One token moves 2 x 4 bytes per state value and computes 6 operations on it: it is bound by the state's stream and, at these sizes (2 MB), by the
// latency of a launch.  A run of columns is bound by its instructions, some 93 vector instructions a column and wavefront (370 cycles of 580 measured; 0.24 us a column
// with one wavefront a SIMD, 0.37 with two on half of them), and by the chain dot -> u -> update; the next columns' q, k, v and gates are requested four columns ahead.  Everything is f32.  A column's arithmetic does not depend on how many columns a
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

// 1 / sqrt(x); SMALL: also where x is subnormal, which the instruction takes for zero.  eps is added to every x, so only an eps near 0 needs that (seven columns of 48 heads: 0.25 us more)
template <bool SMALL>
static __device__ inline float inverse_root(float x) {
  if constexpr (!SMALL) return __builtin_amdgcn_rsqf(x);
  const bool tiny = x < 0x1p-100f;
  return __builtin_amdgcn_rsqf(tiny ? x * 0x1p100f : x) * (tiny ? 0x1p50f : 1.f);
}
enum { PLAIN_NORM = 1, SMALL_NORM = 2 };

// V4: float4 of a row per lane (head_k = 64 V4).  The leading arguments are those that every load needs: they arrive in scalar registers before the wave starts.
template <int V4, bool OUT, int NORM>
__global__ __launch_bounds__(256)
void pa_delta_step_kernel(const float* a_k, const float* a_q, const float* a_v, float* a_state, const float* a_g, const float* a_beta, DeltaParams p) {
  constexpr int AHEAD = 4;
  constexpr uint32_t HK = 64 * V4;
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15;
  const uint32_t tiles = p.hv / 16;
  const uint32_t h = blockIdx.x / tiles, row = (blockIdx.x % tiles) * 16 + wave * 4 + (lane >> 4), kh = h / p.group;
  float* const srow = a_state + ((size_t)h * p.hv + row) * HK + 4 * j;
  f4 S[V4];
#pragma unroll
  for (int i = 0; i < V4; i++) S[i] = *(const f4*)(srow + 64 * i);
  const float* kp = a_k + (size_t)kh * HK + 4 * j;
  const float* qp = a_q + (size_t)kh * HK + 4 * j;
  const float* vp = a_v + (size_t)h * p.hv + row;

  f4 kr[AHEAD][V4], qr[AHEAD][V4];
  float vr[AHEAD];
  auto request = [&](int s) __attribute__((always_inline)) {       // the next column
#pragma unroll
    for (int i = 0; i < V4; i++) kr[s][i] = *(const f4*)(kp + 64 * i);
    if constexpr (OUT) {
#pragma unroll
      for (int i = 0; i < V4; i++) qr[s][i] = *(const f4*)(qp + 64 * i);
    }
    vr[s] = *vp;
    kp += p.k_stride; qp += p.q_stride; vp += p.v_stride;
  };
  // gates of sixteen columns at a time, one a lane: their exponentials are one instruction sequence, and a column takes its own by a lane read
  float gate = 0.f, beta = 0.f;
  auto request_gates = [&](uint32_t t0) __attribute__((always_inline)) {
    const size_t t = min(t0 + j, p.n - 1);
    gate = a_g[t * p.gate_stride + h];
    beta = a_beta[t * p.gate_stride + h];
  };
  request_gates(0);
#pragma unroll
  for (int s = 0; s < AHEAD; s++) if ((uint32_t)s < p.n) request(s);

  for (uint32_t t0 = 0; t0 < p.n; t0 += 16) {
    const float decays = expf(gate), betas = beta;
    if (t0 + 16 < p.n) request_gates(t0 + 16);
    float keep = 0.f;                                              // lane j: the output of column t0 + j
#pragma unroll
    for (int b = 0; b < 4; b++) {
      if (t0 + 4 * b >= p.n) break;
#pragma unroll
      for (int s = 0; s < AHEAD; s++) {
        const uint32_t t = t0 + 4 * b + s;
        if (t >= p.n) break;
        const float decay = readlane_f32(decays, 4 * b + s), bt = readlane_f32(betas, 4 * b + s);
        // with k^ = k / |k|: S' k^ = (S' k) / |k| and u k^ = (u / |k|) k, so the row is used as it came
        float inv_k = 1.f, x = 0.f, y = 0.f;
        if constexpr (NORM != 0) {                                      // off the chain: needs k_t alone
#pragma unroll
          for (int i = 0; i < V4; i++) {
            x = __builtin_fmaf(kr[s][i][0], kr[s][i][0], x); y = __builtin_fmaf(kr[s][i][1], kr[s][i][1], y);
            x = __builtin_fmaf(kr[s][i][2], kr[s][i][2], x); y = __builtin_fmaf(kr[s][i][3], kr[s][i][3], y);
          }
          inv_k = inverse_root<NORM == SMALL_NORM>(row16_sum(x + y) + p.eps);
        }
        x = y = 0.f;
#pragma unroll
        for (int i = 0; i < V4; i++) {
          S[i] = S[i] * decay;
          x = __builtin_fmaf(S[i][0], kr[s][i][0], x); y = __builtin_fmaf(S[i][1], kr[s][i][1], y);
          x = __builtin_fmaf(S[i][2], kr[s][i][2], x); y = __builtin_fmaf(S[i][3], kr[s][i][3], y);
        }
        const float sk = row16_sum(x + y);
        const float u = bt * (NORM != 0 ? __builtin_fmaf(-sk, inv_k, vr[s]) : vr[s] - sk) * inv_k;
#pragma unroll
        for (int i = 0; i < V4; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) S[i][e] = __builtin_fmaf(u, kr[s][i][e], S[i][e]);
        if constexpr (OUT) {
          float scale = p.scale;
          x = y = 0.f;
          if constexpr (NORM != 0) {
#pragma unroll
            for (int i = 0; i < V4; i++) {
              x = __builtin_fmaf(qr[s][i][0], qr[s][i][0], x); y = __builtin_fmaf(qr[s][i][1], qr[s][i][1], y);
              x = __builtin_fmaf(qr[s][i][2], qr[s][i][2], x); y = __builtin_fmaf(qr[s][i][3], qr[s][i][3], y);
            }
            scale *= inverse_root<NORM == SMALL_NORM>(row16_sum(x + y) + p.eps);
            x = y = 0.f;
          }
#pragma unroll
          for (int i = 0; i < V4; i++) {
            x = __builtin_fmaf(S[i][0], qr[s][i][0], x); y = __builtin_fmaf(S[i][1], qr[s][i][1], y);
            x = __builtin_fmaf(S[i][2], qr[s][i][2], x); y = __builtin_fmaf(S[i][3], qr[s][i][3], y);
          }
          const float o = row16_sum(x + y) * scale;
          keep = j == (uint32_t)(4 * b + s) ? o : keep;
        }
        if (t + 1 == p.commit) {
#pragma unroll
          for (int i = 0; i < V4; i++) *(f4*)(srow + 64 * i) = S[i];
        }
        if (t + AHEAD < p.n) request(s);
      }
    }
    if constexpr (OUT) {
      if (t0 + j < p.n) {
        const size_t at = (size_t)(t0 + j) * p.out_stride + (size_t)h * p.hv + row;
        if (p.out_f16) ((_Float16*)p.out)[at] = (_Float16)keep; else ((float*)p.out)[at] = keep;
      }
    }
  }
}

template <int V4>
static void launch_step(const DeltaParams& p, hipStream_t s) {
  const dim3 grid(p.nv * (p.hv / 16)), block(256);
#define STEP(OUT, NORM) hipLaunchKernelGGL((pa_delta_step_kernel<V4, OUT, NORM>), grid, block, 0, s, p.k, p.q, p.v, p.state, p.g, p.beta, p)
  if (!p.l2norm) { if (p.out) STEP(true, 0); else STEP(false, 0); }
  else if (p.eps >= 0x1p-100f) { if (p.out) STEP(true, PLAIN_NORM); else STEP(false, PLAIN_NORM); }
  else { if (p.out) STEP(true, SMALL_NORM); else STEP(false, SMALL_NORM); }
#undef STEP
}
hipError_t pa_launch_delta_step(const DeltaParams& p, hipStream_t s) {
  if (p.hk == 64) launch_step<1>(p, s); else launch_step<2>(p, s);
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
