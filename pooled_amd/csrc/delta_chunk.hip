// The gated delta rule over many columns: chunks of 64 on the matrix cores.
//
// Within a chunk with start state S (here [head_k][head_v]), G_i = g_1 + .. + g_i, the 64 updates solve a triangular system:
//   A_ij = beta_i exp(G_i - G_j) k_i.k_j (i > j),  T = (1 + A)^-1,  X = diag(beta) (V - diag(e^G) K S),  U = T X
//   O = diag(e^G) Q S + P U,  P_ij = exp(G_i - G_j) q_i.k_j (i >= j);   S_next = e^G_64 S + (diag(e^(G_64 - G)) K)^T U
// T depends on keys and gates alone, so it is folded into what multiplies U: with P' = P T and K' = T^T diag(e^(G_64 - G)) K
//   O = diag(e^G) Q S + P' X,   S_next = e^G_64 S + K'^T X.
// Two kernels.  pa_delta_prep_kernel computes K', P' of every chunk and v head, all chunks side by side.  pa_delta_scan_kernel walks the chunks in order, a workgroup
// a v head and 16 columns of its values, S in registers: per chunk K S, then X, then K'^T X, and beside them Q S and P' X.  Only decays between a
// place and a later one occur, never their inverses, so nothing overflows however fast a head forgets; sums of g are kept in 64 bits, because their differences matter.
//
// Precision.  The results are f32 and stay as exact as f32 sums: every operand of the f16 matrix instructions is a pair hi + lo / 2048 of f16 values (22 bits), a product is
// hi hi + (hi lo + lo hi) / 2048 (the dropped lo lo is 2^-22 of it), accumulated in f32.  A pair is exact to 2^-36 of the largest f16 power below it, so it needs operands of known size:
// rows of q are scaled by a power of two to a norm in [0.5, 1), K' by one for its largest element, and S and X, per value column, by one from a bound: the rule over keys no longer than
// one with 0 <= beta <= 2, g <= 0 is a contraction, so |S_next| <= |S| + sum beta |v| =: the bound of S_next, and 2 |S| + sum beta |v| that of X.  A chunk whose inputs leave that
// domain (longer or tiny keys, other gates, infinities, NaN) is marked by the first kernel, or found by the bound, and runs token by token in the second, in f32, with the same
// S: slower (about 1 us a token), but right for every input.
//
// What bounds it: a workgroup's chunk reads K, Q, K' (32 KB each at head_k 128) and P' (16 KB): 112 KB through one CU's 64 bytes a clock, 0.73 us, while its 168
// matrix instructions take 0.3 us of four SIMDs.  The first kernel stores these operands in the order in which lanes load them (a fragment is 1 KB), every
// fragment goes to one wavefront alone, and each is requested a chunk ahead, right behind its last use: no operand passes through LDS but S and X, which change hands
// between the wavefronts twice a chunk.
#include "blocks_internal.h"
#include "glue_math.h"
#include <algorithm>

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

#define CHUNK 64
// per chunk and v head: beta, beta e^G, output factors of Q S and P' X, 1 / |k| and 1 / |q| (or 1), 64 floats each; then e^G_64, the scale of K', the mark
#define SCAL_FLOATS 448
#define SCAL_DECAY 384
#define SCAL_KSCALE 385
#define SCAL_MARK 386
#define LO_SCALE 2048.f
#define LO_INV (1.f / 2048.f)
// operands of magnitude up to one are stored times 4096, so that their low halves are normal f16 numbers too
#define UNIT 4096.f
#define UNIT_INV (1.f / 4096.f)

static __device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// sum / maximum over lanes {i, i ^ 16, i ^ 32, i ^ 48}
static __device__ inline float rows4_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// exp of a 64-bit sum: the part of the argument that f32 drops is put back to first order
static __device__ inline float exp_f64(double x) {
  const float hi = (float)x, e = expf(hi);
  return __builtin_fmaf(e, (float)(x - (double)hi), e);
}
static __device__ inline void split(float x, _Float16& hi, _Float16& lo) {
  asm("" : "+v"(x));      // one f32 number: fused into the product that made it, hi would be rounded once and the difference below from a hi rounded twice, a whole step apart at times
  hi = (_Float16)x;
  lo = (_Float16)((x - (float)hi) * LO_SCALE);
}
struct Pair8 { h8 hi, lo; };
static __device__ inline Pair8 split8(const float (&x)[8]) {
  Pair8 r;
#pragma unroll
  for (int e = 0; e < 8; e++) { _Float16 h, l; split(x[e], h, l); r.hi[e] = h; r.lo[e] = l; }
  return r;
}
// hi hi into `a`, hi lo + lo hi into `b`: the product is a + b / 2048
static __device__ inline void mfma_pair(const h8 ahi, const h8 alo, const h8 bhi, const h8 blo, f4& a, f4& b) {
  a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahi, bhi, a, 0, 0, 0);
  b = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahi, blo, b, 0, 0, 0);
  b = __builtin_amdgcn_mfma_f32_16x16x32_f16(alo, bhi, b, 0, 0, 0);
}
static __device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }          // -126 <= e <= 127
// largest magnitude `m` -> the exponent e with m 2^(13 - e) in [2^13, 2^14), as far as f32 has the powers
static __device__ inline int exponent(float x);
static __device__ inline int scale_exponent(float m) { return m >= 0x1p-100f ? min(exponent(m), 100) : m > 0.f ? -100 : 13; }
static __device__ inline int exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255) - 127; }   // of a positive normal number

// ---- workspace: fragments of 64 lanes x 8 halves (1 KB) --------------------------------------------
// K, Q of a k head: [plane hi, lo][row tile 4][k step HK / 32];  K'^T: [plane][row tile HK / 16][k step 2];  P': [plane][row tile 4][k step 2]
template <int HK> struct Frags {
  static constexpr uint32_t KS = HK / 32, MK = HK / 16;
  static constexpr uint32_t KQ = 2 * 4 * KS * 512, KT = 2 * MK * 2 * 512, P = 2 * 4 * 2 * 512;       // halves
};
struct DeltaWs { _Float16* kq; _Float16* kt; _Float16* pp; float* scal; };

template <int HK>
static DeltaWs ws_at(void* ws, uint32_t chunks, uint32_t nk, uint32_t nv, size_t* bytes) {
  using F = Frags<HK>;
  DeltaWs w;
  unsigned char* b = (unsigned char*)ws;
  size_t at = 0;
  w.kq = (_Float16*)(b + at); at += (size_t)chunks * nk * 2 * F::KQ * 2;
  w.kt = (_Float16*)(b + at); at += (size_t)chunks * nv * F::KT * 2;
  w.pp = (_Float16*)(b + at); at += (size_t)chunks * nv * F::P * 2;
  w.scal = (float*)(b + at); at += (size_t)chunks * nv * SCAL_FLOATS * 4;
  if (bytes) *bytes = at;
  return w;
}
size_t pa_delta_chunk_ws_bytes(uint32_t chunks, uint32_t nk, uint32_t nv, uint32_t hk) {
  size_t b = 0;
  if (hk == 64) ws_at<64>(nullptr, chunks, nk, nv, &b); else ws_at<128>(nullptr, chunks, nk, nv, &b);
  return b;
}

// ---- 1: what does not depend on the state ----------------------------------------------------------
#define TS 68      // floats of a row of A and T in LDS
// LDS, first pair of regions for the products of rows, then the second: K | Q fragments; A | T (f32) | P fragments | T^T fragments
#define PREP_A 0
#define PREP_T (CHUNK * TS * 4)
#define PREP_P (2 * CHUNK * TS * 4)
#define PREP_TT (PREP_P + 16384)
#define PREP_LDS (PREP_TT + 16384)

template <int HK>
__global__ __launch_bounds__(256)
void pa_delta_prep_kernel(DeltaParams p, DeltaWs ws) {
  using F = Frags<HK>;
  constexpr int KS = F::KS, DT = HK / 64;                          // DT: tiles of 16 key dimensions of a wavefront
  __shared__ __attribute__((aligned(16))) unsigned char lds[PREP_LDS];
  __shared__ double Gs[CHUNK];
  __shared__ float beta_s[CHUNK], kfac_s[CHUNK], kinv_s[CHUNK], max_s[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
  const uint32_t h = blockIdx.x, chunk = blockIdx.y, kh = h / p.group, c0 = chunk * CHUNK;
  _Float16* const kq = ws.kq + ((size_t)chunk * p.nk + kh) * 2 * F::KQ;
  float* const scal = ws.scal + ((size_t)chunk * p.nv + h) * SCAL_FLOATS;
  _Float16* const kl = (_Float16*)lds;
  _Float16* const ql = kl + F::KQ;
  bool bad = false;

  // -- rows: lengths, scaled pairs, fragments.  Four lanes a row, eight values each per k step
  {
    const uint32_t row = tid >> 2, part = tid & 3;
    const bool valid = c0 + row < p.n;
    const size_t c = min(c0 + row, p.n - 1);
    const float* kp = p.k + c * p.k_stride + (size_t)kh * HK + 8 * part;
    const float* qp = p.q + c * p.q_stride + (size_t)kh * HK + 8 * part;
    float k[KS][8], q[KS][8], kk = 0.f, qq = 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const f4 a = *(const f4*)(kp + 32 * s + 4 * e), b = *(const f4*)(qp + 32 * s + 4 * e);
#pragma unroll
        for (int j = 0; j < 4; j++) { k[s][4 * e + j] = valid ? a[j] : 0.f; q[s][4 * e + j] = valid ? b[j] : 0.f; }
      }
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 8; e++) { kk = __builtin_fmaf(k[s][e], k[s][e], kk); qq = __builtin_fmaf(q[s][e], q[s][e], qq); }
    kk += dpp_f32<0xB1>(kk); kk += dpp_f32<0x4E>(kk);
    qq += dpp_f32<0xB1>(qq); qq += dpp_f32<0x4E>(qq);
    const float kinv = p.l2norm && valid ? 1.0f / sqrtf(kk + p.eps) : 1.f;
    const float qinv = p.l2norm && valid ? 1.0f / sqrtf(qq + p.eps) : 1.f;
    const float kn = kk * kinv * kinv, qn = qq * qinv * qinv;      // squares of the lengths that the rule sees
    // lengths whose pairs keep their bits: keys in [2^-10, 1], or 0; q of any size whose square is a normal number, or 0
    bad = !(kn <= 1.00002f) || (kn < 0x1p-20f && !(kk == 0.f)) || !(qn < 0x1p100f) || (qn < 0x1p-100f && !(qq == 0.f));
    const int qe = qn >= 0x1p-100f && qn < 0x1p100f ? (exponent(qn) >> 1) + 1 : 0;   // |q| 2^-qe in [0.5, 1)
    const float qs = qinv * pow2(-qe);
    if (part == 0) {
      kinv_s[row] = valid ? kinv : 0.f;
      scal[4 * 64 + row] = kinv;
      scal[5 * 64 + row] = qinv;
      scal[3 * 64 + row] = p.scale * pow2(qe);
    }
    const uint32_t frag = (row >> 4) * KS, at = (part * 16 + (row & 15)) * 8;
    const bool first = h == kh * p.group;                          // one v head of the group stores the k head's fragments
#pragma unroll
    for (int s = 0; s < KS; s++) {
#pragma unroll
      for (int e = 0; e < 8; e++) { k[s][e] *= kinv * UNIT; q[s][e] *= qs * UNIT; }
      const Pair8 kp8 = split8(k[s]), qp8 = split8(q[s]);
      const uint32_t off = (frag + s) * 512 + at;
      *(h8*)(kl + off) = kp8.hi; *(h8*)(kl + F::KQ / 2 + off) = kp8.lo;
      *(h8*)(ql + off) = qp8.hi; *(h8*)(ql + F::KQ / 2 + off) = qp8.lo;
      if (first) {
        *(h8*)(kq + off) = kp8.hi; *(h8*)(kq + F::KQ / 2 + off) = kp8.lo;
        *(h8*)(kq + F::KQ + off) = qp8.hi; *(h8*)(kq + F::KQ + F::KQ / 2 + off) = qp8.lo;
      }
    }
  }
  // -- gates: sums of g in 64 bits by the first wavefront
  if (wave == 0) {
    const bool valid = c0 + lane < p.n;
    const size_t c = min(c0 + lane, p.n - 1);
    const float g = valid ? p.g[c * p.gate_stride + h] : 0.f, b = valid ? p.beta[c * p.gate_stride + h] : 0.f;
    bad = bad || !(g <= 0.f) || !(b >= 0.f && b <= 2.f);
    double G = g > -1e5f ? (double)g : -1e5;                        // exp(-1e5) is 0 as exp(-infinity) is, and differences stay numbers
#pragma unroll
    for (int d = 1; d < 64; d *= 2) { const double o = __shfl_up(G, d); if (lane >= (uint32_t)d) G += o; }
    Gs[lane] = G;
    beta_s[lane] = b;
  }
  const bool mark = __syncthreads_or(bad);
  if (tid < 64) {
    const float eG = exp_f64(Gs[tid]);
    scal[tid] = beta_s[tid];
    scal[64 + tid] = beta_s[tid] * eG;
    kfac_s[tid] = kinv_s[tid] * exp_f64(Gs[63] - Gs[tid]);
    if (tid == 63) { scal[SCAL_DECAY] = eG; scal[SCAL_MARK] = __uint_as_float(mark ? 1u : 0u); }
  } else if (tid < 128) {
    const uint32_t r = tid - 64;
    scal[2 * 64 + r] = exp_f64(Gs[r]);                             // times the factor of P' X, in the second kernel
  }
  if (mark) return;                                                // the chunk runs token by token

  // -- products of rows: tiles (mt <= nt) of K K^T and K Q^T, keys m in rows, keys / queries i in columns; ten tiles dealt to the wavefronts
  f4 ga[3], gp[3];
#pragma unroll
  for (int s = 0; s < 3; s++) {
    const uint32_t id = wave + 4 * s;
    ga[s] = gp[s] = f4{0.f, 0.f, 0.f, 0.f};
    if (id < 10) {
      const uint32_t nt = id >= 6 ? 3 : id >= 3 ? 2 : id >= 1 ? 1 : 0, mt = id - nt * (nt + 1) / 2;
      f4 a1 = ga[s], p1 = ga[s];
#pragma unroll
      for (int ks = 0; ks < KS; ks++) {
        const uint32_t m = (mt * KS + ks) * 512 + lane * 8, i = (nt * KS + ks) * 512 + lane * 8;
        const h8 mh = *(const h8*)(kl + m), ml = *(const h8*)(kl + F::KQ / 2 + m);
        mfma_pair(mh, ml, *(const h8*)(kl + i), *(const h8*)(kl + F::KQ / 2 + i), ga[s], a1);
        mfma_pair(mh, ml, *(const h8*)(ql + i), *(const h8*)(ql + F::KQ / 2 + i), gp[s], p1);
      }
      ga[s] = (ga[s] + a1 * LO_INV) * (UNIT_INV * UNIT_INV);
      gp[s] = (gp[s] + p1 * LO_INV) * (UNIT_INV * UNIT_INV);
    }
  }
  __syncthreads();                                                 // K and Q have been read: their LDS is A, T and P's now
  float* const As = (float*)(lds + PREP_A);
  float* const Tf = (float*)(lds + PREP_T);
  _Float16* const pl = (_Float16*)(lds + PREP_P);
  _Float16* const tt = (_Float16*)(lds + PREP_TT);
  constexpr uint32_t LOP = 4096;                                   // halves from a plane to the other, of P, P' and T^T
#pragma unroll
  for (int s = 0; s < 3; s++) {
    const uint32_t id = wave + 4 * s;
    if (id < 10) {
      const uint32_t nt = id >= 6 ? 3 : id >= 3 ? 2 : id >= 1 ? 1 : 0, mt = id - nt * (nt + 1) / 2;
      const uint32_t i = nt * 16 + l16, m0 = mt * 16 + 4 * lg;
      const double Gi = Gs[i];
      const float b = beta_s[i];
      f4 a;
      h4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float d = m0 + r <= i ? exp_f64(Gi - Gs[m0 + r]) : 0.f;
        a[r] = m0 + r < i ? b * d * ga[s][r] : 0.f;
        _Float16 x, y;
        split(d * gp[s][r] * UNIT, x, y);
        hi[r] = x; lo[r] = y;
      }
      *(f4*)(As + i * TS + m0) = a;
      const uint32_t off = (nt * 2 + (mt >> 1)) * 512 + (l16 + 16 * ((m0 & 31) >> 3)) * 8 + (m0 & 7);
      *(h4*)(pl + off) = hi; *(h4*)(pl + LOP + off) = lo;
    }
  }
  if (wave < 2) {                                                  // the zero halves of fragments that cross the diagonal: tiles (1, 0) and (3, 2)
    const uint32_t nt = 2 * wave, m0 = (nt + 1) * 16 + 4 * lg, off = (nt * 2 + (nt >> 1)) * 512 + (l16 + 16 * ((m0 & 31) >> 3)) * 8 + (m0 & 7);
    *(h4*)(pl + off) = h4{0, 0, 0, 0}; *(h4*)(pl + LOP + off) = h4{0, 0, 0, 0};
  }
  __syncthreads();
  // -- T = (1 + A)^-1: each wavefront its diagonal block by substitution, a lane a column (the four lane groups do the same)
  {
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float s = l16 == (uint32_t)i ? 1.f : 0.f;
#pragma unroll
      for (int m4 = 0; m4 < i; m4 += 4) {
        const f4 a = *(const f4*)(As + (wave * 16 + i) * TS + wave * 16 + m4);
#pragma unroll
        for (int m = 0; m < 4; m++) if (m4 + m < i) s = __builtin_fmaf(-a[m], t[m4 + m], s);
      }
      t[i] = s;
    }
    if (lg == 0) {
#pragma unroll
      for (int i = 0; i < 16; i++) Tf[(wave * 16 + i) * TS + wave * 16 + l16] = t[i];
    }
  }
  __syncthreads();
  // 16 x 16 products in f32; the contraction runs over 4 lg + r, so that a result is the next product's right operand as it stands
  auto left = [&](const float* m, uint32_t br, uint32_t bc) { return *(const f4*)(m + (br * 16 + l16) * TS + bc * 16 + 4 * lg); };
  auto right = [&](const float* m, uint32_t br, uint32_t bc) {
    const float* x = m + (br * 16 + 4 * lg) * TS + bc * 16 + l16;
    return f4{x[0], x[TS], x[2 * TS], x[3 * TS]};
  };
  auto mul = [&](const f4 a, const f4 b, f4 c) {
#pragma unroll
    for (int r = 0; r < 4; r++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
  };
  auto put = [&](uint32_t br, uint32_t bc, const f4 v) {
    float* x = Tf + (br * 16 + 4 * lg) * TS + bc * 16 + l16;
#pragma unroll
    for (int r = 0; r < 4; r++) x[r * TS] = -v[r];
  };
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  if (wave < 2) {
    const uint32_t j = 2 * wave, i = j + 1;
    put(i, j, mul(left(Tf, i, i), mul(left(As, i, j), right(Tf, j, j), zero), zero));
  }
  __syncthreads();
  {
    const uint32_t j = wave & 1, i = 2 + (wave >> 1);
    auto inner = [&](uint32_t row) {                               // row of A T over the first two blocks
      f4 m = mul(left(As, row, j), right(Tf, j, j), zero);
      return j == 0 ? mul(left(As, row, 1), right(Tf, 1, 0), m) : m;
    };
    const f4 m2 = inner(2);
    f4 r;
    if (i == 2) r = mul(left(Tf, 2, 2), m2, zero);
    else r = mul(left(Tf, 3, 3), inner(3), mul(left(Tf, 3, 2), m2, zero));
    put(i, j, r);                                                  // blocks that no other wavefront reads here
  }
  __syncthreads();
  // -- T^T as fragments: rows j, contraction over i
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const uint32_t f = wave * 2 + e, jt = f >> 1, ks = f & 1, j = jt * 16 + l16, i0 = ks * 32 + 8 * lg;
    float x[8];
#pragma unroll
    for (int m = 0; m < 8; m++) x[m] = i0 + m >= j ? Tf[(i0 + m) * TS + j] * UNIT : 0.f;
    const Pair8 s = split8(x);
    *(h8*)(tt + f * 512 + lane * 8) = s.hi; *(h8*)(tt + LOP + f * 512 + lane * 8) = s.lo;
  }
  __syncthreads();
  // -- K' [j][d] = sum_i T_ij e^(G_64 - G_i) k_i[d]
  f4 kt[DT][4];
  float top = 0.f;
#pragma unroll
  for (int x = 0; x < DT; x++) {
    const uint32_t d = (wave * DT + x) * 16 + l16;
    Pair8 b[2];
#pragma unroll
    for (int ks = 0; ks < 2; ks++) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const uint32_t i = ks * 32 + 8 * lg + e;
        v[e] = p.k[(size_t)min(c0 + i, p.n - 1) * p.k_stride + (size_t)kh * HK + d] * (kfac_s[i] * UNIT);
      }
      b[ks] = split8(v);
    }
#pragma unroll
    for (int jt = 0; jt < 4; jt++) {
      f4 a0 = zero, a1 = zero;
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        if (ks < jt / 2) continue;
        const uint32_t f = (jt * 2 + ks) * 512 + lane * 8;
        mfma_pair(*(const h8*)(tt + f), *(const h8*)(tt + LOP + f), b[ks].hi, b[ks].lo, a0, a1);
      }
      kt[x][jt] = (a0 + a1 * LO_INV) * (UNIT_INV * UNIT_INV);
#pragma unroll
      for (int r = 0; r < 4; r++) top = fmaxf(top, fabsf(kt[x][jt][r]));
    }
  }
  // -- P'^T [j][i] = sum_m T_mj P_im: a wavefront a tile of 16 queries
  _Float16* const pp = ws.pp + ((size_t)chunk * p.nv + h) * F::P;
#pragma unroll
  for (int jt = 0; jt < 4; jt++) {
    f4 a0 = zero, a1 = zero;
    if ((uint32_t)jt <= wave) {
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        if (ks < jt / 2 || ks > (int)(wave >> 1)) continue;
        const uint32_t f = (jt * 2 + ks) * 512 + lane * 8, g = (wave * 2 + ks) * 512 + lane * 8;
        mfma_pair(*(const h8*)(tt + f), *(const h8*)(tt + LOP + f), *(const h8*)(pl + g), *(const h8*)(pl + LOP + g), a0, a1);
      }
    }
    h4 hi, lo;
#pragma unroll
    for (int r = 0; r < 4; r++) { _Float16 x, y; split((a0[r] + a1[r] * LO_INV) * UNIT_INV, x, y); hi[r] = x; lo[r] = y; }
    const uint32_t j0 = jt * 16 + 4 * lg, off = (wave * 2 + (jt >> 1)) * 512 + (l16 + 16 * ((j0 & 31) >> 3)) * 8 + (j0 & 7);
    *(h4*)(pp + off) = hi; *(h4*)(pp + LOP + off) = lo;
  }
  // -- K'^T in the order of the second kernel's loads, scaled by the power of two of its largest element
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) max_s[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(max_s[0], max_s[1]), fmaxf(max_s[2], max_s[3]));
  const int ke = top >= 0x1p-100f ? exponent(top) : 13;
  const float ksc = pow2(13 - ke);
  if (tid == 0) scal[SCAL_KSCALE] = pow2(ke - 13);
  _Float16* const kto = ws.kt + ((size_t)chunk * p.nv + h) * F::KT;
#pragma unroll
  for (int x = 0; x < DT; x++)
#pragma unroll
    for (int jt = 0; jt < 4; jt++) {
      h4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; r++) { _Float16 a, b; split(kt[x][jt][r] * ksc, a, b); hi[r] = a; lo[r] = b; }
      const uint32_t j0 = jt * 16 + 4 * lg, off = ((wave * DT + x) * 2 + (jt >> 1)) * 512 + (l16 + 16 * ((j0 & 31) >> 3)) * 8 + (j0 & 7);
      *(h4*)(kto + off) = hi; *(h4*)(kto + F::KT / 2 + off) = lo;
    }
}

// ---- 2: from chunk to chunk -------------------------------------------------------------------------
template <int HK>
__global__ __launch_bounds__(256)
void pa_delta_scan_kernel(DeltaParams p, DeltaWs ws) {
  using F = Frags<HK>;
  constexpr int KS = F::KS, MW = HK / 64;                          // MW: tiles of 16 state rows (key dimensions) of a wavefront
  __shared__ __attribute__((aligned(16))) _Float16 Sl[2][KS * 512], Xl[2][2 * 512];
  __shared__ float norm_s[4][16], value_s[4][16], slow_s[2][2][4][16];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
  const uint32_t h = blockIdx.x % p.nv, v0 = blockIdx.x / p.nv * 16, kh = h / p.group;
  const uint32_t chunks = (p.n + CHUNK - 1) / CHUNK;
  const bool out = p.out != nullptr;

  // state rows 16 (wave MW + x) + 4 lg + r of value column v0 + l16
  float* const sp = p.state + ((size_t)h * p.hv + v0 + l16) * HK + wave * MW * 16 + 4 * lg;
  f4 S[MW];
#pragma unroll
  for (int x = 0; x < MW; x++) S[x] = *(const f4*)(sp + 16 * x);

  // Operands of the wavefront, requested a chunk ahead.  The last chunk requests itself again instead of branching round the loads: a short conditional block between a matrix
  // instruction and the first use of its result makes this compiler (22.0.0git, ROCm 7.2.0) leave out the wait states on the path round the block, and the use then reads the old
  // registers (seen as states 1e-4 off after a last chunk).
  h8 kf[KS][2], qf[KS][2], pf[2][2], tf[MW][2][2];
  struct Rows { f4 sb, sc, se, sq, v; float decay, kscale; uint32_t mark; } now, next;
  auto load_k = [&](uint32_t c) {
    const _Float16* b = ws.kq + ((size_t)c * p.nk + kh) * 2 * F::KQ + wave * KS * 512 + lane * 8;
#pragma unroll
    for (int s = 0; s < KS; s++) { kf[s][0] = *(const h8*)(b + s * 512); kf[s][1] = *(const h8*)(b + F::KQ / 2 + s * 512); }
  };
  auto load_q = [&](uint32_t c) {
    const _Float16* b = ws.kq + ((size_t)c * p.nk + kh) * 2 * F::KQ + F::KQ + wave * KS * 512 + lane * 8;
#pragma unroll
    for (int s = 0; s < KS; s++) { qf[s][0] = *(const h8*)(b + s * 512); qf[s][1] = *(const h8*)(b + F::KQ / 2 + s * 512); }
  };
  auto load_t = [&](uint32_t c) {
    const _Float16* b = ws.kt + ((size_t)c * p.nv + h) * F::KT + wave * MW * 2 * 512 + lane * 8;
#pragma unroll
    for (int x = 0; x < MW; x++)
#pragma unroll
      for (int s = 0; s < 2; s++) { tf[x][s][0] = *(const h8*)(b + (x * 2 + s) * 512); tf[x][s][1] = *(const h8*)(b + F::KT / 2 + (x * 2 + s) * 512); }
  };
  auto load_p = [&](uint32_t c) {
    const _Float16* b = ws.pp + ((size_t)c * p.nv + h) * F::P + wave * 2 * 512 + lane * 8;
#pragma unroll
    for (int s = 0; s < 2; s++) { pf[s][0] = *(const h8*)(b + s * 512); pf[s][1] = *(const h8*)(b + F::P / 2 + s * 512); }
  };
  auto load_rows = [&](uint32_t c) {                               // the wavefront's 16 rows of values, and their gates
    const uint32_t i0 = c * CHUNK + wave * 16 + 4 * lg;
    const float* sg = ws.scal + ((size_t)c * p.nv + h) * SCAL_FLOATS;
    Rows w;
#pragma unroll
    for (int r = 0; r < 4; r++) w.v[r] = i0 + r < p.n ? p.v[(size_t)(i0 + r) * p.v_stride + (size_t)h * p.hv + v0 + l16] : 0.f;
    w.sb = *(const f4*)(sg + wave * 16 + 4 * lg);
    w.sc = *(const f4*)(sg + 64 + wave * 16 + 4 * lg);
    w.se = *(const f4*)(sg + 128 + wave * 16 + 4 * lg);
    w.sq = *(const f4*)(sg + 192 + wave * 16 + 4 * lg);
    w.decay = sg[SCAL_DECAY]; w.kscale = sg[SCAL_KSCALE]; w.mark = __float_as_uint(sg[SCAL_MARK]);
    return w;
  };
  // S as pairs scaled by `sigma`, its column sums |S| (no smaller than the norm, and they neither over- nor underflow before their terms do) and the
  // coming chunk's sums of beta |v|, for everyone
  auto publish = [&](float sigma, const Rows& w) {
    float ss = 0.f, sv = 0.f;
#pragma unroll
    for (int x = 0; x < MW; x++) {
      h4 hi, lo;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        ss += fabsf(S[x][r]);
        _Float16 a, b;
        split(S[x][r] * sigma, a, b);
        hi[r] = a; lo[r] = b;
      }
      const uint32_t d0 = (wave * MW + x) * 16 + 4 * lg, off = (d0 >> 5) * 512 + (l16 + 16 * ((d0 & 31) >> 3)) * 8 + (d0 & 7);
      *(h4*)(&Sl[0][off]) = hi; *(h4*)(&Sl[1][off]) = lo;
    }
#pragma unroll
    for (int r = 0; r < 4; r++) sv += fabsf(w.sb[r] * w.v[r]);
    ss = rows4_sum(ss); sv = rows4_sum(sv);
    if (lg == 0) { norm_s[wave][l16] = ss; value_s[wave][l16] = sv; }
  };

  now = load_rows(0);
  load_k(0); load_t(0);
  if (out) { load_q(0); load_p(0); }
  // the first scale from S itself
  float sigma = 1.f, sigma_inv = 1.f;
  {
    float ss = 0.f;
#pragma unroll
    for (int x = 0; x < MW; x++)
#pragma unroll
      for (int r = 0; r < 4; r++) ss = fmaxf(ss, fabsf(S[x][r]));
#pragma unroll
    for (int o = 16; o < 64; o *= 2) ss = fmaxf(ss, __shfl_xor(ss, o));
    if (lg == 0) norm_s[wave][l16] = ss;
    lds_barrier();
    const float m = fmaxf(fmaxf(norm_s[0][l16], norm_s[1][l16]), fmaxf(norm_s[2][l16], norm_s[3][l16]));
    const int e = scale_exponent(m);
    sigma = pow2(13 - e); sigma_inv = pow2(e - 13);
    lds_barrier();
  }
  publish(sigma, now);

  for (uint32_t c = 0; c < chunks; c++) {
    lds_barrier();
    // bound of X and of the next S, per column; a column that has none sends the chunk the slow way
    const float bound = 1.02f * (2.1f * ((norm_s[0][l16] + norm_s[1][l16]) + (norm_s[2][l16] + norm_s[3][l16])) +
                                 ((value_s[0][l16] + value_s[1][l16]) + (value_s[2][l16] + value_s[3][l16])));
    const bool none = !(bound == 0.f || (bound >= 0x1p-90f && bound < 0x1p90f));
    const uint32_t cn = min(c + 1, chunks - 1);
    const int be = scale_exponent(bound);
    const float to = pow2(13 - be), to_inv = pow2(be - 13);
    next = load_rows(cn);
    if (!now.mark && !__any(none)) {
      // R = K S, X = beta v - beta e^G R
      f4 r0 = {0.f, 0.f, 0.f, 0.f}, r1 = r0, o0 = r0, o1 = r0;
      h8 sh[KS], sl[KS];
#pragma unroll
      for (int s = 0; s < KS; s++) { sh[s] = *(const h8*)(&Sl[0][s * 512 + lane * 8]); sl[s] = *(const h8*)(&Sl[1][s * 512 + lane * 8]); }
#pragma unroll
      for (int s = 0; s < KS; s++) mfma_pair(kf[s][0], kf[s][1], sh[s], sl[s], r0, r1);
      load_k(cn);
      {
        h4 hi, lo;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float x = __builtin_fmaf(-now.sc[r], (r0[r] + r1[r] * LO_INV) * (sigma_inv * UNIT_INV), now.sb[r] * now.v[r]);
          _Float16 a, b;
          split(x * to, a, b);
          hi[r] = a; lo[r] = b;
        }
        const uint32_t i0 = wave * 16 + 4 * lg, off = (i0 >> 5) * 512 + (l16 + 16 * ((i0 & 31) >> 3)) * 8 + (i0 & 7);
        *(h4*)(&Xl[0][off]) = hi; *(h4*)(&Xl[1][off]) = lo;
      }
      if (out) {
#pragma unroll
        for (int s = 0; s < KS; s++) mfma_pair(qf[s][0], qf[s][1], sh[s], sl[s], o0, o1);
        load_q(cn);
      }
      lds_barrier();
      h8 xh[2], xl[2];
#pragma unroll
      for (int s = 0; s < 2; s++) { xh[s] = *(const h8*)(&Xl[0][s * 512 + lane * 8]); xl[s] = *(const h8*)(&Xl[1][s * 512 + lane * 8]); }
      f4 n0[MW], n1[MW];
#pragma unroll
      for (int x = 0; x < MW; x++) {
        n0[x] = n1[x] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 2; s++) mfma_pair(tf[x][s][0], tf[x][s][1], xh[s], xl[s], n0[x], n1[x]);
      }
      load_t(cn);
      const float back = to_inv * now.kscale;
#pragma unroll
      for (int x = 0; x < MW; x++)
#pragma unroll
        for (int r = 0; r < 4; r++) S[x][r] = __builtin_fmaf(S[x][r], now.decay, (n0[x][r] + n1[x][r] * LO_INV) * back);
      publish(to, next);
      if (out) {
        f4 u0 = {0.f, 0.f, 0.f, 0.f}, u1 = u0;
#pragma unroll
        for (int s = 0; s < 2; s++) mfma_pair(pf[s][0], pf[s][1], xh[s], xl[s], u0, u1);
        load_p(cn);
        const uint32_t i0 = c * CHUNK + wave * 16 + 4 * lg;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float o = now.sq[r] * __builtin_fmaf(now.se[r], (o0[r] + o1[r] * LO_INV) * (sigma_inv * UNIT_INV), (u0[r] + u1[r] * LO_INV) * (to_inv * UNIT_INV));
          if (i0 + r < p.n) {
            const size_t at = (size_t)(i0 + r) * p.out_stride + (size_t)h * p.hv + v0 + l16;
            if (p.out_f16) ((_Float16*)p.out)[at] = (_Float16)o; else ((float*)p.out)[at] = o;
          }
        }
      }
      sigma_inv = to_inv;
    } else {
      // token by token, in f32: dot products over the key dimensions of all four wavefronts, one exchange each
      const float* const sg = ws.scal + ((size_t)c * p.nv + h) * SCAL_FLOATS;
      const uint32_t rows = min((uint32_t)CHUNK, p.n - c * CHUNK);
      for (uint32_t t = 0; t < rows; t++) {
        const size_t col = (size_t)c * CHUNK + t;
        const uint32_t d0 = kh * HK + wave * MW * 16 + 4 * lg;
        const float ki = sg[4 * 64 + t], qi = sg[5 * 64 + t];
        const float dec = expf(p.g[col * p.gate_stride + h]), b = p.beta[col * p.gate_stride + h], vt = p.v[col * p.v_stride + (size_t)h * p.hv + v0 + l16];
        f4 k[MW];
        float a = 0.f;
#pragma unroll
        for (int x = 0; x < MW; x++) {
          k[x] = *(const f4*)(p.k + col * p.k_stride + d0 + 16 * x) * ki;
#pragma unroll
          for (int r = 0; r < 4; r++) { S[x][r] *= dec; a = __builtin_fmaf(S[x][r], k[x][r], a); }
        }
        a = rows4_sum(a);
        if (lg == 0) slow_s[0][t & 1][wave][l16] = a;
        lds_barrier();
        const float u = b * (vt - ((slow_s[0][t & 1][0][l16] + slow_s[0][t & 1][1][l16]) + (slow_s[0][t & 1][2][l16] + slow_s[0][t & 1][3][l16])));
#pragma unroll
        for (int x = 0; x < MW; x++)
#pragma unroll
          for (int r = 0; r < 4; r++) S[x][r] = __builtin_fmaf(u, k[x][r], S[x][r]);
        if (out) {
          float o = 0.f;
#pragma unroll
          for (int x = 0; x < MW; x++) {
            const f4 q = *(const f4*)(p.q + col * p.q_stride + d0 + 16 * x) * qi;
#pragma unroll
            for (int r = 0; r < 4; r++) o = __builtin_fmaf(S[x][r], q[r], o);
          }
          o = rows4_sum(o);
          if (lg == 0) slow_s[1][t & 1][wave][l16] = o;
          lds_barrier();
          if (tid < 16) {
            o = p.scale * ((slow_s[1][t & 1][0][l16] + slow_s[1][t & 1][1][l16]) + (slow_s[1][t & 1][2][l16] + slow_s[1][t & 1][3][l16]));
            const size_t at = col * p.out_stride + (size_t)h * p.hv + v0 + l16;
            if (p.out_f16) ((_Float16*)p.out)[at] = (_Float16)o; else ((float*)p.out)[at] = o;
          }
        }
      }
      {
        load_k(cn); load_t(cn);
        if (out) { load_q(cn); load_p(cn); }
        // a scale from S itself, as at the start
        float m = 0.f;
#pragma unroll
        for (int x = 0; x < MW; x++)
#pragma unroll
          for (int r = 0; r < 4; r++) m = fmaxf(m, fabsf(S[x][r]));
#pragma unroll
        for (int o = 16; o < 64; o *= 2) m = fmaxf(m, __shfl_xor(m, o));
        lds_barrier();                                             // everyone has read this chunk's norms
        if (lg == 0) norm_s[wave][l16] = m;
        lds_barrier();
        m = fmaxf(fmaxf(norm_s[0][l16], norm_s[1][l16]), fmaxf(norm_s[2][l16], norm_s[3][l16]));
        const int e = scale_exponent(m);
        sigma = pow2(13 - e); sigma_inv = pow2(e - 13);
        lds_barrier();
        publish(sigma, next);
      }
    }
    now = next;
  }
#pragma unroll
  for (int x = 0; x < MW; x++) *(f4*)(sp + 16 * x) = S[x];
}

template <int HK>
static hipError_t launch_chunks(const DeltaParams& p, void* mem, uint32_t ws_chunks, hipStream_t s) {
  const DeltaWs ws = ws_at<HK>(mem, ws_chunks, p.nk, p.nv, nullptr);
  const uint32_t seg = ws_chunks * CHUNK;
  for (uint32_t c0 = 0; c0 < p.n; c0 += seg) {
    DeltaParams r = p;
    r.n = std::min(seg, p.n - c0); r.commit = r.n;
    r.q += (size_t)c0 * p.q_stride; r.k += (size_t)c0 * p.k_stride; r.v += (size_t)c0 * p.v_stride;
    r.g += (size_t)c0 * p.gate_stride; r.beta += (size_t)c0 * p.gate_stride;
    if (r.out) r.out = (unsigned char*)p.out + (size_t)c0 * p.out_stride * (p.out_f16 ? 2 : 4);
    hipLaunchKernelGGL(pa_delta_prep_kernel<HK>, dim3(p.nv, (r.n + CHUNK - 1) / CHUNK), dim3(256), 0, s, r, ws);
    hipLaunchKernelGGL(pa_delta_scan_kernel<HK>, dim3(p.nv * (p.hv / 16)), dim3(256), 0, s, r, ws);
  }
  return hipGetLastError();
}

hipError_t pa_launch_delta_chunks(const DeltaParams& p, void* ws, uint32_t ws_chunks, hipStream_t s) {
  return p.hk == 64 ? launch_chunks<64>(p, ws, ws_chunks, s) : launch_chunks<128>(p, ws, ws_chunks, s);
}
