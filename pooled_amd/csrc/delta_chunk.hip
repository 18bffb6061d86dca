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
// Precision.  Every operand of the f16 matrix instructions is a pair hi + lo of f16 values (22 bits), a product is hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of it), accumulated
// in f32.  Low halves are stored 2048 times, so that a pair has its 22 bits down to 2^-14 and is exact to 2^-36 below; those of K and Q alone are not (2^-3 and 2^-25).  So operands need a
// known size: rows of q are scaled by a power of two to a norm in [0.5, 1), these, keys, P', T and P by UNIT, K' by a power of two for its largest element, and S and X, per value column, by one
// from a bound: the rule over keys no longer than one with 0 <= beta <= 2, g <= 0 is a contraction, so |S_next| <= |S| + sum beta |v| and |X| <= 2 |S| + beta |v|.  What is small beside the
// bound, by its value or by a decay, loses bits (P' and K' hold decays as S and X hold values), so a chunk with a token that takes in less than HELD = 2^-23 of it goes token by token
// (put_exponent): every token's results are as exact as f32 leaves what that token takes in.  A chunk whose inputs leave the domain (longer or tiny keys, other gates, infinities, NaN)
// is marked by the first kernel, or found by the bound, and goes the same way: token by token in the second kernel, in f32, with the same S.  Slower (0.43 us a token of 32 heads, 0.04
// otherwise), but right for every input.
//
// What bounds it: a workgroup's chunk reads K, Q, K' (32 KB each at head_k 128) and P' (16 KB): 112 KB through one CU's 64 bytes a clock, 0.73 us, while its 168
// matrix instructions take 0.3 us of four SIMDs.  The first kernel stores these operands in the order in which lanes load them (a fragment is 1 KB), every
// fragment goes to one wavefront alone, and each is requested a chunk or two ahead: no operand passes through LDS but S and X, which change hands
// between the wavefronts twice a chunk.
#include "blocks_internal.h"
#include "glue_math.h"
#include <algorithm>

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

#define CHUNK 64
// per chunk and v head: beta, beta e^G, output factors of Q S and P' X, 1 / |k| and 1 / |q| (or 1), 64 floats each; then e^G_64, the scale of K', the mark, and 64 times e^g
#define SCAL_FLOATS 512
#define SCAL_DECAY 384
#define SCAL_KSCALE 385
#define SCAL_MARK 386
#define SCAL_STEP 448
// low halves are stored times 2048 (all but those of K and Q, whose rows have one size): a column's values may be far below its bound, and a row of P, T or K' by its decay below another
#define LO_SCALE 2048.f
#define LO_INV (1.f / 2048.f)
// operands of magnitude up to two are stored times 16384, so that the halves of all but tiny ones are normal f16 numbers
#define UNIT 16384.f
#define UNIT_INV (1.f / 16384.f)
// what a token takes in (see put_exponent) may be this part of the bound of its value columns before its chunk goes token by token
#define HELD 0x1p-23f

static __device__ inline void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// sum over lanes {i, i ^ 16, i ^ 32, i ^ 48}
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
struct Pair8 { h8 hi, lo; };
struct Pair4 { h4 hi, lo; };
// two values at a time: the high halves by one packed conversion, the low ones by a multiply-add each that takes the stored high half as it is
template <bool FAR>
static __device__ inline void split2(float x0, float x1, h2& hi, h2& lo) {
  asm("" : "+v"(x0), "+v"(x1));      // f32 numbers as they are: fused into the product that made them, the high half would be rounded once here and twice there
  uint32_t b;
  const h2 h = {(_Float16)x0, (_Float16)x1};
  __builtin_memcpy(&b, &h, 4);
  asm("" : "+v"(b));
  __builtin_memcpy(&hi, &b, 4);
  float f = FAR ? -LO_SCALE : -1.f;
  asm("" : "+s"(f));                 // not a subtraction: the multiply-add reads a half of `hi` in place and writes one of `lo`
  if constexpr (FAR) { x0 *= LO_SCALE; x1 *= LO_SCALE; }
  lo = h2{(_Float16)__builtin_fmaf((float)hi[0], f, x0), (_Float16)__builtin_fmaf((float)hi[1], f, x1)};
}
template <bool FAR = false>
static __device__ inline Pair4 split4(const f4 x) {
  h2 h0, h1, l0, l1;
  split2<FAR>(x[0], x[1], h0, l0); split2<FAR>(x[2], x[3], h1, l1);
  return {h4{h0[0], h0[1], h1[0], h1[1]}, h4{l0[0], l0[1], l1[0], l1[1]}};
}
static __device__ inline h8 join(const h4 a, const h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// buffers: a base in scalar registers, one vector offset for all fragments of a lane, reads past the end are zero and writes dropped
static __device__ inline __amdgpu_buffer_rsrc_t buffer(const void* p, uint32_t bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)bytes, 0x00020000); }
static __device__ inline f4 load_f4(__amdgpu_buffer_rsrc_t b, uint32_t at, uint32_t base) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(b, (int)at, (int)base, 0);
  f4 r; __builtin_memcpy(&r, &v, 16); return r;
}
static __device__ inline h8 load_h8(__amdgpu_buffer_rsrc_t b, uint32_t at, uint32_t base) {
  const auto v = __builtin_amdgcn_raw_buffer_load_b128(b, (int)at, (int)base, 0);
  h8 r; __builtin_memcpy(&r, &v, 16); return r;
}
static __device__ inline float load_f1(__amdgpu_buffer_rsrc_t b, uint32_t at, uint32_t base) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, (int)at, (int)base, 0)); }
static __device__ inline void store_f32(__amdgpu_buffer_rsrc_t b, uint32_t at, float x) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), b, (int)at, 0, 0); }
static __device__ inline void store_f16(__amdgpu_buffer_rsrc_t b, uint32_t at, float x) {
  const _Float16 h = (_Float16)x;
  uint16_t u; __builtin_memcpy(&u, &h, 2);
  __builtin_amdgcn_raw_buffer_store_b16(u, b, (int)at, 0, 0);
}
static __device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }          // -126 <= e <= 127
// largest magnitude `m` -> the exponent e with m 2^(13 - e) in [2^13, 2^14), as far as f32 has the powers
static __device__ inline int exponent(float x);
static __device__ inline int scale_exponent(float m) { return m >= 0x1p-100f ? min(exponent(m), 100) : m > 0.f ? -100 : 13; }
static __device__ inline int exponent(float x) { return (int)((__float_as_uint(x) >> 23) & 255) - 127; }   // of a positive normal number

// of a row of 16 lanes: the lane before by so many (CTRL), or `other` where there is none; the sum
template <int CTRL> static __device__ inline float dpp_or(float other, float v) { return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(other), __float_as_int(v), CTRL, 0xF, 0xF, false)); }
static __device__ inline float row_sum(float v) {
  v += dpp_f32<0xB1>(v); v += dpp_f32<0x4E>(v); v += dpp_f32<0x141>(v);
  return v + dpp_f32<0x140>(v);
}

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

// inclusive sums over the lanes: within rows of 16, then the rows' last lanes into the rows behind
template <int CTRL, int ROWS> static __device__ inline double dpp_or_zero(double x) {
  uint64_t u; __builtin_memcpy(&u, &x, 8);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
  u = (uint64_t)hi << 32 | lo;
  __builtin_memcpy(&x, &u, 8);
  return x;
}
static __device__ inline double prefix_sum(double x) {
  x += dpp_or_zero<0x111, 0xF>(x); x += dpp_or_zero<0x112, 0xF>(x); x += dpp_or_zero<0x114, 0xF>(x); x += dpp_or_zero<0x118, 0xF>(x);      // 1, 2, 4, 8 lanes to the right
  x += dpp_or_zero<0x142, 0xA>(x);                                 // lane 15 to row 1, 47 to row 3
  x += dpp_or_zero<0x143, 0xC>(x);                                 // lane 31 to rows 2 and 3
  return x;
}

// ---- 1: what does not depend on the state ----------------------------------------------------------
// A wavefront has 16 rows of the chunk ("its tile").  Every product below is laid out so that a result, as the matrix instructions leave it (lane: column l16, rows 4 lg + r), is the
// next product's operand as it stands: contractions run over 4 lg + r, not over 8 lg + j.  So A and P stay in registers from K K^T and K Q^T on; LDS holds the keys, which every
// tile meets, and the blocks of T, which every wavefront needs.
#define TS 20      // floats of a row of a 16 x 16 block in LDS
template <int HK> struct PrepLds {
  union {
    _Float16 k[Frags<HK>::KQ];                                     // keys: [plane][tile][k step][lane][8]
    struct {
      float a[4][16 * TS], t[10][16 * TS];                         // diagonal blocks of A; blocks (i, j) of T at i (i + 1) / 2 + j
      h4 tt[10][2][64];                                            // blocks of T as pairs, in the lanes' order
    };
  };
  double G[CHUNK];
  float beta[CHUNK], kfac[CHUNK], row[CHUNK], col[4][48], top[4];
  int marked;
};

template <int HK>
__global__ __launch_bounds__(256, 4)
void pa_delta_prep_kernel(const float* a_k, const float* a_q, const float* a_g, const float* a_beta, uint32_t n, uint32_t k_stride, uint32_t q_stride, uint32_t gate_stride, uint32_t group,
                          DeltaParams p, DeltaWs ws) {
  using F = Frags<HK>;
  constexpr int KS = F::KS, DT = HK / 64;                          // DT: tiles of 16 key dimensions of a wavefront
  __shared__ __attribute__((aligned(16))) PrepLds<HK> L;
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, lg = lane >> 4;
  const uint32_t h = blockIdx.x, chunk = blockIdx.y, kh = h / group, c0 = chunk * CHUNK;
  const uint32_t w = (wave + chunk + h) & 3;                       // its tile: later tiles are more work, and wavefront i of every workgroup runs on the same SIMD
  _Float16* const kq = ws.kq + ((size_t)chunk * p.nk + kh) * 2 * F::KQ;
  float* const scal = ws.scal + ((size_t)chunk * p.nv + h) * SCAL_FLOATS;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  bool bad = false;
  if (tid == 0) L.marked = 0;
  __syncthreads();

  // -- rows: lengths, scaled pairs.  Lane: row l16 of the tile, values 8 lg .. + 7 of every k step
  const bool gated = c0 + lane < n;
  const size_t gc = (size_t)min(c0 + lane, n - 1) * gate_stride + h;
  const float g_in = a_g[gc], b_in = a_beta[gc];                   // of row `lane`; requested in front of the rows, used while those are on their way
  Pair8 kf[KS], qf[KS];
  {
    const uint32_t row = w * 16 + l16;
    const bool valid = c0 + row < n;
    const size_t c = min(c0 + row, n - 1);
    const float* kp = a_k + c * k_stride + (size_t)kh * HK + 8 * lg;
    const float* qp = a_q + c * q_stride + (size_t)kh * HK + 8 * lg;
    f4 k[KS][2], q[KS][2];
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 2; e++) { k[s][e] = *(const f4*)(kp + 32 * s + 4 * e); q[s][e] = *(const f4*)(qp + 32 * s + 4 * e); }
    // gates: sums of g in 64 bits by one wavefront
    if (w == 0) {
      const float g = gated ? g_in : 0.f, b = gated ? b_in : 0.f;
      bad = !(g <= 0.f) || !(b >= 0.f && b <= 2.f);
      L.G[lane] = prefix_sum(g > -1e5f ? (double)g : -1e5);         // exp(-1e5) is 0 as exp(-infinity) is, and differences stay numbers
      L.beta[lane] = b;
    }
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int j = 0; j < 4; j++) { kk = __builtin_fmaf(k[s][e][j], k[s][e][j], kk); qq = __builtin_fmaf(q[s][e][j], q[s][e][j], qq); }
    kk = valid ? rows4_sum(kk) : 0.f;
    qq = valid ? rows4_sum(qq) : 0.f;
    const float kinv = p.l2norm && valid ? 1.0f / sqrtf(kk + p.eps) : 1.f;
    const float qinv = p.l2norm && valid ? 1.0f / sqrtf(qq + p.eps) : 1.f;
    const float kn = kk * kinv * kinv, qn = qq * qinv * qinv;      // squares of the lengths that the rule sees
    // lengths whose pairs keep their bits: keys in [2^-10, 1], or 0; q of any size whose square is a normal number, or 0
    bad = bad || !(kn <= 1.00002f) || (kn < 0x1p-20f && !(kk == 0.f)) || !(qn < 0x1p100f) || (qn < 0x1p-100f && !(qq == 0.f));
    const int qe = qn >= 0x1p-100f && qn < 0x1p100f ? (exponent(qn) >> 1) + 1 : 0;   // |q| 2^-qe in [0.5, 1)
    if (lg == 0) {
      L.kfac[row] = valid ? kinv : 0.f;
      scal[4 * 64 + row] = kinv;
      scal[5 * 64 + row] = qinv;
      scal[3 * 64 + row] = p.scale * pow2(qe);
    }
    const float ks = valid ? kinv * UNIT : 0.f, qs = valid ? qinv * pow2(-qe) * UNIT : 0.f;
    const bool store_k = h == kh * group, store_q = h == kh * group + (group > 1 ? 1 : 0);      // the k head's fragments are stored by one or two v heads of its group
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const Pair4 k0 = split4(k[s][0] * ks), k1 = split4(k[s][1] * ks), q0 = split4(q[s][0] * qs), q1 = split4(q[s][1] * qs);      // (rows behind the last: a finite one times zero, or the chunk is marked)
      kf[s].hi = join(k0.hi, k1.hi); kf[s].lo = join(k0.lo, k1.lo);
      qf[s].hi = join(q0.hi, q1.hi); qf[s].lo = join(q0.lo, q1.lo);
      const uint32_t off = (w * KS + s) * 512 + lane * 8;
      *(h8*)(L.k + off) = kf[s].hi; *(h8*)(L.k + F::KQ / 2 + off) = kf[s].lo;
      if (store_k) { *(h8*)(kq + off) = kf[s].hi; *(h8*)(kq + F::KQ / 2 + off) = kf[s].lo; }
      if (store_q) { *(h8*)(kq + F::KQ + off) = qf[s].hi; *(h8*)(kq + F::KQ + F::KQ / 2 + off) = qf[s].lo; }
    }
  }
  if (__any(bad) && lane == 0) L.marked = 1;                       // (one barrier; the library's reduction takes three)
  __syncthreads();
  const bool mark = L.marked != 0;
  // decays: of a row from the end of the tile before its own (row), from a row to the end of a later tile's predecessor (col), to the chunk's end (kfac)
  if (tid < 64) {
    const double G = L.G[tid];
    const float eG = exp_f64(G);
    scal[tid] = L.beta[tid];
    scal[64 + tid] = L.beta[tid] * eG;
    scal[2 * 64 + tid] = eG;
    scal[SCAL_STEP + tid] = expf(gated ? g_in : 0.f);
    if (tid == 63) { scal[SCAL_DECAY] = eG; scal[SCAL_MARK] = __uint_as_float(mark ? 1u : 0u); }
    L.row[tid] = tid >= 16 ? exp_f64(G - L.G[(tid & 48) - 1]) : eG;
  } else {
    const uint32_t t = tid >> 6, m = tid & 63;
    if (m < 16 * t) L.col[t][m] = exp_f64(L.G[16 * t - 1] - L.G[m]);
    if (t == 1) L.kfac[m] *= exp_f64(L.G[63] - L.G[m]);
  }
  if (mark) return;                                                // the chunk runs token by token
  __syncthreads();

  // -- tiles (m, w): K K^T and K Q^T, keys m in rows, the wavefront's keys and queries i in columns
  f4 A[4];                                                         // A_im of the tile, i = l16
  h4 Ph[4], Pl[4];                                                 // P_im, as pairs
  const uint32_t i = w * 16 + l16;
#pragma unroll
  for (int m = 0; m < 4; m++) {
    A[m] = zero;
    Ph[m] = Pl[m] = h4{0, 0, 0, 0};
    if ((uint32_t)m <= w) {
      f4 a = zero, q = zero;
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const uint32_t off = (m * KS + s) * 512 + lane * 8;
        const h8 mh = *(const h8*)(L.k + off), ml = *(const h8*)(L.k + F::KQ / 2 + off);
        a = __builtin_amdgcn_mfma_f32_16x16x32_f16(mh, kf[s].hi, a, 0, 0, 0);
        q = __builtin_amdgcn_mfma_f32_16x16x32_f16(mh, qf[s].hi, q, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_16x16x32_f16(mh, kf[s].lo, a, 0, 0, 0);
        q = __builtin_amdgcn_mfma_f32_16x16x32_f16(mh, qf[s].lo, q, 0, 0, 0);
        a = __builtin_amdgcn_mfma_f32_16x16x32_f16(ml, kf[s].hi, a, 0, 0, 0);
        q = __builtin_amdgcn_mfma_f32_16x16x32_f16(ml, qf[s].hi, q, 0, 0, 0);
      }
      const uint32_t m0 = m * 16 + 4 * lg;
      f4 d;
      if ((uint32_t)m < w) {
        d = *(const f4*)(&L.col[w][m0]) * L.row[i];
      } else {
        const double Gi = L.G[i];
#pragma unroll
        for (int r = 0; r < 4; r++) d[r] = m0 + r <= i ? exp_f64(Gi - L.G[m0 + r]) : 0.f;
      }
      d *= UNIT_INV * UNIT_INV;
      const float b = L.beta[i];
      f4 pm;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        A[m][r] = m0 + r < i ? b * d[r] * a[r] : 0.f;
        pm[r] = d[r] * UNIT * q[r];
      }
      const Pair4 s = split4<true>(pm);
      Ph[m] = s.hi; Pl[m] = s.lo;
    }
  }
  __syncthreads();                                                 // the keys have been read: their LDS is A and T's now
  // -- K~ = e^(G_64 - G_i) k_i, right operand: column d, contraction over the chunk's rows.  Requested here, used behind T
  float kt[DT][2][8];
#pragma unroll
  for (int x = 0; x < DT; x++)
#pragma unroll
    for (int ks = 0; ks < 2; ks++)
#pragma unroll
      for (int e = 0; e < 8; e++) kt[x][ks][e] = a_k[(size_t)min(c0 + 32 * ks + 16 * (e >> 2) + 4 * lg + (e & 3), n - 1) * k_stride + (size_t)kh * HK + (w * DT + x) * 16 + l16];

  // -- T = (1 + A)^-1.  The diagonal block by substitution, a lane a column (the four lane groups do the same)
  auto put_block = [&](uint32_t bi, uint32_t bj, const f4 v) {
    const uint32_t b = bi * (bi + 1) / 2 + bj;
#pragma unroll
    for (int r = 0; r < 4; r++) L.t[b][(4 * lg + r) * TS + l16] = v[r];
    const Pair4 s = split4<true>(v * UNIT);
    L.tt[b][0][lane] = s.hi; L.tt[b][1][lane] = s.lo;
  };
  {
    float* const a = L.a[w];
    f4 mine = zero;
#pragma unroll
    for (int m = 0; m < 4; m++) if ((uint32_t)m == w) mine = A[m];
    *(f4*)(a + l16 * TS + 4 * lg) = mine;
    wave_lds_fence();
    float t[16];
#pragma unroll
    for (int r = 0; r < 16; r++) {
      float s = l16 == (uint32_t)r ? 1.f : 0.f;
#pragma unroll
      for (int m4 = 0; m4 < r; m4 += 4) {
        const f4 x = *(const f4*)(a + r * TS + m4);
#pragma unroll
        for (int m = 0; m < 4; m++) if (m4 + m < r) s = __builtin_fmaf(-x[m], t[m4 + m], s);
      }
      t[r] = s;
    }
    f4 v;
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = lg < 2 ? (lg == 0 ? t[r] : t[4 + r]) : (lg == 2 ? t[8 + r] : t[12 + r]);
    put_block(w, w, v);
  }
  __syncthreads();
  // block rows from the top: T_ij = -T_ii sum_k A_ik T_kj, products of 16 x 16 in f32
  auto left = [&](uint32_t b) { return *(const f4*)(&L.t[b * (b + 1) / 2 + b][l16 * TS + 4 * lg]); };                 // T_bb
  auto right = [&](uint32_t bi, uint32_t bj) {
    const float* x = &L.t[bi * (bi + 1) / 2 + bj][4 * lg * TS + l16];
    return f4{x[0], x[TS], x[2 * TS], x[3 * TS]};
  };
  auto mul = [&](const f4 a, const f4 b, f4 c) {
#pragma unroll
    for (int r = 0; r < 4; r++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
    return c;
  };
  f4 m0 = zero, m1 = zero;
  if (w == 1) put_block(1, 0, -mul(left(1), mul(A[0], right(0, 0), zero), zero));
  if (w == 2) {
    m0 = mul(A[0], right(0, 0), zero);
    put_block(2, 1, -mul(left(2), mul(A[1], right(1, 1), zero), zero));
  }
  if (w == 3) {
    m0 = mul(A[0], right(0, 0), zero);
    m1 = mul(A[1], right(1, 1), zero);
    put_block(3, 2, -mul(left(3), mul(A[2], right(2, 2), zero), zero));
  }
  __syncthreads();
  if (w == 2) put_block(2, 0, -mul(left(2), mul(A[1], right(1, 0), m0), zero));
  if (w == 3) {
    m0 = mul(A[1], right(1, 0), m0);
    put_block(3, 1, -mul(left(3), mul(A[2], right(2, 1), m1), zero));
  }
  __syncthreads();
  if (w == 3) put_block(3, 0, -mul(left(3), mul(A[2], right(2, 0), m0), zero));
  // (K~ into pairs while the last block is made)
  Pair8 kb[DT][2];
#pragma unroll
  for (int ks = 0; ks < 2; ks++) {
    const f4 f0 = *(const f4*)(&L.kfac[32 * ks + 4 * lg]), f1 = *(const f4*)(&L.kfac[32 * ks + 16 + 4 * lg]);
#pragma unroll
    for (int x = 0; x < DT; x++) {
      const float* k = kt[x][ks];
      const Pair4 a = split4<true>(f4{k[0], k[1], k[2], k[3]} * (f0 * UNIT)), b = split4<true>(f4{k[4], k[5], k[6], k[7]} * (f1 * UNIT));
      kb[x][ks].hi = join(a.hi, b.hi); kb[x][ks].lo = join(a.lo, b.lo);
    }
  }
  __syncthreads();

  // -- K' [j][d] = sum_i T_ij K~ [i][d] and P'^T [j][i] = sum_m T_mj P_im: T^T the left operand of both
  f4 kr[DT][4], pr[4];
  const h4 none = {0, 0, 0, 0};
  auto t_block = [&](int bi, int bj, int plane) { return bi >= bj ? L.tt[bi * (bi + 1) / 2 + bj][plane][lane] : none; };
#pragma unroll
  for (int jt = 0; jt < 4; jt++) {
    f4 pf = zero, kl[DT];                                          // products with a low half, 2048 times
    pr[jt] = zero;
#pragma unroll
    for (int x = 0; x < DT; x++) kr[x][jt] = kl[x] = zero;
#pragma unroll
    for (int ks = jt / 2; ks < 2; ks++) {
      const h8 th = join(t_block(2 * ks, jt, 0), t_block(2 * ks + 1, jt, 0)), tl = join(t_block(2 * ks, jt, 1), t_block(2 * ks + 1, jt, 1));
      const h8 ph = join(Ph[2 * ks], Ph[2 * ks + 1]), pl = join(Pl[2 * ks], Pl[2 * ks + 1]);
#pragma unroll
      for (int x = 0; x < DT; x++) kr[x][jt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th, kb[x][ks].hi, kr[x][jt], 0, 0, 0);
      pr[jt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th, ph, pr[jt], 0, 0, 0);
#pragma unroll
      for (int x = 0; x < DT; x++) kl[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(th, kb[x][ks].lo, kl[x], 0, 0, 0);
      pf = __builtin_amdgcn_mfma_f32_16x16x32_f16(th, pl, pf, 0, 0, 0);
#pragma unroll
      for (int x = 0; x < DT; x++) kl[x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(tl, kb[x][ks].hi, kl[x], 0, 0, 0);
      pf = __builtin_amdgcn_mfma_f32_16x16x32_f16(tl, ph, pf, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; r++) pr[jt][r] = __builtin_fmaf(pf[r], LO_INV, pr[jt][r]);
#pragma unroll
    for (int x = 0; x < DT; x++)
#pragma unroll
      for (int r = 0; r < 4; r++) kr[x][jt][r] = __builtin_fmaf(kl[x][r], LO_INV, kr[x][jt][r]);
  }
  // -- P' and K'^T in the order of the second kernel's loads, K' scaled by the power of two of its largest element
  float top = 0.f;
#pragma unroll
  for (int x = 0; x < DT; x++)
#pragma unroll
    for (int jt = 0; jt < 4; jt++) top = fmaxf(fmaxf(top, fmaxf(fabsf(kr[x][jt][0]), fabsf(kr[x][jt][1]))), fmaxf(fabsf(kr[x][jt][2]), fabsf(kr[x][jt][3])));
  top = fmaxf(top, dpp_f32<0xB1>(top)); top = fmaxf(top, dpp_f32<0x4E>(top)); top = fmaxf(top, dpp_f32<0x141>(top)); top = fmaxf(top, dpp_f32<0x140>(top));
  top = fmaxf(fmaxf(readlane_f32(top, 0), readlane_f32(top, 16)), fmaxf(readlane_f32(top, 32), readlane_f32(top, 48)));
  if (lane == 0) L.top[w] = top;
  _Float16* const pp = ws.pp + ((size_t)chunk * p.nv + h) * F::P;
  auto frag_at = [&](uint32_t tile, int jt) { return (tile * 2 + (jt >> 1)) * 512 + (l16 + 16 * (2 * (jt & 1) + (lg >> 1))) * 8 + 4 * (lg & 1); };
#pragma unroll
  for (int jt = 0; jt < 4; jt++) {
    const Pair4 s = split4<true>(pr[jt] * UNIT_INV);
    *(h4*)(pp + frag_at(w, jt)) = s.hi; *(h4*)(pp + F::P / 2 + frag_at(w, jt)) = s.lo;
  }
  __syncthreads();
  top = fmaxf(fmaxf(L.top[0], L.top[1]), fmaxf(L.top[2], L.top[3])) * (UNIT_INV * UNIT_INV);
  const int ke = top >= 0x1p-100f ? exponent(top) : 13;
  const float ksc = pow2(13 - ke) * (UNIT_INV * UNIT_INV);
  if (tid == 0) scal[SCAL_KSCALE] = pow2(ke - 13);
  _Float16* const kto = ws.kt + ((size_t)chunk * p.nv + h) * F::KT;
#pragma unroll
  for (int x = 0; x < DT; x++)
#pragma unroll
    for (int jt = 0; jt < 4; jt++) {
      const Pair4 s = split4<true>(kr[x][jt] * ksc);
      *(h4*)(kto + frag_at(w * DT + x, jt)) = s.hi; *(h4*)(kto + F::KT / 2 + frag_at(w * DT + x, jt)) = s.lo;
    }
}

// ---- 2: from chunk to chunk -------------------------------------------------------------------------
// A workgroup has the state of NT x 16 value columns of a head and twelve wavefronts of three roles.  In a chunk's first phase the four KEYS multiply K by S and make X; in the second the
// four of STATE multiply K'^T by X and move the state on; each requests its operands while the other works, one to two chunks ahead.  The four QUERIES, which nothing waits for, have the
// other halves of the phases: Q S while STATE works, P' X of the chunk before while KEYS do, so S and X are there twice.  Two barriers a chunk: S is there | X is there.  Every role has
// a loop of its own, unrolled by two: no register that a load is still filling is ever copied, and no wait is shared.  (NT = 2 has no registers for second sets of operands.)
// What bounds it: the operands, 112 KB a chunk for each workgroup whatever its columns, at 64 bytes a cycle of a CU 1750 of about 3000 cycles, and a chunk's two barriers with
// their exchanges.  2048 columns of 32 heads: 64 us with the operands from the last-level cache, of 48 heads (NT = 2) 87; before the check of a chunk's range
// 63 and 84, and with 32 heads 53 from L2 and 42 alone on the chip.
//
// Scales: E_c is the exponent, per value column, that X of chunk c and the state behind it are scaled by.  It comes from the sums N_c of |S| in front of the chunk before and the
// sums V of beta |v|: |S| in front of chunk c <= N_(c-1) + V_(c-1), so that KEYS find it a chunk ahead (sums of magnitudes are no smaller than norms, and they neither over- nor
// underflow before their terms do).  NO_SCALE in its place sends the chunk the slow way.
enum { KEYS, STATE, QUERIES };
#define NO_SCALE 10000

template <int HK, int NT> struct ScanLds {
  static constexpr int KS = HK / 32, MT = HK / 64, COLS = 16 * NT;
  _Float16 S[2][NT][2][KS * 512], X[2][NT][2][2 * 512];            // pairs, as right operands, of even and odd chunks
  f4 bv[2][NT][4 * 64], cv[2][16];                                 // beta v, beta e^G of a chunk and the next, in the order of KEYS' lanes
  f4 norm[2][COLS], val[2][COLS];                                  // N and V, by wavefront
  float low[2][COLS][16];                                          // the lowest beta |v| of four tokens
  int exps[2][COLS];
  struct {                                                         // a chunk that goes token by token: its rows, scaled, and the wavefronts' partial sums
    float k[CHUNK][HK], q[CHUNK][HK], v[CHUNK][COLS], decay[CHUNK], beta[CHUNK], part[2][2][4][COLS];
  } slow;
};
static __device__ inline float sum4(const f4 x) { return (x[0] + x[1]) + (x[2] + x[3]); }
static __device__ inline float sum_abs4(const f4 x) { return (fabsf(x[0]) + fabsf(x[1])) + (fabsf(x[2]) + fabsf(x[3])); }

template <int HK, int NT, int ROLE>
static __device__ __attribute__((always_inline)) void scan_role(const DeltaParams& p, const DeltaWs& ws, ScanLds<HK, NT>& L, const uint32_t w) {
  using F = Frags<HK>;
  using LD = ScanLds<HK, NT>;
  constexpr int KS = LD::KS, MT = LD::MT, COLS = LD::COLS;
  const uint32_t tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
  const uint32_t h = blockIdx.x % p.nv, v0 = blockIdx.x / p.nv * COLS, kh = h / p.group;
  const uint32_t chunks = (p.n + CHUNK - 1) / CHUNK, last = chunks - 1;
  const bool out = p.out != nullptr;
  const uint32_t ot = p.out_f16 ? 2 : 4;
  const float* const scal = ws.scal + (size_t)h * SCAL_FLOATS;
  const size_t scal_step = (size_t)p.nv * SCAL_FLOATS;
  auto rows_of = [&](uint32_t c) { return min((uint32_t)CHUNK, p.n - c * CHUNK); };

  // ---- state rows 16 (w MT + m) + 4 lg + r of value columns v0 + 16 t + l16
  f4 S[NT][MT];
  float* const sp = p.state + ((size_t)h * p.hv + v0 + l16) * HK + w * MT * 16 + 4 * lg;
  if constexpr (ROLE == STATE) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int m = 0; m < MT; m++) S[t][m] = *(const f4*)(sp + t * 16 * HK + m * 16);
  }

  // ---- requests.  Past the last chunk the last one's is made again instead of branching round the loads: a short conditional block between a matrix
  // instruction and the first use of its result makes this compiler (22.0.0git, ROCm 7.2.0) leave out the wait states on the path round the block, and the use then reads the old
  // registers (seen as states 1e-4 off after a last chunk; tests/test_wait_states.py looks for it in what was built).  No dword is loaded that is not used: its register would be taken for something else, and that would wait for the load.
  // Rows behind the last column read as zero and are not written: the buffers end with the last column.
  struct KF { h8 x[KS][2]; };
  struct GF { h8 x[MT][2][2]; };
  struct PF { h8 x[2][2]; };
  struct StateRows { f4 a, b, v[NT]; float decay, kscale; };       // beta, beta e^G, values
  struct QueryRows { f4 a, b; };                                   // e^G, factor of the output
  const uint32_t at = lane * 16;
  auto load_k = [&](KF& d, uint32_t c) __attribute__((always_inline)) {
    const auto b = buffer(ws.kq + (((size_t)min(c, last) * p.nk + kh) * 2 + (ROLE == QUERIES ? 1 : 0)) * F::KQ, F::KQ * 2);
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
      for (int e = 0; e < 2; e++) d.x[s][e] = load_h8(b, at + s * 1024, w * KS * 1024 + e * F::KQ);
  };
  auto load_g = [&](GF& d, uint32_t c) __attribute__((always_inline)) {
    const auto b = buffer(ws.kt + ((size_t)min(c, last) * p.nv + h) * F::KT, F::KT * 2);
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int s = 0; s < 2; s++)
#pragma unroll
        for (int e = 0; e < 2; e++) d.x[m][s][e] = load_h8(b, at + s * 1024, (w * MT + m) * 2048 + e * F::KT);
  };
  auto load_p = [&](PF& d, uint32_t c) __attribute__((always_inline)) {
    const auto b = buffer(ws.pp + ((size_t)min(c, last) * p.nv + h) * F::P, F::P * 2);
#pragma unroll
    for (int s = 0; s < 2; s++)
#pragma unroll
      for (int e = 0; e < 2; e++) d.x[s][e] = load_h8(b, at + s * 1024, w * 2048 + e * F::P);
  };
  uint32_t row_at[4];                                              // STATE: of the values, QUERIES: of the output
  if constexpr (ROLE != KEYS) {
#pragma unroll
    for (int r = 0; r < 4; r++) row_at[r] = (w * 16 + 4 * lg + r) * (ROLE == STATE ? p.v_stride * 4 : p.out_stride * ot) + l16 * (ROLE == STATE ? 4 : ot);
  }
  const uint32_t gate_at = (w * 16 + 4 * lg) * 4;
  auto load_rows = [&](StateRows& d, uint32_t c) __attribute__((always_inline)) {
    c = min(c, last);
    const auto b = buffer(scal + c * scal_step, SCAL_FLOATS * 4);
    const auto x = buffer(p.v + (size_t)c * CHUNK * p.v_stride + (size_t)h * p.hv + v0, ((rows_of(c) - 1) * p.v_stride + COLS) * 4);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) d.v[t][r] = load_f1(x, row_at[r] + t * 64, 0);
    d.a = load_f4(b, gate_at, 0); d.b = load_f4(b, gate_at, 256);
    d.decay = load_f1(b, 0, SCAL_DECAY * 4); d.kscale = load_f1(b, 0, SCAL_KSCALE * 4);
  };
  auto load_query_rows = [&](QueryRows& d, uint32_t c) __attribute__((always_inline)) {
    const auto b = buffer(scal + min(c, last) * scal_step, SCAL_FLOATS * 4);
    d.a = load_f4(b, gate_at, 512); d.b = load_f4(b, gate_at, 768);
  };
  auto load_steps = [&](uint32_t c) __attribute__((always_inline)) { return load_f4(buffer(scal + min(c, last) * scal_step, SCAL_FLOATS * 4), l16 * 16, SCAL_STEP * 4); };
  auto load_mark = [&](uint32_t c) __attribute__((always_inline)) { return load_f1(buffer(scal + min(c, last) * scal_step, SCAL_FLOATS * 4), 0, SCAL_MARK * 4); };

  // ---- what STATE and KEYS leave for the others
  auto put_norm = [&](uint32_t c) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float x = 0.f;
#pragma unroll
      for (int m = 0; m < MT; m++) x += sum_abs4(S[t][m]);
      x = rows4_sum(x);
      if (lg == 0) L.norm[c & 1][t * 16 + l16][w] = x;
    }
  };
  auto put_state = [&](uint32_t c, const float (&to)[NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const Pair4 s = split4<true>(S[t][m] * to[t]);
        const uint32_t d0 = (w * MT + m) * 16 + 4 * lg, off = (d0 >> 5) * 512 + (l16 + 16 * ((d0 & 31) >> 3)) * 8 + (d0 & 7);
        *(h4*)(&L.S[c & 1][t][0][off]) = s.hi; *(h4*)(&L.S[c & 1][t][1][off]) = s.lo;
      }
  };
  auto put_rows = [&](const StateRows& d, uint32_t c) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const f4 x = d.a * d.v[t];
      L.bv[c & 1][t][w * 64 + lane] = x;
      const float y = rows4_sum(sum_abs4(x));
      if (lg == 0) L.val[c & 1][t * 16 + l16][w] = y;
      f4 z = x;
      if (c >= last) {                                             // rows behind the last column do not count
#pragma unroll
        for (int r = 0; r < 4; r++) z[r] = w * 16 + 4 * lg + r < rows_of(last) ? z[r] : INFINITY;
      }
      L.low[c & 1][t * 16 + l16][w * 4 + lg] = fminf(fminf(fabsf(z[0]), fabsf(z[1])), fminf(fabsf(z[2]), fabsf(z[3])));
    }
    if (l16 == 0) L.cv[c & 1][w * 4 + lg] = d.b;
  };
  // E_c, by the first of KEYS; fresh: the sums of |S| in front of chunk c itself are there.
  // M_i = e^g_i M_(i-1) + beta_i |v_i|, from |S| on, is what token i takes in of a value column.  The pairs hold every term of a column to 22 bits or to a fixed part of its bound, whichever
  // is more, so a chunk with a token whose M, over the columns, is less than HELD of their bounds goes the slow way, and one that leaves such a column.  Nearly always beta_i |v_i| of any two
  // columns is enough by itself, and for every column that of the last token (looked at four tokens at a time); only where that is not so, M is summed up (in every chunk: 22.0 us instead of 19.2 for the walk over 1001 columns of 8 heads of 64 x 96; without any such check 16.8).
  float taken[NT];                                                 // M behind the chunk before, of column l16, where it was summed up
  bool summed = false;
  auto put_exponent = [&](uint32_t c, bool fresh, float mark) __attribute__((always_inline)) {
    if (w != 0 || c > last) return;
    float bound[NT], before[NT];
    bool enough = true, fine = true;
    const uint32_t end = (rows_of(c) - 1) / 4;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const uint32_t j = t * 16 + l16;
      before[t] = fresh ? sum4(L.norm[c & 1][j]) : 1.01f * (sum4(L.norm[(c - 1) & 1][j]) + sum4(L.val[(c - 1) & 1][j]));
      bound[t] = 1.02f * __builtin_fmaf(2.1f, before[t], sum4(L.val[c & 1][j]));
      f4 low = *(const f4*)(&L.low[c & 1][j][4 * lg]);
      enough = enough && L.low[c & 1][j][end] >= HELD * bound[t];
#pragma unroll
      for (int r = 0; r < 4; r++) low[r] += dpp_f32<0xB1>(low[r]);  // no more than any of the four tokens' sum over the column and its neighbour (l16 ^ 1)
      enough = enough && fminf(fminf(low[0], low[1]), fminf(low[2], low[3])) >= HELD * (bound[t] + dpp_f32<0xB1>(bound[t]));
    }
    if (!__all(enough)) {                                          // a lane: four tokens (4 l16 ..) of the columns lg, 4 + lg, 8 + lg, 12 + lg of each tile
      const f4 step = load_steps(c);
      float d[5], all[4] = {0.f, 0.f, 0.f, 0.f}, floors = 0.f;     // decays over the lane's tokens, and those of 1, 3, 7, 15 lanes before it too
      d[0] = (step[0] * step[1]) * (step[2] * step[3]);
      d[1] = d[0] * dpp_or<0x111>(1.f, d[0]); d[2] = d[1] * dpp_or<0x112>(1.f, d[1]); d[3] = d[2] * dpp_or<0x114>(1.f, d[2]); d[4] = d[3] * dpp_or<0x118>(1.f, d[3]);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float next = 0.f, front = taken[t];
        if (!summed) front = fabsf(L.bv[(c - 1) & 1][t][15 * 16 + l16][3]);                          // at least the last token of the chunk before
        if (fresh) front = before[t] * (HK == 64 ? 0.125f : 0.0884f);  // a 2-norm is at least the sum over the root of its length
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
          const int col = 4 * i + lg;
          const f4 v = L.bv[c & 1][t][l16 * 16 + col];
          float m = fabsf(v[0]);
#pragma unroll
          for (int r = 1; r < 4; r++) m = __builtin_fmaf(m, step[r], fabsf(v[r]));
          m = __builtin_fmaf(dpp_or<0x111>(0.f, m), d[0], m); m = __builtin_fmaf(dpp_or<0x112>(0.f, m), d[1], m);
          m = __builtin_fmaf(dpp_or<0x114>(0.f, m), d[2], m); m = __builtin_fmaf(dpp_or<0x118>(0.f, m), d[3], m);
          m = __builtin_fmaf(dpp_or<0x111>(1.f, d[4]), __shfl(front, col), dpp_or<0x111>(0.f, m));
#pragma unroll
          for (int r = 0; r < 4; r++) { m = __builtin_fmaf(m, step[r], fabsf(v[r])); all[r] += m; }
          const float x = __shfl(m, 16 * (l16 & 3) + 15);          // of column 4 i + l16 % 4
          if ((l16 >> 2) == (uint32_t)i) next = x;
        }
        const float floor = HELD * bound[t];
        taken[t] = next;
        floors += floor;
        fine = fine && (next >= floor || next == 0.f);
      }
      floors = row_sum(floors);
#pragma unroll
      for (int r = 0; r < 4; r++) { const float m = rows4_sum(all[r]); fine = fine && (m >= floors || m == 0.f); }
      fine = __all(fine);
      summed = true;
    } else {
      summed = false;
    }
    fine = fine && __float_as_uint(mark) == 0;
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const bool in = fine && (bound[t] == 0.f || (bound[t] >= 0x1p-90f && bound[t] < 0x1p90f));
      if (lg == 0) L.exps[c & 1][t * 16 + l16] = in ? scale_exponent(bound[t]) : NO_SCALE;
    }
  };
  auto own_exponents = [&](uint32_t c, int (&e)[NT]) __attribute__((always_inline)) {               // of S in front of chunk c, from itself
    if constexpr (ROLE == STATE) put_norm(c);
    lds_barrier();
#pragma unroll
    for (int t = 0; t < NT; t++) e[t] = scale_exponent(sum4(L.norm[c & 1][t * 16 + l16]));
  };

  // ---- in front of the first chunk
  KF k0, k1;
  GF g0, g1;
  PF p0, p1;
  StateRows rows1;                                                 // of the coming chunk
  QueryRows q0, q1;
  float m0 = 0.f, m1 = 0.f;
  if constexpr (ROLE == KEYS) { m0 = load_mark(0); m1 = load_mark(1); load_k(k0, 0); load_k(k1, 1); }
  if constexpr (ROLE == STATE) { load_rows(rows1, 0); load_g(g0, 0); put_rows(rows1, 0); }
  if constexpr (ROLE == QUERIES) { load_query_rows(q0, 0); load_query_rows(q1, 1); load_k(k0, 0); load_p(NT > 1 ? p0 : p1, 0); }
  float decay = 0.f, kscale = 0.f, next_decay = 0.f, next_kscale = 0.f;
  if constexpr (ROLE == STATE) { decay = rows1.decay; kscale = rows1.kscale; load_rows(rows1, 1); }
  float sigma_inv[NT];
  {
    int e[NT];
    float to[NT];
    own_exponents(0, e);
#pragma unroll
    for (int t = 0; t < NT; t++) { sigma_inv[t] = pow2(e[t] - 13); to[t] = pow2(13 - e[t]); }
    if constexpr (ROLE == STATE) put_state(0, to);
    if constexpr (ROLE == KEYS) put_exponent(0, true, m0);
  }

  // product with the S of chunk c: keys or queries
  auto times_state = [&](uint32_t c, uint32_t t, const KF& kf, float from) __attribute__((always_inline)) {
    f4 r0 = {0.f, 0.f, 0.f, 0.f}, r1 = r0, r2 = r0, r;              // hi hi | hi lo, 2048 times | lo hi
#pragma unroll
    for (int s = 0; s < KS; s++) {
      const h8 sh = *(const h8*)(&L.S[c & 1][t][0][s * 512 + lane * 8]), sl = *(const h8*)(&L.S[c & 1][t][1][s * 512 + lane * 8]);
      r0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf.x[s][0], sh, r0, 0, 0, 0);
      r1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf.x[s][0], sl, r1, 0, 0, 0);
      r2 = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf.x[s][1], sh, r2, 0, 0, 0);
    }
    const float back = from * UNIT_INV;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_fmaf(r1[i], LO_INV, r0[i] + r2[i]) * back;
    return r;
  };
  // product of a pair of left operands with the X of chunk c
  auto times_x = [&](uint32_t c, uint32_t t, const h8 (&x)[2][2]) __attribute__((always_inline)) {
    f4 n0 = {0.f, 0.f, 0.f, 0.f}, n1 = n0, n;                       // hi hi | hi lo + lo hi, 2048 times
#pragma unroll
    for (int s = 0; s < 2; s++) {
      const h8 xh = *(const h8*)(&L.X[c & 1][t][0][s * 512 + lane * 8]), xl = *(const h8*)(&L.X[c & 1][t][1][s * 512 + lane * 8]);
      n0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[s][0], xh, n0, 0, 0, 0);
      n1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[s][0], xl, n1, 0, 0, 0);
      n1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[s][1], xh, n1, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) n[i] = __builtin_fmaf(n1[i], LO_INV, n0[i]);
    return n;
  };
  // QUERIES: the start state's part of a chunk's output, all factors in, the factor of the other part, and the rows to store; P' X of that chunk comes a phase later
  f4 held[NT], fx[NT];
  uint32_t held_rows = 0;
#pragma unroll
  for (int t = 0; t < NT; t++) held[t] = fx[t] = f4{0.f, 0.f, 0.f, 0.f};
  auto put_out = [&](uint32_t c, const PF& pf) __attribute__((always_inline)) {
    const auto b = buffer((unsigned char*)p.out + ((size_t)c * CHUNK * p.out_stride + (size_t)h * p.hv + v0) * ot, out && held_rows ? ((held_rows - 1) * p.out_stride + COLS) * ot : 0);
#pragma unroll
    for (int t = 0; t < NT; t++) {
      const f4 n = times_x(c, t, pf.x);
      f4 o;
#pragma unroll
      for (int r = 0; r < 4; r++) o[r] = __builtin_fmaf(fx[t][r], n[r], held[t][r]);
      if (p.out_f16) {
#pragma unroll
        for (int r = 0; r < 4; r++) store_f16(b, row_at[r] + t * 32, o[r]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++) store_f32(b, row_at[r] + t * 64, o[r]);
      }
    }
  };

  auto chunk = [&](const uint32_t c, KF& kf, GF& gf, GF& gf_next, KF& kf_next, PF& pf, PF& pf_next, QueryRows& qr, float& mark, const float mark_next) __attribute__((always_inline)) {
    lds_barrier();
    int e[NT];
    bool none = false;
#pragma unroll
    for (int t = 0; t < NT; t++) { e[t] = L.exps[c & 1][t * 16 + l16]; none = none || e[t] == NO_SCALE; }
    const bool slow = __any(none);
    uint32_t rows = rows_of(c);
    if (slow) {
      // token by token, in f32: dot products over the key dimensions of the four wavefronts of STATE, one exchange and one barrier each.  What the matrix instructions below make of this
      // chunk is dropped.
      const float* const sg = scal + c * scal_step;
      const size_t first = (size_t)c * CHUNK;
      auto& Z = L.slow;
      if constexpr (ROLE == KEYS) {                                // (the others have no registers to spare)
#pragma unroll 1
        for (uint32_t x = tid; x < rows * (HK / 4); x += 256) {
          const uint32_t i = x / (HK / 4), d = x % (HK / 4) * 4;
          *(f4*)(&Z.k[i][d]) = *(const f4*)(p.k + (first + i) * p.k_stride + kh * HK + d) * sg[4 * 64 + i];
          if (out) *(f4*)(&Z.q[i][d]) = *(const f4*)(p.q + (first + i) * p.q_stride + kh * HK + d) * sg[5 * 64 + i];
        }
#pragma unroll 1
        for (uint32_t x = tid; x < rows * COLS; x += 256) Z.v[x / COLS][x % COLS] = p.v[(first + x / COLS) * p.v_stride + (size_t)h * p.hv + v0 + x % COLS];
        if (tid < rows) { Z.decay[tid] = expf(p.g[(first + tid) * p.gate_stride + h]); Z.beta[tid] = p.beta[(first + tid) * p.gate_stride + h]; }
      }
      lds_barrier();
      auto put_token = [&](uint32_t i) __attribute__((always_inline)) {
        if (out && w == 0 && lg == 0) {
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const auto& x = Z.part[1][i & 1];
            const uint32_t j = t * 16 + l16;
            const float o = p.scale * ((x[0][j] + x[1][j]) + (x[2][j] + x[3][j]));
            const size_t to = (first + i) * p.out_stride + (size_t)h * p.hv + v0 + j;
            if (p.out_f16) ((_Float16*)p.out)[to] = (_Float16)o; else ((float*)p.out)[to] = o;
          }
        }
      };
#pragma unroll 1
      for (uint32_t i = 0; i < rows; i++) {
        f4 k[MT];
        if constexpr (ROLE == STATE) {
          const float dec = Z.decay[i];
#pragma unroll
          for (int m = 0; m < MT; m++) k[m] = *(const f4*)(&Z.k[i][(w * MT + m) * 16 + 4 * lg]);
#pragma unroll
          for (int t = 0; t < NT; t++) {
            float a = 0.f;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
              for (int r = 0; r < 4; r++) { S[t][m][r] *= dec; a = __builtin_fmaf(S[t][m][r], k[m][r], a); }
            a = rows4_sum(a);
            if (lg == 0) Z.part[0][i & 1][w][t * 16 + l16] = a;
          }
        }
        lds_barrier();
        if constexpr (ROLE == STATE) {
          const float b = Z.beta[i];
#pragma unroll
          for (int t = 0; t < NT; t++) {
            const auto& x = Z.part[0][i & 1];
            const uint32_t j = t * 16 + l16;
            const float u = b * (Z.v[i][j] - ((x[0][j] + x[1][j]) + (x[2][j] + x[3][j])));
            float o = 0.f;
#pragma unroll
            for (int m = 0; m < MT; m++) {
              const f4 q = *(const f4*)(&Z.q[i][(w * MT + m) * 16 + 4 * lg]);
#pragma unroll
              for (int r = 0; r < 4; r++) { S[t][m][r] = __builtin_fmaf(u, k[m][r], S[t][m][r]); o = __builtin_fmaf(S[t][m][r], q[r], o); }
            }
            o = rows4_sum(o);
            if (lg == 0) Z.part[1][i & 1][w][j] = o;
          }
        }
        if constexpr (ROLE == KEYS) { if (i) put_token(i - 1); }
      }
      lds_barrier();
      if constexpr (ROLE == KEYS) put_token(rows - 1);
      rows = 0;
      own_exponents(c + 1, e);
    }
    float to[NT], to_inv[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) { to[t] = pow2(13 - e[t]); to_inv[t] = pow2(e[t] - 13); }
    if constexpr (ROLE == KEYS) {
      const f4 cv = L.cv[c & 1][w * 4 + lg];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const f4 r = times_state(c, t, kf, sigma_inv[t]), bv = L.bv[c & 1][t][w * 64 + lane];
        f4 x;                                                      // X = beta v - beta e^G K S
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __builtin_fmaf(-cv[i], r[i], bv[i]);
        const Pair4 s = split4<true>(x * to[t]);
        const uint32_t i0 = w * 16 + 4 * lg, off = (i0 >> 5) * 512 + (l16 + 16 * ((i0 & 31) >> 3)) * 8 + (i0 & 7);
        *(h4*)(&L.X[c & 1][t][0][off]) = s.hi; *(h4*)(&L.X[c & 1][t][1][off]) = s.lo;
      }
    } else if constexpr (ROLE == QUERIES) {
      if constexpr (NT == 1) load_p(pf_next, c);
      put_out(max(c, 1u) - 1, pf);                                 // (no rows yet in front of the first chunk)
      if constexpr (NT > 1) load_p(pf, c);
    } else {
      if constexpr (NT == 1) load_g(gf_next, c + 1);
      put_rows(rows1, c + 1);
      next_decay = rows1.decay; next_kscale = rows1.kscale;
      load_rows(rows1, c + 2);
    }
    lds_barrier();
    if constexpr (ROLE == KEYS) {
      load_k(kf, c + 2);
      mark = load_mark(c + 2);
      put_exponent(c + 1, slow, mark_next);
    } else if constexpr (ROLE == STATE) {
      f4 n[NT][MT];
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int m = 0; m < MT; m++) n[t][m] = times_x(c, t, gf.x[m]);
      if constexpr (NT > 1) load_g(gf, c + 1);                     // no room for two chunks' operands
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const float fs = to_inv[t] * kscale;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float x = __builtin_fmaf(S[t][m][i], decay, n[t][m][i] * fs);
            S[t][m][i] = slow ? S[t][m][i] : x;
          }
      }
      put_state(c + 1, to);
      put_norm(c + 1);
      decay = next_decay; kscale = next_kscale;
    } else {
      if constexpr (NT == 1) load_k(kf_next, c + 1);
#pragma unroll
      for (int t = 0; t < NT; t++) {
        held[t] = qr.b * (qr.a * times_state(c, t, kf, sigma_inv[t]));
        fx[t] = qr.b * (to_inv[t] * UNIT_INV);
      }
      held_rows = rows;
      if constexpr (NT > 1) load_k(kf, c + 1);
      load_query_rows(qr, c + 2);
    }
#pragma unroll
    for (int t = 0; t < NT; t++) sigma_inv[t] = to_inv[t];
  };
  for (uint32_t c = 0; c < chunks; c += 2) {
    chunk(c, k0, g0, g1, k1, NT > 1 ? p0 : p1, p0, q0, m0, m1);
    if (c + 1 < chunks) chunk(c + 1, ROLE == QUERIES && NT > 1 ? k0 : k1, NT > 1 ? g0 : g1, g0, k0, p0, p1, q1, m1, m0);
  }
  if constexpr (ROLE == QUERIES) { if (NT == 1 && (last & 1)) put_out(last, p1); else put_out(last, p0); }
  if constexpr (ROLE == STATE) {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int m = 0; m < MT; m++) *(f4*)(sp + t * 16 * HK + m * 16) = S[t][m];
  }
}

template <int HK, int NT>
__global__ __launch_bounds__(768)
void pa_delta_scan_kernel(DeltaParams p, DeltaWs ws) {
  __shared__ __attribute__((aligned(16))) ScanLds<HK, NT> lds;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave < 4) scan_role<HK, NT, KEYS>(p, ws, lds, wave);
  else if (wave < 8) scan_role<HK, NT, STATE>(p, ws, lds, wave - 4);
  else scan_role<HK, NT, QUERIES>(p, ws, lds, wave - 8);
}

template <int HK>
static hipError_t launch_chunks(const DeltaParams& p, void* mem, uint32_t ws_chunks, int n_cu, hipStream_t s) {
  const DeltaWs ws = ws_at<HK>(mem, ws_chunks, p.nk, p.nv, nullptr);
  const uint32_t seg = ws_chunks * CHUNK;
  // Two tiles of value columns a workgroup where one each would not fit on the chip at once: the operands are read half as often, but each chunk takes longer.  2048 columns
  // of 48 heads of 128 values: 84 us with two (192 workgroups), 128 with one (384 on 256 CUs); of 32 heads: 75 with two (128 workgroups), 63 with one (256); all before the check of a chunk's range.
  const bool wide = p.hv % 32 == 0 && p.nv * (p.hv / 16) > (uint32_t)n_cu;
  for (uint32_t c0 = 0; c0 < p.n; c0 += seg) {
    DeltaParams r = p;
    r.n = std::min(seg, p.n - c0); r.commit = r.n;
    r.q += (size_t)c0 * p.q_stride; r.k += (size_t)c0 * p.k_stride; r.v += (size_t)c0 * p.v_stride;
    r.g += (size_t)c0 * p.gate_stride; r.beta += (size_t)c0 * p.gate_stride;
    if (r.out) r.out = (unsigned char*)p.out + (size_t)c0 * p.out_stride * (p.out_f16 ? 2 : 4);
    hipLaunchKernelGGL(pa_delta_prep_kernel<HK>, dim3(p.nv, (r.n + CHUNK - 1) / CHUNK), dim3(256), 0, s, r.k, r.q, r.g, r.beta, r.n, r.k_stride, r.q_stride, r.gate_stride, r.group, r, ws);
    const dim3 threads(768);
    if (wide) hipLaunchKernelGGL((pa_delta_scan_kernel<HK, 2>), dim3(p.nv * (p.hv / 32)), threads, 0, s, r, ws);
    else hipLaunchKernelGGL((pa_delta_scan_kernel<HK, 1>), dim3(p.nv * (p.hv / 16)), threads, 0, s, r, ws);
  }
  return hipGetLastError();
}

hipError_t pa_launch_delta_chunks(const DeltaParams& p, void* ws, uint32_t ws_chunks, int n_cu, hipStream_t s) {
  return p.hk == 64 ? launch_chunks<64>(p, ws, ws_chunks, n_cu, s) : launch_chunks<128>(p, ws, ws_chunks, n_cu, s);
}
