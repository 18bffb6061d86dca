// Declarations of the blocks beside attention: the gated delta rule with its pre-step (delta_step.hip, delta_chunk.hip, pa_delta.hip) and the
// mixture of experts (moe_layer.hip, pa_moe.hip).
#pragma once
#include "pa_internal.h"

// ---- gated delta rule ----------------------------------------------------------------------------

struct pa_delta {
  pa_delta_config cfg{};
  pa_ctx* ctx = nullptr;
  float scale = 1.f;               // of q
  uint32_t channels = 0;           // of the convolution: q heads, k heads, v heads
  float* state = nullptr;          // [n_layers][n_v_heads][head_v][head_k]
  float* conv = nullptr;           // [n_layers][conv_width - 1][channels], oldest input first; nullptr with fewer than two taps
  void* ws = nullptr;              // chunked form: the fragments of one segment of chunks
  uint32_t ws_chunks = 0;
};

struct DeltaParams {
  const float* q; const float* k; const float* v; const float* g; const float* beta;
  float* state;                    // this layer's [nv][hv][hk]
  void* out;                       // [n][out_stride] f32 or f16; nullptr: the state alone
  uint32_t q_stride, k_stride, v_stride, gate_stride, out_stride;
  uint32_t n, commit;              // columns, and how many of them the stored state has seen
  uint32_t nk, nv, hk, hv, group;  // group = nv / nk
  float scale, eps;
  uint32_t l2norm;
  int out_f16;
};

struct DeltaGlueParams {
  const float* x; const float* w; const float* bias;    // [n][x_stride]; [channels][W]; [channels] or nullptr
  const float* a; const float* b; const float* a_log; const float* dt_bias;
  float* conv;                                          // this layer's [W - 1][channels]
  float* out; float* g; float* beta;
  uint32_t x_stride, ab_stride, out_stride, gate_stride;
  uint32_t n, commit, channels, nv, width;
};

hipError_t pa_launch_delta_step(const DeltaParams& p, hipStream_t s);
// in chunks, all columns committed; ws: pa_delta_chunk_ws_bytes(ws_chunks, ..) bytes
hipError_t pa_launch_delta_chunks(const DeltaParams& p, void* ws, uint32_t ws_chunks, int n_cu, hipStream_t s);
size_t pa_delta_chunk_ws_bytes(uint32_t chunks, uint32_t nk, uint32_t nv, uint32_t hk);
hipError_t pa_launch_delta_glue(const DeltaGlueParams& p, hipStream_t s);
hipError_t pa_launch_fill_zero(float* p, size_t n, hipStream_t s);

// ---- mixture of experts --------------------------------------------------------------------------

struct pa_moe {
  pa_moe_config cfg{};
  pa_ctx* ctx = nullptr;
  uint32_t slots = 0;              // experts of a token: top_k, + 1 with a shared expert (kept as expert n_experts)
  float* router = nullptr;         // [n_experts (+ 1: the shared expert's gate)][dim]
  unsigned char* gate = nullptr; unsigned char* up = nullptr; unsigned char* down = nullptr;
  uint16_t* gate_s = nullptr; uint16_t* up_s = nullptr; uint16_t* down_s = nullptr;
  float* scratch = nullptr;        // see MoeParams
};

struct MoeParams {
  const float* router; const unsigned char* gate; const unsigned char* up; const unsigned char* down;
  const uint16_t* gate_s; const uint16_t* up_s; const uint16_t* down_s;
  const float* norm_w; const float* x; float* y; uint32_t* ids; float* weights;
  // scratch of the call: normed activations [n][xn_floats] and expert activations [n][h_floats] in the order their readers load them,
  // router logits [n][logit_stride], the experts of a token and their weights [n][slots]
  float* xn; float* h; float* logits; uint32_t* sel; float* sel_w;
  uint32_t xn_floats, h_floats, logit_stride;
  uint32_t batch;                  // tokens that the scratch holds
  uint32_t x_stride, y_stride, n, dim, ffn, n_experts, top_k, slots;
  float eps;
  uint32_t norm_topk;
  int kind;
};

// floats of an activation of so many values in reading order (moe_layer.hip): groups of 64 blocks; f32 weights: natural order
#define MOE_GROUP_FLOATS 2048
static inline uint32_t moe_act_floats(int kind, uint32_t values) { return kind == PA_W_F32 ? values : (values / 32 + 63) / 64 * MOE_GROUP_FLOATS; }
hipError_t pa_launch_moe(const MoeParams& p, int n_cu, hipStream_t s);
