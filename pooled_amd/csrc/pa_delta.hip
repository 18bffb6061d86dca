// Host side of the gated delta rule (include/pooled_attn.h): handles, argument checks, launches.
#include "blocks_internal.h"
#include "blocks_host.h"
#include <cmath>
#include <cstring>
#include <new>

// Columns that pa_delta_prefill takes in one round of its two kernels.  The fragments of a round (2.6 MB a chunk of 64 with 32 v heads of 128 x 128) should stay in the last-level cache
// between them, and each round costs two launches: 8192 columns of 32 heads take 402 us in rounds of 1024, 362 in rounds of 2048, 404 of 4096, 412 at once (before the check of a chunk's range, 1 us more).  So the workspace does not
// grow with the prompt either.
#define SEGMENT_COLS 2048u

// Which form serves a prefill call.  The step kernel takes 0.24 us a column of 32 heads of 128 x 128 (0.37 of 48 or 64), the chunked form 13 to 19 us for any first chunk.  Steps and chunks,
// in us, for 40, 48, 56 and 64 columns: 4 heads 12.0 and 16.2, 13.9 and 16.4, 16.0 and 16.6, 17.9 and 16.8; 8 heads of 64 x 96 10.4 and 13.3, 12.1 and 13.4, 13.7 and 13.5, 15.4 and 13.6; 32 heads 13.1 and
// 17.2, 14.8 and 17.1, 16.7 and 17.2, 18.5 and 17.4; 48 heads 18.5 and 18.7, 21.2 and 19.0, 24.1 and 19.2, 26.5 and 19.4; 64 heads the same within 0.6.  Equal at 42 to 60 columns: one number
// for all heads, at 48 at most 2.5 us behind and at most 2.5 ahead.
static bool chunked(uint32_t n_cols) { return n_cols >= 48; }

extern "C" int pa_delta_destroy(pa_ctx* ctx, pa_delta* dn) {
  if (!ctx) return PA_ERR_INVALID;
  if (!dn) return PA_OK;
  if (dn->ctx != ctx) return block_fail(ctx, PA_ERR_INVALID, "pa_delta_destroy", "the handle belongs to another context");
  DeviceGuard on(ctx->device);
  hipError_t e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) return block_fail_hip(ctx, e, "pa_delta_destroy");
  if (dn->state) (void)hipFree(dn->state);
  if (dn->conv) (void)hipFree(dn->conv);
  if (dn->ws) (void)hipFree(dn->ws);
  delete dn;
  return PA_OK;
}

extern "C" int pa_delta_create(pa_ctx* ctx, const pa_delta_config* cfg, pa_delta** out) {
  const char* who = "pa_delta_create";
  if (!ctx) return PA_ERR_INVALID;
  if (!cfg || !out) return block_fail(ctx, PA_ERR_INVALID, who, "null argument");
  *out = nullptr;
  const pa_delta_config& c = *cfg;
  if (!c.n_k_heads || !c.n_v_heads || c.n_v_heads % c.n_k_heads) return block_fail(ctx, PA_ERR_INVALID, who, "n_v_heads must be a positive multiple of n_k_heads");
  if (c.n_v_heads > 4096u) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "more than 4096 v heads");
  if (c.head_k != 64 && c.head_k != 128) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "head_k must be 64 or 128 on the gfx950 table");
  if (!c.head_v || (c.head_v & 15) || c.head_v > 512) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "head_v must be a multiple of 16, at most 512, on the gfx950 table");
  if (c.conv_width > 4) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "conv_width must be at most 4");
  if (!c.n_layers || c.n_layers > 65536u) return block_fail(ctx, PA_ERR_INVALID, who, "n_layers must be in [1, 65536]");
  if (!std::isfinite(c.scale) || !(c.eps >= 0.f) || !std::isfinite(c.eps)) return block_fail(ctx, PA_ERR_INVALID, who, "scale must be finite, eps finite and >= 0");
  if (c.flags & ~PA_DELTA_L2NORM) return block_fail(ctx, PA_ERR_INVALID, who, "unknown flag");
  pa_delta* dn = new (std::nothrow) pa_delta();
  if (!dn) return block_fail(ctx, PA_ERR_NOMEM, who, "out of host memory");
  dn->cfg = c; dn->ctx = ctx;
  dn->scale = c.scale != 0.f ? c.scale : (float)(1.0 / std::sqrt((double)c.head_k));
  dn->channels = 2 * c.n_k_heads * c.head_k + c.n_v_heads * c.head_v;
  DeviceGuard on(ctx->device);
  const size_t sbytes = pa_delta_state_bytes(dn, 0) * c.n_layers, cbytes = pa_delta_state_bytes(dn, 1) * c.n_layers;
  dn->ws_chunks = (std::min(ctx->cfg.max_cols, SEGMENT_COLS) + 63) / 64;
  hipError_t e = hipMalloc((void**)&dn->state, sbytes);
  if (e == hipSuccess && cbytes) e = hipMalloc((void**)&dn->conv, cbytes);
  if (e == hipSuccess && chunked(ctx->cfg.max_cols)) e = hipMalloc(&dn->ws, pa_delta_chunk_ws_bytes(dn->ws_chunks, c.n_k_heads, c.n_v_heads, c.head_k));
  if (e == hipSuccess) e = pa_launch_fill_zero(dn->state, sbytes / 4, ctx->stream);
  if (e == hipSuccess && cbytes) e = pa_launch_fill_zero(dn->conv, cbytes / 4, ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) {
    if (dn->state) (void)hipFree(dn->state);
    if (dn->conv) (void)hipFree(dn->conv);
    if (dn->ws) (void)hipFree(dn->ws);
    delete dn;
    return block_fail_hip(ctx, e, who);
  }
  *out = dn;
  return PA_OK;
}

// ---- states --------------------------------------------------------------------------------------

extern "C" size_t pa_delta_state_bytes(const pa_delta* dn, int which) {
  if (!dn) return 0;
  const pa_delta_config& c = dn->cfg;
  if (which == 0) return (size_t)c.n_v_heads * c.head_v * c.head_k * sizeof(float);
  if (which == 1) return c.conv_width > 1 ? (size_t)(c.conv_width - 1) * dn->channels * sizeof(float) : 0;
  return 0;
}
extern "C" void* pa_delta_state_ptr(pa_delta* dn, uint32_t layer, int which) {
  if (!dn || layer >= dn->cfg.n_layers || !pa_delta_state_bytes(dn, which)) return nullptr;
  return (unsigned char*)(which ? dn->conv : dn->state) + pa_delta_state_bytes(dn, which) * layer;
}

static int check_handle(pa_ctx* ctx, const char* who, const pa_delta* dn, uint32_t layer) {
  if (!dn) return block_fail(ctx, PA_ERR_INVALID, who, "null handle");
  if (dn->ctx != ctx) return block_fail(ctx, PA_ERR_INVALID, who, "the handle belongs to another context");
  if (layer >= dn->cfg.n_layers) return block_fail(ctx, PA_ERR_INVALID, who, "layer out of range");
  return PA_OK;
}

static int state_copy(pa_ctx* ctx, const char* who, const pa_delta* dn, uint32_t layer, int which, void* host, bool to_host) {
  if (!ctx) return PA_ERR_INVALID;
  int rc = check_handle(ctx, who, dn, layer);
  if (rc) return rc;
  const size_t bytes = pa_delta_state_bytes(dn, which);
  if (!host || !bytes) return block_fail(ctx, PA_ERR_INVALID, who, "null host pointer, or a state the handle does not have");
  DeviceGuard on(ctx->device);
  void* dev = pa_delta_state_ptr(const_cast<pa_delta*>(dn), layer, which);
  hipError_t e = to_host ? hipMemcpyAsync(host, dev, bytes, hipMemcpyDeviceToHost, ctx->stream) : hipMemcpyAsync(dev, host, bytes, hipMemcpyHostToDevice, ctx->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}
extern "C" int pa_delta_read(pa_ctx* ctx, const pa_delta* dn, uint32_t layer, int which, void* h_dst) { return state_copy(ctx, "pa_delta_read", dn, layer, which, h_dst, true); }
extern "C" int pa_delta_write(pa_ctx* ctx, pa_delta* dn, uint32_t layer, int which, const void* h_src) {
  return state_copy(ctx, "pa_delta_write", dn, layer, which, const_cast<void*>(h_src), false);
}

extern "C" int pa_delta_reset(pa_ctx* ctx, pa_delta* dn, uint32_t layer) {
  const char* who = "pa_delta_reset";
  if (!ctx) return PA_ERR_INVALID;
  int rc = check_handle(ctx, who, dn, layer);
  if (rc) return rc;
  DeviceGuard on(ctx->device);
  for (int which = 0; which < 2; which++) {
    hipError_t e = pa_launch_fill_zero((float*)pa_delta_state_ptr(dn, layer, which), pa_delta_state_bytes(dn, which) / 4, ctx->stream);
    if (e != hipSuccess) return block_fail_hip(ctx, e, who);
  }
  return PA_OK;
}

// ---- calls ---------------------------------------------------------------------------------------

extern "C" int pa_delta_glue(pa_ctx* ctx, pa_delta* dn, uint32_t layer, const float* d_qkv, uint32_t qkv_stride, const float* d_conv_w, const float* d_conv_b,
                             const float* d_a, const float* d_b, uint32_t ab_stride, const float* d_a_log, const float* d_dt_bias, uint32_t n_cols,
                             uint32_t n_commit, float* d_out, uint32_t out_stride, float* d_g, float* d_beta, uint32_t gate_stride) {
  const char* who = "pa_delta_glue";
  if (!ctx) return PA_ERR_INVALID;
  int rc = check_handle(ctx, who, dn, layer);
  if (rc) return rc;
  const pa_delta_config& c = dn->cfg;
  if (!c.conv_width) return block_fail(ctx, PA_ERR_INVALID, who, "the handle was made without a convolution");
  if (!d_qkv || !d_conv_w || !d_a || !d_b || !d_a_log || !d_dt_bias || !d_out || !d_g || !d_beta) return block_fail(ctx, PA_ERR_INVALID, who, "null argument");
  if (!n_cols || n_cols > ctx->cfg.max_cols || n_commit > n_cols) return block_fail(ctx, PA_ERR_INVALID, who, "n_cols must be in [1, max_cols] and n_commit at most n_cols");
  if (qkv_stride < dn->channels || out_stride < dn->channels || ab_stride < c.n_v_heads || gate_stride < c.n_v_heads)
    return block_fail(ctx, PA_ERR_INVALID, who, "column stride shorter than a column");
  if (!aligned(d_qkv, 16) || !aligned(d_out, 16) || !aligned(d_conv_w, 16) || !aligned(d_conv_b, 16) || (qkv_stride & 3) || (out_stride & 3))
    return block_fail(ctx, PA_ERR_INVALID, who, "channel columns and weights must be 16-byte aligned, their strides multiples of 4");
  if (!aligned(d_a, 4) || !aligned(d_b, 4) || !aligned(d_a_log, 4) || !aligned(d_dt_bias, 4) || !aligned(d_g, 4) || !aligned(d_beta, 4))
    return block_fail(ctx, PA_ERR_INVALID, who, "gate columns must be 4-byte aligned");
  const Span in[] = {cols(d_qkv, n_cols, qkv_stride, dn->channels, 4), {d_conv_w, (size_t)dn->channels * c.conv_width * 4}, {d_conv_b, (size_t)dn->channels * 4},
                     cols(d_a, n_cols, ab_stride, c.n_v_heads, 4), cols(d_b, n_cols, ab_stride, c.n_v_heads, 4), {d_a_log, c.n_v_heads * 4ul}, {d_dt_bias, c.n_v_heads * 4ul},
                     {pa_delta_state_ptr(dn, layer, 1), pa_delta_state_bytes(dn, 1)}};
  const Span res[] = {cols(d_out, n_cols, out_stride, dn->channels, 4), cols(d_g, n_cols, gate_stride, c.n_v_heads, 4), cols(d_beta, n_cols, gate_stride, c.n_v_heads, 4)};
  for (const Span& o : res) for (const Span& i : in) if (overlap(o, i)) return block_fail(ctx, PA_ERR_INVALID, who, "an output shares memory with an input");
  const Columns res_cols[] = {{d_out, out_stride * 4ul, dn->channels * 4ul}, {d_g, gate_stride * 4ul, c.n_v_heads * 4ul}, {d_beta, gate_stride * 4ul, c.n_v_heads * 4ul}};
  for (int i = 0; i < 3; i++) for (int j = 0; j < i; j++) if (columns_meet(res_cols[i], res_cols[j], n_cols)) return block_fail(ctx, PA_ERR_INVALID, who, "two outputs share memory");
  const Span& state = in[sizeof in / sizeof *in - 1];
  for (const Span& i : in) if (&i != &state && overlap(state, i)) return block_fail(ctx, PA_ERR_INVALID, who, "an input lies in the layer's state");
  DeltaGlueParams p; memset(&p, 0, sizeof p);
  p.x = d_qkv; p.w = d_conv_w; p.bias = d_conv_b; p.a = d_a; p.b = d_b; p.a_log = d_a_log; p.dt_bias = d_dt_bias;
  p.conv = (float*)pa_delta_state_ptr(dn, layer, 1); p.out = d_out; p.g = d_g; p.beta = d_beta;
  p.x_stride = qkv_stride; p.ab_stride = ab_stride; p.out_stride = out_stride; p.gate_stride = gate_stride;
  p.n = n_cols; p.commit = n_commit; p.channels = dn->channels; p.nv = c.n_v_heads; p.width = c.conv_width;
  DeviceGuard on(ctx->device);
  const hipError_t e = pa_launch_delta_glue(p, ctx->stream);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}

static int rule_params(pa_ctx* ctx, const char* who, pa_delta* dn, uint32_t layer, const float* d_q, uint32_t q_stride, const float* d_k, uint32_t k_stride,
                       const float* d_v, uint32_t v_stride, const float* d_g, const float* d_beta, uint32_t gate_stride, uint32_t n_cols, uint32_t n_commit,
                       void* d_out, uint32_t out_stride, int out_dtype, DeltaParams& p) {
  if (!ctx) return PA_ERR_INVALID;
  int rc = check_handle(ctx, who, dn, layer);
  if (rc) return rc;
  const pa_delta_config& c = dn->cfg;
  const uint32_t kd = c.n_k_heads * c.head_k, vd = c.n_v_heads * c.head_v;
  if (!d_k || !d_v || !d_g || !d_beta || (d_out && !d_q)) return block_fail(ctx, PA_ERR_INVALID, who, "null input");
  if (!n_cols || n_cols > ctx->cfg.max_cols || n_commit > n_cols) return block_fail(ctx, PA_ERR_INVALID, who, "n_cols must be in [1, max_cols] and n_commit at most n_cols");
  if (!d_out && !n_commit) return block_fail(ctx, PA_ERR_INVALID, who, "neither an output nor a column to commit");
  if (d_out && out_dtype != PA_OUT_F32 && out_dtype != PA_OUT_F16) return block_fail(ctx, PA_ERR_INVALID, who, "bad out_dtype");
  if (k_stride < kd || v_stride < vd || gate_stride < c.n_v_heads || (d_out && (q_stride < kd || out_stride < vd)))
    return block_fail(ctx, PA_ERR_INVALID, who, "column stride shorter than a column");
  const size_t elem = out_dtype == PA_OUT_F16 ? 2 : 4;
  if (!aligned(d_k, 16) || (k_stride & 3) || (d_out && (!aligned(d_q, 16) || (q_stride & 3))))
    return block_fail(ctx, PA_ERR_INVALID, who, "q and k must be 16-byte aligned, their strides multiples of 4");
  if (!aligned(d_v, 4) || !aligned(d_g, 4) || !aligned(d_beta, 4) || !aligned(d_out, elem)) return block_fail(ctx, PA_ERR_INVALID, who, "unaligned column");
  const Span o = cols(d_out, n_cols, out_stride, vd, elem), state = {pa_delta_state_ptr(dn, layer, 0), pa_delta_state_bytes(dn, 0)};
  const Span in[] = {cols(d_out ? d_q : nullptr, n_cols, q_stride, kd, 4), cols(d_k, n_cols, k_stride, kd, 4), cols(d_v, n_cols, v_stride, vd, 4),
                     cols(d_g, n_cols, gate_stride, c.n_v_heads, 4), cols(d_beta, n_cols, gate_stride, c.n_v_heads, 4)};
  for (const Span& i : in) {
    if (overlap(o, i)) return block_fail(ctx, PA_ERR_INVALID, who, "the output shares memory with an input");
    if (overlap(state, i)) return block_fail(ctx, PA_ERR_INVALID, who, "an input lies in the layer's state");
  }
  if (overlap(o, state)) return block_fail(ctx, PA_ERR_INVALID, who, "the output shares memory with the state");
  memset(&p, 0, sizeof p);
  p.q = d_out ? d_q : d_k; p.k = d_k; p.v = d_v; p.g = d_g; p.beta = d_beta; p.state = (float*)pa_delta_state_ptr(dn, layer, 0); p.out = d_out;
  p.q_stride = d_out ? q_stride : k_stride; p.k_stride = k_stride; p.v_stride = v_stride; p.gate_stride = gate_stride; p.out_stride = d_out ? out_stride : 0;
  p.n = n_cols; p.commit = n_commit; p.nk = c.n_k_heads; p.nv = c.n_v_heads; p.hk = c.head_k; p.hv = c.head_v; p.group = c.n_v_heads / c.n_k_heads;
  p.scale = dn->scale; p.eps = c.eps; p.l2norm = c.flags & PA_DELTA_L2NORM; p.out_f16 = out_dtype == PA_OUT_F16;
  return PA_OK;
}

extern "C" int pa_delta_decode(pa_ctx* ctx, pa_delta* dn, uint32_t layer, const float* d_q, uint32_t q_stride, const float* d_k, uint32_t k_stride, const float* d_v,
                               uint32_t v_stride, const float* d_g, const float* d_beta, uint32_t gate_stride, uint32_t n_cols, uint32_t n_commit, void* d_out,
                               uint32_t out_stride, int out_dtype) {
  const char* who = "pa_delta_decode";
  DeltaParams p;
  int rc = rule_params(ctx, who, dn, layer, d_q, q_stride, d_k, k_stride, d_v, v_stride, d_g, d_beta, gate_stride, n_cols, n_commit, d_out, out_stride, out_dtype, p);
  if (rc) return rc;
  DeviceGuard on(ctx->device);
  const hipError_t e = pa_launch_delta_step(p, ctx->stream);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}

extern "C" int pa_delta_prefill(pa_ctx* ctx, pa_delta* dn, uint32_t layer, const float* d_q, uint32_t q_stride, const float* d_k, uint32_t k_stride, const float* d_v,
                                uint32_t v_stride, const float* d_g, const float* d_beta, uint32_t gate_stride, uint32_t n_cols, void* d_out, uint32_t out_stride,
                                int out_dtype) {
  const char* who = "pa_delta_prefill";
  DeltaParams p;
  int rc = rule_params(ctx, who, dn, layer, d_q, q_stride, d_k, k_stride, d_v, v_stride, d_g, d_beta, gate_stride, n_cols, n_cols, d_out, out_stride, out_dtype, p);
  if (rc) return rc;
  DeviceGuard on(ctx->device);
  // (a chunk's rows of v and of the output are addressed with 32-bit offsets)
  const hipError_t e = chunked(n_cols) && p.v_stride <= (1u << 22) && p.out_stride <= (1u << 22) ? pa_launch_delta_chunks(p, dn->ws, dn->ws_chunks, ctx->n_cu, ctx->stream) : pa_launch_delta_step(p, ctx->stream);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}
