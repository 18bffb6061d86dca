// Host side of the mixture-of-experts layer (include/pooled_attn.h): handles, argument checks, launches.
#include "blocks_internal.h"
#include "blocks_host.h"
#include <cstring>
#include <new>

static void free_moe(pa_moe* m) {
  void* const all[] = {m->router, m->gate, m->up, m->down, m->gate_s, m->up_s, m->down_s, m->scratch};
  for (void* d : all) if (d) (void)hipFree(d);
  delete m;
}

extern "C" int pa_moe_destroy(pa_ctx* ctx, pa_moe* moe) {
  if (!ctx) return PA_ERR_INVALID;
  if (!moe) return PA_OK;
  if (moe->ctx != ctx) return block_fail(ctx, PA_ERR_INVALID, "pa_moe_destroy", "the handle belongs to another context");
  DeviceGuard on(ctx->device);
  hipError_t e = hipStreamSynchronize(ctx->stream);
  if (e != hipSuccess) return block_fail_hip(ctx, e, "pa_moe_destroy");
  free_moe(moe);
  return PA_OK;
}

// tokens that the scratch holds; a wider call takes them in turn (35 KB a token with 9 experts of 512 x 2048: 18 MB, where 65535 columns would be 2.3 GB a layer)
#define BATCH_TOKENS 512u
static uint32_t batch_of(const pa_ctx* ctx) { return ctx->cfg.max_cols < BATCH_TOKENS ? ctx->cfg.max_cols : BATCH_TOKENS; }

static size_t plane_bytes(int kind, size_t values) { return kind == PA_W_F32 ? values * 4 : kind == PA_W_Q8_0 ? values : values / 2; }

// scratch of n tokens, every part 256-byte aligned: sets p's pointers behind `base` and returns the bytes
static size_t lay_scratch(const pa_moe* m, uint32_t n, unsigned char* base, MoeParams& p) {
  size_t at = 0;
  auto take = [&](size_t bytes) { void* r = base + at; at += (bytes + 255) & ~(size_t)255; return r; };
  p.xn_floats = moe_act_floats(m->cfg.kind, m->cfg.dim);
  p.h_floats = moe_act_floats(m->cfg.kind, m->slots * m->cfg.ffn);
  p.logit_stride = m->cfg.n_experts + 1;
  p.xn = (float*)take((size_t)n * p.xn_floats * 4);
  p.h = (float*)take((size_t)n * p.h_floats * 4);
  p.logits = (float*)take((size_t)n * p.logit_stride * 4);
  p.sel = (uint32_t*)take((size_t)n * m->slots * 4);
  p.sel_w = (float*)take((size_t)n * m->slots * 4);
  return at;
}

extern "C" int pa_moe_create(pa_ctx* ctx, const pa_moe_config* cfg, const pa_moe_planes* planes, pa_moe** out) {
  const char* who = "pa_moe_create";
  if (!ctx) return PA_ERR_INVALID;
  if (!cfg || !planes || !out) return block_fail(ctx, PA_ERR_INVALID, who, "null argument");
  *out = nullptr;
  const pa_moe_config& c = *cfg;
  if (c.kind != PA_W_F32 && c.kind != PA_W_Q8_0 && c.kind != PA_W_Q4_0) return block_fail(ctx, PA_ERR_INVALID, who, "unknown weight kind");
  if (!c.dim || (c.dim & 31) || !c.ffn || (c.ffn & 31)) return block_fail(ctx, PA_ERR_INVALID, who, "dim and ffn must be positive multiples of 32");
  if (c.dim > 8192 || c.ffn > 8192) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "dim or ffn beyond the gfx950 table");
  if (!c.n_experts || !c.top_k || c.top_k > c.n_experts) return block_fail(ctx, PA_ERR_INVALID, who, "n_experts must be positive and top_k in [1, n_experts]");
  if (c.n_experts > 1024 || c.top_k > 16) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "n_experts or top_k beyond the gfx950 table");
  if (c.flags & ~(PA_MOE_NORM_TOPK | PA_MOE_SHARED)) return block_fail(ctx, PA_ERR_INVALID, who, "unknown flag");
  const bool shared = (c.flags & PA_MOE_SHARED) != 0, quant = c.kind != PA_W_F32;
  const pa_moe_planes& h = *planes;
  if (!h.h_router || !h.h_gate || !h.h_up || !h.h_down || (quant && (!h.h_gate_s || !h.h_up_s || !h.h_down_s))) return block_fail(ctx, PA_ERR_INVALID, who, "null plane");
  if (shared && (!h.h_shared_gate || !h.h_shared_gate_w || !h.h_shared_up_w || !h.h_shared_down_w || (quant && (!h.h_shared_gate_s || !h.h_shared_up_s || !h.h_shared_down_s))))
    return block_fail(ctx, PA_ERR_INVALID, who, "null plane of the shared expert");
  pa_moe* m = new (std::nothrow) pa_moe();
  if (!m) return block_fail(ctx, PA_ERR_NOMEM, who, "out of host memory");
  m->cfg = c; m->ctx = ctx; m->slots = c.top_k + (shared ? 1 : 0);
  DeviceGuard on(ctx->device);
  const size_t values = (size_t)c.dim * c.ffn, wb = plane_bytes(c.kind, values), sb = quant ? values / 32 * 2 : 0, rb = (size_t)c.dim * 4;
  hipError_t e = hipSuccess;
  // n_experts rows of a plane, then the shared expert's
  auto put = [&](void** dev, const void* host, const void* host_shared, size_t each) {
    if (e != hipSuccess || !each) return;
    e = hipMalloc(dev, each * (c.n_experts + (shared ? 1 : 0)));
    if (e == hipSuccess) e = hipMemcpyAsync(*dev, host, each * c.n_experts, hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess && shared) e = hipMemcpyAsync((unsigned char*)*dev + each * c.n_experts, host_shared, each, hipMemcpyHostToDevice, ctx->stream);
  };
  put((void**)&m->router, h.h_router, h.h_shared_gate, rb);
  put((void**)&m->gate, h.h_gate, h.h_shared_gate_w, wb);
  put((void**)&m->up, h.h_up, h.h_shared_up_w, wb);
  put((void**)&m->down, h.h_down, h.h_shared_down_w, wb);
  put((void**)&m->gate_s, h.h_gate_s, h.h_shared_gate_s, sb);
  put((void**)&m->up_s, h.h_up_s, h.h_shared_up_s, sb);
  put((void**)&m->down_s, h.h_down_s, h.h_shared_down_s, sb);
  MoeParams p;
  const size_t scratch = lay_scratch(m, batch_of(ctx), nullptr, p);
  if (e == hipSuccess) e = hipMalloc((void**)&m->scratch, scratch);
  const hipError_t s = hipStreamSynchronize(ctx->stream);        // the host planes are the caller's again, whatever happened
  if (e == hipSuccess) e = s;
  if (e != hipSuccess) { free_moe(m); return block_fail_hip(ctx, e, who); }
  *out = m;
  return PA_OK;
}

extern "C" int pa_moe_layer(pa_ctx* ctx, pa_moe* moe, const float* d_norm_w, const float* d_x, uint32_t x_stride, uint32_t n_cols, float* d_y, uint32_t y_stride,
                            uint32_t* d_ids, float* d_weights) {
  const char* who = "pa_moe_layer";
  if (!ctx) return PA_ERR_INVALID;
  if (!moe || !d_x || !d_y) return block_fail(ctx, PA_ERR_INVALID, who, "null argument");
  if (moe->ctx != ctx) return block_fail(ctx, PA_ERR_INVALID, who, "the handle belongs to another context");
  const pa_moe_config& c = moe->cfg;
  if (!n_cols || n_cols > ctx->cfg.max_cols) return block_fail(ctx, PA_ERR_INVALID, who, "n_cols must be in [1, max_cols]");
  if (x_stride < c.dim || y_stride < c.dim || (x_stride & 3) || (y_stride & 3)) return block_fail(ctx, PA_ERR_INVALID, who, "strides must be multiples of 4 and at least dim");
  if (!aligned(d_x, 16) || !aligned(d_y, 16) || !aligned(d_norm_w, 16) || !aligned(d_ids, 4) || !aligned(d_weights, 4))
    return block_fail(ctx, PA_ERR_INVALID, who, "columns and norm weights must be 16-byte aligned, ids and weights 4-byte");
  const Span x = cols(d_x, n_cols, x_stride, c.dim, 4), y = cols(d_y, n_cols, y_stride, c.dim, 4), nw = {d_norm_w, c.dim * 4ul};
  const Span ids = {d_ids, (size_t)n_cols * c.top_k * 4}, wts = {d_weights, (size_t)n_cols * c.top_k * 4};
  const bool in_place = d_x == d_y && x_stride == y_stride;
  if ((!in_place && overlap(x, y)) || overlap(y, nw) || overlap(ids, x) || overlap(ids, y) || overlap(ids, nw) || overlap(wts, x) || overlap(wts, y) || overlap(wts, nw) || overlap(ids, wts))
    return block_fail(ctx, PA_ERR_INVALID, who, "an output shares memory with an input (y may be x itself, with the same stride)");
  MoeParams p; memset(&p, 0, sizeof p);
  p.router = moe->router; p.gate = moe->gate; p.up = moe->up; p.down = moe->down; p.gate_s = moe->gate_s; p.up_s = moe->up_s; p.down_s = moe->down_s;
  p.norm_w = d_norm_w; p.x = d_x; p.y = d_y; p.ids = d_ids; p.weights = d_weights;
  p.batch = batch_of(ctx);
  lay_scratch(moe, p.batch, (unsigned char*)moe->scratch, p);
  p.x_stride = x_stride; p.y_stride = y_stride; p.n = n_cols; p.dim = c.dim; p.ffn = c.ffn; p.n_experts = c.n_experts; p.top_k = c.top_k; p.slots = moe->slots;
  p.eps = ctx->cfg.eps; p.norm_topk = (c.flags & PA_MOE_NORM_TOPK) != 0; p.kind = c.kind;
  DeviceGuard on(ctx->device);
  const hipError_t e = pa_launch_moe(p, ctx->n_cu, ctx->stream);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}
