// Host side of the drafted-tree calls (include/pooled_attn.h): attention of a tree over the cache, the pre-step of columns with positions of their own, compaction of the caches.
#include "tree_internal.h"
#include "blocks_host.h"
#include <cmath>
#include <cstring>

static inline uint32_t ceil_div(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a + b - 1) / b); }
static bool kv_q8(const pa_ctx* ctx) { return (ctx->cfg.flags & PA_FLAG_KV_Q8) != 0; }

static int check_columns(pa_ctx* ctx, const char* who, uint32_t layer, uint32_t base, uint32_t n_cols) {
  if (n_cols == 0 || n_cols > ctx->cfg.max_cols) return block_fail(ctx, PA_ERR_INVALID, who, "n_cols must be in [1, max_cols]");
  if ((uint64_t)base + n_cols > ctx->cfg.max_seq) return block_fail(ctx, PA_ERR_INVALID, who, "the columns' rows exceed max_seq");
  if (layer >= ctx->cfg.n_layers) return block_fail(ctx, PA_ERR_INVALID, who, "layer out of range");
  if (!ctx->layers[layer].k) return block_fail(ctx, PA_ERR_INVALID, who, "layer has no cache (call pa_layer_alloc)");
  return PA_OK;
}
static size_t cols_bytes(uint32_t n_cols, uint32_t stride, uint32_t col, size_t elem) { return ((size_t)(n_cols - 1) * stride + col) * elem; }

// ---- pre-step ------------------------------------------------------------------------------------

extern "C" int pa_set_rope_axes(pa_ctx* ctx, uint32_t n_axes, const uint8_t* h_axis_of_pair) {
  const char* who = "pa_set_rope_axes";
  if (!ctx) return PA_ERR_INVALID;
  if (n_axes == 0 || n_axes > 4) return block_fail(ctx, PA_ERR_INVALID, who, "n_axes must be in [1, 4]");
  if (!h_axis_of_pair && n_axes != 1) return block_fail(ctx, PA_ERR_INVALID, who, "several axes need the axis of every pair");
  uint32_t words[8] = {0};
  for (uint32_t i = 0; h_axis_of_pair && i < ctx->cfg.n_rot / 2; i++) {
    if (h_axis_of_pair[i] >= n_axes) return block_fail(ctx, PA_ERR_INVALID, who, "a pair's axis must be below n_axes");
    words[i / 16] |= (uint32_t)h_axis_of_pair[i] << (i % 16 * 2);
  }
  ctx->rope_axes = n_axes;
  memcpy(ctx->axis_of_pair, words, sizeof words);
  return PA_OK;
}

extern "C" int pa_glue_kv_at(pa_ctx* ctx, uint32_t layer, const float* d_q_in, uint32_t q_stride, const float* d_k, uint32_t k_stride, const float* d_v, uint32_t v_stride,
                             const float* d_qw, const float* d_kw, const uint32_t* d_pos, uint32_t pos_stride, uint32_t base_row, uint32_t n_cols) {
  const char* who = "pa_glue_kv_at";
  if (!ctx) return PA_ERR_INVALID;
  int rc = check_columns(ctx, who, layer, base_row, n_cols);
  if (rc) return rc;
  const pa_config& c = ctx->cfg;
  const uint32_t qd = c.n_heads * c.head_dim, qcol = qd * ((c.flags & PA_FLAG_GATE) ? 2 : 1), kvd = c.n_kv_heads * c.head_dim;
  if (!d_q_in || !d_k || !d_v || !d_pos) return block_fail(ctx, PA_ERR_INVALID, who, "null input");
  if ((c.flags & PA_FLAG_QK_NORM) && (!d_qw || !d_kw)) return block_fail(ctx, PA_ERR_INVALID, who, "norm weights required");
  if (q_stride < qcol || k_stride < kvd || v_stride < kvd) return block_fail(ctx, PA_ERR_INVALID, who, "column stride shorter than a column");
  if (ctx->rope_axes > 1 && pos_stride < n_cols) return block_fail(ctx, PA_ERR_INVALID, who, "pos_stride shorter than an axis's positions");
  if (((uintptr_t)d_q_in | (uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_qw | (uintptr_t)d_kw | (uintptr_t)d_pos) & 3) return block_fail(ctx, PA_ERR_INVALID, who, "pointers must be 4-byte aligned");
  const size_t norm = (c.flags & PA_FLAG_QK_NORM) ? c.head_dim * 4 : 0;
  const Span in[6] = {{d_q_in, cols_bytes(n_cols, q_stride, qcol, 4)}, {d_k, cols_bytes(n_cols, k_stride, kvd, 4)}, {d_v, cols_bytes(n_cols, v_stride, kvd, 4)},
                      {d_pos, ((size_t)(ctx->rope_axes - 1) * pos_stride + n_cols) * 4}, {d_qw, norm}, {d_kw, norm}};
  for (const Span& s : in)
    if (overlap(s, {ctx->q_buf, (size_t)n_cols * qd * 4}) || overlap(s, {ctx->gate_buf, (size_t)n_cols * qd * 4}))
      return block_fail(ctx, PA_ERR_INVALID, who, "an input lies in the context's q or gate buffer, which the call writes");
  const pa_layer& L = ctx->layers[layer];
  GlueAtParams p;
  memset(&p, 0, sizeof p);
  p.q_in = d_q_in; p.k_in = d_k; p.v_in = d_v; p.qw = d_qw; p.kw = d_kw;
  p.inv_freq = ctx->inv_freq; p.rope_tab = ctx->rope_tab; p.tab_rows = ctx->rope_tab ? c.max_seq : 0;
  p.pos = d_pos; p.pos_stride = pos_stride;
  p.q_out = ctx->q_buf; p.gate_out = ctx->gate_buf;
  p.k_cache = L.k; p.v_cache = L.v; p.ks_cache = L.ks; p.vs_cache = L.vs; p.head_rows = c.max_seq + 32;
  p.q_stride = q_stride; p.k_stride = k_stride; p.v_stride = v_stride;
  p.n_heads = c.n_heads; p.n_kv_heads = c.n_kv_heads; p.head_dim = c.head_dim; p.n_rot = c.n_rot;
  p.base_row = base_row; p.n_cols = n_cols; p.flags = c.flags; p.eps = c.eps;
  p.n_axes = ctx->rope_axes;
  memcpy(p.axis_of_pair, ctx->axis_of_pair, sizeof p.axis_of_pair);
  DeviceGuard on(ctx->device);
  const hipError_t e = pa_launch_glue_at(p, ctx->stream);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}

// ---- attention -----------------------------------------------------------------------------------

static size_t part_bytes(const pa_config& c, uint32_t n_cols, uint32_t splits) { return (size_t)n_cols * c.n_heads * splits * c.head_dim * 4; }
static size_t ml_bytes(const pa_config& c, uint32_t n_cols, uint32_t splits) { return (size_t)n_cols * c.n_heads * splits * 8; }

// What a call takes, in us, fitted to 463 timed calls (16 / 2-, 24 / 4- and 16 / 8-head shapes, 2 - 64 columns at 64 - 65536 rows, f16 and int8 rows, 64 - 256 rows a workgroup, all CUs busy
// down to an eighth of them; mean error 4 %, nine in ten within 8 %; what it chooses takes 100.8 % of the best plan tried, 109 % at worst).  The launches, the start of a workgroup and its
// outputs; then its tiles, each so long for the barrier and the chain of one wave and so much for every block of 16 rows, or the stream of the cache if that is more; and the
// partials, written and read again (timed as f16; as f32 they take 0.0 - 0.3 us a MB more, and where twice the weight would choose another plan it takes as long: 26 cases, mean of the quotients 1.00).  q's second products came later too: over
// 60 cases of 5 - 63 columns at 300 - 40000 rows the choice takes 102 % of the best cap's time, 125 % at worst, where the best is two blocks a wave of heads of 256, which are without them.
static double tree_us(const pa_config& c, uint32_t n_cu, uint32_t rows, uint32_t tiles, const TreePlan& pl) {
  const bool q8 = (c.flags & PA_FLAG_KV_Q8) != 0, wide = c.head_dim == 256;
  const double fixed = q8 ? (wide ? 10.1 : 7.6) : wide ? 8.6 : 7.2, out = q8 ? (wide ? 0.05 : 0.18) : wide ? 0.29 : 0.19;
  const double tile = q8 ? (wide ? 0.629 : 0.458) : wide ? 0.356 : 0.358, block = q8 ? (wide ? 0.072 : 0.016) : wide ? 0.063 : 0.019;
  const double blocks = pl.group_rows / 16.0, wgs = (double)pl.n_groups * c.n_kv_heads * pl.n_splits;
  const double chain = pl.split_tiles * (tile + block * blocks) * std::ceil(wgs / n_cu);
  const double stream = 1e-6 / 7.0 * tiles * 32.0 * c.n_kv_heads * c.head_dim * (q8 ? 2.25 : 4.0);
  // (a second launch and its trip to memory saved; 168 calls of 1 - 63 columns at 20 - 450 rows: one split is ahead up to some 200 rows of head_dim 128, 130 of 256, 30 - 150 of int8 rows;
  // 24 columns at 100 rows of 16 / 8 heads of 128 6.2 us against 8.5, at 300 9.2 against 8.7)
  const double merge = pl.n_splits > 1 ? 0.0 : q8 ? (wide ? 1.3 : 2.6) : wide ? 1.9 : 2.9;
  const double partials = pl.n_splits > 1 ? 1e-6 * rows * c.n_kv_heads * pl.n_splits * c.head_dim * 4.0 : 0.0;
  return fixed - merge + std::max(chain, stream) + out * blocks + 0.2135 * partials;
}

// Rows of a workgroup: up to 256, a wave two blocks of 16, or 128, 64 and 32, the groups then sharing the stream through their XCD's L2 (two blocks of int8 rows of head_dim 256 do not fit the
// registers).  Splits: a workgroup a CU, or fewer, whose partials are less, or one, which needs no second launch.  most_splits: what a caller that cannot allocate has room for.
static TreePlan plan_tree(const pa_config& c, uint32_t n_cu, uint32_t base, uint32_t n_cols, uint32_t override_splits, uint32_t most_splits) {
  const uint32_t rows = n_cols * (c.n_heads / c.n_kv_heads), tiles = ceil_div(base + n_cols, 32);
  const bool narrow = (c.flags & PA_FLAG_KV_Q8) && c.head_dim == 256;
  TreePlan best{};
  double best_us = -1.0;
  for (uint32_t cap = narrow ? 128 : 256; cap >= 32; cap /= 2) {
    if (cap < 256 && cap / 2 >= rows && cap > 32) continue;                  // the same groups as the next cap's
    TreePlan pl{};
    pl.group_rows = (ceil_div(rows, ceil_div(rows, cap)) + 15) & ~15u;
    pl.nb = ceil_div(pl.group_rows, 16 * TREE_W);
    pl.n_groups = ceil_div(rows, pl.group_rows);
    const uint32_t full = (uint32_t)std::max<uint64_t>(1, n_cu / ((uint64_t)pl.n_groups * c.n_kv_heads));
    for (uint32_t part : {1u, 2u, 4u, 8u, full}) {
      const uint32_t want = std::max(1u, std::min({override_splits ? override_splits : std::max(1u, full / part), tiles, most_splits}));
      pl.split_tiles = ceil_div(tiles, want);
      pl.n_splits = ceil_div(tiles, pl.split_tiles);
      const double us = tree_us(c, n_cu, rows, tiles, pl);
      if (best_us < 0.0 || us < best_us) { best = pl; best_us = us; }
      if (override_splits || pl.n_splits == 1) break;
    }
  }
  return best;
}

// the plan of a call, for the tests: {nb, waves, n_groups, group_rows, n_splits, split_tiles}
extern "C" int pa_rule_tree(const pa_config* cfg, int n_cu, uint32_t base_pos, uint32_t n_cols, uint32_t splits, uint32_t most_splits, uint32_t* out) {
  const TreePlan pl = plan_tree(*cfg, (uint32_t)n_cu, base_pos, n_cols, splits, most_splits);
  const uint32_t v[6] = {pl.nb, TREE_W, pl.n_groups, pl.group_rows, pl.n_splits, pl.split_tiles};
  memcpy(out, v, sizeof v);
  return 0;
}

extern "C" int pa_attn_tree(pa_ctx* ctx, uint32_t layer, const float* d_q, uint32_t q_stride, const float* d_gate, uint32_t gate_stride, const uint32_t* d_mask,
                            uint32_t mask_stride, uint32_t base_pos, uint32_t n_cols, void* d_out, uint32_t out_stride, int out_dtype) {
  const char* who = "pa_attn_tree";
  if (!ctx) return PA_ERR_INVALID;
  int rc = check_columns(ctx, who, layer, base_pos, n_cols);
  if (rc) return rc;
  const pa_config& c = ctx->cfg;
  const uint32_t qd = c.n_heads * c.head_dim;
  if (c.flags & PA_FLAG_VERIFY_EXACT) return block_fail(ctx, PA_ERR_UNSUPPORTED, who, "PA_FLAG_VERIFY_EXACT promises the bits of one-column decodes, which a tree's columns do not have");
  if (!d_mask || !d_out) return block_fail(ctx, PA_ERR_INVALID, who, "null mask or output");
  if (out_dtype != PA_OUT_F32 && out_dtype != PA_OUT_F16) return block_fail(ctx, PA_ERR_INVALID, who, "bad out_dtype");
  if (!d_q) { d_q = ctx->q_buf; q_stride = qd; }
  if (q_stride < qd || out_stride < qd || (d_gate && gate_stride < qd)) return block_fail(ctx, PA_ERR_INVALID, who, "column stride shorter than a column");
  if (mask_stride < ceil_div(n_cols, 32)) return block_fail(ctx, PA_ERR_INVALID, who, "mask_stride shorter than a column's words");
  if ((q_stride & 3) || (out_stride & 3) || (d_gate && (gate_stride & 3)) || ((uintptr_t)d_q & 15) || ((uintptr_t)d_out & 15) || ((uintptr_t)d_gate & 15) || ((uintptr_t)d_mask & 3))
    return block_fail(ctx, PA_ERR_INVALID, who, "buffers must be 16-byte aligned (the mask 4) with strides a multiple of 4 elements");
  const Span out = {d_out, cols_bytes(n_cols, out_stride, qd, out_dtype == PA_OUT_F16 ? 2 : 4)};
  if (overlap(out, {d_q, cols_bytes(n_cols, q_stride, qd, 4)}) || (d_gate && overlap(out, {d_gate, cols_bytes(n_cols, gate_stride, qd, 4)})) ||
      overlap(out, {d_mask, cols_bytes(n_cols, mask_stride, ceil_div(n_cols, 32), 4)}))
    return block_fail(ctx, PA_ERR_INVALID, who, "the output shares memory with an input");
  DeviceGuard on(ctx->device);
  TreePlan pl = plan_tree(c, (uint32_t)ctx->n_cu, base_pos, n_cols, ctx->decode_splits_override, 0xffffffffu);
  if (pl.n_splits > 1 && (part_bytes(c, n_cols, pl.n_splits) > ctx->part_o_bytes || ml_bytes(c, n_cols, pl.n_splits) > ctx->part_ml_bytes)) {
    // the scratch grows, or, under stream capture, where it cannot, the splits become as many as it has room for
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    hipError_t e = hipStreamIsCapturing(ctx->stream, &st);
    if (e != hipSuccess) return block_fail_hip(ctx, e, who);
    if (st != hipStreamCaptureStatusNone) {
      const size_t fit = std::min(ctx->part_o_bytes / part_bytes(c, n_cols, 1), ctx->part_ml_bytes / ml_bytes(c, n_cols, 1));
      pl = plan_tree(c, (uint32_t)ctx->n_cu, base_pos, n_cols, ctx->decode_splits_override, (uint32_t)std::min<size_t>(fit, 0xffffffffu));
    } else if ((rc = pa_ctx_grow(ctx, (void**)&ctx->part_o, &ctx->part_o_bytes, part_bytes(c, n_cols, pl.n_splits))) ||
               (rc = pa_ctx_grow(ctx, (void**)&ctx->part_ml, &ctx->part_ml_bytes, ml_bytes(c, n_cols, pl.n_splits)))) return rc;
  }
  const pa_layer& L = ctx->layers[layer];
  TreeParams p;
  memset(&p, 0, sizeof p);
  p.q = d_q; p.gate = d_gate; p.k_cache = L.k; p.v_cache = L.v; p.k_scale = L.ks; p.v_scale = L.vs; p.mask = d_mask;
  p.part_o = ctx->part_o; p.part_ml = (float2*)ctx->part_ml; p.out = d_out;
  p.q_stride = q_stride; p.gate_stride = gate_stride; p.mask_stride = mask_stride; p.out_stride = out_stride;
  p.n_heads = c.n_heads; p.n_kv_heads = c.n_kv_heads; p.group = c.n_heads / c.n_kv_heads;
  p.base_pos = base_pos; p.n_cols = n_cols; p.max_seq = c.max_seq;
  p.n_splits = pl.n_splits; p.split_tiles = pl.split_tiles; p.n_groups = pl.n_groups; p.group_rows = pl.group_rows;
  p.out_f16 = out_dtype == PA_OUT_F16;
  p.scale = (float)(1.0 / std::sqrt((double)c.head_dim));
  PaTiming tm, tm2;
  if ((rc = pa_ctx_timing(ctx, &tm, &tm2, pl.n_splits > 1))) return rc;
  hipError_t e = pa_launch_tree(p, pl, c.head_dim, ctx->stream, &tm);
  if (e == hipSuccess && pl.n_splits > 1) e = pa_launch_tree_merge(p, c.head_dim, ctx->stream, &tm2);
  return e == hipSuccess ? PA_OK : block_fail_hip(ctx, e, who);
}

// ---- compaction ----------------------------------------------------------------------------------

extern "C" int pa_kv_compact(pa_ctx* ctx, uint32_t dst_row, const uint32_t* d_sel, uint32_t max_rows) {
  const char* who = "pa_kv_compact";
  if (!ctx) return PA_ERR_INVALID;
  const pa_config& c = ctx->cfg;
  if (!d_sel || ((uintptr_t)d_sel & 3)) return block_fail(ctx, PA_ERR_INVALID, who, "the list must be there and 4-byte aligned");
  if (max_rows == 0 || (uint64_t)dst_row + max_rows > c.max_seq) return block_fail(ctx, PA_ERR_INVALID, who, "dst_row + max_rows must be in [dst_row + 1, max_seq]");
  DeviceGuard on(ctx->device);
  CompactParams p;
  memset(&p, 0, sizeof p);
  const uint32_t per = kv_q8(ctx) ? 4 : 2;
  p.sel = d_sel; p.n_planes = c.n_kv_heads; p.head_rows = c.max_seq + 32; p.dst_row = dst_row; p.max_rows = max_rows; p.max_seq = c.max_seq;
  p.row_bytes = kv_q8(ctx) ? c.head_dim : c.head_dim * 2; p.scale_bytes = kv_q8(ctx) ? c.head_dim / 8 : 0;
  uint32_t layers = 0;
  for (const pa_layer& L : ctx->layers) layers += L.k != nullptr;
  if (!layers) return block_fail(ctx, PA_ERR_INVALID, who, "no layer has a cache (call pa_layer_alloc)");
  p.n_layers = std::min(layers, PA_COMPACT_LAYERS);
  if (!pa_compact_one_round(p)) {
    // Flags for the segments of a long list.  A workgroup waits for flags of its launch: two launches at once with the same ones would take one another's tickets, and a wait could be without
    // end.  So every stream, which runs its launches one behind the other, has flags of its own; and a recorded call, which may be replayed on any stream beside any other call, walks the list
    // without, as does one on hipStreamPerThread, which is another stream in every thread.  (One stream's flags in turn with events between the calls cost 3 us a call.)
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    hipError_t e = hipStreamIsCapturing(ctx->stream, &st);
    if (e != hipSuccess) return block_fail_hip(ctx, e, who);
    if (st == hipStreamCaptureStatusNone && ctx->stream != hipStreamPerThread) {
      const size_t need = pa_compact_flags(p) * sizeof(uint32_t);
      CompactFlags* f = nullptr;
      for (CompactFlags& have : ctx->compact_flags) if (have.stream == ctx->stream) f = &have;
      if (!f) {
        try { ctx->compact_flags.push_back(CompactFlags()); } catch (const std::bad_alloc&) { return block_fail(ctx, PA_ERR_NOMEM, who, "out of host memory"); }
        f = &ctx->compact_flags.back();
        f->stream = ctx->stream;
      }
      if (need > f->bytes) {
        const int rc = pa_ctx_grow(ctx, (void**)&f->flags, &f->bytes, need);
        if (rc) return rc;
        // (zero from here on: a call leaves them as it found them)
        if ((e = hipMemsetAsync(f->flags, 0, f->bytes, ctx->stream)) != hipSuccess) { f->bytes = 0; return block_fail_hip(ctx, e, who); }
      }
      p.flags = f->flags;
    }
  }
  p.n_layers = 0;
  hipError_t e = hipSuccess;
  for (const pa_layer& L : ctx->layers) {
    if (!L.k) continue;
    for (uint32_t w = 0; w < per; w++) p.t[p.n_layers * per + w] = L.tensor((int)w);
    layers--;
    if (++p.n_layers == PA_COMPACT_LAYERS || !layers) {
      if ((e = pa_launch_compact(p, ctx->stream)) != hipSuccess) return block_fail_hip(ctx, e, who);
      p.n_layers = 0;
    }
  }
  return PA_OK;
}
