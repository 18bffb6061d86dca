// Declarations shared by the host side of the drafted-tree calls (pa_tree.hip) and their gfx950 kernels.
#pragma once
#include "pa_internal.h"

// n / d for all n below a bound, as mulhi(n, ceil(2^32 / d)), which is exact while bound x d < 2^32; 0 where it is not, or d is 1
static inline uint32_t div_magic(uint64_t bound, uint32_t d) { return d > 1 && bound * d < (1ull << 32) ? (uint32_t)(((1ull << 32) + d - 1) / d) : 0u; }
static __device__ inline uint32_t div_by(uint32_t n, uint32_t d, uint32_t magic) { return magic ? __umulhi(n, magic) : d == 1 ? n : n / d; }

// ---- attention of a tree of drafted tokens (attn_tree.hip) ----
struct TreeParams {
  const float* q; const float* gate;            // f32 [n_cols][stride], heads of head_dim
  const void* k_cache; const void* v_cache;     // f16 or int8, [nKV][max_seq + 32][hd]
  const float* k_scale; const float* v_scale;   // int8 caches: one f32 scale per 32 values
  const uint32_t* mask;                         // [n_cols][mask_stride]: bit j: the column sees row base_pos + j
  float* part_o; float2* part_ml;               // partials of the splits: O / l and (m, l), see attn_tree.hip
  void* out;                                    // [n_cols][out_stride]
  uint32_t q_stride, gate_stride, mask_stride, out_stride;
  uint32_t n_heads, n_kv_heads, group;          // group = nH / nKV
  uint32_t base_pos, n_cols, max_seq;
  uint32_t n_splits, split_tiles;               // splits of the context, 32-row tiles of each
  uint32_t n_groups, group_rows;                // groups of stacked rows of a kv head (row = column x G + head), rows of each
  int out_f16;
  float scale;                                  // 1 / sqrt(hd)
  uint32_t ng_magic, ns_magic, g_magic, rows_magic; // div_magic of n_groups, n_splits, group and n_cols x group (set by the launchers)
};
#define TREE_W 8              // waves of a workgroup, two a SIMD: one wave a SIMD gets half of what the LDS delivers
// what a call runs as: rows a wave holds (16 nb), groups of rows, splits
struct TreePlan { uint32_t nb, n_groups, group_rows, n_splits, split_tiles; };
hipError_t pa_launch_tree(const TreeParams& p, const TreePlan& pl, uint32_t hd, hipStream_t s, const PaTiming* t);
hipError_t pa_launch_tree_merge(const TreeParams& p, uint32_t hd, hipStream_t s, const PaTiming* t);

// ---- pre-step with positions of each column's own (glue_at.hip) ----
struct GlueAtParams {
  const float* q_in; const float* k_in; const float* v_in;
  const float* qw; const float* kw;             // norm weights [hd]
  const float* inv_freq; const float2* rope_tab;  // [n_rot / 2]; [tab_rows][n_rot / 2] (cos, sin) or nullptr
  const uint32_t* pos;                          // [axes][pos_stride]
  float* q_out; float* gate_out;                // [n_cols][nH * hd]
  void* k_cache; void* v_cache;                 // f16 or int8 [nKV][head_rows][hd]
  float* ks_cache; float* vs_cache;
  uint32_t head_rows, tab_rows;
  uint32_t q_stride, k_stride, v_stride, pos_stride;
  uint32_t n_heads, n_kv_heads, head_dim, n_rot;
  uint32_t base_row, n_cols, flags;
  float eps;
  uint32_t n_axes, per_col_magic;               // per_col_magic: set by the launcher
  uint32_t axis_of_pair[8];                     // two bits a pair, sixteen pairs a word
};
hipError_t pa_launch_glue_at(const GlueAtParams& p, hipStream_t s);

// ---- compaction of the caches to a list of rows (kv_compact.hip) ----
#define PA_COMPACT_LAYERS 32u
struct CompactParams {
  void* t[4 * PA_COMPACT_LAYERS];               // a layer's K, V (and their scales): [planes][head_rows][row_bytes or scale_bytes]
  const uint32_t* sel;                          // n, then n rows, ascending
  uint32_t* flags;                              // pa_compact_flags words, zero before and after a call; nullptr: none
  uint32_t n_layers, n_planes, head_rows;
  uint32_t row_bytes, scale_bytes;              // scale_bytes 0: f16 caches
  uint32_t dst_row, max_rows, max_seq;
};
bool pa_compact_one_round(const CompactParams& p);        // a list so short that no segments are needed
size_t pa_compact_flags(const CompactParams& p);          // words of p.flags
hipError_t pa_launch_compact(const CompactParams& p, hipStream_t s);
