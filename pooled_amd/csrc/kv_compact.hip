// Compaction of the caches to a list of their rows, in place, on gfx950: row dst + i of every cache becomes what row list[i] was.
//
// The list ascends and list[i] >= dst + i, so row dst + i is the source of targets at or before i alone.  Hence two forms, neither of which reads a row that was overwritten:
//   walk      a workgroup has a (tensor, kv head) plane and a slice of its rows' bytes and walks the list in order, each round's rows in registers before one of them is
//             stored.  Workgroups share nothing.  For the accepted path of a draft (one round), and for recorded calls, whose replays nothing keeps from running beside another call.
//   segments  a workgroup has 64 KB of a plane's list: it reads its rows into registers, says so in a flag, waits for the flags of the plane's earlier segments and stores.
//             A segment reads without waiting for anybody and waits only for segments in front of it in its plane.  Workgroups take segments by ticket, in the order in which they
//             start, so those in front are with workgroups that run already and every wait ends, whatever else the device runs and in whatever order workgroups start, as long as no other launch has the same flags meanwhile (each stream has its own).  Whole
//             lines in and out, all CUs busy.  Flags and tickets are zero between calls: the plane's last workgroup through its wait clears them.
// Bound by HBM (two transfers of each row that moves) or, for a few rows, by one launch.  8000 of 16003 rows of six layers of 8 heads of 128 (394 MB read and written): 78 us = 5.05 TB/s,
// the rate of a large copy; 10001 of 30011 int8 rows of three layers of 4 heads of 256 (138 MB): 38 us, where the scales' 32 bytes a row cost whole lines of 128 (23 MB read for 8).  Five
// rows in ten layers: 2.9 us.
#include "tree_internal.h"

typedef unsigned int u4 __attribute__((ext_vector_type(4)));

#define CT_ROUND 8            // rows of a thread a round of the walk
#define CT_SEG 16             // 16-byte units of a thread in a segment

struct CompactPlane { unsigned char* base; uint32_t row_bytes, units; };       // units: 16-byte units of a row, a power of two
static __device__ inline CompactPlane plane_of(const CompactParams& p, uint32_t tensor, uint32_t plane, uint32_t scales) {
  const uint32_t per = p.scale_bytes ? 4 : 2, rb = scales ? p.scale_bytes : p.row_bytes;
  return { (unsigned char*)p.t[tensor / 2 * per + 2 * scales + tensor % 2] + (size_t)plane * p.head_rows * rb, rb, rb / 16 };
}

// workgroups: (tensor, plane, 128-byte slice of a row) of the values, then (tensor, plane) of the scales
__global__ __launch_bounds__(256) void pa_compact_walk_kernel(CompactParams p) {
  const uint32_t planes = 2 * p.n_layers * p.n_planes, slices = p.row_bytes / 128;
  const uint32_t scales = blockIdx.x >= planes * slices, wg = scales ? blockIdx.x - planes * slices : blockIdx.x;
  const uint32_t slice = scales ? 0 : wg % slices, pl = scales ? wg : wg / slices;
  const CompactPlane c = plane_of(p, pl / p.n_planes, pl % p.n_planes, scales);
  const uint32_t n = min(p.sel[0], p.max_rows), units = min(c.units, 8u), per = 256 / units;           // rows of the workgroup at a time
  const uint32_t r0 = threadIdx.x / units;
  unsigned char* base = c.base + slice * 128 + threadIdx.x % units * 16;
  for (uint32_t i0 = 0; i0 < n; i0 += per * CT_ROUND) {
    u4 v[CT_ROUND];
#pragma unroll
    for (int k = 0; k < CT_ROUND; k++) {
      const uint32_t i = min(i0 + k * per + r0, n - 1);
      v[k] = *(const u4*)(base + (size_t)min(p.sel[1 + i], p.max_seq - 1) * c.row_bytes);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < CT_ROUND; k++) {
      const uint32_t i = i0 + k * per + r0;
      if (i < n) *(u4*)(base + (size_t)(p.dst_row + i) * c.row_bytes) = v[k];
    }
  }
}

// workgroups: (segment, tensor, plane) of the values, the segment slowest, then those of the scales; flags in the same order, and behind them a line of each plane: tickets taken, and how many
// are through their waits
#define CT_LINE 32            // words of a plane's line
__global__ __launch_bounds__(256) void pa_compact_segment_kernel(CompactParams p, uint32_t value_segs) {
  const uint32_t planes = 2 * p.n_layers * p.n_planes;
  const uint32_t scales = blockIdx.x >= planes * value_segs, pl = blockIdx.x % planes, segs = scales ? gridDim.x / planes - value_segs : value_segs;
  uint32_t* flags = p.flags + (scales ? planes * value_segs : 0) + pl;       // segment k's: flags[k * planes]
  uint32_t* line = p.flags + gridDim.x + (scales * planes + pl) * CT_LINE;
  __shared__ uint32_t ticket;
  if (threadIdx.x == 0) {
    const uint32_t t = __hip_atomic_fetch_add(line, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (t == segs - 1) __hip_atomic_store(line, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    ticket = t;
  }
  __syncthreads();
  const uint32_t seg = __builtin_amdgcn_readfirstlane(ticket);
  const CompactPlane c = plane_of(p, pl / p.n_planes, pl % p.n_planes, scales);
  const uint32_t n = min(p.sel[0], p.max_rows), sh = 31 - __clz(c.units), rows = 256 * CT_SEG >> sh, i0 = seg * rows;
  if (i0 >= n) return;
  unsigned char* base = c.base + (threadIdx.x & (c.units - 1)) * 16;
  const uint32_t step = 256 >> sh, r0 = threadIdx.x >> sh;
  uint32_t src[CT_SEG];
  u4 v[CT_SEG];
#pragma unroll
  for (int k = 0; k < CT_SEG; k++) src[k] = p.sel[1 + min(i0 + k * step + r0, n - 1)];
#pragma unroll
  for (int k = 0; k < CT_SEG; k++) {
    src[k] = min(src[k], p.max_seq - 1);
    v[k] = __builtin_nontemporal_load((const u4*)(base + (size_t)src[k] * c.row_bytes));
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();                                  // the segment's rows are in registers
  if (threadIdx.x == 0) __hip_atomic_store(flags + (size_t)seg * planes, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (uint32_t k = threadIdx.x; k < seg; k += 256)
    while (!__hip_atomic_load(flags + (size_t)k * planes, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) __builtin_amdgcn_s_sleep(1);
  __syncthreads();
  if (threadIdx.x < 64) {
    const uint32_t live = (n + rows - 1) / rows;
    uint32_t* through = line + 1;
    uint32_t before = 0;
    if (threadIdx.x == 0) before = __hip_atomic_fetch_add(through, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane(before) == live - 1) {
      for (uint32_t k = threadIdx.x; k < live; k += 64) __hip_atomic_store(flags + (size_t)k * planes, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (threadIdx.x == 0) __hip_atomic_store(through, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
#pragma unroll
  for (int k = 0; k < CT_SEG; k++) {
    const uint32_t i = i0 + k * step + r0;
    if (i < n && src[k] != p.dst_row + i) __builtin_nontemporal_store(v[k], (u4*)(base + (size_t)(p.dst_row + i) * c.row_bytes));
  }
}

static uint32_t segments(const CompactParams& p, uint32_t row_bytes) { return row_bytes ? (uint32_t)(((uint64_t)p.max_rows * row_bytes + 256 * CT_SEG * 16 - 1) / (256 * CT_SEG * 16)) : 0; }
bool pa_compact_one_round(const CompactParams& p) { return p.max_rows <= 32 * CT_ROUND; }
static size_t segment_wgs(const CompactParams& p) { return (size_t)2 * p.n_layers * p.n_planes * ((size_t)segments(p, p.row_bytes) + segments(p, p.scale_bytes)); }
size_t pa_compact_flags(const CompactParams& p) { return segment_wgs(p) + (size_t)4 * p.n_layers * p.n_planes * CT_LINE; }

hipError_t pa_launch_compact(const CompactParams& p, hipStream_t s) {
  auto power = [](uint32_t b) { return b % 16 == 0 && (b & (b - 1)) == 0; };
  if (!p.n_layers || p.n_layers > PA_COMPACT_LAYERS || !p.n_planes || p.row_bytes < 128 || p.row_bytes > 4096 || !power(p.row_bytes) || p.scale_bytes > 128 || !power(p.scale_bytes) ||
      !p.max_rows || (uint64_t)p.dst_row + p.max_rows > p.max_seq) return hipErrorInvalidValue;
  const uint64_t planes = 2ull * p.n_layers * p.n_planes;
  const bool walk = pa_compact_one_round(p) || !p.flags;
  const uint64_t wgs = walk ? planes * (p.row_bytes / 128 + (p.scale_bytes ? 1 : 0)) : segment_wgs(p);
  if (wgs > 0x7fffff00ull) return hipErrorInvalidValue;
  if (walk) hipLaunchKernelGGL(pa_compact_walk_kernel, dim3((unsigned)wgs), dim3(256), 0, s, p);
  else hipLaunchKernelGGL(pa_compact_segment_kernel, dim3((unsigned)wgs), dim3(256), 0, s, p, segments(p, p.row_bytes));
  return hipGetLastError();
}
