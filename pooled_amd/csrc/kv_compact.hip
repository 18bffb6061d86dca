// Compaction of the caches to a list of their rows, in place, on gfx950: row dst + i of every cache becomes what row list[i] was.
//
// The list ascends and list[i] >= dst + i, so row dst + i is the source of a target at or before i alone: a workgroup that walks the list in order, each round's rows in
// registers before any of them is stored, never reads a row that it has overwritten, whatever the list.  Workgroups share nothing: each has a (tensor, kv head) plane and a slice
// of its rows' bytes.
#include "tree_internal.h"

typedef unsigned int u4 __attribute__((ext_vector_type(4)));

#define CT_ROUND 8            // rows of a thread a round

// units: 16-byte units of a slice of a row; a power of two
__global__ __launch_bounds__(256) void pa_compact_kernel(CompactParams p, uint32_t units) {
  const uint32_t slices = p.row_bytes / 16 / units, wg = blockIdx.x;
  const uint32_t slice = wg % slices, plane = wg / slices % p.n_planes, t = wg / slices / p.n_planes;
  const uint32_t n = min(p.sel[0], p.max_rows), per = 256 / units;           // rows of the workgroup at a time
  const uint32_t r0 = threadIdx.x / units, u = slice * units + threadIdx.x % units;
  unsigned char* base = (unsigned char*)p.t[t] + (size_t)plane * p.head_rows * p.row_bytes + u * 16;
  for (uint32_t i0 = 0; i0 < n; i0 += per * CT_ROUND) {
    u4 v[CT_ROUND];
#pragma unroll
    for (int k = 0; k < CT_ROUND; k++) {
      const uint32_t i = min(i0 + k * per + r0, n - 1);
      v[k] = *(const u4*)(base + (size_t)min(p.sel[1 + i], p.max_seq - 1) * p.row_bytes);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int k = 0; k < CT_ROUND; k++) {
      const uint32_t i = i0 + k * per + r0;
      if (i < n) *(u4*)(base + (size_t)(p.dst_row + i) * p.row_bytes) = v[k];
    }
  }
}

hipError_t pa_launch_compact(const CompactParams& p, hipStream_t s) {
  if (!p.n_tensors || p.n_tensors > PA_COMPACT_TENSORS || !p.row_bytes || p.row_bytes % 16 || (uint64_t)p.dst_row + p.max_rows > p.max_seq) return hipErrorInvalidValue;
  const uint32_t row_units = p.row_bytes / 16, units = row_units < 8 ? row_units : 8;       // slices of 128 bytes, a cache line
  if ((units & (units - 1)) || row_units % units) return hipErrorInvalidValue;
  hipLaunchKernelGGL(pa_compact_kernel, dim3(p.n_tensors * p.n_planes * (row_units / units)), dim3(256), 0, s, p, units);
  return hipGetLastError();
}
