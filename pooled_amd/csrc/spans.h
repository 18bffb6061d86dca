// Memory that a call's arguments take up, for the checks in front of a launch.
#pragma once
#include <cstddef>
#include <cstdint>

struct Span { const void* p; size_t bytes; };
static inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
// n columns of `col` elements, `stride` from one to the next: from the first byte to the last
static inline Span cols(const void* p, uint32_t n, uint32_t stride, uint32_t col, size_t elem) { return {p, ((size_t)(n - 1) * stride + col) * elem}; }
static inline bool overlap(const Span& a, const Span& b) {
  return a.p && b.p && a.bytes && b.bytes && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
}

// n columns of `bytes` bytes, `step` bytes from one to the next (step >= bytes)
struct Columns { const void* p; size_t step, bytes; };
// does [x, x + bytes) meet one of n columns?
static inline bool meets(uintptr_t x, size_t bytes, const Columns& b, uint32_t n) {
  const uintptr_t p = (uintptr_t)b.p;
  const size_t j = x < p + b.bytes ? 0 : (x - p - b.bytes) / b.step + 1;      // the first column that ends behind x
  return j < n && p + j * b.step < x + bytes;
}
// do two sets of n columns share a byte?  Columns may lie between one another.
static inline bool columns_meet(const Columns& a, const Columns& b, uint32_t n) {
  if (!overlap({a.p, (n - 1) * a.step + a.bytes}, {b.p, (n - 1) * b.step + b.bytes})) return false;
  if (a.step == b.step) return meets((uintptr_t)a.p, a.bytes, b, n) || meets((uintptr_t)b.p, b.bytes, a, n);   // column i meets j as 0 meets j - i, or i - j meets 0
  for (uint32_t i = 0; i < n; i++) if (meets((uintptr_t)a.p + i * a.step, a.bytes, b, n)) return true;
  return false;
}
