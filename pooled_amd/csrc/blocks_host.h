// What the host sides of the blocks beside attention share: errors, the context's device, memory ranges.
#pragma once
#include "pa_internal.h"
#include <algorithm>

// the message of a failing call; an allocation that fails on the way leaves the old message
static inline int block_fail(pa_ctx* ctx, int code, const char* who, const char* msg) {
  try { ctx->err = std::string(who) + ": " + msg; } catch (...) {}
  return code;
}
static inline int block_fail_hip(pa_ctx* ctx, hipError_t e, const char* who) {
  return block_fail(ctx, e == hipErrorOutOfMemory ? PA_ERR_NOMEM : PA_ERR_HIP, who, hipGetErrorString(e));
}

// the context's device while a call allocates or launches, whichever device the caller has made current
struct DeviceGuard {
  int before = -1;
  explicit DeviceGuard(int device) {
    int now = -1;
    if (hipGetDevice(&now) == hipSuccess && now != device && hipSetDevice(device) == hipSuccess) before = now;
  }
  ~DeviceGuard() { if (before >= 0) (void)hipSetDevice(before); }
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
};

static inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }
struct Span { const void* p; size_t bytes; };
static inline Span cols(const void* p, uint32_t n, uint32_t stride, uint32_t col, size_t elem) { return {p, ((size_t)(n - 1) * stride + col) * elem}; }
static inline bool overlap(const Span& a, const Span& b) {
  return a.p && b.p && a.bytes && b.bytes && (uintptr_t)a.p < (uintptr_t)b.p + b.bytes && (uintptr_t)b.p < (uintptr_t)a.p + a.bytes;
}
