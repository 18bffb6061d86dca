// What the host sides of the blocks beside attention share: errors, the context's device; with spans.h, memory ranges.
#pragma once
#include "pa_internal.h"
#include "spans.h"
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
