// The drafted-tree mask as the attention kernel reads it (no HIP types: host tests build it alone).
#pragma once
#include <cstdint>
#ifdef __HIP__
#define PA_HOST_DEVICE __host__ __device__
#else
#define PA_HOST_DEVICE
#endif

// Bit i: the column whose mask words these are, of a draft of n rows, sees row off + i of the draft (off above -32).  Rows in front of the draft are the context's and seen, rows from n on are
// not; words from ceil(n / 32) on are not read.
PA_HOST_DEVICE static inline uint32_t mask_window(const uint32_t* words, int off, uint32_t n) {
  const int w0 = off >> 5, sh = off & 31;
  auto word = [&](int w) -> uint32_t {
    if (w < 0) return 0xffffffffu;
    if ((uint32_t)w * 32 >= n) return 0u;
    const uint32_t left = n - (uint32_t)w * 32, v = words[w];
    return left >= 32 ? v : v & ((1u << left) - 1);
  };
  const uint32_t lo = word(w0);
  return sh ? lo >> sh | word(w0 + 1) << (32 - sh) : lo;
}
