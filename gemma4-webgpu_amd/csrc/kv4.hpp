// kv4.hpp — where a row of the 4-bit paged K/V pool lies (g4_kv4_params in g4hip.h).
#pragma once
#include "kv8.hpp"

namespace g4kv4 {

constexpr int BLOCK = 32;  // dims of a scale
constexpr uint32_t BAD = 255;  // the scale byte of a row and head that is not finite

struct Pool {
  uint8_t *k, *v, *ks, *vs;
  float* mass;  // or null
};
// A row is a page's slot of a KV head.
struct Shape {
  uint32_t page_size, nkh, hd;
  __device__ __forceinline__ size_t row(uint32_t page, uint32_t slot, uint32_t h) const {
    return (size_t)page * (page_size * nkh) + (slot * nkh + h);  // (a page has 2^16 rows at most)
  }
  __device__ __forceinline__ size_t code(uint32_t page, uint32_t slot, uint32_t h) const {
    return row(page, slot, h) * (hd / 2);
  }
  __device__ __forceinline__ size_t k_scale(uint32_t page, uint32_t slot, uint32_t h, uint32_t block) const {
    return row(page, slot, h) * (hd / BLOCK) + block;
  }
  __device__ __forceinline__ size_t v_scale(uint32_t page, uint32_t slot, uint32_t h, uint32_t block) const {
    return ((((size_t)page * (page_size / 16) + slot / 16) * nkh + h) * (hd / BLOCK) + block) * 16 + slot % 16;
  }
};

// 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.
__device__ __forceinline__ float value_of(uint32_t code) {
  const uint32_t m = code & 7u;
  const float x = m < 2 ? 0.5f * (float)m : __uint_as_float((((m >> 1) + 126u) << 23) | ((m & 1u) << 22));
  return code & 8u ? -x : x;
}
// 2^(byte - 127); NaN for 255.
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return byte == BAD ? __builtin_nanf("") : byte ? __uint_as_float(byte << 23) : 0x1p-127f;
}

}  // namespace g4kv4
