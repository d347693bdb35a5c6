// Shared by the kernels of the paged 8-bit key/value cache.
//
// The code layouts are those the attention kernels load matrix operands in,
// 16 bytes a lane and no shuffle on the way: a key's 16-byte piece holds 16
// consecutive elements of one token (the product over elements), a value's
// 16 consecutive tokens of one element (the product over tokens), and the
// pieces a wave loads together lie in runs of 256 bytes and more.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "decode_kernel/dk_kv.h"
#include "dk_device.hpp"

namespace dk {

constexpr float kCodeMax = 127.0f;

// Where things are in the cache; page_shift = log2(page_size).
struct KvView {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  int pages, heads, page_shift;
};

__device__ __forceinline__ float bf2f(uint32_t lo16) {
  return __builtin_bit_cast(float, lo16 << 16);
}

// Element `lo`/`hi` of a packed pair of fp16 (kBf16: bf16) as fp32.
template <bool kBf16>
__device__ __forceinline__ float pair_lo(uint32_t w) {
  return kBf16 ? __builtin_bit_cast(float, w << 16) : h2f((uint16_t)w);
}
template <bool kBf16>
__device__ __forceinline__ float pair_hi(uint32_t w) {
  return kBf16 ? __builtin_bit_cast(float, w & 0xFFFF0000u) : h2f((uint16_t)(w >> 16));
}

// fp32 to bf16, to the nearest, ties to even; NaN stays NaN.
__device__ __forceinline__ uint16_t f2bf(float f) {
  return __builtin_bit_cast(uint16_t, (__bf16)f);
}

template <int kDtype>
__device__ __forceinline__ uint16_t to_half_bits(float f) {
  return kDtype == DK_KV_BF16 ? f2bf(f) : f2h(f);
}

// Byte i of a word as a signed integer.
__device__ __forceinline__ int code_of(uint32_t w, int i) {
  return (int32_t)(w << (24 - 8 * i)) >> 24;
}

}  // namespace dk
