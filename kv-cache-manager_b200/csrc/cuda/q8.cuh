// Pages of keys or values in 8 bits, as the kernels around them see them.
//
// Codes are e4m3 (a sign, four bits of exponent, three of fraction; 0x7f and 0xff are not-a-number), a cache is [pages, nkv,
// block_size, hd] bytes and has one float32 scale for each page and KV head, [pages, nkv].  An element stands for scale * code.
// The scale is a power of two, the least 2^e with 448 * 2^e not below the largest finite element of the page and head, e >= -60
// (448 is the largest code).  The codes have exponents of their own, so a power of two costs them no precision, and in return
//   * scale * code is exact in bfloat16 and float32, codes are exact in float16,
//   * a page whose scale grows is brought to the new one by shifting exponents: only elements that fall below 2^-6 of
//     the new scale are rounded again,
//   * the scale of a value can ride on the exponent of its probability:  2^x * 2^e = 2^(x + e).
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace kvcm {
namespace q8 {

constexpr int kMaxBlock = 1 << 16;               // largest page, in rows: counts of keys stay far from 2^31
constexpr int kLeast = -60;                      // exponent of the smallest scale: zeros do not get a scale that float32 sums lose

// Keys that a request's row of the page table has room for: contexts end there (a step that was refused may leave a longer one).
inline int max_keys(int max_blocks, int block_size) {
  const long long n = (long long)max_blocks * block_size;
  return n < (1 << 30) ? int(n) : 1 << 30;
}

// The page of head `kvh`, in pages of one head.  Page ids outside the pool are taken into it: a wrong table reads a wrong page, not
// foreign memory.
__device__ __forceinline__ size_t head_page(int page, int kvh, int nkv, int num_pages) {
  page = min(max(page, 0), num_pages - 1);
  return size_t(page) * nkv + kvh;
}

// The scale for a largest element (finite): 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float largest) {
  const uint32_t b = __float_as_uint(largest);
  const int e = int(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(uint32_t(max(e, kLeast) + 127) << 23);
}
// 1 / scale, of a power of two.
__device__ __forceinline__ float reciprocal(float scale) { return __uint_as_float(0x7f000000u - __float_as_uint(scale)); }

// Two codes of two floats (a in the low byte); beyond 448 they stay at 448, not-a-number becomes not-a-number.
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;\n" : "=h"(r) : "f"(a), "f"(b));
  return r;
}
// Two codes as float16, exact (the low byte first).
__device__ __forceinline__ uint32_t halves2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"(uint16_t(codes)));
  return r;
}
__device__ __forceinline__ float2 floats2(uint32_t codes) {
  const uint32_t h = halves2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Four codes times a power of two.
__device__ __forceinline__ void values4(uint32_t codes, float scale, float* x) {
  const float2 a = floats2(codes & 0xffffu), b = floats2(codes >> 16);
  x[0] = a.x * scale; x[1] = a.y * scale; x[2] = b.x * scale; x[3] = b.y * scale;
}

}  // namespace q8
}  // namespace kvcm
