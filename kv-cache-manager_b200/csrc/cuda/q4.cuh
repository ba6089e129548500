// Pages of keys or values in 4 bits, as the kernels around them see them.
//
// The page of one KV head is `block_size` rows of hd/2 bytes of codes, then `block_size` pairs (scale, zero) in bfloat16, the
// whole rounded up to 16 bytes (so that rows of 32 elements and more start on 16 bytes); a cache is [pages, nkv, page_bytes].
// One row is one key or value of one head and stands for  x[d] = zero + scale * code[d],  code 0..15.
// One scale a row: the products of a row with a query, and of a probability with a row, then need the scale once a score and
// not once an element:   q.x = scale (q.code) + zero sum(q),   sum_j p_j x_j[d] = sum_j (p_j scale_j) code_j[d] + sum_j p_j zero_j,
// and the codes themselves go into the tensor cores, where small whole numbers are exact.
//
// Word m (32 bits) of a row holds element 8m + 2i at bits 4i and element 8m + 2i + 1 at bits 16 + 4i: one shift and one
// and-or give two neighbouring elements as the two bfloat16 of a register (0x4300 | code is 128 + code).
#pragma once
#include "common.cuh"

namespace kvcm {
namespace q4 {

constexpr int kMaxBlock = 1 << 16;               // largest page, in rows: counts of keys stay far from 2^31

__host__ __device__ inline size_t page_bytes(int block_size, int hd) {
  return (size_t(block_size) * (hd / 2 + 4) + 15) & ~size_t(15);
}

// Keys that a request's row of the page table has room for: contexts end there (a step that was refused may leave a longer one).
inline int max_keys(int max_blocks, int block_size) {
  const long long n = (long long)max_blocks * block_size;
  return n < (1 << 30) ? int(n) : 1 << 30;
}

// The page of head `kvh`.  Page ids outside the pool are taken into it: a wrong table reads a wrong page, not foreign memory.
__device__ __forceinline__ size_t page_base(int page, int kvh, int nkv, int num_pages, size_t bytes) {
  page = min(max(page, 0), num_pages - 1);
  return (size_t(page) * nkv + kvh) * bytes;
}

__device__ __forceinline__ float scale_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float zero_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// Elements 2i and 2i + 1 of a word as 128 + code, two bfloat16.
__device__ __forceinline__ uint32_t two_codes_128(uint32_t word, int i) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;\n" : "=r"(r) : "r"(word >> (4 * i)));    // (a & b) | c
  return r;
}
__device__ __forceinline__ float code_of(uint32_t word, int e) { return float((word >> (4 * (e >> 1) + 16 * (e & 1))) & 15u); }

// Eight codes as a word.
__device__ __forceinline__ uint32_t pack_codes(const uint32_t (&c)[8]) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) w |= c[e] << (4 * (e >> 1) + 16 * (e & 1));
  return w;
}

}  // namespace q4
}  // namespace kvcm
