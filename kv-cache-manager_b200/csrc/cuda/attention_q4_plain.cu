// Paged attention over a cache in 4 bits (layout and formulas: q4.cuh), one block per (row, query head), softmax and sums in
// float32 whatever the storage type of q: the attention of float32 rows and of head sizes that the tensor-core kernels do not
// take, and their twin in tests.  Head sizes are multiples of 8 up to 256, any page size, any number of heads and groups, optional window, capped scores
// and sinks (as in attention_plain.cu).
//
// A chunk of 512 keys at a time: a thread forms the scores of whole keys (a key's codes are hd/2 bytes), then the products with
// V are dealt out as words of eight elements, groups of threads taking every n-th key each, joined at the end in the groups'
// order.  What bounds it is instructions: a code costs a shift, a mask, a conversion and a fused multiply-add, and it costs them once for
// every query head and row that reads it.  B200, float32 rows: 8 requests of some 1,536 keys, 32 heads on 4 of 64, 49 us, 64 of 100 to
// 8,192 keys, 32 on 8 of 128, 722 us (0.5 and 16 at the rate of a copy); a portion of 2,048 rows 4.9 ms (7.0 TFLOP/s), of heads of 40,
// 8 on 2, 0.47 ms.
#include "packed.cuh"
#include "pdl.cuh"
#include "q4.cuh"

namespace kvcm {

constexpr int kQ4PlainThreads = 128;
constexpr int kQ4PlainChunk = 512;

struct PlainQ4Params {
  const void* q; long long q_stride;
  void* out; long long out_stride;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const int* block_tables; int max_blocks, max_keys;      // keys that a request's table has pages for
  const int* row_seq; const int* positions;
  int nh, nkv, hd, block_size, num_pages, window;
  float scale, softcap;
  const float* sink;
};

template <typename T>
__global__ void __launch_bounds__(kQ4PlainThreads) attention_q4_plain_kernel(PlainQ4Params p) {
  __shared__ __align__(16) float qs[256];
  __shared__ float weight[kQ4PlainChunk];                          // scores, then probabilities
  __shared__ unsigned head_of[kQ4PlainChunk];                      // page * nkv + kvh of every key of the chunk
  __shared__ __align__(16) float joined[kQ4PlainThreads * 8];
  __shared__ float joined_z[kQ4PlainThreads];
  __shared__ float scratch[33];
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int kvh = h / (p.nh / p.nkv);
  const int position = p.positions[row], ctx = min(position, p.max_keys - 1) + 1;      // (a context ends with its table)
  const int lo = first_visible(position, p.window, 0);
  const int words = p.hd / 8, row_bytes = p.hd / 2;
  const size_t bytes = q4::page_bytes(p.block_size, p.hd);
  const int* table = p.block_tables + size_t(p.row_seq[row]) * p.max_blocks;

  float q_sum = 0.f;
  for (int d = tid; d < p.hd; d += kQ4PlainThreads) {
    qs[d] = ldf(static_cast<const T*>(p.q) + size_t(row) * p.q_stride + size_t(h) * p.hd + d) * p.scale;
    q_sum += qs[d];
  }
  q_sum = block_sum(q_sum, scratch);                               // (its barriers also publish qs)

  const int groups = kQ4PlainThreads / words;                      // words <= 32
  const int group = tid / words, word = tid - group * words;
  float m = p.sink ? p.sink[h] : -INFINITY, l = p.sink ? 1.f : 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, acc_z = 0.f;
  for (int c0 = lo; c0 < ctx; c0 += kQ4PlainChunk) {
    const int n = min(kQ4PlainChunk, ctx - c0);
    float local_max = -INFINITY;
    for (int j = tid; j < n; j += kQ4PlainThreads) {
      const int pi = (c0 + j) / p.block_size, off = c0 + j - pi * p.block_size;
      const int page = min(max(table[pi], 0), p.num_pages - 1);
      head_of[j] = unsigned(page) * p.nkv + kvh;
      const uint8_t* base = p.k_cache + size_t(head_of[j]) * bytes;
      const uint32_t pair = *reinterpret_cast<const uint32_t*>(base + size_t(p.block_size) * row_bytes + off * 4);
      float s = 0.f;
#pragma unroll 2
      for (int w = 0; w < words; ++w) {
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(base + size_t(off) * row_bytes + w * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(qs[w * 8 + e], q4::code_of(codes, e), s);
      }
      s = fmaf(q4::scale_of(pair), s, q4::zero_of(pair) * q_sum);
      if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
      weight[j] = s;
      local_max = fmaxf(local_max, s);
    }
    const float m_new = fmaxf(m, block_max(local_max, scratch));
    const float factor = (m == -INFINITY) ? 0.f : expf(m - m_new);
    float local_sum = 0.f;
    for (int j = tid; j < n; j += kQ4PlainThreads) {
      const float e = expf(weight[j] - m_new);
      weight[j] = e;
      local_sum += e;
    }
    l = l * factor + block_sum(local_sum, scratch);                // (its barriers also publish weight and head_of)
    m = m_new;
    if (group < groups) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= factor;
      acc_z *= factor;
      for (int j = group; j < n; j += groups) {
        const int off = (c0 + j) % p.block_size;
        const uint8_t* base = p.v_cache + size_t(head_of[j]) * bytes;
        const uint32_t pair = *reinterpret_cast<const uint32_t*>(base + size_t(p.block_size) * row_bytes + off * 4);
        const uint32_t codes = *reinterpret_cast<const uint32_t*>(base + size_t(off) * row_bytes + word * 4);
        const float w = weight[j] * q4::scale_of(pair);
        acc_z = fmaf(weight[j], q4::zero_of(pair), acc_z);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, q4::code_of(codes, e), acc[e]);
      }
    }
    __syncthreads();                                               // weight is overwritten by the next chunk
  }
  if (group < groups) {
#pragma unroll
    for (int e = 0; e < 8; ++e) joined[(group * words + word) * 8 + e] = acc[e];
    if (word == 0) joined_z[group] = acc_z;
  }
  __syncthreads();
  const float inv = l > 0.f ? 1.f / l : 0.f;
  for (int d = tid; d < p.hd; d += kQ4PlainThreads) {
    float sum = 0.f, z = 0.f;
    for (int g = 0; g < groups; ++g) {
      sum += joined[g * p.hd + d];
      z += joined_z[g];
    }
    stf(static_cast<T*>(p.out) + size_t(row) * p.out_stride + size_t(h) * p.hd + d, (sum + z) * inv);
  }
}

template <typename T>
int launch_plain_q4(const PlainQ4Params& p, int rows, cudaStream_t s) {
  return pdl_launch(attention_q4_plain_kernel<T>, dim3(rows, p.nh), dim3(kQ4PlainThreads), 0, s, p);
}

}  // namespace kvcm

using namespace kvcm;

#define KVCM_PLAIN_Q4(SUFFIX, T)                                                                                               \
  KVCM_API int kvcm_attention_plain_q4_##SUFFIX(                                                                               \
      const void* q, long long q_stride, void* out, long long out_stride, const void* k_cache, const void* v_cache, int num_pages, \
      const int* block_tables, int max_blocks, const int* row_seq, const int* positions, int rows, int nh, int nkv, int hd,    \
      int block_size, float scale, int window, float softcap, const float* sink, void* stream) {                               \
    if (rows == 0) return 0;                                                                                                   \
    if (nkv <= 0 || nh % nkv || hd < 8 || hd > 256 || hd % 8 || block_size <= 0 || block_size > q4::kMaxBlock || max_blocks <= 0 || num_pages <= 0 || nh > 65535)               \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    PlainQ4Params p;                                                                                                           \
    p.q = q; p.q_stride = q_stride; p.out = out; p.out_stride = out_stride;                                                    \
    p.k_cache = (const uint8_t*)k_cache; p.v_cache = (const uint8_t*)v_cache; p.num_pages = num_pages;                         \
    p.block_tables = block_tables; p.max_blocks = max_blocks; p.max_keys = q4::max_keys(max_blocks, block_size); p.row_seq = row_seq; p.positions = positions;                    \
    p.nh = nh; p.nkv = nkv; p.hd = hd; p.block_size = block_size; p.window = window;                                           \
    p.scale = scale; p.softcap = softcap; p.sink = sink;                                                                       \
    return launch_plain_q4<T>(p, rows, (cudaStream_t)stream);                                                                  \
  }

KVCM_PLAIN_Q4(bf16, bf16)
KVCM_PLAIN_Q4(f32, float)

KVCM_PACKED(kvcm_attention_plain_q4_bf16)
KVCM_PACKED(kvcm_attention_plain_q4_f32)
