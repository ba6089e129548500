// Attention one row and query head a block, in float32 whatever the storage type of q: over a paged cache in 8 bits (format:
// q8.cuh), and of packed prompts over their own rows.  For float32 rows and for sizes that the tensor-core kernels do not take, and
// their twin in tests.  Head sizes are multiples of 8 up to 256, any page size, any number of heads and groups, optional
// window, capped scores and sinks (as in attention_plain.cu).
//
// A chunk of 512 keys at a time: a thread forms the scores of whole keys, then the products with V are dealt out as words of eight
// elements, groups of threads taking every n-th key each, joined at the end in the groups' order.  What bounds it is instructions:
// every row and query head converts a key's elements anew.  B200: single rows of 64 requests of 8,192 keys, 32 heads on 8 of 128, 1.88 ms; four
// portions of about 1,500 rows behind 5,000 keys 80 ms; a prompt of 8,192 rows 550 ms.
#include "packed.cuh"
#include "pdl.cuh"
#include "q8.cuh"

namespace kvcm {

constexpr int kQ8PlainThreads = 128;
constexpr int kQ8PlainChunk = 512;

// Where keys and values are: in pages of 8 bits.
struct Q8Pages {
  const uint8_t* k_codes; const uint8_t* v_codes; const float* k_scale; const float* v_scale;
  const int* block_tables; int max_blocks, max_keys;      // keys that a request's table has pages for
  const int* row_seq; const int* positions;
  int nkv, hd, block_size, num_pages;

  struct Row { const int* table; };
  // The row that block `b` has, its request's keys and its position; false where there is none.
  __device__ __forceinline__ bool row(int b, int, Row& r, int& row, int& position) const {
    row = b;
    position = positions[b];
    r.table = block_tables + size_t(row_seq[b]) * max_blocks;
    return true;
  }
  __device__ __forceinline__ int most() const { return max_keys; }
  __device__ __forceinline__ size_t place(const Row& r, int key, int kvh) const {
    const int pi = key / block_size;
    return q8::head_page(r.table[pi], kvh, nkv, num_pages) * block_size + (key - pi * block_size);
  }
  __device__ __forceinline__ void load(const uint8_t* codes, const float* scale, size_t at, int word, float (&x)[8]) const {
    const uint2 u = *reinterpret_cast<const uint2*>(codes + at * hd + word * 8);
    const float s = scale[at / block_size];
    q8::values4(u.x, s, x);
    q8::values4(u.y, s, x + 4);
  }
  __device__ __forceinline__ void key8(size_t at, int word, float (&x)[8]) const { load(k_codes, k_scale, at, word, x); }
  __device__ __forceinline__ void value8(size_t at, int word, float (&x)[8]) const { load(v_codes, v_scale, at, word, x); }
};

// The rows of prompts that lie one behind another: entries [0, singles) are prompts of one row, the others' rows are named by tiles.
template <typename T> struct PromptRows {
  const T* k; const T* v; long long k_stride, v_stride;
  const int* tile_seq; const int* tile_q0; const int* seq_q_start; const int* seq_q_len;
  int tiles, tile_rows, hd;

  struct Row { int start, kvh; };
  __device__ __forceinline__ bool row(int b, int kvh, Row& r, int& row, int& position) const {
    int seq = b - tiles * tile_rows;
    position = 0;
    if (seq < 0) {
      const int t = b / tile_rows;
      seq = tile_seq[t];
      if (seq < 0) return false;
      position = tile_q0[t] + b - t * tile_rows;
    }
    if (position >= seq_q_len[seq]) return false;
    r.start = seq_q_start[seq];
    r.kvh = kvh;
    row = r.start + position;
    return true;
  }
  __device__ __forceinline__ int most() const { return 0x7fffffff; }
  __device__ __forceinline__ size_t place(const Row& r, int key, int) const { return size_t(r.start) + key; }
  __device__ __forceinline__ void load(const T* from, float (&x)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ldf(from + e);
  }
};

template <typename T, typename Keys, bool PROMPT>
__global__ void __launch_bounds__(kQ8PlainThreads)
attention_q8_plain_kernel(Keys keys, const T* q, long long q_stride, T* out, long long out_stride, int nh, int nkv, int hd, float scale,
                          int window, float softcap, const float* sink) {
  __shared__ __align__(16) float qs[256];
  __shared__ float weight[kQ8PlainChunk];                          // scores, then probabilities
  __shared__ size_t place_of[kQ8PlainChunk];
  __shared__ __align__(16) float joined[kQ8PlainThreads * 8];
  __shared__ float scratch[33];
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, tid = threadIdx.x, kvh = h / (nh / nkv);
  typename Keys::Row r;
  int row, position;
  if (!keys.row(blockIdx.x, kvh, r, row, position)) return;
  const int ctx = min(position, keys.most() - 1) + 1;              // (a context ends with its table)
  const int lo = first_visible(position, window, 0);
  const int words = hd / 8;
  for (int d = tid; d < hd; d += kQ8PlainThreads) qs[d] = ldf(q + size_t(row) * q_stride + size_t(h) * hd + d) * scale;
  __syncthreads();

  auto load = [&](bool key, size_t at, int word, float (&x)[8]) {
    if constexpr (PROMPT) keys.load((key ? keys.k + at * keys.k_stride : keys.v + at * keys.v_stride) + size_t(kvh) * hd + word * 8, x);
    else if (key) keys.key8(at, word, x);
    else keys.value8(at, word, x);
  };
  const int groups = kQ8PlainThreads / words;                      // words <= 32
  const int group = tid / words, word = tid - group * words;
  float m = sink ? sink[h] : -INFINITY, l = sink ? 1.f : 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int c0 = lo; c0 < ctx; c0 += kQ8PlainChunk) {
    const int n = min(kQ8PlainChunk, ctx - c0);
    float local_max = -INFINITY;
    for (int j = tid; j < n; j += kQ8PlainThreads) {
      const size_t at = keys.place(r, c0 + j, kvh);
      place_of[j] = at;
      float s = 0.f, x[8];
#pragma unroll 2
      for (int w = 0; w < words; ++w) {
        load(true, at, w, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(qs[w * 8 + e], x[e], s);
      }
      if (softcap > 0.f) s = softcap * tanhf(s / softcap);
      weight[j] = s;
      local_max = fmaxf(local_max, s);
    }
    const float m_new = fmaxf(m, block_max(local_max, scratch));
    const float factor = (m == -INFINITY) ? 0.f : expf(m - m_new);
    float local_sum = 0.f;
    for (int j = tid; j < n; j += kQ8PlainThreads) {
      const float e = expf(weight[j] - m_new);
      weight[j] = e;
      local_sum += e;
    }
    l = l * factor + block_sum(local_sum, scratch);                // (its barriers also publish weight and place_of)
    m = m_new;
    if (group < groups) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] *= factor;
      for (int j = group; j < n; j += groups) {
        const float w = weight[j];
        float x[8];
        load(false, place_of[j], word, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, x[e], acc[e]);
      }
    }
    __syncthreads();                                               // weight is overwritten by the next chunk
  }
  if (group < groups) {
#pragma unroll
    for (int e = 0; e < 8; ++e) joined[(group * words + word) * 8 + e] = acc[e];
  }
  __syncthreads();
  const bool none = l == 0.f;                                      // no key: zeros
  const float inv = none ? 0.f : 1.f / l;
  for (int d = tid; d < hd; d += kQ8PlainThreads) {
    float sum = 0.f;
    for (int g = 0; g < groups; ++g) sum += joined[g * hd + d];
    stf(out + size_t(row) * out_stride + size_t(h) * hd + d, none ? 0.f : sum * inv);
  }
}

}  // namespace kvcm

using namespace kvcm;

#define KVCM_PLAIN_Q8(SUFFIX, T)                                                                                               \
  KVCM_API int kvcm_attention_plain_q8_##SUFFIX(                                                                               \
      const void* q, long long q_stride, void* out, long long out_stride, const void* k_codes, const void* v_codes,            \
      const float* k_scale, const float* v_scale, int num_pages, const int* block_tables, int max_blocks, const int* row_seq,  \
      const int* positions, int rows, int nh, int nkv, int hd, int block_size, float scale, int window, float softcap,         \
      const float* sink, void* stream) {                                                                                       \
    if (rows <= 0) return 0;                                                                                                   \
    if (nkv <= 0 || nh <= 0 || nh % nkv || hd < 8 || hd > 256 || hd % 8 || block_size <= 0 || block_size > q8::kMaxBlock ||    \
        max_blocks <= 0 || num_pages <= 0 || nh > 65535)                                                                       \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    Q8Pages k;                                                                                                                 \
    k.k_codes = (const uint8_t*)k_codes; k.v_codes = (const uint8_t*)v_codes; k.k_scale = k_scale; k.v_scale = v_scale;        \
    k.block_tables = block_tables; k.max_blocks = max_blocks; k.max_keys = q8::max_keys(max_blocks, block_size);               \
    k.row_seq = row_seq; k.positions = positions; k.nkv = nkv; k.hd = hd; k.block_size = block_size; k.num_pages = num_pages;  \
    return pdl_launch(attention_q8_plain_kernel<T, Q8Pages, false>, dim3(rows, nh), dim3(kQ8PlainThreads), 0,                  \
                      (cudaStream_t)stream, k, (const T*)q, q_stride, (T*)out, out_stride, nh, nkv, hd, scale, window,         \
                      softcap, sink);                                                                                          \
  }                                                                                                                            \
  KVCM_API int kvcm_prompt_attention_plain_##SUFFIX(                                                                           \
      const void* q, long long q_stride, const void* k_rows, long long k_stride, const void* v_rows, long long v_stride,       \
      void* out, long long out_stride, const int* tile_seq, const int* tile_q0, const int* seq_q_start, const int* seq_q_len,  \
      int tiles, int tile_rows, int singles, int nh, int nkv, int hd, float scale, int window, float softcap,                  \
      const float* sink, void* stream) {                                                                                       \
    if (nkv <= 0 || nh <= 0 || nh % nkv || hd < 8 || hd > 256 || hd % 8 || nh > 65535 || tiles < 0 || singles < 0 ||           \
        tile_rows <= 0 || (long long)tiles * tile_rows + singles > 0x7fffffffll)                                               \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    if (tiles * tile_rows + singles == 0) return 0;                                                                            \
    PromptRows<T> k;                                                                                                           \
    k.k = (const T*)k_rows; k.v = (const T*)v_rows; k.k_stride = k_stride; k.v_stride = v_stride;                              \
    k.tile_seq = tile_seq; k.tile_q0 = tile_q0; k.seq_q_start = seq_q_start; k.seq_q_len = seq_q_len;                          \
    k.tiles = tiles; k.tile_rows = tile_rows; k.hd = hd;                                                                       \
    return pdl_launch(attention_q8_plain_kernel<T, PromptRows<T>, true>, dim3(tiles * tile_rows + singles, nh),                \
                      dim3(kQ8PlainThreads), 0, (cudaStream_t)stream, k, (const T*)q, q_stride, (T*)out, out_stride, nh, nkv,  \
                      hd, scale, window, softcap, sink);                                                                       \
  }

KVCM_PLAIN_Q8(bf16, bf16)
KVCM_PLAIN_Q8(f32, float)

KVCM_PACKED(kvcm_attention_plain_q8_bf16)
KVCM_PACKED(kvcm_attention_plain_q8_f32)
KVCM_PACKED(kvcm_prompt_attention_plain_bf16)
KVCM_PACKED(kvcm_prompt_attention_plain_f32)
