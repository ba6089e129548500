// Writing rows of keys and values into pages of 4 bits, and reading them back (layout: q4.cuh).
//
//   zero = bfloat16(min x), scale = bfloat16((max x - min x) / 15), code = round((x - zero) / scale) within 0..15
//
// over the hd elements of one head of one row; K after its rotation (not rounded in between), V as it is.  float32 arithmetic
// with IEEE roundings throughout, so that the codes are a function of the inputs alone.  All equal elements give scale 0 and
// code 0.  A row with an element that is not finite, or whose range is beyond float32, reads back as not-a-number everywhere: loud,
// not wrong.
//
// What bounds it: memory.  A lane has one word of a row (eight elements: one 16-byte load, one 4-byte store of codes); the lanes
// of a head (hd / 8, rounded up to a power of two) sit in one warp and find minimum and maximum by shuffles, and so does a
// rotate-half partner, hd / 16 lanes away.
#include "pdl.cuh"
#include "q4.cuh"

namespace kvcm {

constexpr int kQ4Threads = 256;

__device__ __forceinline__ void load8(const bf16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
__device__ __forceinline__ void store8(bf16* p, const float (&x)[8]) {
  uint4 v;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = v;
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

struct StoreQ4Params {
  const void* qkv; long long row_stride;
  const float* angles;                 // [rows, rotary_dim]: cosines, then sines; null: no rotation
  int rotary_dim, interleaved;
  const int* slot_mapping;
  uint8_t* k_out; uint8_t* v_out;      // caches
  void* q_out; long long q_stride;
  int rows, nh, nkv, hd, block_size, num_pages;
  int lanes;                           // lanes of a head: hd / 8 rounded up to a power of two
};

// One lane a word; item = (row, head, word).
template <typename T>
__global__ void __launch_bounds__(kQ4Threads) store_q4_kernel(StoreQ4Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const long long item = (long long)blockIdx.x * kQ4Threads + threadIdx.x;
  const int heads = p.nh + 2 * p.nkv;
  const int word = int(item) & (p.lanes - 1);                     // (lanes divides 32 and the block)
  const long long rh = item / p.lanes;
  const int row = int(rh / heads), head = int(rh - (long long)row * heads);
  const bool live = row < p.rows && word * 8 < p.hd;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) load8(static_cast<const T*>(p.qkv) + size_t(row) * p.row_stride + size_t(head) * p.hd + word * 8, x);
  // ---- rotation of q and k heads.  Partner lanes take part whether or not they are live.
  if (p.angles != nullptr) {
    const int half = p.rotary_dim / 2;
    const float* cs = p.angles + size_t(live ? row : 0) * p.rotary_dim;
    if (p.interleaved) {
      if (live && head < p.nh + p.nkv) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pair = word * 4 + i;
          if (pair < half) rotate_pair(x[2 * i], x[2 * i + 1], cs[pair], cs[half + pair], x[2 * i], x[2 * i + 1]);
        }
      }
    } else {
      const int away = half / 8;                                   // words between partners
      const bool first = word < away;
      const int lane = threadIdx.x & 31;
      const int partner = word < 2 * away ? (first ? lane + away : lane - away) : lane;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = __shfl_sync(0xffffffffu, x[e], partner);
      if (live && head < p.nh + p.nkv && word < 2 * away) {
        const int j0 = (first ? word : word - away) * 8;
        float c[8], s[8];
        load8(cs + j0, c);
        load8(cs + half + j0, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float ra, rb;
          rotate_pair(first ? x[e] : y[e], first ? y[e] : x[e], c[e], s[e], ra, rb);
          x[e] = first ? ra : rb;
        }
      }
    }
  }
  if (live && head < p.nh) store8(static_cast<T*>(p.q_out) + size_t(row) * p.q_stride + size_t(head) * p.hd + word * 8, x);
  // ---- the row's range (lanes of q heads and dead lanes go along)
  float low = INFINITY, high = -INFINITY;
  int bad = 0;
  if (live) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      low = fminf(low, x[e]);
      high = fmaxf(high, x[e]);
      bad |= !(fabsf(x[e]) <= 3.402823466e38f);
    }
  }
  for (int o = p.lanes >> 1; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    bad |= __shfl_xor_sync(0xffffffffu, bad, o);
  }
  if (!live || head < p.nh) return;
  const int slot = p.slot_mapping[row];
  if (slot < 0) return;
  const int page = slot / p.block_size, off = slot - page * p.block_size;
  if (page >= p.num_pages) return;
  const bool is_k = head < p.nh + p.nkv;
  const int kvh = head - p.nh - (is_k ? 0 : p.nkv);
  bf16 scale = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(high, low), 15.f)), zero = __float2bfloat16_rn(low);
  const float s = __bfloat162float(scale), z = __bfloat162float(zero);
  bad |= !(s <= 3.402823466e38f);
  uint32_t code[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[e], z), s)) : 0.f;
    code[e] = bad ? 0u : uint32_t(fminf(fmaxf(t, 0.f), 15.f));
  }
  if (bad) scale = zero = __ushort_as_bfloat16(0x7fc0);
  const size_t bytes = q4::page_bytes(p.block_size, p.hd);
  uint8_t* base = (is_k ? p.k_out : p.v_out) + (size_t(page) * p.nkv + kvh) * bytes;
  *reinterpret_cast<uint32_t*>(base + size_t(off) * (p.hd / 2) + word * 4) = q4::pack_codes(code);
  if (word == 0)
    *reinterpret_cast<uint32_t*>(base + size_t(p.block_size) * (p.hd / 2) + off * 4) =
        uint32_t(__bfloat16_as_ushort(scale)) | (uint32_t(__bfloat16_as_ushort(zero)) << 16);
}

__device__ __forceinline__ void values8(uint32_t word, uint32_t pair, float (&x)[8]) {
  const float s = q4::scale_of(pair), z = q4::zero_of(pair);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(z, __fmul_rn(s, q4::code_of(word, e)));      // (the product is exact: 8 + 4 bits)
}

// Rows of slots back as values: k_rows and v_rows [rows, nkv * hd].  Rows without a slot stay as they are.
template <typename T>
__global__ void __launch_bounds__(kQ4Threads)
read_q4_kernel(const uint8_t* k_cache, const uint8_t* v_cache, const int* __restrict__ slot_mapping, T* __restrict__ k_rows,
               T* __restrict__ v_rows, long long k_stride, long long v_stride, int rows, int nkv, int hd, int block_size, int num_pages) {
  pdl_launch_dependents();
  pdl_wait();
  const int words = hd / 8;
  const long long item = (long long)blockIdx.x * kQ4Threads + threadIdx.x;
  const long long rh = item / words;
  const int word = int(item - rh * words);
  const int row = int(rh / (2 * nkv)), head = int(rh - (long long)row * 2 * nkv);
  if (row >= rows) return;
  const int slot = slot_mapping[row];
  if (slot < 0) return;
  const int page = slot / block_size, off = slot - page * block_size;
  if (page >= num_pages) return;
  const bool is_k = head < nkv;
  const int kvh = is_k ? head : head - nkv;
  const uint8_t* base = (is_k ? k_cache : v_cache) + (size_t(page) * nkv + kvh) * q4::page_bytes(block_size, hd);
  float x[8];
  values8(*reinterpret_cast<const uint32_t*>(base + size_t(off) * (hd / 2) + word * 4),
          *reinterpret_cast<const uint32_t*>(base + size_t(block_size) * (hd / 2) + off * 4), x);
  store8((is_k ? k_rows + size_t(row) * k_stride : v_rows + size_t(row) * v_stride) + size_t(kvh) * hd + word * 8, x);
}

// The pages of requests `first_seq` .. `first_seq + grid.y` as bfloat16 pages [request, block][nkv, block_size, hd]: those that hold
// positions that the request's rows of this step see, [first visible of the first row, context).
__global__ void __launch_bounds__(kQ4Threads)
unpack_pages_q4_kernel(const uint8_t* k_cache, const uint8_t* v_cache, const int* __restrict__ block_tables, int max_blocks,
                       const int* __restrict__ seq_q_len, const int* __restrict__ seq_ctx_len, bf16* __restrict__ k_pages,
                       bf16* __restrict__ v_pages, int first_seq, int blocks, int nkv, int hd, int block_size, int num_pages, int window) {
  pdl_launch_dependents();
  pdl_wait();
  const int seq = first_seq + blockIdx.y, block = blockIdx.x;
  const int ctx = seq_ctx_len[seq];
  const int lo = first_visible(ctx - seq_q_len[seq], window, 0);
  if (block * block_size >= ctx || (block + 1) * block_size <= lo) return;
  const int words = hd / 8, per_head = block_size * words;
  const size_t bytes = q4::page_bytes(block_size, hd);
  const size_t from = q4::page_base(block_tables[size_t(seq) * max_blocks + block], 0, nkv, num_pages, bytes);
  const size_t to = (size_t(blockIdx.y) * blocks + block) * nkv * block_size * hd;
  for (int i = threadIdx.x; i < 2 * nkv * per_head; i += kQ4Threads) {
    const int head = i / per_head, at = i - head * per_head;
    const int off = at / words, word = at - off * words;
    const bool is_k = head < nkv;
    const int kvh = is_k ? head : head - nkv;
    const uint8_t* base = (is_k ? k_cache : v_cache) + from + kvh * bytes;
    float x[8];
    // (positions behind the context may hold anything; their probabilities are zero, and zero times a value must stay zero)
    if (block * block_size + off < ctx)
      values8(*reinterpret_cast<const uint32_t*>(base + size_t(off) * (hd / 2) + word * 4),
              *reinterpret_cast<const uint32_t*>(base + size_t(block_size) * (hd / 2) + off * 4), x);
    else
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    store8((is_k ? k_pages : v_pages) + to + (size_t(kvh) * block_size + off) * hd + word * 8, x);
  }
}

template <typename T>
int launch_store_q4(const StoreQ4Params& p, cudaStream_t s) {
  const long long items = (long long)p.rows * (p.nh + 2 * p.nkv) * p.lanes;
  return pdl_launch(store_q4_kernel<T>, dim3(unsigned((items + kQ4Threads - 1) / kQ4Threads)), dim3(kQ4Threads), 0, s, p);
}

template <typename T>
int launch_read_q4(const void* k_cache, const void* v_cache, const int* slots, void* k_rows, void* v_rows, long long k_stride,
                   long long v_stride, int rows, int nkv, int hd, int block_size, int num_pages, cudaStream_t s) {
  const long long items = (long long)rows * 2 * nkv * (hd / 8);
  return pdl_launch(read_q4_kernel<T>, dim3(unsigned((items + kQ4Threads - 1) / kQ4Threads)), dim3(kQ4Threads), 0, s,
                    (const uint8_t*)k_cache, (const uint8_t*)v_cache, slots, (T*)k_rows, (T*)v_rows, k_stride, v_stride, rows, nkv, hd,
                    block_size, num_pages);
}

bool q4_sizes_ok(int nkv, int hd, int block_size, int num_pages) {
  return nkv > 0 && hd >= 8 && hd <= 256 && hd % 8 == 0 && block_size > 0 && num_pages > 0;
}

bool items_fit(long long items) { return (items + kQ4Threads - 1) / kQ4Threads <= 0x7fffffffll; }

}  // namespace kvcm

using namespace kvcm;

// Bytes of a page of one KV head.
KVCM_API long long kvcm_q4_page_bytes(int block_size, int hd) { return (long long)q4::page_bytes(block_size, hd); }

// q|k|v rows (nh + 2 nkv heads of hd) -> rotated q rows in q_out, k and v in the pages of their slots (slot < 0: nowhere).
// `angles` [rows, rotary_dim] float32, cosines then sines (null: no rotation).  All rows and addresses on 16 bytes.
#define KVCM_STORE_Q4(SUFFIX, T)                                                                                              \
  KVCM_API int kvcm_rope_cache_q4_##SUFFIX(const void* qkv, long long row_stride, const float* angles, int rotary_dim,         \
                                           int interleaved, const int* slot_mapping, void* k_cache, void* v_cache, void* q_out, \
                                           long long q_stride, int rows, int nh, int nkv, int hd, int block_size, int num_pages, \
                                           void* stream) {                                                                    \
    if (rows == 0) return 0;                                                                                                   \
    if (!q4_sizes_ok(nkv, hd, block_size, num_pages) || nh < 0) return KVCM_ERR_UNSUPPORTED;                                   \
    if (angles != nullptr && (rotary_dim < 2 || rotary_dim > hd || rotary_dim % (interleaved ? 2 : 16)))                       \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    const uintptr_t places = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |                           \
                             uintptr_t(row_stride * sizeof(T)) | uintptr_t(q_stride * sizeof(T));                              \
    if ((places & 15) || ((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |                       \
                           reinterpret_cast<uintptr_t>(angles)) & 15))                                                         \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    StoreQ4Params p;                                                                                                           \
    p.qkv = qkv; p.row_stride = row_stride; p.angles = angles; p.rotary_dim = rotary_dim; p.interleaved = interleaved;         \
    p.slot_mapping = slot_mapping; p.k_out = (uint8_t*)k_cache; p.v_out = (uint8_t*)v_cache; p.q_out = q_out;                  \
    p.q_stride = q_stride; p.rows = rows; p.nh = nh; p.nkv = nkv; p.hd = hd; p.block_size = block_size;                        \
    p.num_pages = num_pages;                                                                                                   \
    p.lanes = 1;                                                                                                               \
    while (p.lanes * 8 < hd) p.lanes *= 2;                                                                                     \
    if (!items_fit((long long)rows * (nh + 2 * nkv) * p.lanes)) return KVCM_ERR_UNSUPPORTED;                                   \
    return launch_store_q4<T>(p, (cudaStream_t)stream);                                                                        \
  }                                                                                                                           \
  KVCM_API int kvcm_read_cache_q4_##SUFFIX(const void* k_cache, const void* v_cache, const int* slot_mapping, void* k_rows,    \
                                           void* v_rows, long long k_stride, long long v_stride, int rows, int nkv, int hd,    \
                                           int block_size, int num_pages, void* stream) {                                     \
    if (rows == 0) return 0;                                                                                                   \
    const uintptr_t places = reinterpret_cast<uintptr_t>(k_rows) | reinterpret_cast<uintptr_t>(v_rows) |                       \
                             uintptr_t(k_stride * sizeof(T)) | uintptr_t(v_stride * sizeof(T));                                \
    if (!q4_sizes_ok(nkv, hd, block_size, num_pages) || (places & 15) || !items_fit((long long)rows * 2 * nkv * (hd / 8)))     \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    return launch_read_q4<T>(k_cache, v_cache, slot_mapping, k_rows, v_rows, k_stride, v_stride, rows, nkv, hd, block_size,    \
                             num_pages, (cudaStream_t)stream);                                                                 \
  }

KVCM_STORE_Q4(bf16, bf16)
KVCM_STORE_Q4(f32, float)

// k_pages, v_pages: room for seqs x blocks pages [nkv, block_size, hd] of bfloat16.
KVCM_API int kvcm_unpack_pages_q4_bf16(const void* k_cache, const void* v_cache, const int* block_tables, int max_blocks,
                                       const int* seq_q_len, const int* seq_ctx_len, void* k_pages, void* v_pages, int first_seq, int seqs,
                                       int blocks, int nkv, int hd, int block_size, int num_pages, int window, void* stream) {
  if (seqs <= 0 || blocks <= 0) return 0;
  if (!q4_sizes_ok(nkv, hd, block_size, num_pages) || blocks > max_blocks || seqs > 65535) return KVCM_ERR_UNSUPPORTED;
  return pdl_launch(unpack_pages_q4_kernel, dim3(blocks, seqs), dim3(kQ4Threads), 0, (cudaStream_t)stream, (const uint8_t*)k_cache,
                    (const uint8_t*)v_cache, block_tables, max_blocks, seq_q_len, seq_ctx_len, (bf16*)k_pages, (bf16*)v_pages, first_seq,
                    blocks, nkv, hd, block_size, num_pages, window);
}
