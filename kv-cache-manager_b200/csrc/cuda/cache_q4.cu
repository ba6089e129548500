// Writing rows of keys and values into pages of 4 bits, and reading them back (layout: q4.cuh).
//
//   zero = bfloat16(min x), scale = bfloat16((max x - min x) / 15), code = round((x - zero) / scale) within 0..15
//
// over the hd elements of one head of one row; K after its rotation (not rounded in between), V as it is.  float32 arithmetic
// with IEEE roundings throughout, so that the codes are a function of the inputs alone.  All equal elements give scale 0 and
// code 0.  A row with an element that is not finite, or whose range is beyond float32, reads back as not-a-number everywhere: loud,
// not wrong.
//
// What bounds it: memory, if little is done for each element.  A lane has two words of a head (eight elements each: a 16-byte load
// and a 4-byte store of codes), in rotate-half pairs the two that turn with one another, so that angles are read once for both and
// nothing is exchanged; the lanes of a head (hd / 16, rounded up to a power of two) sit in one warp and find minimum and
// maximum by shuffles.  A block has up to 256 such pairs of one row (grid: rows x equal pieces of a row), so nothing is divided to
// find one's place, and codes are found without divisions too (see there).  8,192 rows of 48 heads of 128 (180 MB): 43 us, 4.2 TB/s
// (28 us at the rate of a copy); 55 with 16 divisions a lane, 71 with one word a lane and partners exchanged by shuffles, 96 with
// places counted through and taken apart by 64-bit divisions.  What is left is waiting: a block is one load, a few hundred
// instructions and a store; packed pairs of float32 (50 us), other block sizes and cache hints (no change) do not help.  Reading the
// 8 + 8 KV heads back: 11.7 us (43 MB, 6.5 at that rate), 16.7 with a word a lane and codes converted from whole numbers.  float32 rows:
// written in 56 us (53 at that rate), read back in 20 (12).
#include "packed.cuh"
#include "pdl.cuh"
#include "q4.cuh"

namespace kvcm {

constexpr int kQ4Threads = 256;                    // most threads of a block
constexpr float kQ4Finite = 3.402823466e38f;
constexpr float kQ4Magic = 12582912.f;             // 1.5 * 2^23: what is added to it is rounded to a whole number, ties to even
constexpr uint32_t kQ4MagicWord = 0x3f400000u;     // eight words of its bits (0x4b400000) under the shifts of pack_codes, added up

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
  int log2_lanes;                      // lanes of a head: hd / 16 rounded up to a power of two
};

// One lane two words.
template <typename T>
__global__ void __launch_bounds__(kQ4Threads, 5) store_q4_kernel(StoreQ4Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const int item = blockIdx.y * blockDim.x + threadIdx.x;
  const int heads = p.nh + 2 * p.nkv, lanes = 1 << p.log2_lanes, words = p.hd / 8;
  const int i = item & (lanes - 1);                                // (a head's lanes lie in one warp)
  const int row = blockIdx.x, head = item >> p.log2_lanes;
  // words i and i + away turn with one another; the words behind the rotation, and all where pairs are neighbours, by twos
  const int away = p.angles != nullptr && !p.interleaved ? p.rotary_dim / 16 : 0;
  const int word[2] = {i < away ? i : 2 * i, i < away ? i + away : 2 * i + 1};
  const bool live[2] = {head < heads && word[0] < words, head < heads && word[1] < words};
  float x[2][8], c[8], sn[8];                                      // (all loads of the row first: one trip to memory)
  const bool turns = p.angles != nullptr && live[0] && head < p.nh + p.nkv;
  const float* cs = p.angles + size_t(row) * p.rotary_dim;
  const int slot = p.slot_mapping[row], half = p.rotary_dim / 2;
  if (turns && i < away) {
    load8(cs + i * 8, c);
    load8(cs + half + i * 8, sn);
  }
  const T* from = static_cast<const T*>(p.qkv) + size_t(row) * p.row_stride + size_t(head) * p.hd;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
    if (live[k]) load8(from + word[k] * 8, x[k]);
  }
  // ---- rotation of q and k heads
  if (turns) {
    if (p.interleaved) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pair = word[k] * 4 + e;
          if (pair < half) rotate_pair(x[k][2 * e], x[k][2 * e + 1], cs[pair], cs[half + pair], x[k][2 * e], x[k][2 * e + 1]);
        }
    } else if (i < away) {
#pragma unroll
      for (int e = 0; e < 8; ++e) rotate_pair(x[0][e], x[1][e], c[e], sn[e], x[0][e], x[1][e]);
    }
  }
  if (head < p.nh) {
    T* to = static_cast<T*>(p.q_out) + size_t(row) * p.q_stride + size_t(head) * p.hd;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (live[k]) store8(to + word[k] * 8, x[k]);
  }
  if (__all_sync(0xffffffffu, !live[0] || head < p.nh)) return;    // q heads alone
  // ---- the row's range (lanes of q heads and dead lanes go along)
  float low = INFINITY, high = -INFINITY, sick = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (live[k]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        low = fminf(low, x[k][e]);
        high = fmaxf(high, x[k][e]);
        sick = fmaf(x[k][e], 0.f, sick);                           // not a number from the first element on that is not finite
      }
    }
  for (int o = lanes >> 1; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  const uint32_t all_sick = __ballot_sync(0xffffffffu, sick != 0.f);
  bool bad = ((all_sick >> (threadIdx.x & 31 & -lanes)) & ((1u << lanes) - 1u)) != 0u;
  if (!live[0] || head < p.nh) return;
  if (slot < 0) return;
  const int page = slot / p.block_size, off = slot - page * p.block_size;
  if (page >= p.num_pages) return;
  const bool is_k = head < p.nh + p.nkv;
  const int kvh = head - p.nh - (is_k ? 0 : p.nkv);
  bf16 scale = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(high, low), 15.f)), zero = __float2bfloat16_rn(low);
  const float s = __bfloat162float(scale), z = __bfloat162float(zero);
  bad |= !(s <= kQ4Finite);
  const size_t bytes = q4::page_bytes(p.block_size, p.hd);
  uint8_t* base = (is_k ? p.k_out : p.v_out) + (size_t(page) * p.nkv + kvh) * bytes;
  // A product with 1 / scale is at most 2^-18 off the quotient (of 16 and less; three roundings), so it rounds to the same code
  // where it is not that near to a half.  Where one of the lane's is near (one lane in 2,000), or the scale is so small that its
  // reciprocal is none, the divisions are done.
  const float per = s > 1e-30f ? __frcp_rn(s) : 0.f;
  float farthest = s > 1e-30f || s == 0.f ? 0.f : 1.f;                         // from a whole number
  uint32_t codes[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    codes[k] = 0u - kQ4MagicWord;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = fminf(fmaxf(__fsub_rn(x[k][e], z) * per, 0.f), 15.f), n = __fadd_rn(t, kQ4Magic);
      farthest = fmaxf(farthest, fabsf(__fsub_rn(t, __fsub_rn(n, kQ4Magic))));
      codes[k] += __float_as_uint(n) << (4 * (e >> 1) + 16 * (e & 1));
    }
  }
  if (farthest > 0.5f - 1.f / 65536.f) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t code[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float t = s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[k][e], z), s)) : 0.f;
        code[e] = uint32_t(fminf(fmaxf(t, 0.f), 15.f));
      }
      codes[k] = q4::pack_codes(code);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (live[k]) *reinterpret_cast<uint32_t*>(base + size_t(off) * (p.hd / 2) + word[k] * 4) = bad ? 0u : codes[k];
  if (bad) scale = zero = __ushort_as_bfloat16(0x7fc0);
  if (i == 0)
    *reinterpret_cast<uint32_t*>(base + size_t(p.block_size) * (p.hd / 2) + off * 4) =
        uint32_t(__bfloat16_as_ushort(scale)) | (uint32_t(__bfloat16_as_ushort(zero)) << 16);
}

// (code from 128 + code, which a shift and an and-or give two at a time as bfloat16; the product is exact: 8 + 4 bits)
__device__ __forceinline__ void values8(uint32_t word, uint32_t pair, float (&x)[8]) {
  const float s = q4::scale_of(pair), z = q4::zero_of(pair);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t two = q4::two_codes_128(word, i);
    x[2 * i] = __fadd_rn(z, __fmul_rn(s, __uint_as_float(two << 16) - 128.f));
    x[2 * i + 1] = __fadd_rn(z, __fmul_rn(s, __uint_as_float(two & 0xffff0000u) - 128.f));
  }
}

// Rows of slots back as values: k_rows and v_rows [rows, nkv * hd].  Rows without a slot stay as they are.  A lane has two words.
template <typename T>
__global__ void __launch_bounds__(kQ4Threads)
read_q4_kernel(const uint8_t* k_cache, const uint8_t* v_cache, const int* __restrict__ slot_mapping, T* __restrict__ k_rows,
               T* __restrict__ v_rows, long long k_stride, long long v_stride, int nkv, int hd, int block_size, int num_pages, int log2_lanes) {
  pdl_launch_dependents();
  pdl_wait();
  const int item = blockIdx.y * blockDim.x + threadIdx.x;
  const int row = blockIdx.x, head = item >> log2_lanes, word = 2 * (item & ((1 << log2_lanes) - 1));
  if (head >= 2 * nkv || word >= hd / 8) return;
  const int slot = slot_mapping[row];
  if (slot < 0) return;
  const int page = slot / block_size, off = slot - page * block_size;
  if (page >= num_pages) return;
  const bool is_k = head < nkv;
  const int kvh = is_k ? head : head - nkv;
  const uint8_t* base = (is_k ? k_cache : v_cache) + (size_t(page) * nkv + kvh) * q4::page_bytes(block_size, hd);
  const uint32_t pair = *reinterpret_cast<const uint32_t*>(base + size_t(block_size) * (hd / 2) + off * 4);
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(base + size_t(off) * (hd / 2)) + word;
  T* to = (is_k ? k_rows + size_t(row) * k_stride : v_rows + size_t(row) * v_stride) + size_t(kvh) * hd + word * 8;
  const bool second = word + 1 < hd / 8;
  const uint32_t w[2] = {codes[0], second ? codes[1] : 0u};
  float x[8];
  values8(w[0], pair, x);
  store8(to, x);
  if (second) {
    values8(w[1], pair, x);
    store8(to + 8, x);
  }
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
  const int ctx = int(min((long long)seq_ctx_len[seq], (long long)blocks * block_size));      // (a context ends with its table, and so do its rows)
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

// Lanes of a head, as a power of two: hd / 16, rounded up.
int q4_log2_lanes(int hd) {
  int n = 0;
  while ((16 << n) < hd) ++n;
  return n;
}
// A row's items in blocks of like size: (rows, blocks), threads.
void q4_grid(int rows, int items, dim3& grid, dim3& block) {
  const int pieces = (items + kQ4Threads - 1) / kQ4Threads;
  grid = dim3(rows, pieces);
  block = dim3(((items + pieces - 1) / pieces + 31) / 32 * 32);
}

template <typename T>
int launch_store_q4(const StoreQ4Params& p, cudaStream_t s) {
  dim3 grid, block;
  q4_grid(p.rows, (p.nh + 2 * p.nkv) << p.log2_lanes, grid, block);
  return pdl_launch(store_q4_kernel<T>, grid, block, 0, s, p);
}

template <typename T>
int launch_read_q4(const void* k_cache, const void* v_cache, const int* slots, void* k_rows, void* v_rows, long long k_stride,
                   long long v_stride, int rows, int nkv, int hd, int block_size, int num_pages, cudaStream_t s) {
  const int log2_lanes = q4_log2_lanes(hd);
  dim3 grid, block;
  q4_grid(rows, 2 * nkv << log2_lanes, grid, block);
  return pdl_launch(read_q4_kernel<T>, grid, block, 0, s,
                    (const uint8_t*)k_cache, (const uint8_t*)v_cache, slots, (T*)k_rows, (T*)v_rows, k_stride, v_stride, nkv, hd,
                    block_size, num_pages, log2_lanes);
}

bool q4_sizes_ok(int nkv, int hd, int block_size, int num_pages) {
  return nkv > 0 && nkv <= 8192 && hd >= 8 && hd <= 256 && hd % 8 == 0 && block_size > 0 && block_size <= q4::kMaxBlock && num_pages > 0;
}

}  // namespace kvcm

using namespace kvcm;

// q|k|v rows (nh + 2 nkv heads of hd) -> rotated q rows in q_out, k and v in the pages of their slots (slot < 0: nowhere).
// `angles` [rows, rotary_dim] float32, cosines then sines (null: no rotation).  All rows and addresses on 16 bytes.
#define KVCM_STORE_Q4(SUFFIX, T)                                                                                              \
  KVCM_API int kvcm_rope_cache_q4_##SUFFIX(const void* qkv, long long row_stride, const float* angles, int rotary_dim,         \
                                           int interleaved, const int* slot_mapping, void* k_cache, void* v_cache, void* q_out, \
                                           long long q_stride, int rows, int nh, int nkv, int hd, int block_size, int num_pages, \
                                           void* stream) {                                                                    \
    if (rows == 0) return 0;                                                                                                   \
    if (!q4_sizes_ok(nkv, hd, block_size, num_pages) || nh < 0 || nh > 32768) return KVCM_ERR_UNSUPPORTED;                     \
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
    p.log2_lanes = q4_log2_lanes(hd);                                                                                          \
    return launch_store_q4<T>(p, (cudaStream_t)stream);                                                                        \
  }                                                                                                                           \
  KVCM_API int kvcm_read_cache_q4_##SUFFIX(const void* k_cache, const void* v_cache, const int* slot_mapping, void* k_rows,    \
                                           void* v_rows, long long k_stride, long long v_stride, int rows, int nkv, int hd,    \
                                           int block_size, int num_pages, void* stream) {                                     \
    if (rows == 0) return 0;                                                                                                   \
    const uintptr_t places = reinterpret_cast<uintptr_t>(k_rows) | reinterpret_cast<uintptr_t>(v_rows) |                       \
                             uintptr_t(k_stride * sizeof(T)) | uintptr_t(v_stride * sizeof(T));                                \
    if (!q4_sizes_ok(nkv, hd, block_size, num_pages) || (places & 15))                                                         \
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

KVCM_PACKED(kvcm_rope_cache_q4_bf16)
KVCM_PACKED(kvcm_rope_cache_q4_f32)
KVCM_PACKED(kvcm_read_cache_q4_bf16)
KVCM_PACKED(kvcm_read_cache_q4_f32)
KVCM_PACKED(kvcm_unpack_pages_q4_bf16)
