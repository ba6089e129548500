// Writing rows of keys and values into pages of 8 bits with one scale for a page and head, and reading them back (format: q8.cuh).
//
//   scale' = max(kept, least 2^e with 448 2^e >= max |x|),  code = e4m3(x / scale'),  kept codes <- e4m3(code * scale / scale')
//
// where the maximum runs over the rows that a call brings to the page, and `kept` is the page's scale, or nothing where one of
// them is the page's first row (the page begins anew).  K after its rotation (not rounded in between), V as it is.  float32
// arithmetic with IEEE roundings throughout; the divisions are by powers of two.  Not-a-number and infinite elements become
// not-a-number and do not enter the maximum.
//
// Rows of one page stand next to each other in a step, so a page's rows are a run of rows.  One warp takes a run and one KV head:
// it finds the rows' maximum by shuffles, brings the page to its scale where that grows, and reads the rows a second time to write
// them (out of the nearest cache; the first as many rows as a warp has lanes for stay in registers).  A lane has
// two words of eight elements that turn with one another, so that angles are read once for both and nothing is exchanged.
// What bounds it: a warp's chain (slots, scale, rows, rows again) at 64 registers a thread, which let four blocks an SM overlap but spill
// 488 bytes a thread (668 read back) where windows are 8 or 16 rows, 344 (360) where they are one; float32 rows alike.  B200, about 8,400 rows, 32 heads and 8 + 8 KV heads of 128: 70 us (29 at the rate of a copy; 139 with the rows of a page
// kept in 170 registers; four warps a run 96), read back 15; 64 rows 6.1 and 3.9.  All heads q 54 us, all KV heads 87, where copies take 35 and 27.
// Windows: 900 rows 25 us in windows of 16, 21 of 8; 512 single rows 18 in windows of one.
#include "packed.cuh"
#include "pdl.cuh"
#include "q8.cuh"

namespace kvcm {

constexpr int kQ8Threads = 256;
constexpr int kQ8Warps = kQ8Threads / 32;
constexpr float kQ8Finite = 3.402823466e38f;

namespace {

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

}  // namespace

struct StoreQ8Params {
  const void* qkv; long long row_stride;
  const float* angles;                 // [rows, rotary_dim]: cosines, then sines; null: no rotation
  int rotary_dim, interleaved;
  const int* slot_mapping;
  uint8_t* k_codes; uint8_t* v_codes; float* k_scale; float* v_scale;
  void* q_out; long long q_stride;
  int rows, nh, nkv, hd, block_size, num_pages;
  int log2_lanes;                      // lanes of a head: hd / 16 rounded up to a power of two
};

// The two words of a lane: words i and i + away turn with one another, the others go by twos.
struct Q8Words {
  int i, away, at[2];
  bool live[2];
  __device__ __forceinline__ Q8Words(const StoreQ8Params& p, int lane_of_head) {
    const int words = p.hd / 8;
    i = lane_of_head;
    away = p.angles != nullptr && !p.interleaved ? p.rotary_dim / 16 : 0;
    at[0] = i < away ? i : 2 * i;
    at[1] = i < away ? i + away : 2 * i + 1;
    live[0] = at[0] < words;
    live[1] = at[1] < words;
  }
};

// The lane's words of a head of a row, rotated where the head is (q and k).
template <typename T>
__device__ __forceinline__ void q8_load(const StoreQ8Params& p, const Q8Words& w, int row, int head, bool there, float (&x)[2][8]) {
  float c[8], sn[8];
  const bool turns = p.angles != nullptr && there && w.live[0] && head < p.nh + p.nkv;
  const float* cs = p.angles + size_t(row) * p.rotary_dim;
  const int half = p.rotary_dim / 2;
  if (turns && w.i < w.away) {
    load8(cs + w.i * 8, c);
    load8(cs + half + w.i * 8, sn);
  }
  const T* from = static_cast<const T*>(p.qkv) + size_t(row) * p.row_stride + size_t(head) * p.hd;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[k][e] = 0.f;
    if (there && w.live[k]) load8(from + w.at[k] * 8, x[k]);
  }
  if (turns) {
    if (p.interleaved) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int pair = w.at[k] * 4 + e;
          if (pair < half) rotate_pair(x[k][2 * e], x[k][2 * e + 1], cs[pair], cs[half + pair], x[k][2 * e], x[k][2 * e + 1]);
        }
    } else if (w.i < w.away) {
#pragma unroll
      for (int e = 0; e < 8; ++e) rotate_pair(x[0][e], x[1][e], c[e], sn[e], x[0][e], x[1][e]);
    }
  }
}

// Eight elements as codes; not-a-number of what is not finite (`finite`: everything is).
__device__ __forceinline__ uint2 q8_codes(const float (&x)[8], float per, bool finite) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i] * per, b = x[2 * i + 1] * per;
    if (!finite) {                                                 // (x * 0 is zero, or not-a-number)
      a = fmaf(x[2 * i], 0.f, a);
      b = fmaf(x[2 * i + 1], 0.f, b);
    }
    c[i] = q8::codes2(a, b);
  }
  return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}

// Blocks: windows of W rows x groups of eight warps.  A warp has one q head of the window's rows (W == 1: of as many heads as it has
// lanes for), or one KV head of the runs that begin in the window.
template <typename T, int W>
__global__ void __launch_bounds__(kQ8Threads, 4) store_q8_kernel(StoreQ8Params p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, unit = blockIdx.y * kQ8Warps + (threadIdx.x >> 5);
  const int lanes = 1 << p.log2_lanes, R = 32 >> p.log2_lanes, group = lane >> p.log2_lanes;
  const int w0 = blockIdx.x * W;
  const Q8Words words(p, lane & (lanes - 1));
  const int q_units = W == 1 ? (p.nh + R - 1) / R : p.nh;
  if (unit < q_units) {
    const int stop = min(w0 + W, p.rows);
#pragma unroll 2
    for (int r = w0; r < stop; r += W == 1 ? 1 : R) {
      const int row = W == 1 ? r : r + group, head = W == 1 ? unit * R + group : unit;
      const bool there = row < stop && head < p.nh;
      float x[2][8];
      q8_load<T>(p, words, row, head, there, x);
      T* to = static_cast<T*>(p.q_out) + size_t(row) * p.q_stride + size_t(head) * p.hd;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (there && words.live[k]) store8(to + words.at[k] * 8, x[k]);
    }
    return;
  }
  if (unit - q_units >= 2 * p.nkv) return;
  const bool is_k = unit - q_units < p.nkv;
  const int kvh = unit - q_units - (is_k ? 0 : p.nkv), head = p.nh + unit - q_units;
  uint8_t* const codes = is_k ? p.k_codes : p.v_codes;
  float* const scales = is_k ? p.k_scale : p.v_scale;
  // pages of rows w0 - 1 .. w0 + 30 (-1: none)
  auto place = [&](int row, int& off) {
    const int slot = row >= 0 && row < p.rows ? p.slot_mapping[row] : -1;
    const int page = slot < 0 ? -1 : slot / p.block_size;
    off = slot - page * p.block_size;
    return page < p.num_pages ? page : -1;
  };
  float ahead[2][8];                                               // the first rows of a run; where a window is one row, asked for at once
  if (W == 1) q8_load<T>(p, words, w0 + group, head, w0 + group < p.rows, ahead);
  int off;
  const int page = place(w0 - 1 + lane, off);
  const int before = __shfl_up_sync(0xffffffffu, page, 1);
  uint32_t leaders = __ballot_sync(0xffffffffu, lane >= 1 && lane <= W && page >= 0 && page != before);
  while (leaders) {
    const int first = __ffs(leaders) - 1, r0 = w0 - 1 + first, here = __shfl_sync(0xffffffffu, page, first);
    leaders &= leaders - 1;
    const size_t at = size_t(here) * p.nkv + kvh;
    const float old = scales[at];
    // ---- the run: its rows, and whether the page's first is among them
    const uint32_t same = __ballot_sync(0xffffffffu, page == here) >> first;
    int n = __ffs(~same) - 1;                                      // (first >= 1: the topmost bit is clear)
    bool anew = (__ballot_sync(0xffffffffu, page == here && off == 0) >> first) & ((1u << n) - 1u);
    for (bool more = first + n == 32; more;) {
      int o;
      const bool mine = place(r0 + n + lane, o) == here;
      const uint32_t m = __ballot_sync(0xffffffffu, mine), a = __ballot_sync(0xffffffffu, mine && o == 0);
      const int k = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
      anew |= (a & (k == 32 ? 0xffffffffu : (1u << k) - 1u)) != 0u;
      n += k;
      more = k == 32;
    }
    // ---- its largest element
    // (the maximum passes over not-a-number; `sick` is that from the first element on that is not finite)
    float most = 0.f, sick = 0.f;
    auto largest = [&](const float (&v)[2][8]) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          most = fmaxf(most, fabsf(v[k][e]));
          sick = fmaf(v[k][e], 0.f, sick);
        }
    };
    if (W != 1) q8_load<T>(p, words, r0 + group, head, group < n, ahead);
    if (group < n) largest(ahead);
#pragma unroll 1
    for (int r = R + group; r - group < n; r += R) {
      float v[2][8];
      q8_load<T>(p, words, r0 + r, head, r < n, v);
      largest(v);
    }
    const bool finite = !__any_sync(0xffffffffu, sick != 0.f);
    if (!finite) {                                                 // of the finite elements alone
      most = 0.f;
#pragma unroll 1
      for (int r = group; r - group < n; r += R) {
        float v[2][8];
        q8_load<T>(p, words, r0 + r, head, r < n, v);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 8; ++e) most = fabsf(v[k][e]) <= kQ8Finite ? fmaxf(most, fabsf(v[k][e])) : most;
      }
    }
    most = warp_max(most);
    const float need = q8::scale_for(most), scale = !anew && old > need ? old : need, per = __frcp_rn(scale);
    uint8_t* const base = codes + at * p.block_size * p.hd;
    // ---- what the page holds, at the new scale
    if (!anew && !(old >= scale)) {
      const float ratio = old * per;
      for (int k = lane; k < p.block_size * (p.hd / 8); k += 32) {
        uint2* word = reinterpret_cast<uint2*>(base) + k;
        const uint2 u = *word;
        float v[8];
        q8::values4(u.x, ratio, v);
        q8::values4(u.y, ratio, v + 4);
        *word = q8_codes(v, 1.f, true);                            // (codes of not-a-number stay)
      }
      __syncwarp();
    }
    if (lane == 0 && (anew || scale != old)) scales[at] = scale;
    // ---- the rows
    auto write = [&](int r, const float (&v)[2][8]) {
      if (r >= n) return;
      const int slot = p.slot_mapping[r0 + r];
      uint8_t* to = base + size_t(slot - here * p.block_size) * p.hd;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (words.live[k]) *reinterpret_cast<uint2*>(to + words.at[k] * 8) = q8_codes(v[k], per, finite);
    };
    write(group, ahead);
#pragma unroll 1
    for (int r = R + group; r < n; r += R) {
      float v[2][8];
      q8_load<T>(p, words, r0 + r, head, true, v);
      write(r, v);
    }
  }
}

// Rows of slots back as values: k_rows and v_rows [rows, nkv * hd].  Rows without a slot stay as they are.  A lane has two words.
template <typename T>
__global__ void __launch_bounds__(kQ8Threads)
read_q8_kernel(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scale, const float* v_scale,
               const int* slot_mapping, T* __restrict__ k_rows, T* __restrict__ v_rows, long long k_stride, long long v_stride,
               int nkv, int hd, int block_size, int num_pages, int log2_lanes) {
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
  const size_t at = size_t(page) * nkv + kvh;
  const float scale = (is_k ? k_scale : v_scale)[at];
  const uint8_t* from = (is_k ? k_codes : v_codes) + (at * block_size + off) * hd + word * 8;
  T* to = (is_k ? k_rows + size_t(row) * k_stride : v_rows + size_t(row) * v_stride) + size_t(kvh) * hd + word * 8;
  const bool second = word + 1 < hd / 8;
  const uint2 a = *reinterpret_cast<const uint2*>(from);
  const uint2 b = second ? *reinterpret_cast<const uint2*>(from + 8) : make_uint2(0u, 0u);
  float x[8];
  q8::values4(a.x, scale, x);
  q8::values4(a.y, scale, x + 4);
  store8(to, x);
  if (second) {
    q8::values4(b.x, scale, x);
    q8::values4(b.y, scale, x + 4);
    store8(to + 8, x);
  }
}

// The pages of requests `first_seq` .. `first_seq + grid.y` as bfloat16 pages [request, block][nkv, block_size, hd]: those that hold
// positions that the request's rows of this step see, [first visible of the first row, context).  Exact, but for products with
// scales beyond bfloat16's range.
__global__ void __launch_bounds__(kQ8Threads)
unpack_pages_q8_kernel(const uint8_t* k_codes, const uint8_t* v_codes, const float* k_scale, const float* v_scale,
                       const int* block_tables, int max_blocks, const int* seq_q_len, const int* seq_ctx_len, bf16* __restrict__ k_pages,
                       bf16* __restrict__ v_pages, int first_seq, int blocks, int nkv, int hd, int block_size, int num_pages, int window) {
  pdl_launch_dependents();
  pdl_wait();
  const int seq = first_seq + blockIdx.y, block = blockIdx.x;
  const int ctx = seq_ctx_len[seq];
  const int lo = first_visible(max(ctx - seq_q_len[seq], 0), window, 0);
  if (block * block_size >= ctx || (block + 1) * block_size <= lo) return;
  const int words = hd / 8, per_head = block_size * words;
  const size_t page = q8::head_page(block_tables[size_t(seq) * max_blocks + block], 0, nkv, num_pages);
  const size_t to = (size_t(blockIdx.y) * blocks + block) * nkv * block_size * hd;
  for (int i = threadIdx.x; i < 2 * nkv * per_head; i += kQ8Threads) {
    const int head = i / per_head, at = i - head * per_head;
    const int off = at / words, word = at - off * words;
    const bool is_k = head < nkv;
    const int kvh = is_k ? head : head - nkv;
    float x[8];
    // (positions behind the context may hold anything; their probabilities are zero, and zero times a value must stay zero)
    if (block * block_size + off < ctx) {
      const float scale = (is_k ? k_scale : v_scale)[page + kvh];
      const uint2 u = *reinterpret_cast<const uint2*>((is_k ? k_codes : v_codes) + ((page + kvh) * block_size + off) * hd + word * 8);
      q8::values4(u.x, scale, x);
      q8::values4(u.y, scale, x + 4);
    } else {
      for (int e = 0; e < 8; ++e) x[e] = 0.f;
    }
    store8((is_k ? k_pages : v_pages) + to + (size_t(kvh) * block_size + off) * hd + word * 8, x);
  }
}

namespace {

// Lanes of a head, as a power of two: hd / 16, rounded up.
int q8_log2_lanes(int hd) {
  int n = 0;
  while ((16 << n) < hd) ++n;
  return n;
}

bool q8_sizes_ok(int nkv, int hd, int block_size, int num_pages) {
  return nkv > 0 && nkv <= 8192 && hd >= 8 && hd <= 256 && hd % 8 == 0 && block_size > 0 && block_size <= q8::kMaxBlock && num_pages > 0;
}

template <typename T, int W>
int launch_store_q8_as(const StoreQ8Params& p, cudaStream_t s) {
  const int R = 32 >> p.log2_lanes, units = (W == 1 ? (p.nh + R - 1) / R : p.nh) + 2 * p.nkv;
  return pdl_launch(store_q8_kernel<T, W>, dim3((p.rows + W - 1) / W, (units + kQ8Warps - 1) / kQ8Warps), dim3(kQ8Threads), 0, s, p);
}
template <typename T>
int launch_store_q8(const StoreQ8Params& p, cudaStream_t s) {
  // Few rows: a window each, or a warp would take several requests' runs one behind another; many: windows as long as a usual page.
  return p.rows <= 512 ? launch_store_q8_as<T, 1>(p, s) : p.rows <= 2048 ? launch_store_q8_as<T, 8>(p, s) : launch_store_q8_as<T, 16>(p, s);
}

}  // namespace
}  // namespace kvcm

using namespace kvcm;

// q|k|v rows (nh + 2 nkv heads of hd) -> rotated q rows in q_out, k and v in the pages of their slots (slot < 0: nowhere).
// `angles` [rows, rotary_dim] float32, cosines then sines (null: no rotation).  All rows and addresses on 16 bytes.
#define KVCM_STORE_Q8(SUFFIX, T)                                                                                              \
  KVCM_API int kvcm_rope_cache_q8_##SUFFIX(const void* qkv, long long row_stride, const float* angles, int rotary_dim,         \
                                           int interleaved, const int* slot_mapping, void* k_codes, void* v_codes,             \
                                           float* k_scale, float* v_scale, void* q_out, long long q_stride, int rows, int nh,  \
                                           int nkv, int hd, int block_size, int num_pages, void* stream) {                     \
    if (rows <= 0) return 0;                                                                                                   \
    if (!q8_sizes_ok(nkv, hd, block_size, num_pages) || nh < 0 || nh > 32768) return KVCM_ERR_UNSUPPORTED;                     \
    if (angles != nullptr && (rotary_dim < 2 || rotary_dim > hd || rotary_dim % (interleaved ? 2 : 16)))                       \
      return KVCM_ERR_UNSUPPORTED;                                                                                             \
    const uintptr_t places = reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) |                           \
                             uintptr_t(row_stride * sizeof(T)) | uintptr_t(q_stride * sizeof(T)) |                             \
                             reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) |                     \
                             reinterpret_cast<uintptr_t>(angles);                                                              \
    if (places & 15) return KVCM_ERR_UNSUPPORTED;                                                                              \
    StoreQ8Params p;                                                                                                           \
    p.qkv = qkv; p.row_stride = row_stride; p.angles = angles; p.rotary_dim = rotary_dim; p.interleaved = interleaved;         \
    p.slot_mapping = slot_mapping; p.k_codes = (uint8_t*)k_codes; p.v_codes = (uint8_t*)v_codes; p.k_scale = k_scale;          \
    p.v_scale = v_scale; p.q_out = q_out; p.q_stride = q_stride; p.rows = rows; p.nh = nh; p.nkv = nkv; p.hd = hd;             \
    p.block_size = block_size; p.num_pages = num_pages;                                                                        \
    p.log2_lanes = q8_log2_lanes(hd);                                                                                          \
    return launch_store_q8<T>(p, (cudaStream_t)stream);                                                                        \
  }                                                                                                                           \
  KVCM_API int kvcm_read_cache_q8_##SUFFIX(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale, \
                                           const int* slot_mapping, void* k_rows, void* v_rows, long long k_stride,            \
                                           long long v_stride, int rows, int nkv, int hd, int block_size, int num_pages,       \
                                           void* stream) {                                                                    \
    if (rows <= 0) return 0;                                                                                                   \
    const uintptr_t places = reinterpret_cast<uintptr_t>(k_rows) | reinterpret_cast<uintptr_t>(v_rows) |                       \
                             uintptr_t(k_stride * sizeof(T)) | uintptr_t(v_stride * sizeof(T)) |                               \
                             reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes);                      \
    if (!q8_sizes_ok(nkv, hd, block_size, num_pages) || (places & 15)) return KVCM_ERR_UNSUPPORTED;                            \
    const int log2_lanes = q8_log2_lanes(hd), items = 2 * nkv << log2_lanes, pieces = (items + kQ8Threads - 1) / kQ8Threads;   \
    return pdl_launch(read_q8_kernel<T>, dim3(rows, pieces), dim3(((items + pieces - 1) / pieces + 31) / 32 * 32), 0,          \
                      (cudaStream_t)stream, (const uint8_t*)k_codes, (const uint8_t*)v_codes, k_scale, v_scale, slot_mapping,  \
                      (T*)k_rows, (T*)v_rows, k_stride, v_stride, nkv, hd, block_size, num_pages, log2_lanes);                 \
  }

KVCM_STORE_Q8(bf16, bf16)
KVCM_STORE_Q8(f32, float)

// k_pages, v_pages: room for seqs x blocks pages [nkv, block_size, hd] of bfloat16.
KVCM_API int kvcm_unpack_pages_q8_bf16(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                                       const int* block_tables, int max_blocks, const int* seq_q_len, const int* seq_ctx_len,
                                       void* k_pages, void* v_pages, int first_seq, int seqs, int blocks, int nkv, int hd, int block_size,
                                       int num_pages, int window, void* stream) {
  if (seqs <= 0 || blocks <= 0) return 0;
  if (!q8_sizes_ok(nkv, hd, block_size, num_pages) || blocks > max_blocks || seqs > 65535) return KVCM_ERR_UNSUPPORTED;
  return pdl_launch(unpack_pages_q8_kernel, dim3(blocks, seqs), dim3(kQ8Threads), 0, (cudaStream_t)stream, (const uint8_t*)k_codes,
                    (const uint8_t*)v_codes, k_scale, v_scale, block_tables, max_blocks, seq_q_len, seq_ctx_len, (bf16*)k_pages,
                    (bf16*)v_pages, first_seq, blocks, nkv, hd, block_size, num_pages, window);
}

KVCM_PACKED(kvcm_rope_cache_q8_bf16)
KVCM_PACKED(kvcm_rope_cache_q8_f32)
KVCM_PACKED(kvcm_read_cache_q8_bf16)
KVCM_PACKED(kvcm_read_cache_q8_f32)
KVCM_PACKED(kvcm_unpack_pages_q8_bf16)
