// Causal attention of many rows of a request on the fifth-generation tensor cores: portions over a paged cache in 8 bits (format: q8.cuh), and
// whole prompts over their own bfloat16 rows, packed one behind another.  head_dim up to 128.
//
// One block per (256 query rows of a request, query head), as two groups of 128 rows that share every tile of keys and values.  Per
// tile of 128 keys and group:
//     S = Q K^T   accumulator in tensor memory
//     softmax     one thread a row:  p = 2^(x - m), x the scaled scores; P lies in tensor memory over the scores that it was made of
//     O += P V    V as the MN-major operand, O in tensor memory for the whole block
// A row takes its scores 32 at a time, relative to the maximum that it knows, without looking for theirs: where 32 probabilities
// add up to more than 2^12 (or the row has seen nothing yet) their maximum is found, sums, O and the tile's earlier probabilities
// are rescaled, and the 32 are taken again, which after the first tiles hardly ever happens.
// The products of a group run in order: S of the next tile behind O += P V of this one, so one barrier says that S is there, that
// O holds the tile before, and that P has been read.
//
// Prompts: bfloat16 operands, tiles of K and V by TMA straight from the rows (three coordinates: element, head, row, so that elements
// beyond head_dim are zeros and heads of any multiple of 8 fill blocks of 64).
// Pages: float16 operands.  Codes are exact in float16, so seven warps turn them into operands with one conversion for two; scales stay
// out of the products: the key's enters the score's factor, the value's, a power of two, the probability's exponent
// (2^(x - m) scale = 2^(x - m + log2 scale): weights in place of probabilities), one factor for eight keys, which lie in one page.
// m is the reference of the weights, and sums take the weights' scales out again.  q enters as float16 times a power of two for
// each row, exact but for elements 2^-29 as large as the row's largest.  P is rounded to float16 (prompts: bfloat16), and once more where a
// maximum is renewed inside its tile.
//
// Values that are not finite and that some row of a tile does not see would come to it as zero times them.  Rows past the
// last are zeros in shared memory; a row whose result is not finite looks whether an unseen value was the reason, and is then
// attended once more without the tensor cores.
//
// Every wait is bounded; one that runs out sets the error word of the tcgen05 attention family (codes 33 and up) and ends the block.
#include <cuda_fp16.h>

#include "packed.cuh"
#include "pdl.cuh"
#include "q8.cuh"
#include "tcgen05_common.cuh"

extern "C" const int* kvcm_attention_tcgen05_error_address(void);

namespace kvcm {

constexpr int kArGroupRows = 128, kArRows = 256;
constexpr int kArKeys = 128;
constexpr int kArTile = 128 * 128;                 // [128 rows][64 elements of 16 bits]: also a 64-wide block of a tile of keys or values
constexpr int kArStages = 2;                       // tiles of keys, and of values
constexpr int kArRing = 4;                         // tiles' scales
constexpr int kArKeyWarps = 4, kArValueWarps = 3;  // pages: who turns codes into operands
constexpr float kArMost = 4096.f;                  // a row's sum of 32 weights from which its maximum is renewed
// tensor memory: S of group g at column g * 128 (and P in its first 64 columns); O of group g at 256 + g * HD

struct ArScales { float key, value, out; };        // of eight keys: scale, log2 of the value's less the block's, 2^-(that)

struct RowsParams {
  bf16* out; long long out_stride;
  const bf16* q; long long q_stride;
  const bf16* k; long long k_stride; const bf16* v; long long v_stride;                      // prompts
  const uint8_t* k_codes; const uint8_t* v_codes; const float* k_scale; const float* v_scale;      // pages
  const int* block_tables; int max_blocks, max_keys;      // keys that a request's table has pages for
  const int* tile_seq; const int* tile_q0; int tiles;     // tiles of 64 rows; a block takes every fourth and its three successors
  const int* seq_q_start; const int* seq_q_len; const int* seq_ctx_len;
  int nh, nkv, hd, block_size, log2_block, num_pages, window;
  float scale_log2, cap_pre;
  const float* sink;
  int* error;
};

namespace {

__device__ __forceinline__ float ar_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ar_tanh(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(ar_exp2(x * 2.8853900817779268f) + 1.f));
  return fmaf(-2.f, r, 1.f);
}
// a * b + c of two floats at once
__device__ __forceinline__ float2 ar_fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 ar_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// 16 consecutive columns of this thread's lane of tensor memory (no wait).
__device__ __forceinline__ void ar_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                 "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr));
}
__device__ __forceinline__ void ar_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
// Waits for the loads of tensor memory that the thread has asked for; `v` is one of them (nothing of it is used before).
__device__ __forceinline__ void ar_wait32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :: "memory");
  asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                    "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
// The product with its first operand in tensor memory: 16-bit elements, two neighbours of a row to a column.
__device__ __forceinline__ void ar_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t instr, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(instr), "r"(accumulate) : "memory");
}
// A box of [rows][64 elements] of one head: x element, y head, z row.
__device__ __forceinline__ void ar_tma_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n"
               ::"r"(tc5::s32(dst)), "l"(map), "r"(tc5::s32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
template <bool HALF> __device__ __forceinline__ uint32_t ar_pack(float a, float b) {
  uint32_t r;
  if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
template <bool HALF> __device__ __forceinline__ float2 ar_unpack(uint32_t v) {
  if constexpr (HALF) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// What turns a row's products into scores: x = s * factor (capped: tanh(s * factor) * scale_log2).
struct ArRow { float factor, scale_log2; };

// The scores of two keys behind their tanh or factor, plus `add`.
template <bool CAP>
__device__ __forceinline__ float2 ar_scores(uint32_t s0, uint32_t s1, float factor, float scale_log2, float add) {
  const float2 s = make_float2(__uint_as_float(s0), __uint_as_float(s1));
  if constexpr (CAP) return make_float2(fmaf(ar_tanh(s.x * factor), scale_log2, add), fmaf(ar_tanh(s.y * factor), scale_log2, add));
  else return ar_fma2(s, make_float2(factor, factor), make_float2(add, add));
}

// 32 products of a row into weights; `weights` their sum, `sum` that of the probabilities.  MASK: only keys [a, b) of the 32 count.
// AGAIN: the maximum is known, so nothing is above 2^12 but what scores of 2^24 and more are rounded by.
template <bool CAP, bool PAGES, bool MASK, bool AGAIN>
__device__ __forceinline__ void ar_exponentials(const uint32_t (&s)[32], const ArScales* sc, uint32_t (&packed)[16], const ArRow& row, float m,
                                                int a, int b, float& weights, float& sum) {
  float2 w2 = make_float2(0.f, 0.f), l2 = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float factor = row.factor, add = -m, out = 1.f;
    if constexpr (PAGES) {
      factor *= sc[j].key;
      add += sc[j].value;
      out = sc[j].out;
    }
    float2 g0, g1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 8 * j + 2 * k;
      float2 t = ar_scores<CAP>(s[i], s[i + 1], factor, row.scale_log2, add);
      if constexpr (MASK) {
        t.x = i >= a && i < b ? t.x : -INFINITY;
        t.y = i + 1 >= a && i + 1 < b ? t.y : -INFINITY;
      }
      if constexpr (AGAIN) t = make_float2(t.x > 12.f ? 12.f : t.x, t.y > 12.f ? 12.f : t.y);      // (not-a-number stays)
      const float2 e = make_float2(ar_exp2(t.x), ar_exp2(t.y));
      if (k == 0) g0 = e; else if (k == 1) g1 = e; else if (k == 2) g0 = ar_add2(g0, e); else g1 = ar_add2(g1, e);
      packed[i / 2] = ar_pack<PAGES>(e.x, e.y);
    }
    g0 = ar_add2(g0, g1);
    w2 = ar_add2(w2, g0);
    if constexpr (PAGES) l2 = ar_fma2(g0, make_float2(out, out), l2);
  }
  weights = w2.x + w2.y;
  sum = PAGES ? l2.x + l2.y : weights;
}

// The largest of the 32 weights' exponents, less m.
template <bool CAP, bool PAGES>
__device__ __forceinline__ float ar_largest(const uint32_t (&s)[32], const ArScales* sc, const ArRow& row, float m, int a, int b) {
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float factor = PAGES ? row.factor * sc[j].key : row.factor, add = PAGES ? sc[j].value - m : -m;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 8 * j + 2 * k;
      const float2 t = ar_scores<CAP>(s[i], s[i + 1], factor, row.scale_log2, add);
      mx = (i >= a && i < b) ? fmaxf(mx, t.x) : mx;
      mx = (i + 1 >= a && i + 1 < b) ? fmaxf(mx, t.y) : mx;
    }
  }
  return mx;
}

// What a row has in tensor memory times alpha: O, and the first `chunks` pieces of 32 weights, which are rounded once more by
// that (a tile's pieces at most three times, and only where scores climb inside the tile).  The whole warp takes part.
template <int HD, bool HALF>
__device__ __noinline__ void ar_rescale(uint32_t o_addr, bool has_o, uint32_t p_addr, int chunks, float alpha) {
  uint32_t v[16];
#pragma unroll 1
  for (int c = 0; has_o && c < HD / 16; ++c) {
    ar_ld16(o_addr + uint32_t(c * 16), v);
    tc5::ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
    ar_st16(o_addr + uint32_t(c * 16), v);
  }
  if (chunks > 0) tc5::st_wait();                                  // loads of tensor memory pass stores that nobody waited for
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    ar_ld16(p_addr + uint32_t(c * 16), v);
    tc5::ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 f = ar_unpack<HALF>(v[i]);
      v[i] = ar_pack<HALF>(f.x * alpha, f.y * alpha);
    }
    ar_st16(p_addr + uint32_t(c * 16), v);
  }
  tc5::st_wait();
}

// Keys and values of one request and KV head, element by element.
template <bool PAGES> struct ArKeys {
  const RowsParams& p;
  const int* table;
  int start, kvh;
  __device__ __forceinline__ size_t place(int key) const {
    if constexpr (PAGES) {
      const int pi = p.log2_block >= 0 ? key >> p.log2_block : key / p.block_size;
      return q8::head_page(table[pi], kvh, p.nkv, p.num_pages) * p.block_size + (key - pi * p.block_size);
    } else {
      return size_t(start) + key;
    }
  }
  __device__ __forceinline__ float key(size_t at, int d) const {
    if constexpr (PAGES) return q8::floats2(p.k_codes[at * p.hd + d]).x * p.k_scale[at / p.block_size];
    else return ldf(p.k + at * p.k_stride + size_t(kvh) * p.hd + d);
  }
  __device__ __forceinline__ float value(size_t at, int d) const {
    if constexpr (PAGES) return q8::floats2(p.v_codes[at * p.hd + d]).x * p.v_scale[at / p.block_size];
    else return ldf(p.v + at * p.v_stride + size_t(kvh) * p.hd + d);
  }
};

// A row whose result is not finite, by a whole warp: if a value that it does not see, of the keys [from, first) and (pos, to) that its
// products had, is not finite, the row is attended again, key by key.
template <int HD, bool CAP, bool PAGES>
__device__ __noinline__ void ar_again(const RowsParams& p, int seq, int start, int head, int row, int pos, int first, int from, int to) {
  const int lane = threadIdx.x & 31, kvh = head / (p.nh / p.nkv);
  const ArKeys<PAGES> keys{p, PAGES ? p.block_tables + size_t(seq) * p.max_blocks : nullptr, start, kvh};
  bool sick = false;
  for (int j = from + lane; j < to; j += 32) {
    if (j >= first && j <= pos) continue;
    const size_t at = keys.place(j);
    for (int d = 0; d < p.hd; ++d) sick |= !(fabsf(keys.value(at, d)) <= 3.402823466e38f);
  }
  if (!__any_sync(0xffffffffu, sick)) return;
  float q[HD / 32], o[HD / 32], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i) {
    const int d = i * 32 + lane;
    q[i] = d < p.hd ? ldf(p.q + size_t(row) * p.q_stride + size_t(head) * p.hd + d) : 0.f;
    o[i] = 0.f;
  }
  for (int j = first; j <= pos; ++j) {
    const size_t at = keys.place(j);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
      if (i * 32 + lane < p.hd) s = fmaf(q[i], keys.key(at, i * 32 + lane), s);
    s = warp_sum(s);
    const float x = CAP ? ar_tanh(s * p.cap_pre) * p.scale_log2 : s * p.scale_log2;
    const float top = x > m ? x : m, f = m == -INFINITY ? 0.f : ar_exp2(m - top), e = x == -INFINITY ? 0.f : ar_exp2(x - top);
    m = top;
    l = fmaf(l, f, e);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
      if (i * 32 + lane < p.hd) o[i] = fmaf(e, keys.value(at, i * 32 + lane), o[i] * f);
  }
  if (p.sink && m != -INFINITY) l += ar_exp2(p.sink[head] * 1.4426950408889634f - m);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < HD / 32; ++i)
    if (i * 32 + lane < p.hd) stf(p.out + size_t(row) * p.out_stride + size_t(head) * p.hd + i * 32 + lane, l == 0.f ? 0.f : o[i] * inv);
}

// 16 codes (elements 16 ch .. 16 ch + 15 of row r) as float16 into a 128-byte swizzled tile [HD/64][128 rows][64].  The lanes of a
// row's second block write their halves the other way round, so that eight lanes meet in no bank.
template <int HD>
__device__ __forceinline__ void ar_spread(unsigned char* tile, uint4 u, int r, int ch) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint4 half[2];
  uint32_t* h = reinterpret_cast<uint32_t*>(half);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = q8::halves2(w[i] & 0xffffu);
    h[2 * i + 1] = q8::halves2(w[i] >> 16);
  }
  unsigned char* row = tile + (ch >> 2) * kArTile + r * 128;
  const int c = (ch & 3) * 2, swap = HD > 64 ? ch >> 2 : 0;
  *reinterpret_cast<uint4*>(row + (((c + swap) ^ (r & 7)) * 16)) = swap ? half[1] : half[0];
  *reinterpret_cast<uint4*>(row + (((c + 1 - swap) ^ (r & 7)) * 16)) = swap ? half[0] : half[1];
}

template <int HD, bool PAGES> constexpr size_t ar_smem() {
  return size_t(2 + 2 * kArStages) * (HD / 64) * kArTile + (PAGES ? kArRing * (kArKeys / 8) * sizeof(ArScales) : 0);
}
template <bool PAGES> constexpr int ar_threads() { return PAGES ? 512 : 320; }

template <int HD, bool CAP, bool PAGES>
__global__ void __launch_bounds__(ar_threads<PAGES>(), 1)
attention_rows_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int KB = HD / 64;                                      // 64-wide blocks of a head
  constexpr int kMmaWarp = PAGES ? 15 : 9;
  constexpr int kPieces = HD / 16;                                 // pages: 16-byte pieces of a row of codes
  unsigned char* q_s = smem_raw;                                   // [2][KB][128 rows][64]
  unsigned char* k_s = q_s + 2 * KB * kArTile;                     // [stages][KB][128 keys][64]
  unsigned char* v_s = k_s + kArStages * KB * kArTile;
  ArScales* scales = reinterpret_cast<ArScales*>(v_s + kArStages * KB * kArTile);          // [ring][16 groups of eight keys]
  __shared__ __align__(8) uint64_t q_full, q_ready, k_full[kArStages], v_full[kArStages], k_free[kArStages], v_free[kArStages], v_tail,
      sc_full[kArRing], s_full[2], p_full[2], o_full;
  __shared__ uint32_t tmem_base;
  __shared__ float value_base;                                     // log2 of the value scale that weights are relative to
  __shared__ volatile int abort_flag;

  // heads fastest and the last tiles, which see most keys, first
  const int tile = int(gridDim.y) - 1 - int(blockIdx.y), head = blockIdx.x;
  int* const error = p.error;
  // Tiles and lengths may come from a kernel of the same step, so they are read behind the wait.  (Whoever leaves waits as
  // well: a launch of nothing but empty tiles would else be over before the kernel in front of it.)
  pdl_wait();
  int seq, q0, most = kArRows;
  if (!PAGES && tile >= p.tiles) {                                 // a prompt of one row
    seq = tile - p.tiles;
    q0 = 0;
    most = 1;
  } else {
    seq = p.tile_seq[tile];
    q0 = p.tile_q0[tile];
  }
  if (seq < 0 || (q0 & (kArRows - 1))) return;                     // no tile, or one that belongs to a block before
  const int q_start = p.seq_q_start[seq], q_len = p.seq_q_len[seq];
  const int rows_here = min(most, q_len - q0);
  if (rows_here <= 0) return;
  if (tc5::s32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicExch(error, (33 << 16) | int(blockIdx.y & 0xffff));
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctx = PAGES ? min(p.seq_ctx_len[seq], p.max_keys) : q_len;       // (a context ends with its table)
  const int pos0 = ctx - q_len + q0;                               // position of the block's first row
  const int hi = pos0 + rows_here;                                 // keys [lo, hi) matter to the block
  const int lo = first_visible(pos0, p.window, 0);
  const int j0 = lo / kArKeys;
  const int groups = rows_here > kArGroupRows ? 2 : 1;
  // a group's keys end with its last row's own, and so do its tiles
  const int hi_first = groups == 1 ? hi : pos0 + kArGroupRows;
  const int n_tiles = (hi - 1) / kArKeys - j0 + 1, n_first = (hi_first - 1) / kArKeys - j0 + 1;
  const int kvh = head / (p.nh / p.nkv);

  if (threadIdx.x == 0) {
    abort_flag = 0;
    tc5::mbar_init(&q_full, 1);
    tc5::mbar_init(&q_ready, 4 * groups);
    for (int i = 0; i < kArStages; ++i) {
      tc5::mbar_init(&k_full[i], PAGES ? kArKeyWarps : 1);
      tc5::mbar_init(&v_full[i], PAGES ? kArValueWarps : 1);
      tc5::mbar_init(&k_free[i], 1);
      tc5::mbar_init(&v_free[i], 1);
    }
    tc5::mbar_init(&v_tail, 1);
    for (int i = 0; i < kArRing; ++i) tc5::mbar_init(&sc_full[i], 1);
    for (int g = 0; g < 2; ++g) {
      tc5::mbar_init(&s_full[g], 1);
      tc5::mbar_init(&p_full[g], 4);                               // a group's four warps
    }
    tc5::mbar_init(&o_full, 1);
    tc5::mbar_init_fence();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5::s32(&tmem_base)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  tc5::fence_before();
  __syncthreads();
  tc5::fence_after();
  const uint32_t tmem = tmem_base;
  pdl_launch_dependents();                                         // (only with the tensor memory in hand, see attention_tcgen05.cu)

  auto fail = [&](int code) {
    atomicExch(error, (code << 16) | int(blockIdx.y & 0xffff));
    abort_flag = 1;
  };
  auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {  // the warp stays together whatever a lane saw
    if (__all_sync(0xffffffffu, tc5::mbar_wait(bar, parity))) return true;
    if (!abort_flag && lane == 0) fail(code);                      // (the first to give up says so; the others' waits run out too)
    return false;
  };

  if (warp == kMmaWarp) {
    // ---- one thread: the products
    if (lane == 0) {
      if (PAGES) {
        tc5::mbar_expect_tx(&q_full, groups * KB * kArTile);
        for (int g = 0; g < groups; ++g)
          for (int kb = 0; kb < KB; ++kb)
            ar_tma_3d(q_s + (g * KB + kb) * kArTile, &map_q, &q_full, kb * 64, head, q_start + q0 + g * kArGroupRows);
      }
      constexpr uint32_t kTypes = PAGES ? ~((7u << 7) | (7u << 10)) : ~0u;       // float16 or bfloat16
      constexpr uint32_t idesc_s = tc5::idesc(kArGroupRows, kArKeys, false) & kTypes;
      constexpr uint32_t idesc_o = tc5::idesc(kArGroupRows, HD, true) & kTypes;
      constexpr uint64_t kStageStep = (KB * kArTile) >> 4;          // (descriptor addresses count units of 16 bytes)
      const uint64_t dk = tc5::smem_desc(tc5::s32(k_s));
      // values, MN-major: 64-wide blocks a leading offset apart
      const uint64_t dv = (tc5::smem_desc(tc5::s32(v_s)) & ~(uint64_t(0x3fff) << 16)) | (uint64_t(kArTile >> 4) << 16);
      bool ok = tc5::mbar_wait(PAGES ? &q_ready : &q_full, 0);
      if (!ok) fail(34);
      tc5::fence_after();
      for (int n = 0; ok && n <= n_tiles; ++n) {
        for (int g = 0; g < groups; ++g) {
          const int mine = g == 0 ? n_first : n_tiles;
          if (n >= 1 && n <= mine) {                               // O += P_(n-1) V_(n-1)
            const int m = n - 1, st = m % kArStages;
            if (!tc5::mbar_wait(&v_full[st], (m / kArStages) & 1)) { fail(35); ok = false; break; }
            if (!tc5::mbar_wait(&p_full[g], m & 1)) { fail(36); ok = false; break; }
            tc5::fence_after();
            // (of the last tile only the steps of 16 keys that some row of the group sees)
            const int steps = min(kArKeys, (g == 0 ? hi_first : hi) - (j0 + m) * kArKeys + 15) / 16;
            for (int j = 0; j < steps; ++j)                        // 16 keys: 8 columns of P, 16 rows down V
              ar_mma_ts(tmem + 256 + g * HD, tmem + g * kArKeys + j * 8, dv + st * kStageStep + uint64_t(j * (16 * 128 >> 4)), idesc_o,
                        (m > 0 || j > 0) ? 1u : 0u);
          }
          if (n < mine) {                                          // S_n, over P_(n-1)
            const int st = n % kArStages;
            if (!tc5::mbar_wait(&k_full[st], (n / kArStages) & 1)) { fail(37); ok = false; break; }
            tc5::fence_after();
            const uint64_t dq = tc5::smem_desc(tc5::s32(q_s + g * KB * kArTile));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc5::mma(tmem + uint32_t(g * kArKeys), dq + uint64_t(kb * (kArTile >> 4) + 2 * j),
                         dk + st * kStageStep + uint64_t(kb * (kArTile >> 4) + 2 * j), idesc_s, (kb > 0 || j > 0) ? 1u : 0u);
            tc5::commit(&s_full[g]);                               // and O += P_(n-1) V_(n-1) before it
          }
        }
        if (!ok) break;
        if (n < n_tiles) tc5::commit(&k_free[n % kArStages]);      // tile n of the keys is read,
        if (n >= 1) tc5::commit(&v_free[(n - 1) % kArStages]);     // and n - 1 of the values
      }
      tc5::commit(&o_full);
    }
  } else if (!PAGES && warp == 8) {
    // ---- prompts: one thread asks for Q, K and V
    const int tail = hi - (j0 + n_tiles - 1) * kArKeys;            // keys of the last tile
    bool ok = true;
    for (int n = 0; ok && n < n_tiles; ++n) {
      const int st = n % kArStages, key = q_start + (j0 + n) * kArKeys;
      const uint32_t parity = ((n / kArStages) & 1) ^ 1;
      // (the product of the last tile takes 16 keys at a time; behind the prompt's last come zeros)
      const bool ends = n == n_tiles - 1 && tail % 16 != 0;
      if (lane == 0) {
        ok = tc5::mbar_wait(&k_free[st], parity);
        if (ok) {
          if (n == 0) {
            tc5::mbar_expect_tx(&q_full, groups * KB * kArTile);
            for (int g = 0; g < groups; ++g)
              for (int kb = 0; kb < KB; ++kb)
                ar_tma_3d(q_s + (g * KB + kb) * kArTile, &map_q, &q_full, kb * 64, head, q_start + q0 + g * kArGroupRows);
          }
          tc5::mbar_expect_tx(&k_full[st], KB * kArTile);
          for (int kb = 0; kb < KB; ++kb) ar_tma_3d(k_s + (st * KB + kb) * kArTile, &map_k, &k_full[st], kb * 64, kvh, key);
          ok = tc5::mbar_wait(&v_free[st], parity);
        }
        if (ok) {
          uint64_t* const bar = ends ? &v_tail : &v_full[st];
          tc5::mbar_expect_tx(bar, KB * kArTile);
          for (int kb = 0; kb < KB; ++kb) ar_tma_3d(v_s + (st * KB + kb) * kArTile, &map_v, bar, kb * 64, kvh, key);
        }
        if (!ok && !abort_flag) fail(38);
      }
      ok = __shfl_sync(0xffffffffu, int(ok), 0);
      if (ok && ends) {
        ok = wait_all(&v_tail, 0, 39);
        const int to = (tail + 15) / 16 * 16;
        for (int kb = 0; ok && kb < KB; ++kb)
          for (int i = tail * 8 + lane; i < to * 8; i += 32)
            *reinterpret_cast<uint4*>(v_s + (st * KB + kb) * kArTile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (ok && lane == 0) tc5::mbar_arrive(&v_full[st]);
      }
    }
  } else if (PAGES && warp >= 8 && warp < 8 + kArKeyWarps + kArValueWarps) {
    // ---- pages: codes into operands; four warps the keys, three the values.  A thread asks for its pieces of the next tile behind
    // those of this one.
    const bool is_k = warp < 8 + kArKeyWarps;
    const int threads = 32 * (is_k ? kArKeyWarps : kArValueWarps), t = threadIdx.x - (is_k ? 256 : 256 + 32 * kArKeyWarps);
    constexpr int kMost = (kArKeys * kPieces + 32 * kArValueWarps - 1) / (32 * kArValueWarps);
    const uint8_t* const codes = is_k ? p.k_codes : p.v_codes;
    unsigned char* const to = is_k ? k_s : v_s;
    const ArKeys<true> keys{p, p.block_tables + size_t(seq) * p.max_blocks, 0, kvh};
    uint4 held[kMost];
    float2 of_group;                                               // scales of the eight keys that a lane of the first warp has
    auto ask = [&](int n) {
      const int key0 = (j0 + n) * kArKeys;
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const int piece = i * threads + t, r = piece / kPieces, ch = piece % kPieces;
        held[i] = make_uint4(0u, 0u, 0u, 0u);                      // (keys of nobody: zero times them stays zero)
        if (piece < kArKeys * kPieces && key0 + r >= lo && key0 + r < hi)
          held[i] = *reinterpret_cast<const uint4*>(codes + keys.place(key0 + r) * HD + ch * 16);
      }
      of_group = make_float2(0.f, 1.f);
      if (warp == 8 && lane < kArKeys / 8) {
        const int key = max(key0 + lane * 8, lo);
        if (key < min(hi, key0 + lane * 8 + 8)) {
          const size_t at = keys.place(key) / p.block_size;
          of_group = make_float2(p.k_scale[at], p.v_scale[at]);
        }
      }
    };
    ask(0);
    float base = 0.f;
    for (int n = 0; n < n_tiles; ++n) {
      const int st = n % kArStages;
      if (n >= kArStages && !wait_all(is_k ? &k_free[st] : &v_free[st], ((n / kArStages) & 1) ^ 1, is_k ? 40 : 41)) break;
      if (warp == 8) {
        // (S_(n-2) is complete, so the weights of tile n - 3 are made, and the place of tile n - 4 is free)
        const float log_v = log2f(fmaxf(of_group.y, 1.17549435e-38f));
        if (n == 0) {
          base = __shfl_sync(0xffffffffu, log_v, (lo % kArKeys) / 8);
          if (lane == 0) value_base = base;
        }
        if (lane < kArKeys / 8) {
          const bool there = (j0 + n) * kArKeys + lane * 8 < hi && (j0 + n) * kArKeys + lane * 8 + 8 > lo;
          ArScales s;
          s.key = of_group.x;
          s.value = there ? log_v - base : 0.f;
          s.out = there ? exp2f(base - log_v) : 0.f;
          scales[(n % kArRing) * (kArKeys / 8) + lane] = s;
        }
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&sc_full[n % kArRing]);
      }
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const int piece = i * threads + t;
        if (piece < kArKeys * kPieces) ar_spread<HD>(to + st * KB * kArTile, held[i], piece / kPieces, piece % kPieces);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(is_k ? &k_full[st] : &v_full[st]);
      if (n + 1 < n_tiles) ask(n + 1);
    }
  } else if (warp < 8 && (warp >> 2) < groups) {
    // ---- softmax and output: this thread owns row r of its group (lane r of tensor memory)
    const int g = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int mine = g == 0 ? n_first : n_tiles, hi_mine = g == 0 ? hi_first : hi;
    const int row = g * kArGroupRows + r, pos = pos0 + row;        // rows beyond rows_here compute and store nothing
    const uint32_t lane_addr = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + g * kArKeys, o_addr = lane_addr + 256 + g * HD;
    const int first = first_visible(pos, p.window, 0);
    const int group_pos = pos0 + g * kArGroupRows;                 // of the group's first row
    const int last_first = first_visible(group_pos + kArGroupRows - 1, p.window, 0);
    bool alive = true;
    ArRow rf{CAP ? p.cap_pre : p.scale_log2, p.scale_log2};
    if constexpr (PAGES) {                                         // q as float16, its largest element between 2^14 and 2^15
      alive = wait_all(&q_full, 0, 42);
      if (alive) {
        unsigned char* const at = q_s + g * KB * kArTile + r * 128;
        float largest = 0.f, bad = 0.f;
#pragma unroll 4
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(at + (c >> 3) * kArTile + (((c & 7) ^ (r & 7)) * 16));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = ar_unpack<false>(w[i]);
            largest = fmaxf(largest, fmaxf(fabsf(f.x), fabsf(f.y)));
            bad = fmaf(f.x, 0.f, fmaf(f.y, 0.f, bad));             // not-a-number where an element is not finite
          }
        }
        // 2^(14 - exponent of the largest), and its reciprocal
        const int e = min(max(int(__float_as_uint(largest) >> 23), 15), 254);
        const float up = __uint_as_float(uint32_t(min(127 + 14 + 127 - e, 254)) << 23);
        rf.factor *= __uint_as_float(uint32_t(254 - min(127 + 14 + 127 - e, 253)) << 23) + bad;
#pragma unroll 4
        for (int c = 0; c < HD / 8; ++c) {
          uint4* const u = reinterpret_cast<uint4*>(at + (c >> 3) * kArTile + (((c & 7) ^ (r & 7)) * 16));
          uint32_t w[4] = {u->x, u->y, u->z, u->w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 f = ar_unpack<false>(w[i]);
            w[i] = ar_pack<true>(f.x * up, f.y * up);
          }
          *u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&q_ready);
      }
    }
    float m = -INFINITY;                                           // the maximum the row currently scales by
    bool fresh = true;                                             // some row of the warp has none
    float l = 0.f;
    for (int n = 0; n < mine; ++n) {
      alive = alive && wait_all(&s_full[g], n & 1, 43) && (!PAGES || wait_all(&sc_full[n % kArRing], (n / kArRing) & 1, 44));
      if (!alive) break;
      tc5::fence_after();
      const ArScales* sc = scales + (n % kArRing) * (kArKeys / 8);
      const int key0 = (j0 + n) * kArKeys;
      // the keys of this tile that the row may see: [a, b) relative to it; masks only where some row of the group needs one
      const int a = max(first, lo) - key0, b = min(pos + 1, hi) - key0;
      const bool full = key0 + kArKeys - 1 <= group_pos && key0 >= last_first;
      const int chunks = (min(kArKeys, hi_mine - key0) + 31) / 32;
      float sum = 0.f;
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        uint32_t s[32], packed[16];
        tc5::ld32(s_addr + uint32_t(c * 32), s);
        ar_wait32(s);
        const ArScales* scc = sc + c * 4;
        const int ac = a - c * 32, bc = b - c * 32;
        float part, weights;
        for (int pass = 0;; ++pass) {
          const float m_use = (m == -INFINITY) ? 0.f : m;
          bool renew = fresh;                                      // some row of the warp has seen nothing yet
          if (!fresh) {
            if (pass > 0) ar_exponentials<CAP, PAGES, true, true>(s, scc, packed, rf, m_use, ac, bc, weights, part);
            else if (full) ar_exponentials<CAP, PAGES, false, false>(s, scc, packed, rf, m_use, ac, bc, weights, part);
            else ar_exponentials<CAP, PAGES, true, false>(s, scc, packed, rf, m_use, ac, bc, weights, part);
            renew = pass == 0 && weights > kArMost;                // (behind a renewal a part is at most 32)
          }
          if (!__any_sync(0xffffffffu, renew)) break;
          const float mx = ar_largest<CAP, PAGES>(s, scc, rf, m_use, ac, bc);
          const bool grows = renew && mx != -INFINITY && (m == -INFINITY || mx > 0.f);
          const float alpha = grows && m != -INFINITY ? ar_exp2(-mx) : 1.f;
          if (grows) m = m_use + mx;
          sum *= alpha;
          l *= alpha;
          if (__any_sync(0xffffffffu, alpha != 1.f)) ar_rescale<HD, PAGES>(o_addr, n > 0, s_addr, c, alpha);
          if (fresh) {
            ar_exponentials<CAP, PAGES, true, true>(s, scc, packed, rf, (m == -INFINITY) ? 0.f : m, ac, bc, weights, part);
            fresh = __any_sync(0xffffffffu, m == -INFINITY);
            break;
          }
        }
        sum += part;
        ar_st16(s_addr + uint32_t(c * 16), packed);                // over products that are read
      }
      l += sum;
      tc5::st_wait();
      tc5::fence_before();
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(&p_full[g]);
    }
    if (alive) alive = wait_all(&o_full, 0, 45);
    tc5::fence_after();
    if (alive) {
      if (p.sink && m != -INFINITY) l += ar_exp2(p.sink[head] * 1.4426950408889634f - m);
      const bool none = l == 0.f;                                  // no key: zeros
      float inv = none ? 0.f : 1.f / l;
      if constexpr (PAGES) inv *= exp2f(value_base);
      inv = inv > 3.402823466e38f ? 3.402823466e38f : inv;         // (scores of 2^24 and more: sums may be next to nothing, and O too)
      bf16* dst = p.out + size_t(q_start + q0 + row) * p.out_stride + size_t(head) * p.hd;
      float sick = 0.f;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t ov[32];
        tc5::ld32(o_addr + uint32_t(c * 32), ov);                  // (all lanes of the warp take part in the load)
        ar_wait32(ov);
        if (row < rows_here) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 h;
            uint32_t* hw = reinterpret_cast<uint32_t*>(&h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = none ? 0.f : __uint_as_float(ov[e * 8 + 2 * i]) * inv, y = none ? 0.f : __uint_as_float(ov[e * 8 + 2 * i + 1]) * inv;
              sick = fmaf(x, 0.f, fmaf(y, 0.f, sick));
              hw[i] = ar_pack<false>(x, y);
            }
            if (c * 32 + e * 8 < p.hd) *reinterpret_cast<uint4*>(dst + c * 32 + e * 8) = h;
          }
        }
      }
      // (the keys that the products of this row's group had: whole tiles, up to the last one's steps of 16 and the block's own)
      uint32_t odd = __ballot_sync(0xffffffffu, sick != 0.f);
      const int from = PAGES ? lo : j0 * kArKeys, to = min(hi, (hi_mine + 15) / 16 * 16);
      while (odd) {
        const int who = __ffs(odd) - 1;
        odd &= odd - 1;
        const int its = __shfl_sync(0xffffffffu, row, who);
        ar_again<HD, CAP, PAGES>(p, seq, q_start, head, q_start + q0 + its, pos0 + its, first_visible(pos0 + its, p.window, 0), from, to);
        __syncwarp();
      }
    }
    tc5::fence_before();
  }
  // every role ends here; after a wait that ran out, copies in flight get time to land before the shared memory is given up
  if (abort_flag) {
    const unsigned long long t0 = tc5::now_ns();
    while (tc5::now_ns() - t0 < 100000ull) {}
  }
  tc5::fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc5::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
  }
}

template <int HD, bool CAP, bool PAGES>
int launch_rows_as(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const RowsParams& p, dim3 grid, cudaStream_t s) {
  static OncePerDevice once;
  const int rc = allow_shared_memory(once, attention_rows_kernel<HD, CAP, PAGES>, ar_smem<HD, PAGES>());
  if (rc != 0) return rc;
  return pdl_launch(attention_rows_kernel<HD, CAP, PAGES>, grid, dim3(ar_threads<PAGES>()), ar_smem<HD, PAGES>(), s, mq, mk, mv, p);
}
template <bool PAGES>
int launch_rows(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const RowsParams& p, dim3 grid, cudaStream_t s) {
  const bool cap = p.cap_pre > 0.f;
  if (p.hd <= 64) return cap ? launch_rows_as<64, true, PAGES>(mq, mk, mv, p, grid, s) : launch_rows_as<64, false, PAGES>(mq, mk, mv, p, grid, s);
  return cap ? launch_rows_as<128, true, PAGES>(mq, mk, mv, p, grid, s) : launch_rows_as<128, false, PAGES>(mq, mk, mv, p, grid, s);
}

// bfloat16 rows of heads as [rows][heads][hd], boxes of [128 rows][1 head][64 elements], 128-byte swizzle, zeros outside.
int rows_map(CUtensorMap* map, const void* base, long long rows, int heads, int hd, long long stride) {
  tc5::EncodeTiledFn enc = tc5::encode_tiled();
  if (!enc) return KVCM_ERR_UNSUPPORTED;
  cuuint64_t dims[3] = {cuuint64_t(hd), cuuint64_t(heads), cuuint64_t(rows)};
  cuuint64_t strides[2] = {cuuint64_t(hd) * 2, cuuint64_t(stride) * 2};
  cuuint32_t box[3] = {64u, 1u, 128u};
  cuuint32_t elem[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 20000 + int(r);
}

bool aligned16(const void* at, long long stride) { return (reinterpret_cast<uintptr_t>(at) & 15) == 0 && stride % 8 == 0; }

}  // namespace
}  // namespace kvcm

using namespace kvcm;

// q: [total_rows, >= nh * hd]; tiles of 64 query rows as the batch builder makes them (tile_seq < 0: no tile); hd 64 or 128, block_size a
// multiple of 8.
KVCM_API int kvcm_attention_prefill_q8_bf16(const void* q, long long q_stride, int total_rows, void* out, long long out_stride,
                                            const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                                            int num_pages, const int* block_tables, int max_blocks, const int* tile_seq, const int* tile_q0,
                                            const int* seq_q_start, const int* seq_q_len, const int* seq_ctx_len, int tiles, int nh, int nkv,
                                            int hd, int block_size, float scale, int window, float softcap, const float* sink,
                                            void* stream) {
  if (tiles <= 0) return 0;
  if ((hd != 64 && hd != 128) || nkv <= 0 || nh <= 0 || nh % nkv || block_size <= 0 || block_size % 8 || block_size > q8::kMaxBlock ||
      max_blocks <= 0 || num_pages <= 0 || total_rows <= 0 || tiles > 65535)
    return KVCM_ERR_UNSUPPORTED;
  if (!aligned16(q, q_stride) || !aligned16(out, out_stride) || !aligned16(k_codes, 0) || !aligned16(v_codes, 0)) return KVCM_ERR_UNSUPPORTED;
  CUtensorMap mq;
  const int rc = rows_map(&mq, q, total_rows, nh, hd, q_stride);
  if (rc) return rc;
  RowsParams p = {};
  p.out = (bf16*)out; p.out_stride = out_stride; p.q = (const bf16*)q; p.q_stride = q_stride;
  p.k_codes = (const uint8_t*)k_codes; p.v_codes = (const uint8_t*)v_codes; p.k_scale = k_scale; p.v_scale = v_scale; p.num_pages = num_pages;
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.max_keys = q8::max_keys(max_blocks, block_size);
  p.tile_seq = tile_seq; p.tile_q0 = tile_q0; p.tiles = tiles;
  p.seq_q_start = seq_q_start; p.seq_q_len = seq_q_len; p.seq_ctx_len = seq_ctx_len;
  p.nh = nh; p.nkv = nkv; p.hd = hd; p.block_size = block_size; p.window = window;
  p.scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f;
  p.cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  p.sink = sink;
  p.error = const_cast<int*>(kvcm_attention_tcgen05_error_address());
  if (p.error == nullptr) return KVCM_ERR_UNSUPPORTED;
  p.log2_block = -1;
  for (int b = 0; b < 31; ++b) if ((1 << b) == block_size) p.log2_block = b;
  return launch_rows<true>(mq, mq, mq, p, dim3(nh, tiles), (cudaStream_t)stream);
}

// q, k and v: rows of the prompts, one behind another; entries [0, singles) are prompts of one row, tiles name the others'.
KVCM_API int kvcm_prompt_attention_bf16(const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                        int total_rows, void* out, long long out_stride, const int* tile_seq, const int* tile_q0,
                                        const int* seq_q_start, const int* seq_q_len, int tiles, int singles, int nh, int nkv, int hd,
                                        float scale, int window, float softcap, const float* sink, void* stream) {
  if (tiles < 0 || singles < 0 || (long long)tiles + singles > 65535) return KVCM_ERR_UNSUPPORTED;
  if (tiles + singles == 0) return 0;
  if (hd <= 0 || hd % 8 || hd > 128 || nkv <= 0 || nh <= 0 || nh % nkv || total_rows <= 0) return KVCM_ERR_UNSUPPORTED;
  if (!aligned16(q, q_stride) || !aligned16(k, k_stride) || !aligned16(v, v_stride) || !aligned16(out, out_stride)) return KVCM_ERR_UNSUPPORTED;
  CUtensorMap mq, mk, mv;
  int rc = rows_map(&mq, q, total_rows, nh, hd, q_stride);
  if (!rc) rc = rows_map(&mk, k, total_rows, nkv, hd, k_stride);
  if (!rc) rc = rows_map(&mv, v, total_rows, nkv, hd, v_stride);
  if (rc) return rc;
  RowsParams p = {};
  p.out = (bf16*)out; p.out_stride = out_stride; p.q = (const bf16*)q; p.q_stride = q_stride;
  p.k = (const bf16*)k; p.k_stride = k_stride; p.v = (const bf16*)v; p.v_stride = v_stride;
  p.tile_seq = tile_seq; p.tile_q0 = tile_q0; p.tiles = tiles; p.seq_q_start = seq_q_start; p.seq_q_len = seq_q_len;
  p.nh = nh; p.nkv = nkv; p.hd = hd; p.block_size = 1; p.window = window;
  p.scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f;
  p.cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  p.sink = sink;
  p.error = const_cast<int*>(kvcm_attention_tcgen05_error_address());
  if (p.error == nullptr) return KVCM_ERR_UNSUPPORTED;
  return launch_rows<false>(mq, mk, mv, p, dim3(nh, tiles + singles), (cudaStream_t)stream);
}

KVCM_PACKED(kvcm_attention_prefill_q8_bf16)
KVCM_PACKED(kvcm_prompt_attention_bf16)
