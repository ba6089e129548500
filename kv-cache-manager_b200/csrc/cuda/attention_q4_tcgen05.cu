// Causal prefill attention over a paged cache in 4 bits (layout and formulas: q4.cuh) on the fifth-generation tensor cores,
// head_dim 64 or 128.
//
// One block per (256 query rows of a request, query head), as two groups of 128 rows that share every tile of keys and values.  Per
// tile of 128 keys and group:
//     S = Q C^T   C = the key's codes - 8 (bfloat16, exact), accumulator in tensor memory
//     softmax     one thread a row:  x = scale_k S + (zero_k + 8 scale_k) sum(q),  p = 2^(x - m),  P = bfloat16(p scale_v)
//     O += P W    W = the value's codes - 8 (exact), MN-major operand, O in tensor memory for the whole block
// and at the end  o = (O + sum p (zero_v + 8 scale_v)) / sum p.
// (Codes enter around zero: 128 + code would spare the subtraction, 1,097 us instead of 1,119 for four portions behind long prefixes,
// but the float32 sums would then carry terms ten times as large as the score's, which are taken out again behind them.)
// Keys and values are never rounded; P is, to bfloat16, and once more where a maximum is renewed inside its tile.  (With V =
// bfloat16(zero + scale code) as the operand three instructions for two scores fall away, 5 % less time; but the result is then 1.7
// times as far off as its own rounding, with P's alone 1.4 times.)
// A row takes its products 32 at a time, relative to the maximum that it knows, without looking for theirs: where 32 probabilities
// add up to more than 2^12 (or the row has seen nothing yet) their maximum is found, sums, O and the tile's earlier probabilities
// are rescaled, and the 32 are taken again, which after the first tiles hardly ever happens.  The largest probability then lies
// between 1 and 2^12, which float32 sums and the exponents of bfloat16 do not mind.
// P lies in tensor memory over the products that it was made of (32 columns of S become 16 of P), as the first operand of O += P V.
// The products of a group run in order: S of the next tile behind O += P V of this one, so one barrier says that S is there, that
// O holds the tile before, and that P has been read.
//
// Roles (16 warps, 128 registers a thread): 0-3 and 4-7 softmax and output of the two groups; 8-11 turn keys into operands and
// their pairs into scales, 12-14 values; one thread of warp 15 brings Q and issues the products, the groups in turn, so that the
// products of one run under the softmax of the other.
// What bounds it: at head_dim 128 a tile of 256 x 128 takes some 5,500 cycles.  Its exponentials (16 a cycle) and its products each
// take 2,048; shared memory is busy 3,300 by count (the products' operands 1,540, the keys' scales, read by every row's warp,
// 1,020, unpacking 770); a handshake between roles takes some 250, and four of them lie between two softmaxes of a group.  Two
// threads a row, each half of a tile's keys (16 softmax warps at 80 registers), took 1,438 us where one took 1,100.  B200, 32 heads
// on 8 of 128: 2,048 rows 77 us (445 TFLOP/s causal), four portions of 1,500 rows behind 6,000 keys 1,119 us (660 TFLOP/s); 148 rows of
// heads of 64 11.3 us.  Reading tiles and lengths behind the dependency wait is some 2 us of the 77.
// A thread of warps 8-14 copies what it unpacks itself (cp.async into shared memory, a tile ahead) and so waits for nobody else's.
// Masks: key <= position, optional window.  Every wait is bounded; one that runs out sets the error word of the tcgen05 attention
// family (codes 17 and up) and ends the block.
#include "packed.cuh"
#include "pdl.cuh"
#include "q4.cuh"
#include "tcgen05_common.cuh"

extern "C" const int* kvcm_attention_tcgen05_error_address(void);

namespace kvcm {

constexpr int kQfThreads = 512;
constexpr int kQfGroupRows = 128, kQfRows = 256;
constexpr int kQfKeys = 128;
constexpr int kQfKeyWarps = 4, kQfValueWarps = 3;
constexpr int kQfTile = 128 * 128;                 // [128 rows][64 bf16]: also a 64-wide block of a tile of keys or values
constexpr int kQfStages = 2;                       // tiles of keys, and of values, as operands
constexpr int kQfScaleRing = 4;
constexpr float kQfMost = 4096.f;                  // a row's sum of 32 probabilities from which its maximum is renewed
// tensor memory: S of group g at column g * 128 (and P in its first 64 columns); O of group g at 256 + g * head_dim

struct PrefillQ4Params {
  bf16* out; long long out_stride;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const int* block_tables; int max_blocks, max_keys;      // keys that a request's table has pages for
  const int* tile_seq; const int* tile_q0;         // tiles of 64 rows; a block takes every fourth and its three successors
  const int* seq_q_start; const int* seq_q_len; const int* seq_ctx_len;
  int nh, nkv, block_size, log2_block, num_pages, window;
  float scale_log2, cap_pre;
  const float* sink;
  int* error;
};

__device__ __forceinline__ float qf_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float qf_tanh(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(qf_exp2(x * 2.8853900817779268f) + 1.f));
  return fmaf(-2.f, r, 1.f);
}
__device__ __forceinline__ void qf_copy16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(tc5::s32(smem)), "l"(gmem) : "memory");
}
__device__ __forceinline__ void qf_copy4(void* smem, const void* gmem) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(tc5::s32(smem)), "l"(gmem) : "memory");
}
// 16 consecutive columns of this thread's lane of tensor memory (no wait).
__device__ __forceinline__ void qf_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                 "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
               : "r"(taddr));
}
__device__ __forceinline__ void qf_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
// The product with its first operand in tensor memory: 16-bit elements, two neighbours of a row to a column.
__device__ __forceinline__ void qf_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t instr, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(instr), "r"(accumulate) : "memory");
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// a * b + c of two floats at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

struct QfScales { float2 k_scale, k_zero, v_scale, v_zero; };      // of two neighbouring keys, as they meet scores and probabilities

// The scores of two keys, less m, from their products.
template <bool CAP>
__device__ __forceinline__ float2 qf_scores(uint32_t s0, uint32_t s1, const QfScales* sc, float2 qs2, float2 less_m, float cap_pre, float scale_log2) {
  const float4 f = *reinterpret_cast<const float4*>(sc);
  float2 t = fma2(make_float2(__uint_as_float(s0), __uint_as_float(s1)), make_float2(f.x, f.y), fma2(make_float2(f.z, f.w), qs2, CAP ? make_float2(0.f, 0.f) : less_m));
  if constexpr (CAP) {
    t.x = fmaf(qf_tanh(t.x * cap_pre), scale_log2, less_m.x);
    t.y = fmaf(qf_tanh(t.y * cap_pre), scale_log2, less_m.y);
  }
  return t;
}

// 32 products of a row into probabilities times the values' scales, as bfloat16 pairs; returns the probabilities' sum and adds what
// the values' zeros come to to z2.  MASK: only keys [a, b) of the 32 count.
template <bool CAP, bool MASK>
__device__ __forceinline__ float qf_exponentials(const uint32_t (&s)[32], const QfScales* sc, uint32_t (&packed)[16], float qs, float m,
                                                 float cap_pre, float scale_log2, int a, int b, float2& z2) {
  const float2 qs2 = make_float2(qs, qs), less_m = make_float2(-m, -m);
  float2 l0 = make_float2(0.f, 0.f), l1 = make_float2(0.f, 0.f);
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    float2 t = qf_scores<CAP>(s[2 * k], s[2 * k + 1], &sc[k], qs2, less_m, cap_pre, scale_log2);
    float4 f = *(reinterpret_cast<const float4*>(&sc[k]) + 1);
    if constexpr (MASK) {                                          // (a masked value may be no number: zero times it has to be zero)
      const bool x = 2 * k >= a && 2 * k < b, y = 2 * k + 1 >= a && 2 * k + 1 < b;
      t.x = x ? t.x : -INFINITY; f.x = x ? f.x : 0.f; f.z = x ? f.z : 0.f;
      t.y = y ? t.y : -INFINITY; f.y = y ? f.y : 0.f; f.w = y ? f.w : 0.f;
    }
    const float2 ex = make_float2(qf_exp2(t.x), qf_exp2(t.y));
    if (k & 1) l1 = add2(l1, ex); else l0 = add2(l0, ex);
    z2 = fma2(ex, make_float2(f.z, f.w), z2);
    const float2 w = mul2(ex, make_float2(f.x, f.y));
    const __nv_bfloat162 pk = __floats2bfloat162_rn(w.x, w.y);
    packed[k] = *reinterpret_cast<const uint32_t*>(&pk);
  }
  l0 = add2(l0, l1);
  return l0.x + l0.y;
}

// The largest score, less m, of the 32.
template <bool CAP>
__device__ __forceinline__ float qf_largest(const uint32_t (&s)[32], const QfScales* sc, float qs, float m, float cap_pre, float scale_log2, int a, int b) {
  const float2 qs2 = make_float2(qs, qs), less_m = make_float2(-m, -m);
  float mx = -INFINITY;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float2 t = qf_scores<CAP>(s[2 * k], s[2 * k + 1], &sc[k], qs2, less_m, cap_pre, scale_log2);
    mx = (2 * k >= a && 2 * k < b) ? fmaxf(mx, t.x) : mx;
    mx = (2 * k + 1 >= a && 2 * k + 1 < b) ? fmaxf(mx, t.y) : mx;
  }
  return mx;
}

// What a row has in tensor memory times alpha: O, and the first `chunks` pieces of 32 probabilities, which are rounded to bfloat16
// once more by that (a tile's pieces at most three times, and only where scores climb inside the tile).  The whole warp takes part.
template <int HD>
__device__ __noinline__ void qf_rescale(uint32_t o_addr, bool has_o, uint32_t p_addr, int chunks, float alpha) {
  uint32_t v[16];
#pragma unroll 1
  for (int c = 0; has_o && c < HD / 16; ++c) {
    qf_ld16(o_addr + uint32_t(c * 16), v);
    tc5::ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
    qf_st16(o_addr + uint32_t(c * 16), v);
  }
  if (chunks > 0) tc5::st_wait();                                  // loads of tensor memory pass stores that nobody waited for
#pragma unroll 1
  for (int c = 0; c < chunks; ++c) {
    qf_ld16(p_addr + uint32_t(c * 16), v);
    tc5::ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[i] << 16) * alpha, __uint_as_float(v[i] & 0xffff0000u) * alpha);
      v[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    qf_st16(p_addr + uint32_t(c * 16), v);
  }
  tc5::st_wait();
}

// 16 bytes of codes (elements 32 ch .. 32 ch + 31 of row r) as bfloat16 into a 128-byte swizzled tile [HD/64][128 rows][64]: code - 8.
__device__ __forceinline__ void qf_spread(unsigned char* tile, const unsigned char* from, int r, int ch) {
  const uint4 u = *reinterpret_cast<const uint4*>(from);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  unsigned char* row = tile + (ch >> 1) * kQfTile + r * 128;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = q4::two_codes_128(w[j], i);
      asm("sub.rn.bf16x2 %0, %0, %1;\n" : "+r"(e[i]) : "r"(0x43084308u));
    }
    *reinterpret_cast<uint4*>(row + ((((ch & 1) * 4 + j) ^ (r & 7)) * 16)) = make_uint4(e[0], e[1], e[2], e[3]);
  }
}

// The codes of a tile's keys (or values) on their way through shared memory into operands: WARPS warps, each lane its own pieces.
// Neighbouring lanes take neighbouring keys, whose swizzled rows differ in every bank.
template <int HD, int WARPS>
struct QfUnpacker {
  static constexpr int kPieces = HD / 32;                          // 16-byte pieces of a row
  static constexpr int kGroups8 = kQfKeys * kPieces / 8;           // groups of eight pieces
  static constexpr int kPerThread = (kGroups8 + 4 * WARPS - 1) / (4 * WARPS);
  int wq, lane;
  __device__ __forceinline__ bool piece(int i, int& r, int& ch) const {
    const int group = (i * WARPS + wq) * 4 + (lane >> 3);
    r = (group / kPieces) * 8 + (lane & 7);
    ch = group % kPieces;
    return group < kGroups8;
  }
};

template <int HD> constexpr size_t qf_smem() {
  constexpr int KB = HD / 64;
  return size_t(2 + 2 * kQfStages) * KB * kQfTile + size_t(kQfScaleRing) * (kQfKeys / 2) * sizeof(QfScales) + kQfKeys * HD + 2 * kQfKeys * 4;
}

template <int HD, bool CAP>
__global__ void __launch_bounds__(kQfThreads, 1) attn_prefill_q4_kernel(const __grid_constant__ CUtensorMap map_q, PrefillQ4Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int KB = HD / 64;                                      // 64-wide blocks of head_dim
  unsigned char* q_s = smem_raw;                                   // [2][KB][128 rows][64]
  unsigned char* k_s = q_s + 2 * KB * kQfTile;                     // [stages][KB][128 keys][64]
  unsigned char* v_s = k_s + kQfStages * KB * kQfTile;
  QfScales* scales = reinterpret_cast<QfScales*>(v_s + kQfStages * KB * kQfTile);          // [ring][64 pairs of keys]
  unsigned char* raw = reinterpret_cast<unsigned char*>(scales + kQfScaleRing * (kQfKeys / 2));     // codes [2][128][HD/2], pairs [2][128]
  __shared__ __align__(8) uint64_t q_full, k_full[kQfStages], v_full[kQfStages], sc_full[kQfScaleRing], s_full[2], p_full[2], done[kQfStages], o_full;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;

  // heads fastest and the last tiles, which see most keys, first
  const int tile = int(gridDim.y) - 1 - int(blockIdx.y), head = blockIdx.x;
  int* const error = p.error;
  // The tiles and lengths too may come from a kernel of the same step, so they are read behind the wait.  (Whoever leaves waits as
  // well: a launch of nothing but empty tiles would else be over before the kernel in front of it, and the one behind it waits
  // for this launch alone.)
  pdl_wait();
  const int seq = p.tile_seq[tile], q0 = p.tile_q0[tile];
  if (seq < 0 || (q0 & (kQfRows - 1))) return;                     // no tile, or one that belongs to a block before
  if (tc5::s32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicExch(error, (17 << 16) | int(blockIdx.y & 0xffff));
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_start = p.seq_q_start[seq], q_len = p.seq_q_len[seq], ctx = min(p.seq_ctx_len[seq], p.max_keys);     // (a context ends with its table)
  const int rows_here = min(kQfRows, q_len - q0);
  const int pos0 = ctx - q_len + q0;                               // position of the block's first row
  const int hi = pos0 + rows_here;                                 // keys [lo, hi) matter to the block
  const int lo = first_visible(pos0, p.window, 0);
  const int j0 = lo / kQfKeys;
  const int groups = rows_here > kQfGroupRows ? 2 : 1;
  // a group's tiles: up to the one with its last row's own key
  const int n_tiles = (hi - 1) / kQfKeys - j0 + 1;
  const int n_first = groups == 1 ? n_tiles : (pos0 + kQfGroupRows - 1) / kQfKeys - j0 + 1;     // of the first group
  const int kvh = head / (p.nh / p.nkv);

  if (threadIdx.x == 0) {
    abort_flag = 0;
    tc5::mbar_init(&q_full, 1);
    for (int i = 0; i < kQfStages; ++i) {
      tc5::mbar_init(&k_full[i], kQfKeyWarps);
      tc5::mbar_init(&v_full[i], kQfValueWarps);
      tc5::mbar_init(&done[i], 1);
    }
    for (int i = 0; i < kQfScaleRing; ++i) tc5::mbar_init(&sc_full[i], kQfKeyWarps);
    for (int g = 0; g < 2; ++g) {
      tc5::mbar_init(&s_full[g], 1);
      tc5::mbar_init(&p_full[g], 4);                               // a group's four warps
    }
    tc5::mbar_init(&o_full, 1);
    tc5::mbar_init_fence();
  }
  if (warp == 15) {
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
  const size_t bytes = q4::page_bytes(p.block_size, HD);
  const int* table = p.block_tables + size_t(seq) * p.max_blocks;
  auto page_of = [&](int key, int& off) {
    const int pi = p.log2_block >= 0 ? key >> p.log2_block : key / p.block_size;
    off = key - pi * p.block_size;
    return q4::page_base(table[pi], kvh, p.nkv, p.num_pages, bytes);
  };
  const int pairs_at = p.block_size * (HD / 2);

  if (warp == 15) {
    // ---- one thread: Q once, then the products
    if (lane == 0) {
      tc5::mbar_expect_tx(&q_full, groups * KB * kQfTile);
      for (int g = 0; g < groups; ++g)
        for (int kb = 0; kb < KB; ++kb)
          tc5::tma_load_2d(q_s + (g * KB + kb) * kQfTile, &map_q, &q_full, head * HD + kb * 64, q_start + q0 + g * kQfGroupRows);
      constexpr uint32_t idesc_s = tc5::idesc(kQfGroupRows, kQfKeys, false);
      constexpr uint32_t idesc_o = tc5::idesc(kQfGroupRows, HD, true);
      constexpr uint64_t kStageStep = (KB * kQfTile) >> 4;          // (descriptor addresses count units of 16 bytes)
      const uint64_t dk = tc5::smem_desc(tc5::s32(k_s));
      // values, MN-major: 64-wide blocks a leading offset apart
      const uint64_t dv = (tc5::smem_desc(tc5::s32(v_s)) & ~(uint64_t(0x3fff) << 16)) | (uint64_t(kQfTile >> 4) << 16);
      bool ok = tc5::mbar_wait(&q_full, 0);
      if (!ok) fail(18);
      for (int n = 0; ok && n <= n_tiles; ++n) {
        for (int g = 0; g < groups; ++g) {
          const int mine = g == 0 ? n_first : n_tiles;
          if (n >= 1 && n <= mine) {                               // O += P_(n-1) V_(n-1)
            const int m = n - 1, st = m % kQfStages;
            if (!tc5::mbar_wait(&v_full[st], (m / kQfStages) & 1)) { fail(21); ok = false; break; }
            if (!tc5::mbar_wait(&p_full[g], m & 1)) { fail(22); ok = false; break; }
            tc5::fence_after();
#pragma unroll
            for (int j = 0; j < kQfKeys / 16; ++j)                 // 16 keys: 8 columns of P, 16 rows down V
              qf_mma_ts(tmem + 256 + g * HD, tmem + g * kQfKeys + j * 8, dv + st * kStageStep + uint64_t(j * (16 * 128 >> 4)), idesc_o,
                        (m > 0 || j > 0) ? 1u : 0u);
          }
          if (n < mine) {                                          // S_n, over P_(n-1)
            const int st = n % kQfStages;
            if (!tc5::mbar_wait(&k_full[st], (n / kQfStages) & 1)) { fail(19); ok = false; break; }
            tc5::fence_after();
            const uint64_t dq = tc5::smem_desc(tc5::s32(q_s + g * KB * kQfTile));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc5::mma(tmem + uint32_t(g * kQfKeys), dq + uint64_t(kb * (kQfTile >> 4) + 2 * j),
                         dk + st * kStageStep + uint64_t(kb * (kQfTile >> 4) + 2 * j), idesc_s, (kb > 0 || j > 0) ? 1u : 0u);
            tc5::commit(&s_full[g]);                               // and O += P_(n-1) V_(n-1) before it
            if (g == groups - 1) tc5::commit(&done[st]);           // tile n of the keys and n - 1 of the values are read
          }
        }
      }
      tc5::commit(&o_full);
    }
  } else if (warp >= 8 && warp < 8 + kQfKeyWarps) {
    // ---- keys into operands, their pairs into scales.  Where S_n of the last group is issued, both groups are done with the
    // scales of tile n - 1: three places would do.
    const QfUnpacker<HD, kQfKeyWarps> unpack{warp - 8, lane};
    const int t = threadIdx.x - 256;                               // this thread's key of the tile
    unsigned char* pair = raw + kQfKeys * HD + t * 4;
    auto ask = [&](int n) {
      const int key0 = (j0 + n) * kQfKeys;
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch, off;
        if (unpack.piece(i, r, ch) && key0 + r >= lo && key0 + r < hi) {
          const size_t at = page_of(key0 + r, off);
          qf_copy16(raw + r * (HD / 2) + ch * 16, p.k_cache + at + size_t(off) * (HD / 2) + ch * 16);
        }
      }
      if (key0 + t >= lo && key0 + t < hi) {
        int off;
        const size_t at = page_of(key0 + t, off);
        qf_copy4(pair, p.k_cache + at + pairs_at + off * 4);
        qf_copy4(pair + kQfKeys * 4, p.v_cache + at + pairs_at + off * 4);
      } else {                                                     // zero: zero times it stays zero (codes are finite whatever they are)
        *reinterpret_cast<uint32_t*>(pair) = 0u;
        *reinterpret_cast<uint32_t*>(pair + kQfKeys * 4) = 0u;
      }
    };
    ask(0);
    for (int n = 0; n < n_tiles; ++n) {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      if (n >= kQfStages && !wait_all(&done[n % kQfStages], ((n - kQfStages) / kQfStages) & 1, 23)) break;
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(pair), vp = *reinterpret_cast<const uint32_t*>(pair + kQfKeys * 4);
      float* f = reinterpret_cast<float*>(scales + (n % kQfScaleRing) * (kQfKeys / 2) + (t >> 1)) + (t & 1);
      const float unit = CAP ? 1.f : p.scale_log2, ks = q4::scale_of(kp), vs = q4::scale_of(vp);
      f[0] = ks * unit;
      f[2] = fmaf(8.f, ks, q4::zero_of(kp)) * unit;
      f[4] = vs;
      f[6] = fmaf(8.f, vs, q4::zero_of(vp));
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch;
        if (unpack.piece(i, r, ch)) qf_spread(k_s + (n % kQfStages) * KB * kQfTile, raw + r * (HD / 2) + ch * 16, r, ch);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        tc5::mbar_arrive(&sc_full[n % kQfScaleRing]);
        tc5::mbar_arrive(&k_full[n % kQfStages]);
      }
      if (n + 1 < n_tiles) ask(n + 1);
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  } else if (warp >= 8 && warp < 8 + kQfKeyWarps + kQfValueWarps) {
    // ---- values into operands
    const QfUnpacker<HD, kQfValueWarps> unpack{warp - 8 - kQfKeyWarps, lane};
    unsigned char* codes = raw + kQfKeys * (HD / 2);
    auto ask = [&](int n) {
      const int key0 = (j0 + n) * kQfKeys;
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch, off;
        if (unpack.piece(i, r, ch) && key0 + r >= lo && key0 + r < hi) {
          const size_t at = page_of(key0 + r, off);
          qf_copy16(codes + r * (HD / 2) + ch * 16, p.v_cache + at + size_t(off) * (HD / 2) + ch * 16);
        }
      }
    };
    ask(0);
    for (int n = 0; n < n_tiles; ++n) {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      if (n >= kQfStages && !wait_all(&done[(n - 1) % kQfStages], ((n - 1) / kQfStages) & 1, 24)) break;
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch;
        if (unpack.piece(i, r, ch)) qf_spread(v_s + (n % kQfStages) * KB * kQfTile, codes + r * (HD / 2) + ch * 16, r, ch);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(&v_full[n % kQfStages]);
      if (n + 1 < n_tiles) ask(n + 1);
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  } else {
    // ---- softmax and output: this thread owns row r of its group (lane r of tensor memory)
    const int g = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int mine = g == 0 ? n_first : n_tiles;
    const int row = g * kQfGroupRows + r, pos = pos0 + row;        // rows beyond rows_here compute and store nothing
    const uint32_t lane_addr = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + g * kQfKeys, o_addr = lane_addr + 256 + g * HD;
    if (g < groups) {
      const int first = first_visible(pos, p.window, 0);
      const int group_pos = pos0 + g * kQfGroupRows;               // of the group's first row
      const int last_first = first_visible(group_pos + kQfGroupRows - 1, p.window, 0);
      bool alive = wait_all(&q_full, 0, 25);
      float qs = 0.f;                                              // sum of q over the row
      if (alive) {
#pragma unroll 4
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(q_s + (g * KB + (c >> 3)) * kQfTile + r * 128 + (((c & 7) ^ (r & 7)) * 16));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) qs += __uint_as_float(w[i] << 16) + __uint_as_float(w[i] & 0xffff0000u);
        }
      }
      float m = -INFINITY;                                         // the maximum the row currently scales by
      bool fresh = true;                                           // some row of the warp has none
      float l = 0.f;
      float2 z2 = make_float2(0.f, 0.f);                           // what the values' zeros come to
      for (int n = 0; n < mine; ++n) {
        alive = alive && wait_all(&s_full[g], n & 1, 26) && wait_all(&sc_full[n % kQfScaleRing], (n / kQfScaleRing) & 1, 27);
        if (!alive) break;
        tc5::fence_after();
        const QfScales* sc = scales + (n % kQfScaleRing) * (kQfKeys / 2);
        const int key0 = (j0 + n) * kQfKeys;
        // the keys of this tile that the row may see: [a, b) relative to it; masks only where some row of the group needs one
        const int a = max(first, lo) - key0, b = min(pos + 1, hi) - key0;
        const bool full = key0 + kQfKeys - 1 <= group_pos && key0 >= last_first;
        float sum = 0.f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t s[32], packed[16];
          tc5::ld32(s_addr + uint32_t(c * 32), s);
          tc5::ld_wait();
          const QfScales* scc = sc + c * 16;
          const int ac = a - c * 32, bc = b - c * 32;
          float part;
          float2 z_part;
          for (int pass = 0;; ++pass) {
            z_part = make_float2(0.f, 0.f);
            const float m_use = (m == -INFINITY) ? 0.f : m;
            bool renew = fresh;                                    // some row of the warp has seen nothing yet
            if (!fresh) {
              part = full ? qf_exponentials<CAP, false>(s, scc, packed, qs, m_use, p.cap_pre, p.scale_log2, ac, bc, z_part)
                          : qf_exponentials<CAP, true>(s, scc, packed, qs, m_use, p.cap_pre, p.scale_log2, ac, bc, z_part);
              renew = pass == 0 && part > kQfMost;                 // (behind a renewal a part is at most 32)
            }
            if (!__any_sync(0xffffffffu, renew)) break;
            const float mx = qf_largest<CAP>(s, scc, qs, m_use, p.cap_pre, p.scale_log2, ac, bc);
            const bool grows = renew && mx != -INFINITY && (m == -INFINITY || mx > 0.f);
            const float alpha = grows && m != -INFINITY ? qf_exp2(-mx) : 1.f;
            if (grows) m = m_use + mx;
            sum *= alpha;
            l *= alpha;
            z2.x *= alpha;
            z2.y *= alpha;
            if (__any_sync(0xffffffffu, alpha != 1.f)) qf_rescale<HD>(o_addr, n > 0, s_addr, c, alpha);
            if (fresh) {
              part = qf_exponentials<CAP, true>(s, scc, packed, qs, (m == -INFINITY) ? 0.f : m, p.cap_pre, p.scale_log2, ac, bc, z_part);
              fresh = __any_sync(0xffffffffu, m == -INFINITY);
              break;
            }
          }
          sum += part;
          z2 = add2(z2, z_part);
          qf_st16(s_addr + uint32_t(c * 16), packed);              // over products that are read
        }
        l += sum;
        tc5::st_wait();
        tc5::fence_before();
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&p_full[g]);
      }
      if (alive) alive = wait_all(&o_full, 0, 29);
      tc5::fence_after();
      if (alive) {
        if (p.sink && m != -INFINITY) l += qf_exp2(p.sink[head] * 1.4426950408889634f - m);
        const bool none = l == 0.f;                                // no key: zeros (a group without a tile has nothing in tensor memory)
        const float inv = none ? 0.f : 1.f / l, z = z2.x + z2.y;
        bf16* dst = p.out + size_t(q_start + q0 + row) * p.out_stride + size_t(head) * HD;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t ov[32];
          tc5::ld32(o_addr + uint32_t(c * 32), ov);                // (all lanes of the warp take part in the load)
          tc5::ld_wait();
          if (row < rows_here) {
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = none ? 0u : ov[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              __nv_bfloat162 h[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                h[i] = __floats2bfloat162_rn((__uint_as_float(ov[e * 8 + 2 * i]) + z) * inv, (__uint_as_float(ov[e * 8 + 2 * i + 1]) + z) * inv);
              *reinterpret_cast<uint4*>(dst + c * 32 + e * 8) = *reinterpret_cast<const uint4*>(h);
            }
          }
        }
      }
      tc5::fence_before();
    }
  }
  // every role ends here; after a wait that ran out, copies in flight get time to land before the shared memory is given up
  if (abort_flag) {
    const unsigned long long t0 = tc5::now_ns();
    while (tc5::now_ns() - t0 < 100000ull) {}
  }
  tc5::fence_before();
  __syncthreads();
  if (warp == 15) {
    tc5::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
  }
}

template <int HD, bool CAP>
int launch_prefill_q4(const CUtensorMap& mq, const PrefillQ4Params& p, dim3 grid, cudaStream_t s) {
  static OncePerDevice once;
  const int rc = allow_shared_memory(once, attn_prefill_q4_kernel<HD, CAP>, qf_smem<HD>());
  if (rc != 0) return rc;
  return pdl_launch(attn_prefill_q4_kernel<HD, CAP>, grid, dim3(kQfThreads), qf_smem<HD>(), s, mq, p);
}

}  // namespace kvcm

using namespace kvcm;

// 1 if this kernel takes the head size (any page size).
KVCM_API int kvcm_attention_prefill_q4_supports(int hd) { return hd == 64 || hd == 128; }

// q: [total_rows, >= nh * hd]; tiles of 64 query rows as the batch builder makes them (tile_seq < 0: no tile).
KVCM_API int kvcm_attention_prefill_q4_bf16(const void* q, long long q_stride, int total_rows, void* out, long long out_stride,
                                            const void* k_cache, const void* v_cache, int num_pages, const int* block_tables, int max_blocks,
                                            const int* tile_seq, const int* tile_q0, const int* seq_q_start, const int* seq_q_len,
                                            const int* seq_ctx_len, int tiles, int nh, int nkv, int hd, int block_size, float scale,
                                            int window, float softcap, const float* sink, void* stream) {
  if (tiles <= 0) return 0;
  if (!kvcm_attention_prefill_q4_supports(hd) || nkv <= 0 || nh <= 0 || nh % nkv || block_size <= 0 || block_size > q4::kMaxBlock || max_blocks <= 0 || num_pages <= 0 || total_rows <= 0 ||
      tiles > 65535)
    return KVCM_ERR_UNSUPPORTED;
  if ((q_stride % 8) || (out_stride % 8) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                                               reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15))
    return KVCM_ERR_UNSUPPORTED;
  CUtensorMap mq;
  const int rc = tc5::make_map(&mq, q, total_rows, (long long)nh * hd, q_stride, kQfGroupRows);
  if (rc) return rc;
  PrefillQ4Params p;
  p.out = (bf16*)out; p.out_stride = out_stride;
  p.k_cache = (const uint8_t*)k_cache; p.v_cache = (const uint8_t*)v_cache; p.num_pages = num_pages;
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.max_keys = q4::max_keys(max_blocks, block_size); p.tile_seq = tile_seq; p.tile_q0 = tile_q0;
  p.seq_q_start = seq_q_start; p.seq_q_len = seq_q_len; p.seq_ctx_len = seq_ctx_len;
  p.nh = nh; p.nkv = nkv; p.block_size = block_size; p.window = window;
  p.scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f;
  p.cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  p.sink = sink;
  p.error = const_cast<int*>(kvcm_attention_tcgen05_error_address());
  if (p.error == nullptr) return KVCM_ERR_UNSUPPORTED;
  p.log2_block = -1;
  for (int b = 0; b < 31; ++b) if ((1 << b) == block_size) p.log2_block = b;
  const dim3 grid(nh, tiles);
  cudaStream_t s = (cudaStream_t)stream;
  if (hd == 64) return softcap > 0.f ? launch_prefill_q4<64, true>(mq, p, grid, s) : launch_prefill_q4<64, false>(mq, p, grid, s);
  return softcap > 0.f ? launch_prefill_q4<128, true>(mq, p, grid, s) : launch_prefill_q4<128, false>(mq, p, grid, s);
}

KVCM_PACKED(kvcm_attention_prefill_q4_bf16)
