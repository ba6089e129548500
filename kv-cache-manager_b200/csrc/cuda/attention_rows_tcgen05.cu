// Causal attention of many rows of a request on the fifth-generation tensor cores: portions over a paged cache in 8 bits (format: q8.cuh), and
// whole prompts over their own bfloat16 rows, packed one behind another.  head_dim up to 128.
//
// One block per (256 query rows of a request, query head), as two groups of 128 rows that share every tile of keys and values.  Per
// tile of 128 keys and group:
//     S = Q K^T   accumulator in tensor memory
//     softmax     one thread a row (prompts: two):  p = 2^(x - m), x the scaled scores; P lies in tensor memory over its scores
//     O += P V    V as the MN-major operand, O in tensor memory for the whole block
// A row takes a tile's scores relative to the maximum that it knows, without looking for theirs: where their probabilities add up
// to more than 2^12 (prompts: leave 2^-40 .. 2^20; or the row has seen nothing yet) their maximum is found, sum and O are rescaled, and the tile is taken
// again, which after the first tiles hardly ever happens.
// The products of a group run in order: S of the next tile behind O += P V of this one, so one barrier says that S is there, that
// O holds the tile before, and that P has been read.
//
// Prompts: bfloat16 operands, tiles of K and V by TMA straight from the rows (three coordinates: element, head, row, so that elements
// beyond head_dim are zeros and heads of any multiple of 8 fill blocks of 64).
// Pages: float16 operands.  Codes are exact in float16, so seven warps turn them into operands with one conversion for two; scales stay
// out of the products: the key's enters the score's factor, the value's, a power of two, the probability's exponent
// (2^(x - m) scale = 2^(x - m + log2 scale): weights in place of probabilities), one factor for eight keys, which lie in one page.
// m is the reference of the weights, and sums take the weights' scales out again (rows of blocks whose values' scales are more than 2^100 apart,
// which float32's exponents cannot hold that way, are attended once more without the tensor cores).  q enters as float16 times a power of two for
// each row, exact but for elements 2^-29 as large as the row's largest.  P is rounded to float16 (prompts: bfloat16).
//
// Values that are not finite and that some row of a tile does not see would come to it as zero times them.  Rows past the
// last are zeros in shared memory; a row whose result is not finite looks whether an unseen value was the reason, or (prompts)
// whether sums relative to no maximum were too large for float32, and is then attended once more without the tensor cores.
//
// Prompts' blocks stay: three tiles before its end a block asks for another that has not begun and takes its work, so that Q, K and V come
// while rows are written (16 ragged prompts 78 us in place of 104 without cap, asked for at a block's beginning 94).
//
// What bounds it: a group's chain of softmax and products, of which two groups' overlap.  A tile of 256 x 128 takes some 3,200 cycles at
// prompts of heads of 128, the products 2,048 of them, and the exponential units as many; the issuing warp's instructions between
// products, of which a barrier's wait or a commit is some hundred cycles, are the gap (four commits a tile in place of five, two barriers in place of
// four: 468 -> 444 us).  A product of 128 x 64 takes as long as one of 128 x 128, so smaller tiles that would
// let S run ahead of the softmax lose (720 us for 8,192 rows against 640 at the time).  B200, 32 heads on 8 of 128:
// a prompt of 8,192 rows 445 us (1,235 TFLOP/s; 520 after seconds of it, under the power cap), four portions of about 1,500 rows behind
// 5,000 keys 683 (740 TFLOP/s); 16 ragged prompts of some 600 rows, 16 heads, window, capped, sinks 103; five of 110 rows of heads of 64 17.
//
// Every wait for a barrier in memory is bounded (a second, in which no warp of the block has said that it is attending rows once more); one that
// runs out sets the error word of the tcgen05 attention family (codes 33 and up) and ends the block.  Warps that wait for one another at named
// barriers, which have no limit, take every such step together whatever they saw.
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
constexpr float kArMost = 4096.f;                  // pages: a row's sum of a tile's weights from which its maximum is renewed
constexpr int kArFarApart = 100;                   // pages: exponents by which the scales of a block's values may differ
constexpr float kArMostPrompt = 1048576.f, kArLeast = 9.094947e-13f;      // prompts: 2^20, and 2^-40
// tensor memory: S of group g at column g * 128 (and P in its first 64 columns); O of group g at 256 + g * HD

struct alignas(16) ArScales { float key, value, out; };        // of eight keys: scale, log2 of the value's less the block's, 2^-(that)

struct RowsParams {
  bf16* out; long long out_stride;
  const bf16* q; long long q_stride;
  const bf16* k; long long k_stride; const bf16* v; long long v_stride;                      // prompts
  const uint8_t* k_codes; const uint8_t* v_codes; const float* k_scale; const float* v_scale;      // pages
  const int* block_tables; int max_blocks, max_keys;      // keys that a request's table has pages for (prompts: no end)
  const int* tile_seq; const int* tile_q0; int tiles, blocks;      // tiles of 64 rows; a block takes one and its three successors
  const int* seq_q_start; const int* seq_q_len; const int* seq_ctx_len;
  int nh, nkv, hd, block_size, log2_block, num_pages, window;
  float scale_log2, cap_pre;
  const float* sink;
  int* error;
};

namespace {

typedef volatile uint32_t ArBeat;                  // counts on while a warp of the block is at work that may take longer than a wait's limit

// tc5::mbar_wait for waits of a microsecond: the thread sleeps in the instruction and does not take its scheduler's turns.
__device__ __forceinline__ bool ar_wait(uint64_t* bar, uint32_t parity, const ArBeat* beat) {
  uint32_t start = 0, seen = 0;
  for (;;) {
    uint32_t done, now;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done) : "r"(tc5::s32(bar)), "r"(parity), "r"(100000u) : "memory");
    if (done) return true;
    asm volatile("mov.u32 %0, %globaltimer_lo;\n" : "=r"(now));
    if (start == 0) {
      start = now | 1u;
    } else if (int(now - start) > int(tc5::kWaitLimitNs)) {        // (start may be one ahead of now)
      if (*beat == seen) return false;                             // nobody has been at work since it was looked at last
      seen = *beat;
      start = now | 1u;
    }
  }
}

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
__device__ __forceinline__ float2 ar_mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float ar_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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
__device__ __forceinline__ void ar_wait16(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :: "memory");
}
__device__ __forceinline__ void ar_wait32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :: "memory");
  asm volatile("" : "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                    "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}
// The products and their commit, as one thread of a warp that stays together issues them (`one`: it is this thread): addresses and
// descriptors are then the same in all lanes, which the compiler may keep where the instruction wants them.
__device__ __forceinline__ void ar_mma_ss(uint32_t one, uint32_t d_tmem, uint64_t da, uint64_t db, uint32_t instr, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d_tmem), "l"(da), "l"(db), "r"(instr), "r"(accumulate), "r"(one) : "memory");
}
// With the first operand in tensor memory: 16-bit elements, two neighbours of a row to a column.
__device__ __forceinline__ void ar_mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t db, uint32_t instr, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
               ::"r"(d_tmem), "r"(a_tmem), "l"(db), "r"(instr), "r"(accumulate), "r"(one) : "memory");
}
__device__ __forceinline__ void ar_commit(uint32_t one, uint64_t* bar) {
  asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %1, 0;\n"
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(tc5::s32(bar)), "r"(one) : "memory");
}
__device__ __forceinline__ uint32_t ar_elect() {
  uint32_t one;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(one));
  return one;
}
__device__ __forceinline__ int ar_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
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

// The scores of two keys behind their tanh or factor, plus `add`.  SMALL: behind a factor that brought them into [-1, 1], where tanh is
// an odd polynomial of degree 11 (least largest error, 5.8e-7, from an exchange algorithm), which costs no exponentials.
template <bool CAP, bool SMALL = false>
__device__ __forceinline__ float2 ar_scores(uint32_t s0, uint32_t s1, float factor, float scale_log2, float add) {
  const float2 s = make_float2(__uint_as_float(s0), __uint_as_float(s1));
  if constexpr (CAP && SMALL) {
    constexpr float c[6] = {0.999999463558197f, -0.33329397439956665f, 0.13284258544445038f, -0.05168433114886284f, 0.016832629218697548f, -0.0031027502845972776f};
    const float2 y = ar_mul2(s, make_float2(factor, factor)), z = ar_mul2(y, y);
    float2 t = ar_fma2(z, make_float2(c[5], c[5]), make_float2(c[4], c[4]));
#pragma unroll
    for (int i = 3; i >= 0; --i) t = ar_fma2(z, t, make_float2(c[i], c[i]));
    return ar_fma2(ar_mul2(t, y), make_float2(scale_log2, scale_log2), make_float2(add, add));
  } else if constexpr (CAP) return make_float2(fmaf(ar_tanh(s.x * factor), scale_log2, add), fmaf(ar_tanh(s.y * factor), scale_log2, add));
  else return ar_fma2(s, make_float2(factor, factor), make_float2(add, add));
}

// N products of a row into weights, added to `w2`, and probabilities, added to `l2` (pages).  MASK: only the `seen` of them count.
// Prompts' rows with few keys have them in masked tiles, whose sums take the weights as they were rounded: a row of one key is its value, and of
// a few the roundings cancel in part (rows with many see no difference, and full tiles keep the two instructions a pair).
// AGAIN: the maximum is known, so nothing is above 2^12 but what scores of 2^24 and more are rounded by.
template <bool CAP, bool PAGES, bool MASK, bool AGAIN, bool SMALL, int N>
__device__ __forceinline__ void ar_exponentials(const uint32_t (&s)[N], const ArScales* sc, uint32_t* packed, const ArRow& row, float m,
                                                uint32_t seen, float2& w2, float2& l2) {
  if constexpr (MASK) asm volatile("" : "+r"(seen));               // (its bits are looked at here, not ahead of the branches before)
#pragma unroll
  for (int j = 0; j < N / 8; ++j) {
    float factor = row.factor, add = -m, out = 1.f;
    if constexpr (PAGES) {
      const float4 f = *reinterpret_cast<const float4*>(sc + j);
      factor *= f.x;
      add += f.y;
      out = f.z;
    }
    float2 g0, g1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 8 * j + 2 * k;
      float2 t = ar_scores<CAP, SMALL>(s[i], s[i + 1], factor, row.scale_log2, add);
      if constexpr (MASK) {
        t.x = seen & (1u << i) ? t.x : -INFINITY;
        t.y = seen & (2u << i) ? t.y : -INFINITY;
      }
      if constexpr (AGAIN) t = make_float2(t.x > 12.f ? 12.f : t.x, t.y > 12.f ? 12.f : t.y);      // (not-a-number stays)
      float2 e = make_float2(ar_exp2(t.x), ar_exp2(t.y));
      packed[i / 2] = ar_pack<PAGES>(e.x, e.y);
      if constexpr (MASK && !PAGES) e = ar_unpack<false>(packed[i / 2]);
      if (k == 0) g0 = e; else if (k == 1) g1 = e; else if (k == 2) g0 = ar_add2(g0, e); else g1 = ar_add2(g1, e);
    }
    g0 = ar_add2(g0, g1);
    w2 = ar_add2(w2, g0);
    if constexpr (PAGES) l2 = ar_fma2(g0, make_float2(out, out), l2);
  }
}

// Bits [a, b) of a word.
__device__ __forceinline__ uint32_t ar_bits(int a, int b) {
  const uint32_t below_b = b >= 32 ? 0xffffffffu : b <= 0 ? 0u : (1u << b) - 1u, below_a = a >= 32 ? 0xffffffffu : a <= 0 ? 0u : (1u << a) - 1u;
  return below_b & ~below_a;
}

// Whether the factor brings all of the warp's products into [-1, 1].
template <bool PAGES, int N>
__device__ __forceinline__ bool ar_small(const uint32_t (&s)[N], const ArScales* sc, float row_factor) {
  float largest = 0.f;
#pragma unroll
  for (int j = 0; j < N / 8; ++j) {
    const float factor = PAGES ? row_factor * sc[j].key : row_factor;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 y = ar_mul2(make_float2(__uint_as_float(s[8 * j + 2 * k]), __uint_as_float(s[8 * j + 2 * k + 1])), make_float2(factor, factor));
      const float2 z = ar_mul2(y, y);
      largest = ar_max3(largest, z.x, z.y);
    }
  }
  return !__any_sync(0xffffffffu, largest > 1.f);
}

// A thread's products of a tile into weights, two to a register.  Of `chunks` 32.  A thread with all of a row's products takes them by
// 16, the next ones under way while 16 are worked on; of two, which run under each other, each has the registers for 32 at once, or for
// 16 and the polynomial of capped scores (16 ragged prompts 130 us in place of 160).
template <int CHUNKS, bool CAP, bool PAGES, bool MASK, bool AGAIN>
__device__ __forceinline__ void ar_tile(uint32_t s_addr, const ArScales* sc, uint32_t (&packed)[16 * CHUNKS], const ArRow& row, float m, int a, int b,
                                        int chunks, float& weights, float& sum) {
  float2 w2 = make_float2(0.f, 0.f), l2 = make_float2(0.f, 0.f);
  if constexpr (CHUNKS == 4 || CAP) {
    constexpr int kAhead = CHUNKS == 4 ? 1 : 0;
    uint32_t s[kAhead + 1][16];
    if (kAhead) ar_ld16(s_addr, s[0]);
#pragma unroll
    for (int c = 0; c < 2 * CHUNKS; ++c) {
      if (MASK && c >= 2 * chunks) {
#pragma unroll
        for (int i = 0; i < 8; ++i) packed[c * 8 + i] = 0u;
        continue;
      }
      if (!kAhead) ar_ld16(s_addr + uint32_t(c * 16), s[0]);
      ar_wait16(s[c & kAhead]);
      if (kAhead && c < 2 * CHUNKS - 1) ar_ld16(s_addr + uint32_t(c * 16 + 16), s[(c + 1) & kAhead]);
      const uint32_t seen = MASK ? ar_bits(a - c * 16, b - c * 16) : 0u;
      if (CAP && ar_small<PAGES>(s[c & kAhead], sc + c * 2, row.factor))
        ar_exponentials<CAP, PAGES, MASK, AGAIN, true>(s[c & kAhead], sc + c * 2, packed + c * 8, row, m, seen, w2, l2);
      else
        ar_exponentials<CAP, PAGES, MASK, AGAIN, false>(s[c & kAhead], sc + c * 2, packed + c * 8, row, m, seen, w2, l2);
    }
    if (kAhead && MASK) tc5::ld_wait();
  } else {
    uint32_t s[32];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if (!MASK || c < chunks) {
        tc5::ld32(s_addr + uint32_t(c * 32), s);
        ar_wait32(s);
        const uint32_t seen = MASK ? ar_bits(a - c * 32, b - c * 32) : 0u;
        if (CAP && ar_small<PAGES>(s, sc + c * 4, row.factor))
          ar_exponentials<CAP, PAGES, MASK, AGAIN, true>(s, sc + c * 4, packed + c * 16, row, m, seen, w2, l2);
        else
          ar_exponentials<CAP, PAGES, MASK, AGAIN, false>(s, sc + c * 4, packed + c * 16, row, m, seen, w2, l2);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) packed[c * 16 + i] = 0u;
      }
    }
  }
  weights = w2.x + w2.y;
  sum = PAGES ? l2.x + l2.y : weights;
}

// The largest of the 32 weights' exponents, less m.
template <bool CAP, bool PAGES>
__device__ __forceinline__ float ar_largest(const uint32_t (&s)[32], const ArScales* sc, const ArRow& row, float m, uint32_t seen) {
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float factor = PAGES ? row.factor * sc[j].key : row.factor, add = PAGES ? sc[j].value - m : -m;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = 8 * j + 2 * k;
      const float2 t = ar_scores<CAP>(s[i], s[i + 1], factor, row.scale_log2, add);
      mx = seen & (1u << i) ? fmaxf(mx, t.x) : mx;
      mx = seen & (2u << i) ? fmaxf(mx, t.y) : mx;
    }
  }
  return mx;
}

// `columns` of what a row has in O times alpha.  The whole warp takes part.
__device__ __noinline__ void ar_rescale(uint32_t o_addr, int columns, float alpha) {
  uint32_t v[16];
#pragma unroll 1
  for (int c = 0; c < columns; c += 16) {
    ar_ld16(o_addr + uint32_t(c), v);
    tc5::ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
    ar_st16(o_addr + uint32_t(c), v);
  }
  tc5::st_wait();
}

// A barrier of the warps that share rows, and whether any of their threads said so.
template <int SPLIT> __device__ __forceinline__ bool ar_either(int id, bool mine) {
  if (SPLIT == 1) return __any_sync(0xffffffffu, mine);
  uint32_t any;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.b32 p, %1, 0;\nbarrier.cta.red.or.pred.aligned q, %2, 64, p;\nselp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(any) : "r"(uint32_t(mine)), "r"(id) : "memory");
  return any != 0u;
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
  __device__ __forceinline__ static void floats8(uint4 u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = ar_unpack<false>(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  // Elements 8 c .. 8 c + 7.
  __device__ __forceinline__ void key8(size_t at, int c, float (&x)[8]) const { eight(true, at, c, x); }
  __device__ __forceinline__ void value8(size_t at, int c, float (&x)[8]) const { eight(false, at, c, x); }
  __device__ __forceinline__ void eight(bool is_k, size_t at, int c, float (&x)[8]) const {
    if constexpr (PAGES) {
      const uint2 u = *reinterpret_cast<const uint2*>((is_k ? p.k_codes : p.v_codes) + at * p.hd + c * 8);
      const float scale = (is_k ? p.k_scale : p.v_scale)[at / p.block_size];
      q8::values4(u.x, scale, x);
      q8::values4(u.y, scale, x + 4);
    } else {
      floats8(*reinterpret_cast<const uint4*>((is_k ? p.k + at * p.k_stride : p.v + at * p.v_stride) + size_t(kvh) * p.hd + c * 8), x);
    }
  }
  // Elements N lane .. N lane + N - 1 of a value, N = 2 or 4; zeros behind the head's.
  template <int N> __device__ __forceinline__ void value(size_t at, float (&x)[N]) const {
    const int d = N * int(threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = 0.f;
    if (d >= p.hd) return;
    if constexpr (PAGES) {
      const float scale = p.v_scale[at / p.block_size];
      const uint8_t* const from = p.v_codes + at * p.hd + d;
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 f = q8::floats2(*reinterpret_cast<const uint16_t*>(from + i));
        x[i] = f.x * scale;
        x[i + 1] = f.y * scale;
      }
    } else {
      const bf16* const from = p.v + at * p.v_stride + size_t(kvh) * p.hd + d;
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float2 f = ar_unpack<false>(*reinterpret_cast<const uint32_t*>(from + i));
        x[i] = f.x;
        x[i + 1] = f.y;
      }
    }
  }
};

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

// A block's work: up to 256 rows of a request and a head.  rows 0: none.
struct ArItem { int seq, head, q0, q_start, q_len, rows, ctx; };

// The work of block (x, y), looked up by a whole warp: heads fastest; the last tiles, which see most keys, first, and prompts of one row last.
template <bool PAGES>
__device__ __forceinline__ ArItem ar_item(const RowsParams& p, int x, int y) {
  const int tile = p.blocks - 1 - y;
  ArItem it{-1, x, 0, 0, 0, 0, 0};
  int most = kArRows;
  if (!PAGES && tile < 0) {                                        // a prompt of one row
    it.seq = -1 - tile;
    most = 1;
  } else {                                                         // the tile-th of those that begin a block
    for (int t0 = 0, before = 0; t0 < p.tiles; t0 += 128) {
      int s[4], q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * 32 + int(threadIdx.x & 31);
        s[i] = t < p.tiles ? p.tile_seq[t] : -1;
        q[i] = t < p.tiles ? p.tile_q0[t] : -1;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool begins = s[i] >= 0 && (q[i] & (kArRows - 1)) == 0;
        const uint32_t leads = __ballot_sync(0xffffffffu, begins);
        const int at = tile - before;
        before += __popc(leads);
        if (it.seq < 0 && at >= 0 && tile < before) {
          const int from = __ffs(__ballot_sync(0xffffffffu, begins && __popc(leads & ((1u << (threadIdx.x & 31)) - 1u)) == at)) - 1;
          it.seq = __shfl_sync(0xffffffffu, s[i], from);
          it.q0 = __shfl_sync(0xffffffffu, q[i], from);
        }
      }
      if (it.seq >= 0) break;
    }
  }
  if (it.seq < 0) return it;                                       // fewer than the host had to reckon with
  it.q_start = p.seq_q_start[it.seq];
  it.q_len = p.seq_q_len[it.seq];
  it.rows = max(min(most, it.q_len - it.q0), 0);
  it.ctx = PAGES ? p.seq_ctx_len[it.seq] : it.q_len;
  return it;
}

// What it has to do with keys.  Pages: a context that is longer than its table leaves the rows where they are, and their keys end with the table
// (rows, groups of rows and whole blocks may then see none; what is said of tiles holds for blocks that see some).
struct ArSpan {
  int pos0, hi, lo, j0, groups, hi_first, n_tiles, n_first, kvh;
  __device__ __forceinline__ ArSpan(const RowsParams& p, const ArItem& it) {
    const int keys = p.max_keys;
    pos0 = it.ctx - it.q_len + it.q0;                              // position of the block's first row
    hi = min(pos0 + it.rows, keys);                                // keys [lo, hi) matter to the block
    lo = first_visible(pos0, p.window, 0);
    j0 = lo / kArKeys;
    groups = it.rows > kArGroupRows ? 2 : 1;
    // a group's keys end with its last row's own, and so do its tiles
    hi_first = groups == 1 ? hi : min(pos0 + kArGroupRows, keys);
    n_tiles = (hi - 1) / kArKeys - j0 + 1;
    n_first = (hi_first - 1) / kArKeys - j0 + 1;
    kvh = it.head / (p.nh / p.nkv);
  }
};

// A row without the tensor cores, by a whole warp: 32 keys at a time, a lane a key for the scores and a lane two or four elements for the output,
// which is kept as the mean that it is so far, so that it is finite where the values are.  That takes its time (32 rows behind 100,000 keys
// half a second), so the warp says now and then that it is at work, and nobody's wait runs out meanwhile.
template <int HD, bool CAP, bool PAGES>
__device__ __forceinline__ void ar_again(const RowsParams& p, ArBeat* beat, int seq, int start, int head, int row, int first, int last) {
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31, kvh = head / (p.nh / p.nkv), words = p.hd / 8;
  const ArKeys<PAGES> keys{p, PAGES ? p.block_tables + size_t(seq) * p.max_blocks : nullptr, start, kvh};
  const uint4* const q = reinterpret_cast<const uint4*>(p.q + size_t(row) * p.q_stride + size_t(head) * p.hd);
  float o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll 1
  for (int j0 = first; j0 <= last; j0 += 32) {
    const int n = min(32, last - j0 + 1);
    if (lane == 0) *beat = *beat + 1;
    float x = -INFINITY;
    size_t at = 0;
    if (lane < n) {
      at = keys.place(j0 + lane);
      float s = 0.f;
#pragma unroll 1
      for (int c = 0; c < words; ++c) {
        float k[8], w[8];
        keys.key8(at, c, k);
        keys.floats8(q[c], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(w[e], k[e], s);
      }
      x = CAP ? ar_tanh(s * p.cap_pre) * p.scale_log2 : s * p.scale_log2;
    }
    const float top = fmaxf(m, warp_max(x)), f = m == -INFINITY ? 0.f : ar_exp2(m - top), e = x == -INFINITY ? 0.f : ar_exp2(x - top);
    const float before = m == -INFINITY ? 0.f : l * f, sum = before + warp_sum(e), per = sum == 0.f ? 0.f : 1.f / sum;
    m = top;
    l = sum;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= before * per;
#pragma unroll 4
    for (int k = 0; k < n; ++k) {                                  // (more at once take registers from the kernel around the call: 2 % of packed prompts)
      float v[N];
      keys.template value<N>(__shfl_sync(0xffffffffu, (unsigned long long)at, k), v);
      const float w = __shfl_sync(0xffffffffu, e * per, k);
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(w, v[i], o[i]);
    }
  }
  const float share = p.sink && m != -INFINITY ? l / (l + ar_exp2(p.sink[head] * 1.4426950408889634f - m)) : 1.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (N * lane < p.hd) stf(p.out + size_t(row) * p.out_stride + size_t(head) * p.hd + N * lane + i, l == 0.f ? 0.f : o[i] * share);
}

// The rows `odd` of the warp's 32 rows of group g, whose results are not finite.  Those are attended again that do not see a value that is
// not finite but came beside (of the keys that the group's products had).  Pages: and those of `counts`, whose values' scales are too far
// apart.  Prompts: and, where some value is large, those whose weights are numbers (`counts`): their weights add up to 2^37 at most, so sums of values from 2^90 on may have left float32 although their mean does not.
constexpr float kArLarge = 1.2379400392853803e27f;      // 2^90
template <int HD, bool CAP, bool PAGES>
__device__ __noinline__ void ar_redo(const RowsParams& p, ArBeat* beat, const ArItem& it, int g, uint32_t odd, uint32_t counts) {
  const ArSpan w(p, it);
  const ArKeys<PAGES> keys{p, PAGES ? p.block_tables + size_t(it.seq) * p.max_blocks : nullptr, it.q_start, w.kvh};
  const int lane = threadIdx.x & 31, row0 = g * kArGroupRows + int(threadIdx.x >> 5 & 3) * 32, pos = w.pos0 + row0 + lane;
  const int first = first_visible(pos, p.window, 0), last = min(pos, w.hi - 1);
  // (keys of whole tiles, up to the last one's steps of 16 and the block's own)
  const int from = PAGES ? w.lo : w.j0 * kArKeys, to = min(w.hi, ((g == 0 ? w.hi_first : w.hi) + 15) / 16 * 16);
  const bool all = !PAGES && (odd & counts) != 0u;
  const bool mine = odd >> lane & 1u;
  const int seen_from = __reduce_max_sync(0xffffffffu, mine ? first : 0), seen_to = __reduce_min_sync(0xffffffffu, mine ? last : 0x7fffffff);
  bool beside = false, large = false;
#pragma unroll 1
  for (int j0 = from; j0 < to; j0 += 32) {
    if (!all && j0 >= seen_from && j0 + 31 <= seen_to) continue;   // (every row sees them)
    if (lane == 0) *beat = *beat + 1;
    bool bad = false;
    if (j0 + lane < to) {
      const size_t at = keys.place(j0 + lane);
#pragma unroll 1
      for (int c = 0; c < p.hd / 8; ++c) {
        float x[8];
        keys.value8(at, c, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool finite = fabsf(x[e]) <= 3.402823466e38f;
          bad |= !finite;
          large |= finite && fabsf(x[e]) >= kArLarge;
        }
      }
    }
    beside |= (__ballot_sync(0xffffffffu, bad) & ~ar_bits(first - j0, last + 1 - j0)) != 0u;
  }
  odd &= __ballot_sync(0xffffffffu, beside) | (PAGES || (all && __any_sync(0xffffffffu, large)) ? counts : 0u);
#pragma unroll 1
  while (odd) {
    const int who = __ffs(odd) - 1;
    odd &= odd - 1;
    ar_again<HD, CAP, PAGES>(p, beat, it.seq, it.q_start, it.head, it.q_start + it.q0 + row0 + who, __shfl_sync(0xffffffffu, first, who),
                             __shfl_sync(0xffffffffu, last, who));
    __syncwarp();
  }
}

// Asks for the work of a block of the grid that has not begun, in its place (the answer in 16 bytes of shared memory, counted on `bar`).
__device__ __forceinline__ void ar_ask_block(uint4* answer, uint64_t* bar) {
  tc5::mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n"
               ::"r"(tc5::s32(answer)), "r"(tc5::s32(bar)) : "memory");
}
// Whether there was one, and which.
__device__ __forceinline__ bool ar_block_answer(const uint4* answer, int& x, int& y) {
  uint32_t is, bx = 0, by = 0;
  asm volatile("{\n.reg .pred p;\n.reg .b128 r;\nld.shared.b128 r, [%3];\n"
               "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\nselp.u32 %2, 1, 0, p;\n"
               "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, _, _}, r;\n}\n"
               : "+r"(bx), "+r"(by), "=r"(is) : "r"(tc5::s32(answer)) : "memory");
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  x = int(bx);
  y = int(by);
  return is != 0u;
}

// Rows that see no key: zeros.
__device__ __noinline__ void ar_no_key(const RowsParams& p, int row0, int rows, int head) {
  const int words = p.hd / 8;
  for (int i = threadIdx.x; i < rows * words; i += blockDim.x) {
    const int row = i / words, d = (i - row * words) * 8;
    *reinterpret_cast<uint4*>(p.out + size_t(row0 + row) * p.out_stride + size_t(head) * p.hd + d) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int HD, bool PAGES> constexpr size_t ar_smem() {
  return size_t(2 + 2 * kArStages) * (HD / 64) * kArTile + (PAGES ? kArRing * (kArKeys / 8) * sizeof(ArScales) : 0);
}
template <bool PAGES> constexpr int ar_split() { return PAGES ? 1 : 2; }         // threads of a row
template <bool PAGES> constexpr int ar_threads() { return 256 * ar_split<PAGES>() + (PAGES ? 256 : 64); }


template <int HD, bool CAP, bool PAGES>
__global__ void __launch_bounds__(ar_threads<PAGES>(), 1)
attention_rows_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                      const __grid_constant__ CUtensorMap map_v, const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int KB = HD / 64;                                      // 64-wide blocks of a head
  constexpr int SPLIT = ar_split<PAGES>(), kSoftmaxWarps = 8 * SPLIT, CHUNKS = 4 / SPLIT, kSpan = kArKeys / SPLIT;
  constexpr int kMmaWarp = ar_threads<PAGES>() / 32 - 1;
  constexpr int kPieces = HD / 16;                                 // pages: 16-byte pieces of a row of codes
  unsigned char* q_s = smem_raw;                                   // [2][KB][128 rows][64]
  unsigned char* k_s = q_s + 2 * KB * kArTile;                     // [stages][KB][128 keys][64]
  unsigned char* v_s = k_s + kArStages * KB * kArTile;
  ArScales* scales = reinterpret_cast<ArScales*>(v_s + kArStages * KB * kArTile);          // [ring][16 groups of eight keys]
  __shared__ __align__(8) uint64_t q_full, q_ready, k_full[kArStages], v_full[kArStages], kv_free[kArStages], v_tail,
      sc_full[kArRing], s_full[2], p_full[2], o_full[2], next_told, item_full[2], item_free[2];
  __shared__ __align__(16) uint4 next_block;
  __shared__ ArItem items[2];                                      // the work in hand; prompts: and what comes behind it
  __shared__ uint32_t tmem_base;
  __shared__ float told[SPLIT][kArRows];                           // what the threads of a row tell each other
  __shared__ int left[8][2];                                       // that a warp gave up
  __shared__ size_t group_at[2][2][PAGES ? kArKeys / 8 : 1];       // pages: where keys, and values, of a tile are, by eights
  __shared__ float value_base;                                     // log2 of the value scale that weights are relative to
  __shared__ volatile int far_apart[2];                            // pages: that a group's value scales are further apart than sums of weights can hold
  __shared__ volatile int abort_flag;
  __shared__ ArBeat beat;

  int* const error = p.error;
  // Tiles and lengths may come from a kernel of the same step, so they are read behind the wait.  (Whoever leaves waits as
  // well: a launch of nothing but empty tiles would else be over before the kernel in front of it.)
  pdl_wait();
  const ArItem begin = ar_item<PAGES>(p, blockIdx.x, blockIdx.y);
  if (begin.rows == 0) return;
  if constexpr (PAGES) {
    const ArSpan w(p, begin);
    if (w.hi <= w.lo) {
      ar_no_key(p, begin.q_start + begin.q0, begin.rows, begin.head);
      return;
    }
  }
  if (tc5::s32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicExch(error, (33 << 16) | int(blockIdx.y & 0xffff));
    return;
  }
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

  if (threadIdx.x < 16) left[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    far_apart[0] = far_apart[1] = 0;
    beat = 0;
    items[0] = begin;
    tc5::mbar_init(&q_full, 1);
    tc5::mbar_init(&q_ready, 4 * SPLIT * (begin.rows > kArGroupRows ? 2 : 1));
    for (int i = 0; i < kArStages; ++i) {
      tc5::mbar_init(&k_full[i], PAGES ? kArKeyWarps : 1);
      tc5::mbar_init(&v_full[i], PAGES ? kArValueWarps : 1);
      tc5::mbar_init(&kv_free[i], 1);
    }
    tc5::mbar_init(&v_tail, 1);
    for (int i = 0; i < kArRing; ++i) tc5::mbar_init(&sc_full[i], 1);
    for (int g = 0; g < 2; ++g) {
      tc5::mbar_init(&s_full[g], 1);
      tc5::mbar_init(&o_full[g], 1);
      tc5::mbar_init(&p_full[g], 4 * SPLIT);                       // a group's warps
    }
    tc5::mbar_init(&next_told, 1);
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&item_full[i], 1);
      tc5::mbar_init(&item_free[i], kSoftmaxWarps + 1);            // softmax and products
    }
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
    if (__all_sync(0xffffffffu, ar_wait(bar, parity, &beat))) return true;
    if (!abort_flag && lane == 0) fail(code);                      // (the first to give up says so; the others' waits run out too)
    return false;
  };

  // Prompts' blocks stay and take the work of blocks that have not begun, so that its Q, K and V come while the rows before are attended and
  // written.  Whether there is work with number `n` of the block, in items[n & 1] until all have left it.
  auto there_is_item = [&](int n) {
    if (n == 0) return true;
    return !PAGES && wait_all(&item_full[n & 1], ((n - 1) >> 1) & 1, 47) && items[n & 1].rows > 0;
  };
  auto leave_item = [&](int n) {
    __syncwarp();
    if (!PAGES && lane == 0) tc5::mbar_arrive(&item_free[n & 1]);
  };

  if (warp == kMmaWarp) {
    // ---- the products: the warp stays together, one thread of it issues.  Step n is O += P_(n-1) V_(n-1) and S_n of either group.
    const uint32_t one = ar_elect();
    if (PAGES && one) {
      const ArSpan w(p, begin);
      tc5::mbar_expect_tx(&q_full, w.groups * KB * kArTile);
      for (int g = 0; g < w.groups; ++g)
        for (int kb = 0; kb < KB; ++kb)
          ar_tma_3d(q_s + (g * KB + kb) * kArTile, &map_q, &q_full, kb * 64, begin.head, begin.q_start + begin.q0 + g * kArGroupRows);
    }
    __syncwarp();
    constexpr uint32_t kTypes = PAGES ? ~((7u << 7) | (7u << 10)) : ~0u;         // float16 or bfloat16
    constexpr uint32_t idesc_s = tc5::idesc(kArGroupRows, kArKeys, false) & kTypes;
    constexpr uint32_t idesc_o = tc5::idesc(kArGroupRows, HD, true) & kTypes;
    constexpr uint64_t kStageStep = (KB * kArTile) >> 4;            // (descriptor addresses count units of 16 bytes)
    const uint64_t dq = tc5::smem_desc(tc5::s32(q_s)), dk = tc5::smem_desc(tc5::s32(k_s));
    // values, MN-major: 64-wide blocks a leading offset apart
    const uint64_t dv = (tc5::smem_desc(tc5::s32(v_s)) & ~(uint64_t(0x3fff) << 16)) | (uint64_t(kArTile >> 4) << 16);
    const uint32_t base = uint32_t(ar_uniform(int(tmem)));
    bool ok = true;
    uint32_t step = 0, odd = 0;                                     // steps so far; bit g: whether the group's tiles of weights so far are odd
    for (int number = 0; ok && there_is_item(number); ++number) {
      const ArSpan w(p, items[number & 1]);
      leave_item(number);
      const int tiles = ar_uniform(w.n_tiles), tiles_first = ar_uniform(w.n_first), both = ar_uniform(w.groups);
      // (of a group's last tile only the steps of 16 keys that some row of it sees)
      const int last_steps = ar_uniform((w.hi - (w.j0 + w.n_tiles - 1) * kArKeys + 15) / 16);
      const int last_first = ar_uniform((w.hi_first - (w.j0 + w.n_first - 1) * kArKeys + 15) / 16);
      ok = wait_all(PAGES ? &q_ready : &q_full, number & 1, 34);
      for (int n = 0; ok && n <= tiles; ++n, ++step) {
        const int st = step & 1;                                    // of tile n of the keys and tile n - 1 of the values
        static_assert(kArStages == 2, "stages by parity");
        const uint32_t parity = (step >> 1) & 1;
        ok = PAGES ? (n == 0 || wait_all(&v_full[st], ((n - 1) >> 1) & 1, 35)) : wait_all(&k_full[st], parity, 37);
        for (int g = 0; ok && g < both; ++g) {
          const int mine = g == 0 ? tiles_first : tiles;
          if (n > mine) continue;
          if (n >= 1) {                                             // O += P_(n-1) V_(n-1)
            ok = wait_all(&p_full[g], (odd >> g) & 1, 36);
            if (!ok) break;
            odd ^= 1u << g;
            tc5::fence_after();
            const uint64_t v = dv + st * kStageStep;
            const uint32_t d = base + 256 + g * HD, a = base + g * kArKeys;
            const int steps = n < mine ? 8 : g == 0 ? last_first : last_steps;
            // 16 keys: 8 columns of P (every thread's over its own products), 16 rows down V
            if (steps == 8) {
#pragma unroll
              for (int j = 0; j < 8; ++j) ar_mma_ts(one, d, a + (SPLIT == 2 ? (j & 3) * 8 + (j >> 2) * 64 : j * 8), v + uint64_t(j * (16 * 128 >> 4)), idesc_o, (n > 1 || j > 0) ? 1u : 0u);
            } else {
#pragma unroll 1
              for (int j = 0; j < steps; ++j) ar_mma_ts(one, d, a + (SPLIT == 2 ? (j & 3) * 8 + (j >> 2) * 64 : j * 8), v + uint64_t(j * (16 * 128 >> 4)), idesc_o, (n > 1 || j > 0) ? 1u : 0u);
            }
          }
          if (n < mine) {                                           // S_n, over P_(n-1)
            if (PAGES && !wait_all(&k_full[st], parity, 37)) { ok = false; break; }
            tc5::fence_after();
            const uint64_t q = dq + g * kStageStep, k = dk + st * kStageStep;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                ar_mma_ss(one, base + g * kArKeys, q + uint64_t(kb * (kArTile >> 4) + 2 * j), k + uint64_t(kb * (kArTile >> 4) + 2 * j), idesc_s,
                          (kb > 0 || j > 0) ? 1u : 0u);
          }
          ar_commit(one, n < mine ? &s_full[g] : &o_full[g]);       // (s_full: and O += P_(n-1) V_(n-1) before it)
        }
        if (ok) ar_commit(one, &kv_free[st]);
      }
      if (PAGES) break;
    }
  } else if (!PAGES && warp == kSoftmaxWarps) {
    // ---- prompts: one thread asks for Q, K, V and more work, which the warp looks up
    bool ok = true;
    int tails = 0, asked = 0;                                      // ends with zeros, questions
    uint32_t step = 0;                                             // of the products
    ArItem it = begin;
    for (int number = 0; ok && it.rows > 0; ++number) {
      const ArSpan w(p, it);
      const int tail = w.hi - (w.j0 + w.n_tiles - 1) * kArKeys;    // keys of the last tile
      // tile n of the keys and tile n - 1 of the values come, and are read, together
      for (int n = 0; ok && n <= w.n_tiles; ++n, ++step) {
        const int st = step & 1, key = it.q_start + (w.j0 + n) * kArKeys;
        const bool has_k = n < w.n_tiles, has_v = n > 0;
        // (the product of the last tile takes 16 keys at a time; behind the prompt's last come zeros)
        const bool ends = n == w.n_tiles && tail % 16 != 0;
        if (lane == 0) {
          if (n == max(w.n_tiles - 3, 0)) ar_ask_block(&next_block, &next_told);        // (the later, the better blocks' ends fit)
          ok = ar_wait(&kv_free[st], ((step >> 1) & 1) ^ 1, &beat);
          if (ok && n == 0) {                                      // (the work before has had its last scores one step ago)
            tc5::mbar_expect_tx(&q_full, w.groups * KB * kArTile);
            for (int g = 0; g < w.groups; ++g)
              for (int kb = 0; kb < KB; ++kb)
                ar_tma_3d(q_s + (g * KB + kb) * kArTile, &map_q, &q_full, kb * 64, it.head, it.q_start + it.q0 + g * kArGroupRows);
          }
          if (ok) {
            uint64_t* const bar = ends ? &v_tail : &k_full[st];
            tc5::mbar_expect_tx(bar, (int(has_k) + int(has_v)) * KB * kArTile);
            for (int kb = 0; has_k && kb < KB; ++kb) ar_tma_3d(k_s + (st * KB + kb) * kArTile, &map_k, bar, kb * 64, w.kvh, key);
            for (int kb = 0; has_v && kb < KB; ++kb) ar_tma_3d(v_s + (st * KB + kb) * kArTile, &map_v, bar, kb * 64, w.kvh, key - kArKeys);
          }
          if (!ok && !abort_flag) fail(38);
        }
        ok = __shfl_sync(0xffffffffu, int(ok), 0);
        if (ok && ends) {
          ok = wait_all(&v_tail, tails & 1, 39);
          ++tails;
          const int to = (tail + 15) / 16 * 16;
          for (int kb = 0; ok && kb < KB; ++kb)
            for (int i = tail * 8 + lane; i < to * 8; i += 32)
              *reinterpret_cast<uint4*>(v_s + (st * KB + kb) * kArTile + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
          __syncwarp();
          if (ok && lane == 0) tc5::mbar_arrive(&k_full[st]);
        }
      }
      // ---- the work behind it: of the next block that has some
      for (;;) {
        int x, y;
        if (!wait_all(&next_told, asked & 1, 48)) { ok = false; it.rows = 0; break; }      // (also where a wait above ran out: an answer has to land)
        ++asked;
        if (!ar_block_answer(&next_block, x, y) || !ok) { it.rows = 0; break; }
        it = ar_item<PAGES>(p, x, y);
        if (it.rows > 0) break;
        __syncwarp();
        if (lane == 0) ar_ask_block(&next_block, &next_told);
      }
      const int to = (number + 1) & 1;
      if (!wait_all(&item_free[to], (((number + 1) >> 1) & 1) ^ 1, 49)) break;
      if (lane == 0) {
        items[to] = it;
        tc5::mbar_arrive(&item_full[to]);
      }
      __syncwarp();
    }
  } else if (PAGES && warp >= kSoftmaxWarps && warp < kSoftmaxWarps + kArKeyWarps + kArValueWarps) {
    // ---- pages: codes into operands; four warps the keys, three the values.  The first warp of each says where a tile's groups of eight
    // keys lie; a thread asks for its pieces of the next tile behind those of this one.
    const ArSpan w(p, begin);
    const int lo = w.lo, hi = w.hi, j0 = w.j0, n_tiles = w.n_tiles;
    const bool is_k = warp < kSoftmaxWarps + kArKeyWarps;
    const int warps = is_k ? kArKeyWarps : kArValueWarps, wq = warp - kSoftmaxWarps - (is_k ? 0 : kArKeyWarps);
    constexpr int kRows = 32 / kPieces, kParts = 8 / kRows;        // rows of a warp's piece, pieces of eight keys
    constexpr int kAll = kArKeys / kRows, kMost = (kAll + kArValueWarps - 1) / kArValueWarps;
    const uint8_t* const codes = (is_k ? p.k_codes : p.v_codes) + (lane % kPieces) * 16 + (lane / kPieces) * HD;
    unsigned char* const to = is_k ? k_s : v_s;
    const ArKeys<true> keys{p, p.block_tables + size_t(begin.seq) * p.max_blocks, 0, w.kvh};
    uint4 held[kMost];
    float2 of_group = make_float2(0.f, 1.f);                       // scales of the eight keys that a lane of the first warp has
    // where the eight keys of a lane of a first warp are in tile n, counted in rows of a head, and their scales
    auto look = [&](int n) {
      const int key0 = (j0 + n) * kArKeys + lane * 8, key = max(key0, lo);
      if (wq != 0 || lane >= kArKeys / 8 || n >= n_tiles) return;
      of_group = make_float2(0.f, 1.f);
      size_t at = 0;
      if (key < min(hi, key0 + 8)) {
        at = keys.place(key);
        if (is_k) of_group = make_float2(p.k_scale[at / p.block_size], p.v_scale[at / p.block_size]);
        at -= key - key0;
      }
      group_at[is_k ? 0 : 1][n & 1][lane] = at;
    };
    auto ask = [&](int n) {
      const int key0 = (j0 + n) * kArKeys;
      const size_t* const at = group_at[is_k ? 0 : 1][n & 1];
      const bool inside = key0 >= lo && key0 + kArKeys <= hi;
#pragma unroll
      for (int i = 0; i < kMost; ++i) {
        const int piece = i * warps + wq, r = piece * kRows + lane / kPieces;
        held[i] = make_uint4(0u, 0u, 0u, 0u);                      // (keys of nobody: zero times them stays zero)
        if (piece < kAll && (inside || (key0 + r >= lo && key0 + r < hi)))
          held[i] = *reinterpret_cast<const uint4*>(codes + (at[piece / kParts] + (piece % kParts) * kRows) * HD);
      }
    };
    auto together = [&]() { asm volatile("barrier.cta.sync.aligned %0, %1;\n" ::"r"(is_k ? 9 : 10), "r"(32 * warps) : "memory"); };
    look(0);
    together();
    ask(0);
    float base = 0.f;
    int least = 255, most = 0;                                     // exponents of the values' scales so far, in a lane's groups of eight
    bool there_is = true;                                          // room for the tile
    for (int n = 0; n < n_tiles; ++n) {
      // tile n of the keys is read in step n of the products, of the values in the one behind it
      const int at_step = is_k ? n : n + 1, st = at_step & 1;
      const float2 scale = of_group;
      look(n + 1);
      there_is = there_is && wait_all(&kv_free[st], ((at_step >> 1) & 1) ^ 1, is_k ? 40 : 41);
      if (warp == kSoftmaxWarps) {
        // (S_(n-2) is complete, so the weights of tile n - 3 are made, and the place of tile n - 4 is free)
        const float log_v = log2f(fmaxf(scale.y, 1.17549435e-38f));
        if (n == 0) {
          base = __shfl_sync(0xffffffffu, log_v, (lo % kArKeys) / 8);
          if (lane == 0) value_base = base;
        }
        if (lane < kArKeys / 8) {
          const bool there = (j0 + n) * kArKeys + lane * 8 < hi && (j0 + n) * kArKeys + lane * 8 + 8 > lo;
          ArScales s;
          s.key = scale.x;
          s.value = there ? log_v - base : 0.f;
          s.out = there ? exp2f(base - log_v) : 0.f;
          scales[(n % kArRing) * (kArKeys / 8) + lane] = s;
          if (there) {
            const int e = int(__float_as_uint(scale.y) >> 23);
            least = min(least, e);
            most = max(most, e);
          }
        }
        if (n == w.n_first - 1 || n == n_tiles - 1) {              // (ahead of the barrier that a group's last weights wait for)
          least = __reduce_min_sync(0xffffffffu, least);
          most = __reduce_max_sync(0xffffffffu, most);
          if (lane == 0 && most - least > kArFarApart) {
            if (n == w.n_first - 1) far_apart[0] = 1;
            if (n == n_tiles - 1) far_apart[1] = 1;
          }
        }
        __syncwarp();
        if (there_is && lane == 0) tc5::mbar_arrive(&sc_full[n % kArRing]);
      }
      if (there_is) {
#pragma unroll
        for (int i = 0; i < kMost; ++i) {
          const int piece = i * warps + wq;
          if (piece < kAll) ar_spread<HD>(to + st * KB * kArTile, held[i], piece * kRows + lane / kPieces, lane % kPieces);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(is_k ? &k_full[st] : &v_full[st]);
      }
      together();                                                  // (whoever gave up comes along to the end, and the others' waits run out too)
      if (n + 1 < n_tiles) ask(n + 1);
    }
  } else if (warp < kSoftmaxWarps) {
    // ---- softmax and output: one or two threads own row r of their group (lane r of tensor memory).  Two, each with half of a tile's
    // keys, give a scheduler two warps of a group, whose exponentials, products and conversions run under each other's.
    const int half = warp >> 3, g = (warp >> 2) & 1, quarter = warp & 3, r = quarter * 32 + lane, pair = 1 + (warp & 7);
    int before = 0, works = 0;                                     // tiles of the group in the work before, and how much work it had
    bool alive = true;
    const uint32_t lane_addr = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t s_addr = lane_addr + g * kArKeys + half * kSpan, o_addr = lane_addr + 256 + g * HD + half * (HD / SPLIT);
    const int row = g * kArGroupRows + r;                          // rows beyond the work's compute and store nothing
    float* const mine_told = &told[half][row];
    const float* const other_told = &told[half ^ (SPLIT - 1)][row];
    for (int number = 0; alive; ++number) {
      // (the two warps of the same rows go on or leave together: each waits for the other at their barrier, and that wait has no limit)
      if (ar_either<SPLIT>(pair, !there_is_item(number))) break;
      const ArItem& it = items[number & 1];
      int mine, hi_mine, key0, a, b, full_from, full_to;
      {
        const ArSpan w(p, it);
        if (g >= w.groups) {
          leave_item(number);
          if (PAGES) break;
          continue;
        }
        mine = g == 0 ? w.n_first : w.n_tiles;
        // the keys of this half of the tile that the row may see: [a, b) relative to it; masks only where some row of the group needs one
        key0 = w.j0 * kArKeys + half * kSpan;
        a = max(first_visible(w.pos0 + row, p.window, 0), w.lo) - key0;
        b = min(w.pos0 + row + 1, w.hi) - key0;
        hi_mine = (g == 0 ? w.hi_first : w.hi) - key0;
        full_to = min(w.pos0 + g * kArGroupRows + 1, w.hi) - kSpan - key0;      // of the group's first row
        full_from = first_visible(w.pos0 + (g + 1) * kArGroupRows - 1, p.window, 0) - key0;
      }
      ArRow rf{CAP ? p.cap_pre : p.scale_log2, p.scale_log2};
      if constexpr (PAGES) {                                         // q as float16, its largest element between 2^14 and 2^15
        alive = wait_all(&q_full, 0, 42);
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
            bad = fmaf(f.x, 0.f, fmaf(f.y, 0.f, bad));               // not-a-number where an element is not finite
          }
        }
        ar_either<SPLIT>(pair, false);                                      // (both have read the row)
        // 2^(14 - exponent of the largest), and its reciprocal
        const int e = min(max(int(__float_as_uint(largest) >> 23), 15), 254);
        const float up = __uint_as_float(uint32_t(268 - e) << 23);
        rf.factor *= __uint_as_float(uint32_t(e - 14) << 23) + bad;
#pragma unroll 4
        for (int c = half * (HD / 8 / SPLIT); c < (half + 1) * (HD / 8 / SPLIT); ++c) {
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
      // What the row currently scales by, alike in its two threads: a maximum of its scores.  Prompts begin at zero, which is near enough to
      // most rows' (weights of bfloat16 are as exact anywhere): their maximum is looked for where weights leave 2^-40 .. 2^20.
      float m = PAGES ? -INFINITY : 0.f;
      bool fresh = PAGES;                                            // some row of the warp has none
      bool settled = PAGES;                                          // the row's was looked for
      float l = 0.f;                                                 // of this thread's keys
      for (int n = 0; n < mine; ++n) {
        alive = alive && wait_all(&s_full[g], (before + n) & 1, 43) && (!PAGES || wait_all(&sc_full[n % kArRing], (n / kArRing) & 1, 44));
        tc5::fence_after();
        const ArScales* sc = scales + (n % kArRing) * (kArKeys / 8) + half * (kSpan / 8);
        const bool full = full_to >= 0 && full_from <= 0;
        const int chunks = min(max(hi_mine + 31, 0) / 32, CHUNKS);
        uint32_t packed[16 * CHUNKS];
        float weights = 0.f, sum = 0.f;
        if (alive && !fresh && chunks > 0) {
          const float m_use = (m == -INFINITY) ? 0.f : m;
          if (full) ar_tile<CHUNKS, CAP, PAGES, false, false>(s_addr, sc, packed, rf, m_use, a, b, chunks, weights, sum);
          else ar_tile<CHUNKS, CAP, PAGES, true, false>(s_addr, sc, packed, rf, m_use, a, b, chunks, weights, sum);
        }
        // (a warp that gave up says so here, and both leave)
        const bool small = !settled && max(a, 0) < min(b, kSpan) && l + weights < kArLeast;
        if (ar_either<SPLIT>(pair, fresh || small || weights > (PAGES ? kArMost : kArMostPrompt) || !alive)) {      // hardly ever
          const float m_use = (m == -INFINITY) ? 0.f : m;
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; alive && c < chunks; ++c) {
            uint32_t s[32];
            tc5::ld32(s_addr + uint32_t(c * 32), s);
            ar_wait32(s);
            mx = fmaxf(mx, ar_largest<CAP, PAGES>(s, sc + c * 4, rf, m_use, ar_bits(a - c * 32, b - c * 32)));
          }
          if (!settled && l >= kArLeast) mx = fmaxf(mx, 0.f);        // (what has weight already is not scaled up)
          *mine_told = mx;
          if (lane == 0) left[warp & 7][half] = !alive;
          ar_either<SPLIT>(pair, false);
          if (left[warp & 7][0] | left[warp & 7][1]) { alive = false; break; }
          mx = fmaxf(mx, *other_told);
          // (a reference that was not looked for may also come down, where nothing of weight has been added)
          const bool grows = mx != -INFINITY && (m == -INFINITY || mx > 0.f || !settled);
          const float alpha = grows && m != -INFINITY ? ar_exp2(fminf(-mx, 100.f)) : 1.f;
          settled = settled || mx != -INFINITY;
          if (grows) m = m_use + mx;
          l *= alpha;
          if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) ar_rescale(o_addr, HD / SPLIT, alpha);
          if (chunks > 0) ar_tile<CHUNKS, CAP, PAGES, true, true>(s_addr, sc, packed, rf, (m == -INFINITY) ? 0.f : m, a, b, chunks, weights, sum);
          fresh = __any_sync(0xffffffffu, m == -INFINITY);           // some row of the warp has seen nothing yet
        }
        l += sum;
        if (chunks > 0) {                                            // over products that are read
          tc5::st32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(packed));
          if constexpr (SPLIT == 1) tc5::st32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(packed + 32));
        }
        tc5::st_wait();
        tc5::fence_before();
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&p_full[g]);
        a -= kArKeys;
        b -= kArKeys;
        hi_mine -= kArKeys;
        full_from -= kArKeys;
        full_to -= kArKeys;
      }
      if (alive) alive = wait_all(&o_full[g], works & 1, 45);
      before += mine;
      ++works;
      *mine_told = l;
      const bool both_alive = !ar_either<SPLIT>(pair, !alive);
      tc5::fence_after();
      if (both_alive) {
        const int first_row = it.q_start + it.q0, head = it.head, rows_here = it.rows;
        if constexpr (SPLIT == 2) l = half == 0 ? l + *other_told : *other_told + l;
        if (p.sink && m != -INFINITY) l += ar_exp2(p.sink[head] * 1.4426950408889634f - m);
        const bool none = l == 0.f;                                  // no key: zeros
        float inv = none ? 0.f : 1.f / l;
        if constexpr (PAGES) inv *= exp2f(value_base);
        inv = inv > 3.402823466e38f ? 3.402823466e38f : inv;         // (scores of 2^24 and more: sums may be next to nothing, and O too)
        bf16* dst = p.out + size_t(first_row + row) * p.out_stride + size_t(head) * p.hd;
        float sick = 0.f;
#pragma unroll 1
        for (int c = 0; c < HD / 32 / SPLIT; ++c) {
          uint32_t ov[32];
          tc5::ld32(o_addr + uint32_t(c * 32), ov);                  // (all lanes of the warp take part in the load)
          ar_wait32(ov);
          if (row < rows_here) {
            const int d0 = half * (HD / SPLIT) + c * 32;
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
              if (d0 + e * 8 < p.hd) *reinterpret_cast<uint4*>(dst + d0 + e * 8) = h;
            }
          }
        }
        if (PAGES && far_apart[g]) {                                    // (a warp's rows are its own: nothing to tell)
          ar_redo<HD, CAP, PAGES>(p, &beat, it, g, __ballot_sync(0xffffffffu, row < rows_here), ~0u);
        } else if (ar_either<SPLIT>(pair, sick != 0.f)) {            // (and every element of the rows is written)
          *mine_told = sick;
          ar_either<SPLIT>(pair, false);
          const uint32_t odd = half == 0 ? __ballot_sync(0xffffffffu, sick != 0.f || *other_told != 0.f) : 0u;
          if (odd) ar_redo<HD, CAP, PAGES>(p, &beat, it, g, odd, PAGES ? 0u : __ballot_sync(0xffffffffu, l == l));
        }
      }
      tc5::fence_before();
      alive = both_alive;
      leave_item(number);
      if (PAGES) break;
    }
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
int launch_rows(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const RowsParams& p, bool cap, dim3 grid, cudaStream_t s) {
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

// Blocks of 256 rows that `tiles` tiles of `portions` requests are at most: of each the last block may be of one tile.
int rows_blocks(int tiles, int portions) {
  const long long n = ((long long)tiles + 3ll * portions) / 4;
  return n < tiles ? int(n) : tiles;
}

bool aligned16(const void* at, long long stride) { return (reinterpret_cast<uintptr_t>(at) & 15) == 0 && stride % 8 == 0; }

}  // namespace
}  // namespace kvcm

using namespace kvcm;

// q: [total_rows, >= nh * hd]; tiles of 64 query rows as the batch builder makes them (tile_seq < 0: no tile), of at most `portions` requests;
// hd 64 or 128, block_size a multiple of 8.
KVCM_API int kvcm_attention_prefill_q8_bf16(const void* q, long long q_stride, int total_rows, void* out, long long out_stride,
                                            const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                                            int num_pages, const int* block_tables, int max_blocks, const int* tile_seq, const int* tile_q0,
                                            const int* seq_q_start, const int* seq_q_len, const int* seq_ctx_len, int tiles, int portions,
                                            int nh, int nkv, int hd, int block_size, float scale, int window, float softcap,
                                            const float* sink, void* stream) {
  if (tiles <= 0 || portions <= 0) return 0;
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
  p.blocks = rows_blocks(tiles, portions);
  return launch_rows<true>(mq, mq, mq, p, softcap > 0.f, dim3(nh, p.blocks), (cudaStream_t)stream);
}

// q, k and v: rows of the prompts, one behind another; entries [0, singles) are prompts of one row, tiles name those of at most `portions`
// others.
KVCM_API int kvcm_prompt_attention_bf16(const void* q, long long q_stride, const void* k, long long k_stride, const void* v, long long v_stride,
                                        int total_rows, void* out, long long out_stride, const int* tile_seq, const int* tile_q0,
                                        const int* seq_q_start, const int* seq_q_len, int tiles, int portions, int singles, int nh, int nkv, int hd,
                                        float scale, int window, float softcap, const float* sink, void* stream) {
  if (tiles < 0 || portions < 0 || singles < 0 || (long long)tiles + singles > 65535) return KVCM_ERR_UNSUPPORTED;
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
  p.max_keys = 0x7fffffff;
  p.scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f;
  p.cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  p.sink = sink;
  p.error = const_cast<int*>(kvcm_attention_tcgen05_error_address());
  if (p.error == nullptr) return KVCM_ERR_UNSUPPORTED;
  p.blocks = rows_blocks(tiles, portions);
  return p.blocks + singles == 0 ? 0 : launch_rows<false>(mq, mk, mv, p, softcap > 0.f, dim3(nh, p.blocks + singles), (cudaStream_t)stream);
}

KVCM_PACKED(kvcm_attention_prefill_q8_bf16)
KVCM_PACKED(kvcm_prompt_attention_bf16)
