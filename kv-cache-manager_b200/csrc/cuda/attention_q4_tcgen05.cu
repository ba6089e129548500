// Causal prefill attention over a paged cache in 4 bits (layout and formulas: q4.cuh) on the fifth-generation tensor cores,
// head_dim 64 or 128.
//
// One block per (256 query rows of a request, query head), as two groups of 128 rows that share every tile of keys and values.  Per
// tile of 128 keys and group:
//     S = Q C^T   C = 128 + the key's codes (bfloat16, exact), accumulator in tensor memory
//     softmax     one thread a row:  x = scale S + (zero - 128 scale) sum(q),  P = bfloat16(2^(x - m))
//     O += P V    V = bfloat16(zero + scale code), MN-major operand, O in tensor memory for the whole block
// A key is never rounded: its scale and zero meet the score, which costs two packed multiply-adds for two scores.  A value is, once, to
// bfloat16, as P is: applied to P instead, its scale and zero were three more instructions for two scores in the loop that
// bounds the kernel (four portions behind long prefixes: 1,270 us against DONE_US).
// A row takes its tile relative to the maximum that it knew before, without looking for the tile's own: where the tile's sum comes
// out above 2^12 (or the row has seen nothing yet) the tile's maximum is found, sums and O are rescaled, and the tile is taken
// again, S being still there.  The largest probability therefore lies between 1 and 2^12 times 1, which float32 sums and the
// exponents of bfloat16 do not mind.
//
// Roles (16 warps, 128 registers a thread): 0-3 and 4-7 softmax and output of the two groups; 8-11 turn keys into operands and
// pairs into scales, 12-14 values; one thread of warp 15 brings Q and issues the products, S of a group's next tile before O += P W
// of this one, the groups in turn, so that the products of one run under the softmax of the other.
// What bounds it: at head_dim 128 a tile's exponentials (256 x 128 at 16 a cycle) and its products each take 2,048 cycles, and the
// handshakes between roles, some 150 cycles each, come on top where they are not hidden: tiles of 64 keys, with twice as many
// of them, took 4,100 cycles for half the work.
// A thread of warps 8-14 copies what it unpacks itself (cp.async into shared memory, a tile ahead) and so waits for nobody else's.
// Masks: key <= position, optional window.  Every wait is bounded; one that runs out sets the error word of the tcgen05 attention
// family (codes 17 and up) and ends the block.
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
constexpr float kQfMost = 4096.f;                  // a row's sum of one tile from which its maximum is renewed
// tensor memory: S of group g at column g * 128; O of group g at 256 + g * head_dim

struct PrefillQ4Params {
  bf16* out; long long out_stride;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const int* block_tables; int max_blocks;
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

struct QfScales { float2 scale, zero; };           // of two neighbouring keys, as they meet a score

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

// A row's 128 products into probabilities in P (128-byte swizzled, two blocks of 64 keys); returns their sum.  MASK: only keys
// [a, b) count.
template <bool CAP, bool MASK>
__device__ __forceinline__ float qf_softmax_tile(uint32_t s_addr, const QfScales* sc, unsigned char* rowp, int r, float qs, float m, float cap_pre,
                                                 float scale_log2, int a, int b) {
  const float2 qs2 = make_float2(qs, qs), less_m = make_float2(-m, -m);
  float2 l0 = make_float2(0.f, 0.f), l1 = make_float2(0.f, 0.f);
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t s[32];
    tc5::ld32(s_addr + uint32_t(c * 32), s);
    tc5::ld_wait();
#pragma unroll
    for (int e = 0; e < 4; ++e) {                                  // 16-byte pieces of the row of P
      uint32_t packed[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = e * 4 + i;
        float2 t = qf_scores<CAP>(s[2 * k], s[2 * k + 1], &sc[c * 16 + k], qs2, less_m, cap_pre, scale_log2);
        if constexpr (MASK) {
          const int j = c * 32 + 2 * k;
          t.x = (j >= a && j < b) ? t.x : -INFINITY;
          t.y = (j + 1 >= a && j + 1 < b) ? t.y : -INFINITY;
        }
        const float2 ex = make_float2(qf_exp2(t.x), qf_exp2(t.y));
        if (i & 1) l1 = add2(l1, ex); else l0 = add2(l0, ex);
        const __nv_bfloat162 pk = __floats2bfloat162_rn(ex.x, ex.y);
        packed[i] = *reinterpret_cast<const uint32_t*>(&pk);
      }
      const int piece = c * 4 + e;
      *reinterpret_cast<uint4*>(rowp + (piece >> 3) * kQfTile + (((piece & 7) ^ (r & 7)) * 16)) =
          make_uint4(packed[0], packed[1], packed[2], packed[3]);
    }
  }
  l0 = add2(l0, l1);
  return l0.x + l0.y;
}

// The largest score of a row's 128 products, keys [a, b).
template <bool CAP>
__device__ __noinline__ float qf_largest(uint32_t s_addr, const QfScales* sc, float qs, float cap_pre, float scale_log2, int a, int b) {
  const float2 qs2 = make_float2(qs, qs), none = make_float2(0.f, 0.f);
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    uint32_t s[32];
    tc5::ld32(s_addr + uint32_t(c * 32), s);
    tc5::ld_wait();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 t = qf_scores<CAP>(s[2 * k], s[2 * k + 1], &sc[c * 16 + k], qs2, none, cap_pre, scale_log2);
      const int j = c * 32 + 2 * k;
      mx = (j >= a && j < b) ? fmaxf(mx, t.x) : mx;
      mx = (j + 1 >= a && j + 1 < b) ? fmaxf(mx, t.y) : mx;
    }
  }
  return mx;
}

// 16 bytes of codes (elements 32 ch .. 32 ch + 31 of row r) as bfloat16 into a 128-byte swizzled tile [HD/64][128 rows][64]:
// 128 + code, or the values.
template <bool VALUES>
__device__ __forceinline__ void qf_spread(unsigned char* tile, const unsigned char* from, int r, int ch, float scale, float zero_128) {
  const uint4 u = *reinterpret_cast<const uint4*>(from);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  unsigned char* row = tile + (ch >> 1) * kQfTile + r * 128;
  const float2 s2 = make_float2(scale, scale), z2 = make_float2(zero_128, zero_128);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = q4::two_codes_128(w[j], i);
      if (VALUES) {
        const float2 v = fma2(make_float2(__uint_as_float(e[i] << 16), __uint_as_float(e[i] & 0xffff0000u)), s2, z2);
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        e[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
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
  return size_t(2 + 1 + 1) * KB * kQfTile + size_t(4) * kQfTile + size_t(2) * (kQfKeys / 2) * sizeof(QfScales) + kQfKeys * HD + kQfKeys * 4 +
         QfUnpacker<HD, kQfValueWarps>::kPerThread * kQfValueWarps * 32 * 4;
}

template <int HD, bool CAP>
__global__ void __launch_bounds__(kQfThreads, 1) attn_prefill_q4_kernel(const __grid_constant__ CUtensorMap map_q, PrefillQ4Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int KB = HD / 64;                                      // 64-wide blocks of head_dim
  unsigned char* q_s = smem_raw;                                   // [2][KB][128 rows][64]
  unsigned char* k_s = q_s + 2 * KB * kQfTile;                     // [KB][128 keys][64]
  unsigned char* v_s = k_s + KB * kQfTile;
  unsigned char* p_s = v_s + KB * kQfTile;                         // [2 groups][2][128 rows][64 keys]
  QfScales* scales = reinterpret_cast<QfScales*>(p_s + 4 * kQfTile);       // [2][64 pairs of keys]
  unsigned char* raw = reinterpret_cast<unsigned char*>(scales + 2 * (kQfKeys / 2));      // codes [2][128][HD/2]; the keys' pairs [128]; of each value piece
  __shared__ __align__(8) uint64_t q_full, k_full, v_full, sc_full[2], s_full[2], s_free[2], p_full[2], p_free[2], o_full;
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;

  // heads fastest and the last tiles, which see most keys, first
  const int tile = int(gridDim.y) - 1 - int(blockIdx.y), head = blockIdx.x;
  int* const error = p.error;
  const int seq = p.tile_seq[tile], q0 = p.tile_q0[tile];
  if (seq < 0 || (q0 & (kQfRows - 1))) return;                     // no tile, or one that belongs to a block before
  if (tc5::s32(smem_raw) & 1023) {
    if (threadIdx.x == 0) atomicExch(error, (17 << 16) | int(blockIdx.y & 0xffff));
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q_start = p.seq_q_start[seq], q_len = p.seq_q_len[seq], ctx = p.seq_ctx_len[seq];
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
    tc5::mbar_init(&k_full, kQfKeyWarps);
    tc5::mbar_init(&v_full, kQfValueWarps);
    for (int i = 0; i < 2; ++i) {
      tc5::mbar_init(&sc_full[i], kQfKeyWarps);
      tc5::mbar_init(&s_full[i], 1);
      tc5::mbar_init(&s_free[i], 4);                               // a group's four warps
      tc5::mbar_init(&p_full[i], 4);
      tc5::mbar_init(&p_free[i], 1);
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
  pdl_wait();

  auto fail = [&](int code) {
    atomicExch(error, (code << 16) | int(blockIdx.y & 0xffff));
    abort_flag = 1;
  };

  auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {  // the warp stays together whatever a lane saw
    const bool ok = !abort_flag && tc5::mbar_wait(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return true;
    if (!abort_flag && lane == 0) fail(code);
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
      const uint64_t dk = tc5::smem_desc(tc5::s32(k_s));
      // values, MN-major: 64-wide blocks a leading offset apart
      const uint64_t dv = (tc5::smem_desc(tc5::s32(v_s)) & ~(uint64_t(0x3fff) << 16)) | (uint64_t(kQfTile >> 4) << 16);
      bool ok = tc5::mbar_wait(&q_full, 0);
      if (!ok) fail(18);
      for (int n = 0; ok && n <= n_tiles && !abort_flag; ++n) {
        if (n < n_tiles && !tc5::mbar_wait(&k_full, n & 1)) { fail(19); break; }
        for (int g = 0; ok && g < groups; ++g) {
          const int mine = g == 0 ? n_first : n_tiles;
          if (n < mine) {                                          // S_n
            if (!tc5::mbar_wait(&s_free[g], (n & 1) ^ 1)) { fail(20); ok = false; break; }
            tc5::fence_after();
            const uint64_t dq = tc5::smem_desc(tc5::s32(q_s + g * KB * kQfTile));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc5::mma(tmem + uint32_t(g * kQfKeys), dq + uint64_t(kb * (kQfTile >> 4) + 2 * j), dk + uint64_t(kb * (kQfTile >> 4) + 2 * j),
                         idesc_s, (kb > 0 || j > 0) ? 1u : 0u);
            tc5::commit(&s_full[g]);
          }
          if (n >= 1 && n <= mine) {                               // O += P_(n-1) W_(n-1)
            const int m = n - 1;
            if (!tc5::mbar_wait(&p_full[g], m & 1)) { fail(22); ok = false; break; }
            if (!tc5::mbar_wait(&v_full, m & 1)) { fail(21); ok = false; break; }
            tc5::fence_after();
            const uint64_t dp = tc5::smem_desc(tc5::s32(p_s + 2 * g * kQfTile));
#pragma unroll
            for (int j = 0; j < kQfKeys / 16; ++j)                 // 16 keys: 32 bytes along a row of P, 16 rows down W
              tc5::mma(tmem + 256 + g * HD, dp + uint64_t((j >> 2) * (kQfTile >> 4) + 2 * (j & 3)), dv + uint64_t(j * (16 * 128 >> 4)), idesc_o,
                       (m > 0 || j > 0) ? 1u : 0u);
            tc5::commit(&p_free[g]);
          }
        }
      }
      tc5::commit(&o_full);
    }
  } else if (warp >= 8 && warp < 8 + kQfKeyWarps) {
    // ---- keys into operands, pairs of both into scales.  S of the last group is the last to read a tile of keys; and where it
    // is asked for, every row has taken the tile before, so two places for scales are enough.
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
      } else {
        *reinterpret_cast<uint32_t*>(pair) = 0u;                   // (a masked score, finite whatever the codes are)
      }
    };
    ask(0);
    for (int n = 0; n < n_tiles; ++n) {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      if (n > 0 && !wait_all(&s_full[groups - 1], (n - 1) & 1, 23)) break;
      const uint32_t two = *reinterpret_cast<const uint32_t*>(pair);
      float* f = reinterpret_cast<float*>(scales + (n & 1) * (kQfKeys / 2) + (t >> 1)) + (t & 1);
      const float unit = CAP ? 1.f : p.scale_log2, scale = q4::scale_of(two);
      f[0] = scale * unit;
      f[2] = fmaf(-128.f, scale, q4::zero_of(two)) * unit;
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch;
        if (unpack.piece(i, r, ch)) qf_spread<false>(k_s, raw + r * (HD / 2) + ch * 16, r, ch, 0.f, 0.f);
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        tc5::mbar_arrive(&sc_full[n & 1]);
        tc5::mbar_arrive(&k_full);
      }
      if (n + 1 < n_tiles) ask(n + 1);
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
  } else if (warp >= 8 && warp < 8 + kQfKeyWarps + kQfValueWarps) {
    // ---- values into operands; each piece with its own copy of its row's pair
    const QfUnpacker<HD, kQfValueWarps> unpack{warp - 8 - kQfKeyWarps, lane};
    unsigned char* codes = raw + kQfKeys * (HD / 2);
    unsigned char* pair = raw + kQfKeys * HD + kQfKeys * 4 + (threadIdx.x - 32 * (8 + kQfKeyWarps)) * 4;
    constexpr int kPairStep = kQfValueWarps * 32 * 4;
    auto ask = [&](int n) {
      const int key0 = (j0 + n) * kQfKeys;
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch, off;
        if (!unpack.piece(i, r, ch)) continue;
        if (key0 + r >= lo && key0 + r < hi) {
          const size_t at = page_of(key0 + r, off);
          qf_copy16(codes + r * (HD / 2) + ch * 16, p.v_cache + at + size_t(off) * (HD / 2) + ch * 16);
          qf_copy4(pair + i * kPairStep, p.v_cache + at + pairs_at + off * 4);
        } else {
          *reinterpret_cast<uint32_t*>(pair + i * kPairStep) = 0u; // a value of zero: zero times it stays zero
        }
      }
    };
    ask(0);
    for (int n = 0; n < n_tiles; ++n) {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      if (n > 0 && !wait_all(&p_free[groups - 1], (n - 1) & 1, 24)) break;
#pragma unroll
      for (int i = 0; i < unpack.kPerThread; ++i) {
        int r, ch;
        if (!unpack.piece(i, r, ch)) continue;
        const uint32_t two = *reinterpret_cast<const uint32_t*>(pair + i * kPairStep);
        const float scale = q4::scale_of(two);
        qf_spread<true>(v_s, codes + r * (HD / 2) + ch * 16, r, ch, scale, fmaf(-128.f, scale, q4::zero_of(two)));
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(&v_full);
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
      float l = 0.f;
      unsigned char* const rowp = p_s + 2 * g * kQfTile + r * 128;
      for (int n = 0; alive && n < mine; ++n) {
        if (!wait_all(&s_full[g], n & 1, 26) || !wait_all(&sc_full[n & 1], (n >> 1) & 1, 27)) { alive = false; break; }
        // P's buffer was last read by O += P_(n-1) W_(n-1); O must hold that tile where it is rescaled
        if (n > 0 && !wait_all(&p_free[g], (n - 1) & 1, 28)) { alive = false; break; }
        tc5::fence_after();
        const QfScales* sc = scales + (n & 1) * (kQfKeys / 2);
        const int key0 = (j0 + n) * kQfKeys;
        // the keys of this tile that the row may see: [a, b) relative to it; masks only where some row of the group needs one
        const int a = max(first, lo) - key0, b = min(pos + 1, hi) - key0;
        const bool full = key0 + kQfKeys - 1 <= group_pos && key0 >= last_first;
        float sum = 0.f;
        bool again = m == -INFINITY;                               // nothing seen yet: the maximum first
        for (int pass = 0; pass < 2; ++pass) {
          if (__any_sync(0xffffffffu, again)) {
            const float mx = qf_largest<CAP>(s_addr, sc, qs, p.cap_pre, p.scale_log2, a, b);
            const bool renew = again && mx > m;
            const float alpha = renew && m != -INFINITY ? qf_exp2(m - mx) : 1.f;
            if (renew) m = mx;
            l *= alpha;
            if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
              uint32_t ov[32];
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                tc5::ld32(o_addr + uint32_t(c * 32), ov);
                tc5::ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                tc5::st32(o_addr + uint32_t(c * 32), ov);
              }
              tc5::st_wait();
            }
          }
          const float m_use = (m == -INFINITY) ? 0.f : m;
          sum = full ? qf_softmax_tile<CAP, false>(s_addr, sc, rowp, r, qs, m_use, p.cap_pre, p.scale_log2, a, b)
                     : qf_softmax_tile<CAP, true>(s_addr, sc, rowp, r, qs, m_use, p.cap_pre, p.scale_log2, a, b);
          again = !again && sum > kQfMost;                         // (after a look at the maximum it is at most 128)
          if (!__any_sync(0xffffffffu, again)) break;
        }
        l += sum;
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        tc5::fence_before();
        __syncwarp();
        if (lane == 0) {
          tc5::mbar_arrive(&s_free[g]);                            // S_(n+1) may be written
          tc5::mbar_arrive(&p_full[g]);
        }
      }
      if (alive) alive = wait_all(&o_full, 0, 29);
      tc5::fence_after();
      if (alive) {
        if (p.sink && m != -INFINITY) l += qf_exp2(p.sink[head] * 1.4426950408889634f - m);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bf16* dst = p.out + size_t(q_start + q0 + row) * p.out_stride + size_t(head) * HD;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t ov[32];
          tc5::ld32(o_addr + uint32_t(c * 32), ov);                // (all lanes of the warp take part in the load)
          tc5::ld_wait();
          if (row < rows_here) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              __nv_bfloat162 h[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                h[i] = __floats2bfloat162_rn(__uint_as_float(ov[e * 8 + 2 * i]) * inv, __uint_as_float(ov[e * 8 + 2 * i + 1]) * inv);
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
  if (!kvcm_attention_prefill_q4_supports(hd) || nkv <= 0 || nh <= 0 || nh % nkv || block_size <= 0 || num_pages <= 0 || total_rows <= 0 ||
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
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.tile_seq = tile_seq; p.tile_q0 = tile_q0;
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
