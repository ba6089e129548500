// Causal prefill attention over a paged cache in 4 bits (layout and formulas: q4.cuh) on the fifth-generation tensor cores,
// head_dim 64 or 128.
//
// One block per (256 query rows of a request, query head), as two groups of 128 rows that share every tile of keys and values.  Per
// tile of 64 keys and group:
//     S = Q C^T   C = 128 + the key's codes (bfloat16, exact), accumulator in tensor memory, two buffers
//     softmax     one thread a row:  x = scale_k S + (zero_k - 128 scale_k) sum(q),  p = 2^(x - m),  P = bfloat16(p scale_v)
//     O += P W    W = the value's codes - 8 (exact), MN-major operand, O in tensor memory for the whole block
// and at the end  o = (O + sum p (zero_v + 8 scale_v)) / sum p.  Keys and values are never rounded: what is rounded is P, to bfloat16.
// Reference maximum renewed only when it is 2^8 behind, as in attention_tcgen05.cu.
//
// Roles (12 warps): 0-3 and 4-7 softmax and output of the two groups; 8-10 turn pages into operands: a thread takes 16 bytes of
// codes (32 elements of a key), writes four 16-byte pieces of a 128-byte swizzled row, and asks for the next tile's codes before
// it waits; one thread of warp 11 brings Q and issues the products, S one tile ahead of O.
// Two groups to a tile because unpacking is then paid once for 256 rows, and because the softmax of one covers the products of
// the other: the exponentials of a tile and a group (128 x 64 at 16 a cycle) take as long as its two products at head_dim 128.
// Scales and zeros lie in a ring of five tiles beside the operands: a thread of the softmax may still read those of tile n while
// tile n + 4 is unpacked, but not n + 5 (its products ask for S_(n+3), which wants every row's S_(n+1) read).
// Masks: key <= position, optional window.  Every wait is bounded; one that runs out sets the error word of the tcgen05 attention
// family (codes 17 and up) and ends the block.
#include "pdl.cuh"
#include "q4.cuh"
#include "tcgen05_common.cuh"

extern "C" const int* kvcm_attention_tcgen05_error_address(void);

namespace kvcm {

constexpr int kQfThreads = 384;                   // (twelve warps, three to a scheduler: 168 registers a thread)
constexpr int kQfUnpackWarps = 3;
constexpr int kQfGroupRows = 128, kQfRows = 256;
constexpr int kQfKeys = 64;
constexpr int kQfStages = 2;                       // tiles of K operands, and of V operands
constexpr int kQfScaleRing = 5;
constexpr int kQfTile = 128 * 128;                 // [128 rows][64 bf16]
constexpr int kQfBlock = kQfKeys * 128;            // [64 keys][64 bf16]
constexpr float kQfRescaleStep = 8.f;              // in log2 units
// tensor memory: S of group g in buffer b at column (2 g + b) * 64; O of group g at 256 + g * head_dim

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
__device__ __forceinline__ float qf_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 128 + code -> code - 8, two at a time.
__device__ __forceinline__ uint32_t qf_centred(uint32_t v) {
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(v), "r"(0x43084308u));
  return r;
}
// a * b + c of two floats at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}\n"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

struct QfScales { float2 k_scale, k_zero, v_scale, v_zero; };      // of two neighbouring keys

template <int HD> constexpr size_t qf_smem() {
  constexpr int KB = HD / 64;
  return size_t(2) * KB * kQfTile + size_t(2) * kQfStages * KB * kQfBlock + size_t(4) * kQfTile + size_t(kQfScaleRing) * (kQfKeys / 2) * sizeof(QfScales);
}

template <int HD, bool CAP>
__global__ void __launch_bounds__(kQfThreads, 1) attn_prefill_q4_kernel(const __grid_constant__ CUtensorMap map_q, PrefillQ4Params p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  constexpr int KB = HD / 64;                                      // 64-wide blocks of head_dim
  constexpr int kStage = KB * kQfBlock;
  constexpr int kPieces = HD / 32;                                 // 16-byte pieces of a row of codes
  constexpr int kGroups8 = kQfKeys * kPieces / 8;                  // groups of eight pieces of K (and of V)
  constexpr int kPerThread = (kGroups8 + 4 * kQfUnpackWarps - 1) / (4 * kQfUnpackWarps);
  unsigned char* q_s = smem_raw;                                   // [2][KB][128 rows][64]
  unsigned char* k_s = q_s + 2 * KB * kQfTile;                     // [stages][KB][64 keys][64]
  unsigned char* v_s = k_s + kQfStages * kStage;
  unsigned char* p_s = v_s + kQfStages * kStage;                   // [2 groups][2][128 rows][64 keys]
  QfScales* scales = reinterpret_cast<QfScales*>(p_s + 4 * kQfTile);       // [ring][32 pairs of keys]
  __shared__ __align__(8) uint64_t q_full, k_full[kQfStages], k_empty[kQfStages], v_full[kQfStages], v_empty[kQfStages], sc_full[kQfScaleRing],
      s_full[2][2], s_free[2][2], p_full[2][2], p_free[2][2], o_full;
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
    for (int i = 0; i < kQfStages; ++i) {
      tc5::mbar_init(&k_full[i], kQfUnpackWarps);
      tc5::mbar_init(&v_full[i], kQfUnpackWarps);
      tc5::mbar_init(&k_empty[i], 1);
      tc5::mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kQfScaleRing; ++i) tc5::mbar_init(&sc_full[i], kQfUnpackWarps);
    for (int g = 0; g < 2; ++g)
      for (int i = 0; i < 2; ++i) {
        tc5::mbar_init(&s_full[g][i], 1);
        tc5::mbar_init(&s_free[g][i], 4);                          // a group's four warps
        tc5::mbar_init(&p_full[g][i], 4);
        tc5::mbar_init(&p_free[g][i], 1);
      }
    tc5::mbar_init(&o_full, 1);
    tc5::mbar_init_fence();
  }
  if (warp == 11) {
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

  if (warp == 11) {
    // ---- one thread: Q once, then the products
    if (lane == 0) {
      tc5::mbar_expect_tx(&q_full, groups * KB * kQfTile);
      for (int g = 0; g < groups; ++g)
        for (int kb = 0; kb < KB; ++kb)
          tc5::tma_load_2d(q_s + (g * KB + kb) * kQfTile, &map_q, &q_full, head * HD + kb * 64, q_start + q0 + g * kQfGroupRows);
      constexpr uint32_t idesc_s = tc5::idesc(kQfGroupRows, kQfKeys, false);
      constexpr uint32_t idesc_o = tc5::idesc(kQfGroupRows, 64, true);
      bool ok = tc5::mbar_wait(&q_full, 0);
      if (!ok) fail(18);
      for (int n = 0; ok && n <= n_tiles && !abort_flag; ++n) {
        if (n < n_tiles) {                                         // S_n of both groups
          const int st = n % kQfStages;
          if (!tc5::mbar_wait(&k_full[st], (n / kQfStages) & 1)) { fail(19); break; }
          const uint64_t dk = tc5::smem_desc(tc5::s32(k_s + st * kStage));
          for (int g = 0; g < groups; ++g) {
            if (g == 0 && n >= n_first) continue;
            if (!tc5::mbar_wait(&s_free[g][n & 1], ((n >> 1) & 1) ^ 1)) { fail(20); ok = false; break; }
            tc5::fence_after();
            const uint64_t dq = tc5::smem_desc(tc5::s32(q_s + g * KB * kQfTile));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc5::mma(tmem + uint32_t((2 * g + (n & 1)) * kQfKeys), dq + uint64_t(kb * (kQfTile >> 4) + 2 * j),
                         dk + uint64_t(kb * (kQfBlock >> 4) + 2 * j), idesc_s, (kb > 0 || j > 0) ? 1u : 0u);
            tc5::commit(&s_full[g][n & 1]);
          }
          if (!ok) break;
          tc5::commit(&k_empty[st]);
        }
        if (n >= 1) {                                              // O += P_m W_m of both groups
          const int m = n - 1, st = m % kQfStages;
          if (!tc5::mbar_wait(&v_full[st], (m / kQfStages) & 1)) { fail(21); break; }
          const uint32_t v_addr = tc5::s32(v_s + st * kStage);
          for (int g = 0; g < groups; ++g) {
            if (g == 0 && m >= n_first) continue;
            if (!tc5::mbar_wait(&p_full[g][m & 1], (m >> 1) & 1)) { fail(22); ok = false; break; }
            tc5::fence_after();
            const uint64_t dp = tc5::smem_desc(tc5::s32(p_s + (2 * g + (m & 1)) * kQfTile));
#pragma unroll
            for (int j = 0; j < kQfKeys / 16; ++j)
#pragma unroll
              for (int nb = 0; nb < KB; ++nb)
                tc5::mma(tmem + 256 + g * HD + nb * 64, dp + uint64_t(2 * j), tc5::smem_desc(v_addr + nb * kQfBlock + j * 16 * 128), idesc_o,
                         (m > 0 || j > 0) ? 1u : 0u);
            tc5::commit(&p_free[g][m & 1]);
          }
          if (!ok) break;
          tc5::commit(&v_empty[st]);
        }
      }
      tc5::commit(&o_full);
    }
  } else if (warp >= 8) {
    // ---- pages into operands
    const int t = threadIdx.x - 256, wq = warp - 8;
    const size_t bytes = q4::page_bytes(p.block_size, HD);
    const int pairs_at = p.block_size * (HD / 2);
    const int* table = p.block_tables + size_t(seq) * p.max_blocks;
    auto page_of = [&](int key, int& off) {
      const int pi = p.log2_block >= 0 ? key >> p.log2_block : key / p.block_size;
      off = key - pi * p.block_size;
      return q4::page_base(table[pi], kvh, p.nkv, p.num_pages, bytes);
    };
    // this thread's pieces: neighbouring lanes take neighbouring keys (their swizzled rows differ in every bank)
    int key_of[kPerThread], ch_of[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int group = (i * kQfUnpackWarps + wq) * 4 + (lane >> 3);       // eight lanes: eight keys, one piece
      key_of[i] = group < kGroups8 ? (group / kPieces) * 8 + (lane & 7) : -1;
      ch_of[i] = group % kPieces;
    }
    uint4 kc[kPerThread], vc[kPerThread];
    uint32_t kp = 0, vp = 0;                                       // the pair of key t (t < 64)
    auto ask = [&](int n) {
      const int key0 = (j0 + n) * kQfKeys;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        const int key = key0 + key_of[i];
        kc[i] = vc[i] = make_uint4(0u, 0u, 0u, 0u);
        if (key_of[i] >= 0 && key >= lo && key < hi) {
          int off;
          size_t at = page_of(key, off);
          at += size_t(off) * (HD / 2) + ch_of[i] * 16;
          kc[i] = *reinterpret_cast<const uint4*>(p.k_cache + at);
          vc[i] = *reinterpret_cast<const uint4*>(p.v_cache + at);
        }
      }
      if (t < kQfKeys) {
        const int key = key0 + t;
        kp = vp = 0u;                                              // zero: zero times it stays zero
        if (key >= lo && key < hi) {
          int off;
          size_t at = page_of(key, off);
          at += pairs_at + off * 4;
          kp = *reinterpret_cast<const uint32_t*>(p.k_cache + at);
          vp = *reinterpret_cast<const uint32_t*>(p.v_cache + at);
        }
      }
    };
    // element 32 ch + 8 j of key r: 16 bytes at swizzled piece (32 ch + 8 j) % 64 / 8 of row r of block ch / 2
    auto spread = [&](unsigned char* base, const uint4& codes, int r, int ch, bool centre) {
      const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
      unsigned char* row = base + (ch >> 1) * kQfBlock + r * 128;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = q4::two_codes_128(w[j], i);
          if (centre) e[i] = qf_centred(e[i]);
        }
        *reinterpret_cast<uint4*>(row + ((((ch & 1) * 4 + j) ^ (r & 7)) * 16)) = make_uint4(e[0], e[1], e[2], e[3]);
      }
    };
    auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
      const bool ok = !abort_flag && tc5::mbar_wait(bar, parity);
      if (__all_sync(0xffffffffu, ok)) return true;
      if (!abort_flag && lane == 0) fail(code);
      return false;
    };
    ask(0);
    for (int n = 0; n < n_tiles; ++n) {
      const int st = n % kQfStages;
      const uint32_t round = ((n / kQfStages) & 1) ^ 1;
      if (!wait_all(&k_empty[st], round, 23)) break;
      if (t < kQfKeys) {
        float* f = reinterpret_cast<float*>(scales + (n % kQfScaleRing) * (kQfKeys / 2) + (t >> 1)) + (t & 1);
        const float unit = CAP ? 1.f : p.scale_log2;
        const float ks = q4::scale_of(kp), vs = q4::scale_of(vp);
        f[0] = ks * unit;
        f[2] = fmaf(-128.f, ks, q4::zero_of(kp)) * unit;
        f[4] = vs;
        f[6] = fmaf(8.f, vs, q4::zero_of(vp));
      }
#pragma unroll
      for (int i = 0; i < kPerThread; ++i)
        if (key_of[i] >= 0) spread(k_s + st * kStage, kc[i], key_of[i], ch_of[i], false);
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        tc5::mbar_arrive(&sc_full[n % kQfScaleRing]);
        tc5::mbar_arrive(&k_full[st]);
      }
      if (!wait_all(&v_empty[st], round, 24)) break;
#pragma unroll
      for (int i = 0; i < kPerThread; ++i)
        if (key_of[i] >= 0) spread(v_s + st * kStage, vc[i], key_of[i], ch_of[i], true);
      if (n + 1 < n_tiles) ask(n + 1);
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
      __syncwarp();
      if (lane == 0) tc5::mbar_arrive(&v_full[st]);
    }
  } else {
    // ---- softmax and output: this thread owns row r of its group (lane r of tensor memory)
    const int g = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const int mine = g == 0 ? n_first : n_tiles;
    const int row = g * kQfGroupRows + r, pos = pos0 + row;        // rows beyond rows_here compute and store nothing
    const uint32_t lane_addr = tmem + (uint32_t(quarter * 32) << 16);
    const uint32_t o_addr = lane_addr + 256 + g * HD;
    if (g < groups) {
      const int first = first_visible(pos, p.window, 0);
      const int group_pos = pos0 + g * kQfGroupRows;               // of the group's first row
      const int last_first = first_visible(group_pos + kQfGroupRows - 1, p.window, 0);
      auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
        const bool ok = !abort_flag && tc5::mbar_wait(bar, parity);
        if (__all_sync(0xffffffffu, ok)) return true;
        if (!abort_flag && lane == 0) fail(code);
        return false;
      };
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
      const float2 qs2 = make_float2(qs, qs);
      float m = -INFINITY;                                         // the maximum the row currently scales by
      float2 l2 = make_float2(0.f, 0.f), z2 = make_float2(0.f, 0.f);
      for (int n = 0; alive && n < mine; ++n) {
        if (!wait_all(&s_full[g][n & 1], (n >> 1) & 1, 26)) { alive = false; break; }
        tc5::fence_after();
        uint32_t v[2][32];                                         // the row's 64 products
#pragma unroll
        for (int c = 0; c < 2; ++c) tc5::ld32(lane_addr + uint32_t((2 * g + (n & 1)) * kQfKeys + c * 32), v[c]);
        tc5::ld_wait();
        tc5::fence_before();
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&s_free[g][n & 1]);        // S_(n+2) may be written
        if (!wait_all(&sc_full[n % kQfScaleRing], (n / kQfScaleRing) & 1, 27)) { alive = false; break; }
        const QfScales* sc = scales + (n % kQfScaleRing) * (kQfKeys / 2);
        float* x = reinterpret_cast<float*>(&v[0][0]);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float4 s = *reinterpret_cast<const float4*>(&sc[i]);       // scales, then zeros, of keys 2i and 2i + 1
          float2 t = fma2(make_float2(x[2 * i], x[2 * i + 1]), make_float2(s.x, s.y), mul2(make_float2(s.z, s.w), qs2));
          if constexpr (CAP) {
            t.x = qf_tanh(t.x * p.cap_pre) * p.scale_log2;
            t.y = qf_tanh(t.y * p.cap_pre) * p.scale_log2;
          }
          x[2 * i] = t.x;
          x[2 * i + 1] = t.y;
        }
        const int key0 = (j0 + n) * kQfKeys;
        // the keys of this tile that the row may see: [a, b) relative to it; masks only where some row of the group needs one
        const int a = max(first, lo) - key0, b = min(pos + 1, hi) - key0;
        const bool full = key0 + kQfKeys - 1 <= group_pos && key0 >= last_first;
        if (!full) {
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = (i >= a && i < b) ? x[i] : -INFINITY;
        }
        float part[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float t = qf_max3(x[8 * e], x[8 * e + 1], x[8 * e + 2]);
          t = qf_max3(t, x[8 * e + 3], x[8 * e + 4]);
          t = qf_max3(t, x[8 * e + 5], x[8 * e + 6]);
          part[e] = fmaxf(t, x[8 * e + 7]);
        }
        const float m_tile = fmaxf(qf_max3(qf_max3(part[0], part[1], part[2]), part[3], part[4]), qf_max3(part[5], part[6], part[7]));
        float alpha = 1.f;
        bool rescale = false;
        if (m == -INFINITY) {
          m = m_tile;                                              // nothing was added yet
        } else if (m_tile > m + kQfRescaleStep) {
          alpha = qf_exp2(m - m_tile);
          m = m_tile;
          rescale = true;
        }
        if (__any_sync(0xffffffffu, rescale)) {
          // O must hold tile n - 1 completely; nothing newer is issued before this warp has delivered P_n
          if (n > 0 && !wait_all(&p_free[g][(n - 1) & 1], ((n - 1) >> 1) & 1, 28)) { alive = false; break; }
          tc5::fence_after();
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
          l2.x *= alpha; l2.y *= alpha; z2.x *= alpha; z2.y *= alpha;
        }
        // P_n's buffer was last read by O += P_(n-2) W_(n-2), issued before S_n: having seen S_n, it may be written
        const float m_use = (m == -INFINITY) ? 0.f : m;
        unsigned char* rowp = p_s + (2 * g + (n & 1)) * kQfTile + r * 128;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t packed[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = c * 4 + i;
            const float4 s = *(reinterpret_cast<const float4*>(&sc[k]) + 1);
            const float2 e = make_float2(qf_exp2(x[2 * k] - m_use), qf_exp2(x[2 * k + 1] - m_use));
            l2 = add2(l2, e);
            z2 = fma2(e, make_float2(s.z, s.w), z2);
            const float2 w = mul2(e, make_float2(s.x, s.y));
            const __nv_bfloat162 h = __floats2bfloat162_rn(w.x, w.y);
            packed[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *reinterpret_cast<uint4*>(rowp + ((c ^ (r & 7)) * 16)) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        tc5::fence_before();
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive(&p_full[g][n & 1]);
      }
      if (alive) alive = wait_all(&o_full, 0, 29);
      tc5::fence_after();
      if (alive) {
        float l = l2.x + l2.y;
        const float z = z2.x + z2.y;
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
  if (warp == 11) {
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
