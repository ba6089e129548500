// Decode attention over a paged cache in 4 bits (layout and formulas: q4.cuh): one query row a request, bfloat16 rows.
//
// One block per (context partition, KV head x 8 query heads, request), four warps; a warp takes every fourth step of 32 keys of the
// partition and needs no other warp until the end.  The products are transposed, so that the query heads are the 8 columns of an
// m16n8k16 product and a group of at most eight heads wastes nothing of the 16 rows, which are keys (S^T = K Q^T) and then
// elements of the head (O^T = V^T P^T):
//   S^T: a lane's codes of a key are hd/4 elements in a row, any order of the contraction being as good as another if q is read
//        in the same one; they enter as 128 + code (bfloat16, exact), and  q.k = scale (q.(128 + code)) + (zero - 128 scale) sum(q).
//        In float32 the offset costs four bits of 24, in an error of a score of about 2e-5 at hd 128.
//   O^T: an element of two neighbouring keys is one register (the words of the two keys, half by half), as code - 8 (exact), and
//        sum p x = sum (p scale)(code - 8) + sum p (zero + 8 scale).  p scale enters as the sum of two bfloat16 (16 bits): with one,
//        its rounding would meet the offset zero, which the exact sum of p does not share, and double the error of the result.
//   P goes from accumulators to operands by a transposing register move (movmatrix): no shared memory in between.
// Pages come by 16-byte asynchronous copies into a ring of steps per warp: no barriers between warps, pages of any size.
//
// What bounds it: a step of 32 keys at hd 128 is 4.25 KB of memory and about 480 warp instructions, 120 cycles of an SM's four
// schedulers against 190 that the memory takes for it: memory, if enough warps are there to cover each other's latencies.
// More than eight heads on one KV head: a block for each eight, which read the same pages from L2.
// Partitions of a request: at most 8 are the blocks of one cluster and merge through distributed shared memory; more go
// through scratch memory and a second kernel (as in attention_fast.cu).
#include <cooperative_groups.h>

#include "attention_mma.cuh"
#include "pdl.cuh"
#include "q4.cuh"

namespace kvcm {

constexpr int kQ4Warps = 4;
constexpr int kQ4DecodeThreads = 32 * kQ4Warps;
constexpr int kQ4Step = 32;                        // keys of a warp's step
constexpr int kQ4Heads = 8;                        // query heads of a block
constexpr int kQ4TabMax = 512;                     // page-table entries of a partition kept in shared memory
constexpr int kQ4ClusterParts = 8;

struct DecodeQ4Params {
  const bf16* q; long long q_stride;
  bf16* out; long long out_stride;
  const uint8_t* k_cache; const uint8_t* v_cache;
  const int* block_tables; int max_blocks;
  const int* seq_ctx_len;
  float* part_o; float* part_ml;
  int nh, nkv, block_size, log2_block, num_pages, window, part_size, num_parts, cluster_merge;
  float scale_log2;                    // what a score is multiplied by on its way into exp2
  float cap_pre;                       // > 0: s <- tanh(s * cap_pre) first
  const float* sink;
};

template <int HD> struct Q4Shape {
  static_assert(HD % 32 == 0 && HD <= 256, "heads of 32 to 256 elements in steps of 32");
  static constexpr int kChunks = HD / 32;                          // 16-byte pieces of a row of codes
  static constexpr int kKeyWords = HD / 32;                        // words of a key that a lane multiplies with q
  static constexpr int kFull = HD / 64;                            // whole words of a value that a lane turns into operands
  static constexpr int kHalf = (HD / 32) & 1;                      // and one half of a word where hd is an odd multiple of 32
  static constexpr int kTiles = HD / 16;                           // tiles of 16 elements of the output
  static constexpr int kCodeBytes = kQ4Step * HD / 2;
  static constexpr int kStageBytes = 2 * kCodeBytes + 2 * kQ4Step * 4;

  // Where 16-byte piece c of row r lies in a stage.  The pieces are moved inside their row (inside 128 bytes at hd 64) so that
  // neither the reads of keys (rows side by side) nor those of values (every second row) meet in a bank.
  __device__ static __forceinline__ int at(int r, int c) {
    if constexpr (HD == 64) return (r * 32 + c * 16) ^ ((r & 4) << 4);
    else if constexpr (HD == 128) return r * 64 + ((c ^ ((r >> 1) & 2)) * 16);
    else if constexpr (HD == 256) return r * 128 + ((c ^ ((r & 6) ^ ((r & 1) << 2))) * 16);
    else return r * (HD / 2) + c * 16;
  }
  // The row (of eight) that is row r of a product.
  __device__ static __forceinline__ int row(int r) {
    if constexpr (HD == 64) return (r >> 1) | ((r & 1) << 2);
    else if constexpr (HD == 128) return r ^ ((r >> 1) & 1);
    else return r;
  }
};

__device__ __forceinline__ void cp_async4(void* smem_dst, const void* gmem_src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(smem_dst)), "l"(gmem_src));
}
// The 8 x 8 matrix of 16-bit elements that the warp holds, one row a group of four lanes, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// 128 + code -> code - 8, two at a time (whole numbers: exact).
__device__ __forceinline__ uint32_t centred(uint32_t v) {
  const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));     // 136
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int HD, int STAGES> constexpr size_t q4_decode_core_smem() {
  const size_t ring = size_t(kQ4Warps) * STAGES * Q4Shape<HD>::kStageBytes;
  const size_t merge = (size_t(kQ4Warps + 1) * kQ4Heads * HD + size_t(2 * kQ4Warps + 2) * kQ4Heads) * sizeof(float);
  return ring > merge ? ring : merge;
}
template <int HD, int STAGES> constexpr size_t q4_decode_smem() { return q4_decode_core_smem<HD, STAGES>() + kQ4TabMax * sizeof(int); }

// The partitions of a cluster: every block has its partial result in its own shared memory (bo [8][HD], bm maximum, bl sum; an
// empty partition has bm = -inf and no bo).  The outputs are dealt out over the blocks, four adjacent elements an item; each adds
// the partitions up in their order.
template <int HD>
__device__ __forceinline__ void q4_cluster_tail(const DecodeQ4Params& p, int seq, int head0, int heads_here, float* bo, float* bm, float* bl) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int P = p.num_parts;
  constexpr int Q = HD / 4;
  for (int it = int(cluster.block_rank()) * kQ4DecodeThreads + threadIdx.x; it < heads_here * Q; it += P * kQ4DecodeThreads) {
    const int r = it / Q, d = (it - r * Q) * 4;
    float m[kQ4ClusterParts], l[kQ4ClusterParts], top = -INFINITY;
    float4 o[kQ4ClusterParts];
#pragma unroll
    for (int i = 0; i < kQ4ClusterParts; ++i) {
      m[i] = -INFINITY; l[i] = 0.f; o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < P) {
        m[i] = *cluster.map_shared_rank(bm + r, i);
        l[i] = *cluster.map_shared_rank(bl + r, i);
        o[i] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(bo + r * HD + d, i));
      }
    }
#pragma unroll
    for (int i = 0; i < kQ4ClusterParts; ++i) top = fmaxf(top, m[i]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kQ4ClusterParts; ++i) {
      if (l[i] == 0.f) continue;                                   // nothing there, and its bo is not written
      const float f = fast_exp2(m[i] - top);
      acc.x = fmaf(f, o[i].x, acc.x); acc.y = fmaf(f, o[i].y, acc.y); acc.z = fmaf(f, o[i].z, acc.z); acc.w = fmaf(f, o[i].w, acc.w);
      sum = fmaf(f, l[i], sum);
    }
    if (p.sink && top != -INFINITY) sum += fast_exp2(p.sink[head0 + r] * 1.4426950408889634f - top);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bf16* dst = p.out + size_t(seq) * p.out_stride + size_t(head0 + r) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
  cluster.sync();                                                  // nobody leaves while its memory is read
}

template <int HD, int STAGES>
__global__ void __launch_bounds__(kQ4DecodeThreads, HD <= 128 ? 4 : 2) attn_decode_q4_kernel(DecodeQ4Params p) {
  typedef Q4Shape<HD> S;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  int* stab = reinterpret_cast<int*>(smem_raw + q4_decode_core_smem<HD, STAGES>());
  const int part = blockIdx.x, G = p.nh / p.nkv, head_tiles = (G + kQ4Heads - 1) / kQ4Heads;
  const int kvh = blockIdx.y / head_tiles, ht = blockIdx.y - kvh * head_tiles;
  const int head0 = kvh * G + ht * kQ4Heads, heads_here = min(kQ4Heads, G - ht * kQ4Heads);
  const int seq = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  float* mo = reinterpret_cast<float*>(smem_raw);                  // after the key loop: [warps][8][HD]
  float* mm = mo + kQ4Warps * kQ4Heads * HD;                       // [warps][8] maximum
  float* ml = mm + kQ4Warps * kQ4Heads;                            // [warps][8] sum
  float* bo = ml + kQ4Warps * kQ4Heads;                            // [8][HD] the block's result
  float* bm = bo + kQ4Heads * HD;                                  // [8]
  float* bl = bm + kQ4Heads;                                       // [8]

  pdl_launch_dependents();
  // The step's integers are there before the step's kernels; keys, also old ones, only behind the wait: a caller may have
  // written a whole prompt by the kernel before this one.
  const int ctx = p.seq_ctx_len[seq];
  const int lo = ctx > 0 ? first_visible(ctx - 1, p.window, 0) : 0;
  const int pbeg = lo / kQ4Step * kQ4Step + part * p.part_size;
  const int begin = max(lo, pbeg), end = min(ctx, pbeg + p.part_size);
  const bool nothing = begin >= end;
  const int* table = p.block_tables + size_t(seq) * p.max_blocks;
  int tab0 = 0;
  bool staged = false;
  if (!nothing) {
    tab0 = begin / p.block_size;
    const int n = (end - 1) / p.block_size - tab0 + 1;
    staged = n <= kQ4TabMax;
    if (staged)
      for (int j = tid; j < n; j += kQ4DecodeThreads) stab[j] = table[tab0 + j];
  }
  pdl_wait();
  if (nothing) {
    if (p.cluster_merge) {
      if (tid < kQ4Heads) { bm[tid] = -INFINITY; bl[tid] = 0.f; }
      q4_cluster_tail<HD>(p, seq, head0, heads_here, bo, bm, bl);
    } else if (p.num_parts == 1) {
      for (int i = tid; i < heads_here * HD; i += kQ4DecodeThreads)
        p.out[size_t(seq) * p.out_stride + size_t(head0) * HD + i] = __float2bfloat16_rn(0.f);
    } else if (tid < heads_here) {
      float* pair = p.part_ml + ((size_t(seq) * p.nh + head0 + tid) * p.num_parts + part) * 2;
      pair[0] = -INFINITY;
      pair[1] = 0.f;
    }
    return;
  }
  // ---- q of head g as the second operand: elements in the order in which a lane's codes lie
  uint32_t qb[S::kKeyWords][4];
  float qs[2];                                                     // sum of q over the elements, heads 2 t4 and 2 t4 + 1
  {
    float sum = 0.f;
    const bf16* row = p.q + size_t(seq) * p.q_stride + size_t(head0 + g) * HD;
#pragma unroll
    for (int i = 0; i < S::kKeyWords; ++i) {
      const int word = (S::kKeyWords % 4 == 0) ? (i / 4) * 16 + t4 * 4 + (i & 3) : t4 * S::kKeyWords + i;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (g < heads_here) v = *reinterpret_cast<const uint4*>(row + word * 8);
      qb[i][0] = v.x; qb[i][1] = v.y; qb[i][2] = v.z; qb[i][3] = v.w;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += __uint_as_float(qb[i][e] << 16) + __uint_as_float(qb[i][e] & 0xffff0000u);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    qs[0] = __shfl_sync(0xffffffffu, sum, t4 * 8);
    qs[1] = __shfl_sync(0xffffffffu, sum, t4 * 8 + 4);
  }
  __syncthreads();                                                 // the page-table slice is there

  // ---- the warp's steps: keys first + 32 (4 i + warp)
  const int first = begin / kQ4Step * kQ4Step;
  const int steps_all = (end - first + kQ4Step - 1) / kQ4Step;
  const int steps = (steps_all - warp + kQ4Warps - 1) / kQ4Warps;
  unsigned char* ring = smem_raw + size_t(warp) * STAGES * S::kStageBytes;
  const size_t head_bytes = q4::page_bytes(p.block_size, HD);
  const int pairs_at = p.block_size * (HD / 2);
  auto place = [&](int key, size_t& base, int& off) {              // where a key's page and row are
    const int pi = p.log2_block >= 0 ? key >> p.log2_block : key / p.block_size;
    off = key - pi * p.block_size;
    base = q4::page_base(staged ? stab[pi - tab0] : table[pi], kvh, p.nkv, p.num_pages, head_bytes);
  };
  auto load_step = [&](int i) {
    if (i < steps) {
      unsigned char* st = ring + (i % STAGES) * S::kStageBytes;
      const int key0 = first + (i * kQ4Warps + warp) * kQ4Step;
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c) {
        const int piece = c * 32 + lane, r = piece / S::kChunks, ch = piece - r * S::kChunks;
        const int key = key0 + r;
        if (key >= begin && key < end) {
          size_t base;
          int off;
          place(key, base, off);
          base += size_t(off) * (HD / 2) + ch * 16;
          const int at = S::at(r, ch);
          cp_async16(st + at, p.k_cache + base);
          cp_async16(st + S::kCodeBytes + at, p.v_cache + base);
        }
      }
      unsigned char* pairs = st + 2 * S::kCodeBytes + lane * 4;
      const int key = key0 + lane;
      if (key >= begin && key < end) {
        size_t base;
        int off;
        place(key, base, off);
        base += pairs_at + off * 4;
        cp_async4(pairs, p.k_cache + base);
        cp_async4(pairs + kQ4Step * 4, p.v_cache + base);
      } else {                                                     // zero, so that zero times it stays zero (codes are finite whatever they are)
        *reinterpret_cast<uint32_t*>(pairs) = 0u;
        *reinterpret_cast<uint32_t*>(pairs + kQ4Step * 4) = 0u;
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load_step(i);

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, zacc[2] = {0.f, 0.f};       // heads 2 t4, 2 t4 + 1; this lane's keys
  float o[S::kTiles][4];
#pragma unroll
  for (int i = 0; i < S::kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  const int row_g = S::row(g), row_a = S::row(2 * t4), row_b = S::row(2 * t4 + 1);

  for (int i = 0; i < steps; ++i) {
    load_step(i + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const unsigned char* st = ring + (i % STAGES) * S::kStageBytes;
    const uint32_t* kpair = reinterpret_cast<const uint32_t*>(st + 2 * S::kCodeBytes);
    const uint32_t* vpair = kpair + kQ4Step;
    const int key0 = first + (i * kQ4Warps + warp) * kQ4Step;
    const bool inside = key0 >= begin && key0 + kQ4Step <= end;

    float x[2][4];                                                 // scores in log2 units: [16 keys][key g, head 2t | 2t+1; key g + 8]
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      uint32_t ka[S::kKeyWords], kb[S::kKeyWords];
      const int ra = mt * 16 + row_g, rb = ra + 8;
      if constexpr (S::kKeyWords % 4 == 0) {
#pragma unroll
        for (int w = 0; w < S::kKeyWords / 4; ++w) {
          const uint4 a = *reinterpret_cast<const uint4*>(st + S::at(ra, w * 4 + t4));
          const uint4 b = *reinterpret_cast<const uint4*>(st + S::at(rb, w * 4 + t4));
          ka[4 * w] = a.x; ka[4 * w + 1] = a.y; ka[4 * w + 2] = a.z; ka[4 * w + 3] = a.w;
          kb[4 * w] = b.x; kb[4 * w + 1] = b.y; kb[4 * w + 2] = b.z; kb[4 * w + 3] = b.w;
        }
      } else if constexpr (HD == 64) {
        const uint2 a = *reinterpret_cast<const uint2*>(st + S::at(ra, t4 >> 1) + (t4 & 1) * 8);
        const uint2 b = *reinterpret_cast<const uint2*>(st + S::at(rb, t4 >> 1) + (t4 & 1) * 8);
        ka[0] = a.x; ka[1] = a.y; kb[0] = b.x; kb[1] = b.y;
      } else {
#pragma unroll
        for (int w = 0; w < S::kKeyWords; ++w) {
          ka[w] = *reinterpret_cast<const uint32_t*>(st + S::at(ra, 0) + (t4 * S::kKeyWords + w) * 4);
          kb[w] = *reinterpret_cast<const uint32_t*>(st + S::at(rb, 0) + (t4 * S::kKeyWords + w) * 4);
        }
      }
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < S::kKeyWords; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t a[4] = {q4::two_codes_128(ka[w], 2 * h), q4::two_codes_128(kb[w], 2 * h), q4::two_codes_128(ka[w], 2 * h + 1),
                                 q4::two_codes_128(kb[w], 2 * h + 1)};
          mma_bf16(c, a, qb[w][2 * h], qb[w][2 * h + 1]);
        }
      const uint32_t pa = kpair[ra], pb = kpair[rb];
      const float sa = q4::scale_of(pa), za = fmaf(-128.f, sa, q4::zero_of(pa));
      const float sb = q4::scale_of(pb), zb = fmaf(-128.f, sb, q4::zero_of(pb));
      x[mt][0] = fmaf(sa, c[0], za * qs[0]);
      x[mt][1] = fmaf(sa, c[1], za * qs[1]);
      x[mt][2] = fmaf(sb, c[2], zb * qs[0]);
      x[mt][3] = fmaf(sb, c[3], zb * qs[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[mt][j] = (p.cap_pre > 0.f ? fast_tanh(x[mt][j] * p.cap_pre) : x[mt][j]) * p.scale_log2;
      if (!inside) {
        const bool in_a = key0 + ra >= begin && key0 + ra < end, in_b = key0 + rb >= begin && key0 + rb < end;
        x[mt][0] = in_a ? x[mt][0] : -INFINITY; x[mt][1] = in_a ? x[mt][1] : -INFINITY;
        x[mt][2] = in_b ? x[mt][2] : -INFINITY; x[mt][3] = in_b ? x[mt][3] : -INFINITY;
      }
    }
    // ---- running maximum, sum
    float grown[2];
    bool moved = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float top = fmaxf(fmaxf(x[0][h], x[0][h + 2]), fmaxf(x[1][h], x[1][h + 2]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
      const float m_new = fmaxf(m[h], top);
      grown[h] = m[h] == m_new ? 1.f : fast_exp2(m[h] - m_new);    // (-inf to -inf: nothing seen yet, nothing to rescale)
      moved |= m[h] != m_new;
      m[h] = m_new;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) { l[h] *= grown[h]; zacc[h] *= grown[h]; }
#pragma unroll
      for (int k = 0; k < S::kTiles; ++k) {
        o[k][0] *= grown[0]; o[k][1] *= grown[1]; o[k][2] *= grown[0]; o[k][3] *= grown[1];
      }
    }
    const float m0 = m[0] == -INFINITY ? 0.f : m[0], m1 = m[1] == -INFINITY ? 0.f : m[1];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint32_t pa = vpair[mt * 16 + row_g], pb = vpair[mt * 16 + row_g + 8];
      const float sa = q4::scale_of(pa), za = fmaf(8.f, sa, q4::zero_of(pa));
      const float sb = q4::scale_of(pb), zb = fmaf(8.f, sb, q4::zero_of(pb));
      const float e0 = fast_exp2(x[mt][0] - m0), e1 = fast_exp2(x[mt][1] - m1);
      const float e2 = fast_exp2(x[mt][2] - m0), e3 = fast_exp2(x[mt][3] - m1);
      l[0] += e0 + e2;
      l[1] += e1 + e3;
      zacc[0] = fmaf(e0, za, fmaf(e2, zb, zacc[0]));
      zacc[1] = fmaf(e1, za, fmaf(e3, zb, zacc[1]));
      const float w0 = e0 * sa, w1 = e1 * sa, w2 = e2 * sb, w3 = e3 * sb;
      uint32_t hi[2] = {pack_bf16(w0, w1), pack_bf16(w2, w3)};
      uint32_t low[2] = {pack_bf16(w0 - __uint_as_float(hi[0] << 16), w1 - __uint_as_float(hi[0] & 0xffff0000u)),
                         pack_bf16(w2 - __uint_as_float(hi[1] << 16), w3 - __uint_as_float(hi[1] & 0xffff0000u))};
#pragma unroll
      for (int k = 0; k < 2; ++k) { hi[k] = transposed(hi[k]); low[k] = transposed(low[k]); }
      // ---- values: keys 2 t4, 2 t4 + 1 and the same eight further
      const unsigned char* vt = st + S::kCodeBytes;
      const int r0 = mt * 16 + row_a, r1 = mt * 16 + row_b;
      uint32_t v[4][S::kFull > 0 ? S::kFull : 1];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = ((k & 1) ? r1 : r0) + (k >> 1) * 8;
        if constexpr (HD == 64) {
          v[k][0] = *reinterpret_cast<const uint32_t*>(vt + S::at(r, g >> 2) + (g & 3) * 4);
        } else if constexpr (HD == 128) {
          const uint2 u = *reinterpret_cast<const uint2*>(vt + S::at(r, g >> 1) + (g & 1) * 8);
          v[k][0] = u.x; v[k][1] = u.y;
        } else if constexpr (HD == 256) {
          const uint4 u = *reinterpret_cast<const uint4*>(vt + S::at(r, g));
          v[k][0] = u.x; v[k][1] = u.y; v[k][2] = u.z; v[k][3] = u.w;
        } else {
#pragma unroll
          for (int w = 0; w < S::kFull; ++w) v[k][w] = *reinterpret_cast<const uint32_t*>(vt + S::at(r, 0) + (g * S::kFull + w) * 4);
        }
      }
#pragma unroll
      for (int w = 0; w < S::kFull; ++w) {
        const uint32_t ea = __byte_perm(v[0][w], v[1][w], 0x5410), oa = __byte_perm(v[0][w], v[1][w], 0x7632);    // even, odd elements
        const uint32_t eb = __byte_perm(v[2][w], v[3][w], 0x5410), ob = __byte_perm(v[2][w], v[3][w], 0x7632);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a[4] = {centred(q4::two_codes_128(ea, k)), centred(q4::two_codes_128(oa, k)), centred(q4::two_codes_128(eb, k)),
                                 centred(q4::two_codes_128(ob, k))};
          mma_bf16(o[4 * w + k], a, hi[0], hi[1]);
          mma_bf16(o[4 * w + k], a, low[0], low[1]);
        }
      }
      if constexpr (S::kHalf) {                                    // the last four words: lane groups 2w and 2w + 1 take the halves of word w
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          u[k] = *reinterpret_cast<const uint32_t*>(vt + S::at(((k & 1) ? r1 : r0) + (k >> 1) * 8, 0) + (8 * S::kFull + (g >> 1)) * 4);
        const uint32_t pick = (g & 1) ? 0x7632 : 0x5410;
        const uint32_t a_ = __byte_perm(u[0], u[1], pick), b_ = __byte_perm(u[2], u[3], pick);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t a[4] = {centred(q4::two_codes_128(a_, 2 * k)), centred(q4::two_codes_128(a_, 2 * k + 1)),
                                 centred(q4::two_codes_128(b_, 2 * k)), centred(q4::two_codes_128(b_, 2 * k + 1))};
          mma_bf16(o[4 * S::kFull + k], a, hi[0], hi[1]);
          mma_bf16(o[4 * S::kFull + k], a, low[0], low[1]);
        }
      }
    }
    __syncwarp();                                                  // the step's place is loaded again next round
  }
  cp_async_wait<0>();
  __syncthreads();                                                 // the rings give way to the merge

  // ---- the warp's partial result: lanes over keys joined, the zeros' part added to every element
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int off = 4; off <= 16; off *= 2) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
      zacc[h] += __shfl_xor_sync(0xffffffffu, zacc[h], off);
    }
  float* row0 = mo + (warp * kQ4Heads + 2 * t4) * HD;
  float* row1 = row0 + HD;
#pragma unroll
  for (int w = 0; w < S::kFull; ++w)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int d = 8 * (g * S::kFull + w) + 2 * k;
      *reinterpret_cast<float2*>(row0 + d) = make_float2(o[4 * w + k][0] + zacc[0], o[4 * w + k][2] + zacc[0]);
      *reinterpret_cast<float2*>(row1 + d) = make_float2(o[4 * w + k][1] + zacc[1], o[4 * w + k][3] + zacc[1]);
    }
  if constexpr (S::kHalf) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int d = 8 * (8 * S::kFull + (g >> 1)) + 4 * k + (g & 1);
      const float (&c)[4] = o[4 * S::kFull + k];
      row0[d] = c[0] + zacc[0]; row0[d + 2] = c[2] + zacc[0];
      row1[d] = c[1] + zacc[1]; row1[d + 2] = c[3] + zacc[1];
    }
  }
  if (g == 0) {
    mm[warp * kQ4Heads + 2 * t4] = m[0]; mm[warp * kQ4Heads + 2 * t4 + 1] = m[1];
    ml[warp * kQ4Heads + 2 * t4] = l[0]; ml[warp * kQ4Heads + 2 * t4 + 1] = l[1];
  }
  __syncthreads();
  // ---- the four warps, four adjacent elements an item
  constexpr int Q = HD / 4;
  for (int it = tid; it < heads_here * Q; it += kQ4DecodeThreads) {
    const int r = it / Q, d = (it - r * Q) * 4;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kQ4Warps; ++w) top = fmaxf(top, mm[w * kQ4Heads + r]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kQ4Warps; ++w) {
      const float lw = ml[w * kQ4Heads + r];
      if (lw == 0.f) continue;                                     // a warp without keys
      const float f = fast_exp2(mm[w * kQ4Heads + r] - top);
      const float4 v = *reinterpret_cast<const float4*>(mo + (w * kQ4Heads + r) * HD + d);
      acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
      sum = fmaf(f, lw, sum);
    }
    const int head = head0 + r;
    if (p.cluster_merge) {
      *reinterpret_cast<float4*>(bo + r * HD + d) = acc;
      if (d == 0) { bm[r] = top; bl[r] = sum; }
    } else if (p.num_parts == 1) {
      if (p.sink && top != -INFINITY) sum += fast_exp2(p.sink[head] * 1.4426950408889634f - top);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      bf16* dst = p.out + size_t(seq) * p.out_stride + size_t(head) * HD + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    } else {
      const size_t at = (size_t(seq) * p.nh + head) * p.num_parts + part;
      *reinterpret_cast<float4*>(p.part_o + at * HD + d) = acc;
      if (d == 0) { p.part_ml[at * 2] = top; p.part_ml[at * 2 + 1] = sum; }
    }
  }
  if (p.cluster_merge) q4_cluster_tail<HD>(p, seq, head0, heads_here, bo, bm, bl);
}

// More partitions than a cluster merges, out of scratch memory, in their order.
__global__ void attn_decode_q4_merge_kernel(const float* part_o, const float* part_ml, bf16* __restrict__ out, long long out_stride, int nh,
                                            int hd, int num_parts, const float* __restrict__ sink) {
  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.x, head = blockIdx.y;
  const size_t base = (size_t(seq) * nh + head) * num_parts;
  float top = -INFINITY;
  for (int i = 0; i < num_parts; ++i) top = fmaxf(top, part_ml[(base + i) * 2]);
  for (int d = threadIdx.x; d < hd; d += blockDim.x) {
    float acc = 0.f, sum = 0.f;
    for (int i = 0; i < num_parts; ++i) {
      const float li = part_ml[(base + i) * 2 + 1];
      if (li == 0.f) continue;
      const float f = exp2f(part_ml[(base + i) * 2] - top);
      acc = fmaf(f, part_o[(base + i) * hd + d], acc);
      sum = fmaf(f, li, sum);
    }
    if (sink && top != -INFINITY) sum += exp2f(sink[head] * 1.4426950408889634f - top);
    out[size_t(seq) * out_stride + size_t(head) * hd + d] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc / sum);
  }
}

template <int HD> constexpr int q4_decode_stages() { return HD <= 128 ? 3 : 2; }

template <int HD>
int launch_decode_q4(const DecodeQ4Params& p, int seqs, cudaStream_t s) {
  constexpr int STAGES = q4_decode_stages<HD>();
  auto kernel = attn_decode_q4_kernel<HD, STAGES>;
  constexpr size_t smem = q4_decode_smem<HD, STAGES>();
  static OncePerDevice once;
  if (smem > 48 * 1024) {
    const int rc = allow_shared_memory(once, kernel, smem);
    if (rc != 0) return rc;
  }
  const int G = p.nh / p.nkv;
  const dim3 grid(p.num_parts, p.nkv * ((G + kQ4Heads - 1) / kQ4Heads), seqs);
  if (p.cluster_merge) return pdl_launch_cluster(kernel, grid, dim3(kQ4DecodeThreads), smem, s, p.num_parts, p);
  return pdl_launch(kernel, grid, dim3(kQ4DecodeThreads), smem, s, p);
}

template <int HD> int q4_blocks_per_sm() {
  constexpr int STAGES = q4_decode_stages<HD>();
  auto kernel = attn_decode_q4_kernel<HD, STAGES>;
  constexpr size_t smem = q4_decode_smem<HD, STAGES>();
  int n = 0;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kQ4DecodeThreads, smem) != cudaSuccess) return 0;
  return n;
}

#define KVCM_FOR_Q4_HEAD_DIMS(X) X(32) X(64) X(96) X(128) X(160) X(192) X(224) X(256)

}  // namespace kvcm

using namespace kvcm;

// 1 if the tensor-core kernels take this head size.
KVCM_API int kvcm_attention_q4_decode_supports(int hd) { return hd > 0 && hd <= 256 && hd % 32 == 0; }

// Blocks of the kernel that an SM of the current device holds at once (0: it cannot say).
KVCM_API int kvcm_attention_decode_q4_blocks_per_sm(int hd) {
#define X(N) if (hd == N) return q4_blocks_per_sm<N>();
  KVCM_FOR_Q4_HEAD_DIMS(X)
#undef X
  return 0;
}

// num_parts partitions of part_size keys (a multiple of 128) cover [first visible key rounded down to 32, context).  More than 8 of
// them, or cluster_merge == 0, want scratch: seqs * nh * num_parts * (hd + 2) floats.
KVCM_API int kvcm_attention_decode_q4_bf16(const void* q, long long q_stride, void* out, long long out_stride, const void* k_cache,
                                           const void* v_cache, int num_pages, const int* block_tables, int max_blocks,
                                           const int* seq_ctx_len, int seqs, int nh, int nkv, int hd, int block_size, float scale,
                                           int window, int part_size, int num_parts, float* scratch, int cluster_merge, float softcap,
                                           const float* sink, void* stream) {
  if (seqs == 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || block_size <= 0 || num_pages <= 0 || part_size <= 0 || part_size % (kQ4Step * kQ4Warps) ||
      num_parts < 1 || seqs > 65535 || nh > 65535)
    return KVCM_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(q) | uintptr_t(q_stride * 2) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) ||
      ((reinterpret_cast<uintptr_t>(out) | uintptr_t(out_stride * 2)) & 7))
    return KVCM_ERR_UNSUPPORTED;
  if (cluster_merge && (num_parts < 2 || num_parts > kQ4ClusterParts)) cluster_merge = 0;
  if (num_parts > 1 && !cluster_merge && scratch == nullptr) return KVCM_ERR_UNSUPPORTED;
  DecodeQ4Params p;
  p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.out_stride = out_stride;
  p.k_cache = (const uint8_t*)k_cache; p.v_cache = (const uint8_t*)v_cache; p.num_pages = num_pages;
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.seq_ctx_len = seq_ctx_len;
  p.part_o = scratch; p.part_ml = scratch ? scratch + (size_t)seqs * nh * num_parts * hd : nullptr;
  p.nh = nh; p.nkv = nkv; p.block_size = block_size; p.window = window;
  p.part_size = part_size; p.num_parts = num_parts; p.cluster_merge = cluster_merge;
  p.scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f;
  p.cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  p.sink = sink;
  p.log2_block = -1;
  for (int b = 0; b < 31; ++b) if ((1 << b) == block_size) p.log2_block = b;
  int rc = KVCM_ERR_UNSUPPORTED;
#define X(N) if (hd == N) rc = launch_decode_q4<N>(p, seqs, (cudaStream_t)stream);
  KVCM_FOR_Q4_HEAD_DIMS(X)
#undef X
  if (rc != 0 || num_parts == 1 || cluster_merge) return rc;
  return pdl_launch(attn_decode_q4_merge_kernel, dim3(seqs, nh), dim3(hd < 64 ? 32 : 64), 0, (cudaStream_t)stream, (const float*)p.part_o,
                    (const float*)p.part_ml, p.out, out_stride, nh, hd, num_parts, p.sink);
}
