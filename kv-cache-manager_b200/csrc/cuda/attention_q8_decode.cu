// Decode attention over a paged cache in 8 bits (format: q8.cuh): one query row a request, bfloat16 rows.
//
// One block per piece of work (keys of one request, KV head x up to 8 query heads), four warps; a warp takes every fourth step of keys
// and needs no other warp until the end.  The products are transposed, so that the query heads are the columns of the
// products and the rows are keys (S^T = K Q^T) and then elements of the head (O^T = V^T P^T): a group of few heads wastes little.
// Both are products of float16, m16n8k16, in which codes are exact:
//   S^T  a lane's codes of a key are hd/4 elements (any order of the contraction is as good as another if q is read in the same
//        one), two of which one conversion turns into an operand.  q enters as float16 times a power of two for each head, exact
//        but for elements 2^-29 as large as the head's largest.  The key's scale meets the sum.
//   O^T  an element of two neighbouring keys is one register (their codes byte by byte, then one conversion).  Weights p scale enter
//        in units of the power of two in the head's largest weight that the warp has seen, so a weight is rounded by 2^-11 of
//        itself at most, and by 2^-25 of that unit where it is smaller than 2^-14 of it.
//   P goes from accumulators to operands by a transposing register move (movmatrix): no shared memory in between.
// The scores of the next step are formed under the softmax of this one.  Pages come by 16-byte asynchronous copies into a ring of
// steps per warp: no barriers between warps, pages of any size.
//
// Pieces of work: partitions of every request (of the grid), of which up to 8 are the blocks of a cluster that merges through
// distributed shared memory, or equal shares of all requests' tiles of 128 keys, for batches of ragged or many requests: a share
// begins and ends inside a request, the two pieces go through scratch memory, and a second kernel joins them (decode_join.cuh).
//
// What bounds it, B200: memory, where there is enough to read: 64 requests of 8,192 keys, 32 heads on 8 of 128 elements, 1.07 GB: 187 us, 5.7 TB/s
// (164 at the rate of a copy) with two blocks of four warps an SM and three steps of 8 KB a warp, one of them under way.  8 requests of some
// 1,536 keys, 32 heads on 4 of 64: 9.7 us: launch, lengths, table, q and keys behind one another, and the cluster's merge.
#include <cuda_fp16.h>

#include "decode_join.cuh"
#include "packed.cuh"
#include "q8.cuh"

namespace kvcm {

constexpr int kQ8DWarps = 4;
constexpr int kQ8DStep = 32;                       // keys of a warp's step
constexpr int kQ8DTile = kQ8DStep * kQ8DWarps;     // keys of a round of the block
constexpr int kQ8DTabMax = 512;                    // page-table entries of a partition kept in shared memory
constexpr float kQ8DLowest = 3.402823466e38f;
constexpr float kQ8DLeast = 1.17549435e-38f;       // 2^-126
// What it costs to start on a request and head, in tiles of 128 keys, for the shares: its table, its q, an empty ring.  (1, 2, 4, 6 and 8, heads of
// 128: 64 ragged requests up to 8,192 keys 65, 59, 57, 59 and 59 us with a cold cache; 100 shorter ones 49, 43, 41, 43 and 45.)
constexpr int kQ8DStart = 4;
// Exponents (of float32) by which a weight may be above its unit before the unit is formed anew: 2^12 is far from float16's end, and
// a unit that is too small costs no bits.
constexpr uint32_t kQ8DUnitRoom = 12u << 23;

struct DecodeQ8Params {
  const bf16* q; long long q_stride;
  bf16* out; long long out_stride;
  const uint8_t* k_codes; const uint8_t* v_codes; const float* k_scale; const float* v_scale;
  const int* block_tables; int max_blocks, max_keys;      // keys that a request's table has pages for
  const int* seq_ctx_len;
  float* part_o; float* part_ml;
  int* part_first;                     // shares: [seqs * head tiles][2]
  int seqs, nh, nkv, block_size, log2_block, num_pages, window;
  int part_size, num_parts, cluster_merge;      // num_parts 0: equal shares of all keys
  float scale_log2;                    // what a score is multiplied by on its way into exp2
  float cap_pre;                       // > 0: s <- tanh(s * cap_pre) first
  const float* sink;
};

namespace {

template <int HD> struct Q8Shape {
  static_assert(HD % 32 == 0 && HD <= 256, "heads of 32 to 256 elements in steps of 32");
  static constexpr int kChunks = HD / 16;                          // 16-byte pieces of a row of codes
  static constexpr int kKeyWords = HD / 16;                        // words (four codes) of a key that a lane multiplies with q
  static constexpr int kWords = HD / 32;                           // words of a value that a lane turns into operands
  static constexpr int kTiles = HD / 16;                           // tiles of 16 elements of the output
  static constexpr int kCodeBytes = kQ8DStep * HD;
  static constexpr int kStageBytes = 2 * kCodeBytes + 2 * kQ8DStep * 4;

  // Where 16-byte piece c of row r lies in a stage.  The pieces are moved inside their row (inside 128 bytes at hd 32) so that
  // neither the reads of keys (rows side by side) nor those of values (every second row) meet in a bank.
  __device__ static __forceinline__ int at(int r, int c) {
    if constexpr (HD == 32) return (r * 32 + c * 16) ^ ((r & 4) << 4);
    else if constexpr (HD == 64) return r * 64 + ((c ^ ((r >> 1) & 2)) * 16);
    else if constexpr (HD == 128 || HD == 256) return r * HD + ((c ^ ((r & 6) ^ ((r & 1) << 2))) * 16);
    else return r * HD + c * 16;
  }
  // The row (of eight) that is row r of a product.
  __device__ static __forceinline__ int row(int r) {
    if constexpr (HD == 32) return (r >> 1) | ((r & 1) << 2);
    else if constexpr (HD == 64) return r ^ ((r >> 1) & 1);
    else return r;
  }
  // The first of the four elements in word i of lane t4's part of a key, and in word j of lane g's part of a value.
  __device__ static __forceinline__ int key_element(int t4, int i) {
    if constexpr (HD % 64 == 0 && (HD & (HD - 1)) == 0) return ((i >> 2) * 4 + t4) * 16 + (i & 3) * 4;
    else return t4 * (HD / 4) + i * 4;
  }
  __device__ static __forceinline__ int value_element(int g, int j) {
    if constexpr (HD == 256) return ((j >> 2) * 8 + g) * 16 + (j & 3) * 4;
    else return g * (HD / 8) + j * 4;
  }
  // A lane's words of row r of keys, of row r of values.
  __device__ static __forceinline__ void key_words(const unsigned char* st, int r, int t4, uint32_t (&w)[kKeyWords]) {
    if constexpr (HD % 64 == 0 && (HD & (HD - 1)) == 0) {
#pragma unroll
      for (int j = 0; j < HD / 64; ++j) {
        const uint4 u = *reinterpret_cast<const uint4*>(st + at(r, j * 4 + t4));
        w[4 * j] = u.x; w[4 * j + 1] = u.y; w[4 * j + 2] = u.z; w[4 * j + 3] = u.w;
      }
    } else if constexpr (HD == 32) {
      const uint2 u = *reinterpret_cast<const uint2*>(st + at(r, t4 >> 1) + (t4 & 1) * 8);
      w[0] = u.x; w[1] = u.y;
    } else {
#pragma unroll
      for (int j = 0; j < HD / 32; ++j) {
        const uint2 u = *reinterpret_cast<const uint2*>(st + at(r, 0) + t4 * (HD / 4) + j * 8);
        w[2 * j] = u.x; w[2 * j + 1] = u.y;
      }
    }
  }
  __device__ static __forceinline__ void value_words(const unsigned char* st, int r, int g, uint32_t (&w)[kWords]) {
    if constexpr (HD == 128 || HD == 256) {
#pragma unroll
      for (int j = 0; j < HD / 128; ++j) {
        const uint4 u = *reinterpret_cast<const uint4*>(st + at(r, j * 8 + g));
        w[4 * j] = u.x; w[4 * j + 1] = u.y; w[4 * j + 2] = u.z; w[4 * j + 3] = u.w;
      }
    } else if constexpr (HD == 64) {
      const uint2 u = *reinterpret_cast<const uint2*>(st + at(r, g >> 1) + (g & 1) * 8);
      w[0] = u.x; w[1] = u.y;
    } else if constexpr (HD == 32) {
      w[0] = *reinterpret_cast<const uint32_t*>(st + at(r, g >> 2) + (g & 3) * 4);
    } else {
#pragma unroll
      for (int j = 0; j < kWords; ++j) w[j] = *reinterpret_cast<const uint32_t*>(st + at(r, 0) + (g * kWords + j) * 4);
    }
  }
};

__device__ __forceinline__ void q8_cp_async4(void* smem_dst, const void* gmem_src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(smem_dst)), "l"(gmem_src));
}
// The 8 x 8 matrix of 16-bit elements that the warp holds, one row a group of four lanes, transposed.
__device__ __forceinline__ uint32_t q8_transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// The largest power of two in a positive number, as a float's bits.
__device__ __forceinline__ uint32_t q8_power_of_two(float x) { return __float_as_uint(x) & 0x7f800000u; }
__device__ __forceinline__ uint32_t q8_pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ void q8_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int HD, int STAGES> constexpr size_t q8_decode_core_smem() {
  const size_t ring = size_t(kQ8DWarps) * STAGES * Q8Shape<HD>::kStageBytes;
  const size_t merge = (size_t(kQ8DWarps + 1) * kDecodeHeads * HD + size_t(2 * kQ8DWarps + 2) * kDecodeHeads) * sizeof(float);
  return ring > merge ? ring : merge;
}
template <int HD, int STAGES> constexpr size_t q8_decode_smem() { return q8_decode_core_smem<HD, STAGES>() + kQ8DTabMax * sizeof(int); }

// A block's piece of work: keys [begin, end) of one request for eight query heads of a KV head.
struct Q8Segment {
  int seq, kvh, head0, heads_here, begin, end;
  int slot;                            // >= 0: where the partial result goes; < 0: the result itself
};

// A lane of a warp has the sums of heads 2 t4 and 2 t4 + 1.
template <int HD, int STAGES, bool CAP>
__global__ void __launch_bounds__(kDecodeThreads, HD > 128 ? 1 : 2) attn_decode_q8_kernel(DecodeQ8Params p) {
  typedef Q8Shape<HD> S;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned* stab = reinterpret_cast<unsigned*>(smem_raw + q8_decode_core_smem<HD, STAGES>());     // pages of the head, counted over all heads
  __shared__ int found[2];
  const int G = p.nh / p.nkv, head_tiles = (G + kDecodeHeads - 1) / kDecodeHeads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  float* mo = reinterpret_cast<float*>(smem_raw);                  // after the key loop: [warps][8][HD]
  float* mm = mo + kQ8DWarps * kDecodeHeads * HD;                       // [warps][8] maximum
  float* ml = mm + kQ8DWarps * kDecodeHeads;                            // [warps][8] sum
  float* bo = ml + kQ8DWarps * kDecodeHeads;                            // [8][HD] the block's result
  float* bm = bo + kDecodeHeads * HD;                                  // [8]
  float* bl = bm + kDecodeHeads;                                       // [8]
  const bool shares = p.num_parts == 0;

  // Everything is read behind the wait: a caller may have written a whole prompt by the kernel before this one, and the lengths by
  // one of the same step (step_tables, or a sum of its own), which nothing else makes visible here.
  pdl_launch_dependents();
  pdl_wait();
  auto length = [&](int s) { return p.seq_ctx_len[s]; };
  auto first_key = [&](int ctx) { return ctx > 0 ? first_visible(ctx - 1, p.window, 0) : 0; };
  // (keys end with the table, wherever the row is)
  auto keys_of = [&](int ctx) { return min(ctx, p.max_keys); };
  // a request's cost for each head: its tiles of keys behind the start (no key, no cost)
  auto cost_of = [&](int ctx) {
    const int keys = keys_of(ctx), lo = first_key(ctx);
    return keys > lo ? kQ8DStart + (keys - lo / kQ8DStep * kQ8DStep + kQ8DTile - 1) / kQ8DTile : 0;
  };
  const int H = p.nkv * head_tiles;
  // ---- where the block's work starts
  int seq, unit_h = 0, at_cost = 0;                                // shares: request, head tile of it, how far in
  long long left = 0, U = 0, before = 0;                           // cost left of the share; of all; of one head of the requests before
  long long takers = 0;                                            // blocks that have a share
  if (!shares) {
    seq = blockIdx.z;
  } else {
    // every block adds up all lengths; the thread whose requests hold the share's first tile says where
    int* sums = reinterpret_cast<int*>(smem_raw);                  // [threads] (the rings are not in use yet)
    const int per = (p.seqs + kDecodeThreads - 1) / kDecodeThreads;
    const int s0 = min(tid * per, p.seqs), s1 = min(s0 + per, p.seqs);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += cost_of(length(s));
    int up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    if (lane == 31) sums[warp] = up;
    __syncthreads();
    int total = 0, in_front = up - mine;
#pragma unroll
    for (int w = 0; w < kQ8DWarps; ++w) {
      if (w < warp) in_front += sums[w];
      total += sums[w];
    }
    U = (long long)total * H;
    takers = min((long long)gridDim.x, U);                         // (a block between two that share a request then has a piece of it)
    if (blockIdx.x >= takers) return;
    const long long u0 = U * blockIdx.x / takers, u1 = U * (blockIdx.x + 1) / takers;
    left = u1 - u0;
    if ((long long)in_front * H <= u0 && u0 < (long long)(in_front + mine) * H) {
      int s = s0, f = in_front, n = cost_of(length(s));
      while ((long long)(f + n) * H <= u0) { f += n; ++s; n = cost_of(length(s)); }
      found[0] = s;
      found[1] = f;
    }
    __syncthreads();
    seq = found[0];
    before = found[1];
    const int n = cost_of(length(seq));
    const long long at = u0 - before * H;
    unit_h = int(at / n);
    at_cost = int(at - (long long)unit_h * n);
  }

  const unsigned head_units = unsigned(p.block_size) * S::kChunks;  // of 16 bytes, in a page of a head
  const int row_g = S::row(g), row_a = S::row(2 * t4), row_b = S::row(2 * t4 + 1);
  unsigned char* const ring = smem_raw + size_t(warp) * STAGES * S::kStageBytes;

  for (;;) {
    // ---- the next piece of work
    Q8Segment w;
    const int ctx = length(seq), keys = keys_of(ctx), lo = first_key(ctx), base = lo / kQ8DStep * kQ8DStep;
    w.seq = seq;
    w.slot = -1;
    int of_h;
    bool empty;
    if (!shares) {
      of_h = blockIdx.y;
      const int from = base + int(blockIdx.x) * p.part_size;
      w.begin = max(lo, from);
      w.end = int(blockIdx.x) + 1 == p.num_parts ? keys : min(keys, from + p.part_size);     // (the last one takes what is left)
      if (p.num_parts > 1 && !p.cluster_merge) w.slot = blockIdx.x;
    } else {
      of_h = unit_h;
      const int n = cost_of(ctx), take = int(min((long long)(n - at_cost), left));
      const int tile0 = max(0, at_cost - kQ8DStart), tile1 = max(0, at_cost + take - kQ8DStart);
      w.begin = max(lo, base + tile0 * kQ8DTile);
      w.end = min(keys, base + tile1 * kQ8DTile);
      empty = tile1 <= tile0;                                      // the start alone: the next block takes it
      if (tile0 > 0 || tile1 < n - kQ8DStart) w.slot = 2 * int(blockIdx.x) + (tile0 == 0 ? 1 : 0);
      if (!empty && tile0 == 0 && tid == 0) {                      // who reads the pieces of this request and head: blocks first .. last
        const long long last_unit = before * H + (long long)unit_h * n + n - 1;
        p.part_first[(seq * H + unit_h) * 2] = blockIdx.x;
        p.part_first[(seq * H + unit_h) * 2 + 1] = int(((last_unit + 1) * takers - 1) / U);
      }
      left -= take;
      at_cost += take;
      if (at_cost == n) {
        at_cost = 0;
        if (++unit_h == H) {
          unit_h = 0;
          before += n;
          if (left > 0)
            do ++seq; while (cost_of(length(seq)) == 0);    // (there is more, so there is such a request)
        }
      }
      if (empty) {
        if (left <= 0) return;
        continue;
      }
    }
    w.kvh = of_h / head_tiles;
    const int ht = of_h - w.kvh * head_tiles;
    w.head0 = w.kvh * G + ht * kDecodeHeads;
    w.heads_here = min(kDecodeHeads, G - ht * kDecodeHeads);

    // heads 2 t4, 2 t4 + 1; sums over this lane's keys (the maximum starts finite: no difference to it is not-a-number)
    float m[2] = {-kQ8DLowest, -kQ8DLowest}, l[2] = {0.f, 0.f};
    float o[S::kTiles][4];
#pragma unroll
    for (int i = 0; i < S::kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float heaviest[2] = {kQ8DLeast, kQ8DLeast};                    // weight of a head so far; the power of two in it is their unit
    if (w.begin < w.end) {
      // ---- q as the second operand: column g is head g, elements in the order in which a lane's codes lie
      uint32_t qb[S::kKeyWords][2];
      float step[2];                                               // of heads 2 t4 (+ 1): what their products count
      {
        const bf16* row = p.q + size_t(w.seq) * p.q_stride + size_t(w.head0 + g) * HD;
        uint2 v[S::kKeyWords];
        float largest = 0.f, bad = 0.f;
#pragma unroll
        for (int i = 0; i < S::kKeyWords; ++i) {
          v[i] = make_uint2(0u, 0u);
          if (g < w.heads_here) v[i] = *reinterpret_cast<const uint2*>(row + S::key_element(t4, i));
          const uint32_t e[2] = {v[i].x, v[i].y};
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float lo16 = __uint_as_float(e[j] << 16), hi16 = __uint_as_float(e[j] & 0xffff0000u);
            largest = fmaxf(largest, fmaxf(fabsf(lo16), fabsf(hi16)));
            bad = fmaf(lo16, 0.f, fmaf(hi16, 0.f, bad));           // not-a-number where an element is not finite
          }
        }
#pragma unroll
        for (int off = 1; off <= 2; off *= 2) {
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, off));
          bad += __shfl_xor_sync(0xffffffffu, bad, off);
        }
        // times 2^(14 - exponent of the largest)
        const int e = min(max(int(__float_as_uint(largest) >> 23), 15), 254);
        const float up = __uint_as_float(uint32_t(268 - e) << 23), down = __uint_as_float(uint32_t(e - 14) << 23);
#pragma unroll
        for (int i = 0; i < S::kKeyWords; ++i) {
          qb[i][0] = q8_pack_half(__uint_as_float(v[i].x << 16) * up, __uint_as_float(v[i].x & 0xffff0000u) * up);
          qb[i][1] = q8_pack_half(__uint_as_float(v[i].y << 16) * up, __uint_as_float(v[i].y & 0xffff0000u) * up);
        }
        const float mine = (CAP ? p.cap_pre : p.scale_log2) * down + bad;
#pragma unroll
        for (int h = 0; h < 2; ++h) step[h] = __shfl_sync(0xffffffffu, mine, (2 * t4 + h) * 4);
      }
      const int* table = p.block_tables + size_t(w.seq) * p.max_blocks;
      // rounds of 128 keys; as many at a time as the table slice has pages for
      const int first = w.begin / kQ8DStep * kQ8DStep;
      const int rounds_at_once = max(1, (kQ8DTabMax - 1) * min(p.block_size, 65536) / kQ8DTile);
      for (int at = first; at < w.end; at += rounds_at_once * kQ8DTile) {
        const int stop = min(w.end, at + rounds_at_once * kQ8DTile);
        const int tab0 = max(at, w.begin) / p.block_size, pages = (stop - 1) / p.block_size - tab0 + 1;
        if (at != first) __syncthreads();                          // the slice before is read
        for (int j = tid; j < pages; j += kDecodeThreads)
          stab[j] = unsigned(min(max(table[tab0 + j], 0), p.num_pages - 1)) * unsigned(p.nkv) + unsigned(w.kvh);
        __syncthreads();

        // the warp's steps of keys: at + step (4 i + warp)
        const int steps = ((stop - at + kQ8DStep - 1) / kQ8DStep - warp + kQ8DWarps - 1) / kQ8DWarps;
        unsigned char* load_to = ring;
        int load_key = at + warp * kQ8DStep, loads = steps;
        auto load_step = [&]() {
          if (loads > 0) {
            unsigned char* const scales = load_to + 2 * S::kCodeBytes + lane * 4;
            const unsigned* const tab = stab - tab0;
            if (p.log2_block >= 0 && load_key >= w.begin && load_key + kQ8DStep <= w.end) {      // the usual step
              const int lb = p.log2_block, in_page = p.block_size - 1;
#pragma unroll
              for (int c = 0; c < S::kChunks * kQ8DStep / 32; ++c) {
                const int piece = c * 32 + lane, r = piece / S::kChunks, ch = piece - r * S::kChunks;
                const int key = load_key + r, to = S::at(r, ch);
                const unsigned u = tab[key >> lb] * head_units + unsigned((key & in_page) * S::kChunks + ch);
                cp_async16(load_to + to, p.k_codes + size_t(u) * 16);
                cp_async16(load_to + S::kCodeBytes + to, p.v_codes + size_t(u) * 16);
              }
              if (lane < kQ8DStep) {
                const unsigned page = tab[(load_key + lane) >> lb];
                q8_cp_async4(scales, p.k_scale + page);
                q8_cp_async4(scales + kQ8DStep * 4, p.v_scale + page);
              }
            } else {                                               // pages of any size, keys outside the piece of work
#pragma unroll 1
              for (int piece = lane; piece < kQ8DStep * S::kChunks; piece += 32) {
                const int r = piece / S::kChunks, ch = piece - r * S::kChunks, key = load_key + r, to = S::at(r, ch);
                if (key < w.begin || key >= w.end) {               // zeros, so that zero times them stays zero
                  *reinterpret_cast<uint4*>(load_to + S::kCodeBytes + to) = make_uint4(0u, 0u, 0u, 0u);
                  continue;
                }
                const int pi = key / p.block_size, off = key - pi * p.block_size;
                const size_t u = size_t(tab[pi] * head_units + unsigned(off * S::kChunks + ch)) * 16;
                cp_async16(load_to + to, p.k_codes + u);
                cp_async16(load_to + S::kCodeBytes + to, p.v_codes + u);
              }
              const int key = load_key + lane;
              if (lane < kQ8DStep && key >= w.begin && key < w.end) {
                const unsigned page = tab[key / p.block_size];
                q8_cp_async4(scales, p.k_scale + page);
                q8_cp_async4(scales + kQ8DStep * 4, p.v_scale + page);
              } else if (lane < kQ8DStep) {
                *reinterpret_cast<uint32_t*>(scales) = 0u;
                *reinterpret_cast<uint32_t*>(scales + kQ8DStep * 4) = 0u;
              }
            }
            --loads;
            load_key += kQ8DTile;
            load_to = load_to + S::kStageBytes == ring + STAGES * S::kStageBytes ? ring : load_to + S::kStageBytes;
          }
          cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) load_step();

        // scores of a step in log2 units: x[16 keys][key g, key g + 8][head 2 t4, 2 t4 + 1]
        auto scores = [&](const unsigned char* st, float (&x)[2][2][2]) {
          const float* scale = reinterpret_cast<const float*>(st + 2 * S::kCodeBytes);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            uint32_t ka[S::kKeyWords], kb[S::kKeyWords];
            const int ra = mt * 16 + row_g, rb = ra + 8;
            S::key_words(st, ra, t4, ka);
            S::key_words(st, rb, t4, kb);
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < S::kKeyWords; ++j)
              q8_mma(c, q8::halves2(ka[j] & 0xffffu), q8::halves2(kb[j] & 0xffffu), q8::halves2(ka[j] >> 16), q8::halves2(kb[j] >> 16), qb[j][0], qb[j][1]);
            const float sa = scale[ra], sb = scale[rb];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              x[mt][0][h] = c[h] * (sa * step[h]);                 // (large keys and small queries, or the reverse, meet first)
              x[mt][1][h] = c[2 + h] * (sb * step[h]);
              if constexpr (CAP) {
                x[mt][0][h] = fast_tanh(x[mt][0][h]) * p.scale_log2;
                x[mt][1][h] = fast_tanh(x[mt][1][h]) * p.scale_log2;
              }
            }
          }
        };
        // The scores of step i + 1 are formed while the softmax of step i, whose steps wait for one another, is under way.
        const unsigned char* st = ring;
        int key0 = at + warp * kQ8DStep;
        float x[2][2][2], ahead[2][2][2];
        if (steps > 0) {
          cp_async_wait<STAGES - 2>();
          __syncwarp();
          scores(st, ahead);
        }
        for (int i = 0; i < steps; ++i) {
          load_step();
          cp_async_wait<STAGES - 2>();
          __syncwarp();
          const float* v_scale = reinterpret_cast<const float*>(st + 2 * S::kCodeBytes) + kQ8DStep;
          const unsigned char* const next = st + S::kStageBytes == ring + STAGES * S::kStageBytes ? ring : st + S::kStageBytes;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h) x[mt][k][h] = ahead[mt][k][h];
          if (key0 < w.begin || key0 + kQ8DStep > w.end) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int key = key0 + mt * 16 + row_g + k * 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) x[mt][k][h] = key >= w.begin && key < w.end ? x[mt][k][h] : -INFINITY;
              }
          }
          scores(next, ahead);                                     // (behind the last step: of what lies there, and nobody reads it)
          // ---- running maximum
          float top[2];
          bool moved = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(fmaxf(x[0][0][h], x[0][1][h]), fmaxf(x[1][0][h], x[1][1][h]));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 4));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 8));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 16));
            moved |= top[h] > m[h];
          }
          auto rescale = [&](const float (&f)[2]) {
#pragma unroll
            for (int k = 0; k < S::kTiles; ++k) {
              o[k][0] *= f[0]; o[k][2] *= f[0];
              o[k][1] *= f[1]; o[k][3] *= f[1];
            }
          };
          if (__any_sync(0xffffffffu, moved)) {
            float grown[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float m_new = fmaxf(m[h], top[h]);
              grown[h] = fast_exp2(m[h] - m_new);                  // (zero where nothing was seen yet)
              m[h] = m_new;
              l[h] *= grown[h];
              // the weights so far have become `grown` of what they were, and so has the largest of them
              const uint32_t unit = q8_power_of_two(heaviest[h]);
              heaviest[h] = fmaxf(heaviest[h] * grown[h], kQ8DLeast);
              if (grown[h] > 0.f) grown[h] *= __uint_as_float(0x3f800000u + (unit - q8_power_of_two(heaviest[h])));     // (old unit / new unit)
            }
            rescale(grown);
          }
          // ---- weights p scale, and their unit
          float most_of[2] = {0.f, 0.f};
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const float sa = v_scale[mt * 16 + row_g], sb = v_scale[mt * 16 + row_g + 8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float ea = fast_exp2(x[mt][0][h] - m[h]), eb = fast_exp2(x[mt][1][h] - m[h]);
              l[h] += ea + eb;
              x[mt][0][h] = ea * sa;
              x[mt][1][h] = eb * sb;
              most_of[h] = fmaxf(most_of[h], fmaxf(x[mt][0][h], x[mt][1][h]));
            }
          }
          bool beyond = false;
#pragma unroll
          for (int h = 0; h < 2; ++h) beyond |= __float_as_uint(most_of[h]) >= q8_power_of_two(heaviest[h]) + kQ8DUnitRoom;
          if (__any_sync(0xffffffffu, beyond)) {
            float f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int off = 4; off <= 16; off *= 2) most_of[h] = fmaxf(most_of[h], __shfl_xor_sync(0xffffffffu, most_of[h], off));
              // (up to 2^126: its reciprocal is a normal number)
              const float now = fmaxf(heaviest[h], fminf(most_of[h], 1.f / kQ8DLeast));
              const uint32_t apart = q8_power_of_two(now) - q8_power_of_two(heaviest[h]);
              f[h] = __uint_as_float(0x3f800000u - min(apart, 0x3f800000u));                   // old unit / new unit; zero below 2^-126
              heaviest[h] = now;
            }
            rescale(f);
          }
          float per_unit[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) per_unit[h] = __uint_as_float(0x7f000000u - q8_power_of_two(heaviest[h]));
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint32_t b0 = q8_transposed(q8_pack_half(x[mt][0][0] * per_unit[0], x[mt][0][1] * per_unit[1]));
            const uint32_t b1 = q8_transposed(q8_pack_half(x[mt][1][0] * per_unit[0], x[mt][1][1] * per_unit[1]));
            // ---- values: keys 2 t4, 2 t4 + 1 and the same eight further
            const unsigned char* vt = st + S::kCodeBytes;
            const int r0 = mt * 16 + row_a, r1 = mt * 16 + row_b;
            uint32_t v[4][S::kWords];
            S::value_words(vt, r0, g, v[0]);
            S::value_words(vt, r1, g, v[1]);
            S::value_words(vt, r0 + 8, g, v[2]);
            S::value_words(vt, r1 + 8, g, v[3]);
#pragma unroll
            for (int j = 0; j < S::kWords; ++j) {
              // codes of two keys, element by element: elements 0 and 1 of the word, then 2 and 3
              const uint32_t a = __byte_perm(v[0][j], v[1][j], 0x5140), b = __byte_perm(v[2][j], v[3][j], 0x5140);
              q8_mma(o[2 * j], q8::halves2(a & 0xffffu), q8::halves2(a >> 16), q8::halves2(b & 0xffffu), q8::halves2(b >> 16), b0, b1);
              const uint32_t c = __byte_perm(v[0][j], v[1][j], 0x7362), d = __byte_perm(v[2][j], v[3][j], 0x7362);
              q8_mma(o[2 * j + 1], q8::halves2(c & 0xffffu), q8::halves2(c >> 16), q8::halves2(d & 0xffffu), q8::halves2(d >> 16), b0, b1);
            }
          }
          __syncwarp();                                            // the step's place is loaded again next round
          key0 += kQ8DTile;
          st = next;
        }
        cp_async_wait<0>();
      }
    }
    __syncthreads();                                               // the rings give way to the merge

    // ---- the warp's partial result: lanes over keys joined, units taken out
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int off = 4; off <= 16; off *= 2) l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
    const float unit[2] = {__uint_as_float(q8_power_of_two(heaviest[0])), __uint_as_float(q8_power_of_two(heaviest[1]))};
    float* row0 = mo + (warp * kDecodeHeads + 2 * t4) * HD;
    float* row1 = row0 + HD;
#pragma unroll
    for (int j = 0; j < S::kWords; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = S::value_element(g, j) + 2 * k;
        const float (&c)[4] = o[2 * j + k];
        *reinterpret_cast<float2*>(row0 + d) = make_float2(c[0] * unit[0], c[2] * unit[0]);
        *reinterpret_cast<float2*>(row1 + d) = make_float2(c[1] * unit[1], c[3] * unit[1]);
      }
    if (g == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mm[warp * kDecodeHeads + 2 * t4 + h] = m[h];
        ml[warp * kDecodeHeads + 2 * t4 + h] = l[h];
      }
    }
    __syncthreads();
    // ---- the four warps, four adjacent elements an item
    constexpr int Q = HD / 4;
    for (int it = tid; it < w.heads_here * Q; it += kDecodeThreads) {
      const int r = it / Q, d = (it - r * Q) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kQ8DWarps; ++k) top = fmaxf(top, mm[k * kDecodeHeads + r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kQ8DWarps; ++k) {
        const float lk = ml[k * kDecodeHeads + r];
        if (lk == 0.f) continue;                                   // a warp without keys
        const float f = fast_exp2(mm[k * kDecodeHeads + r] - top);
        const float4 v = *reinterpret_cast<const float4*>(mo + (k * kDecodeHeads + r) * HD + d);
        acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
        sum = fmaf(f, lk, sum);
      }
      const int head = w.head0 + r;
      if (p.cluster_merge) {
        *reinterpret_cast<float4*>(bo + r * HD + d) = acc;
        if (d == 0) { bm[r] = top; bl[r] = sum; }
      } else if (w.slot < 0) {
        if (p.sink && sum != 0.f) sum += fast_exp2(p.sink[head] * 1.4426950408889634f - top);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        bf16* dst = p.out + size_t(w.seq) * p.out_stride + size_t(head) * HD + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
      } else {
        const size_t at = shares ? size_t(w.slot) * kDecodeHeads + r : (size_t(w.seq) * p.nh + head) * p.num_parts + w.slot;
        *reinterpret_cast<float4*>(p.part_o + at * HD + d) = acc;
        if (d == 0) { p.part_ml[at * 2] = top; p.part_ml[at * 2 + 1] = sum; }
      }
    }
    if (!shares) {
      if (p.cluster_merge) decode_cluster_tail<HD>(p, w.seq, w.head0, w.heads_here, bo, bm, bl);
      return;
    }
    if (left <= 0) return;
    __syncthreads();                                               // the merge gives way to the rings
  }
}

// Steps in flight, and blocks an SM.
template <int HD> constexpr int q8_decode_stages() { return 3; }

template <int HD, bool CAP>
int launch_decode_q8(const DecodeQ8Params& p, int shares, cudaStream_t s) {
  constexpr int STAGES = q8_decode_stages<HD>();
  auto kernel = attn_decode_q8_kernel<HD, STAGES, CAP>;
  constexpr size_t smem = q8_decode_smem<HD, STAGES>();
  static OncePerDevice once;
  if (smem > 48 * 1024) {
    const int rc = allow_shared_memory(once, kernel, smem);
    if (rc != 0) return rc;
  }
  const int tiles = (p.nh / p.nkv + kDecodeHeads - 1) / kDecodeHeads;
  const dim3 grid = p.num_parts == 0 ? dim3(shares) : dim3(p.num_parts, p.nkv * tiles, p.seqs);
  if (p.cluster_merge) return pdl_launch_cluster(kernel, grid, dim3(kDecodeThreads), smem, s, p.num_parts, p);
  return pdl_launch(kernel, grid, dim3(kDecodeThreads), smem, s, p);
}

template <int HD> int q8_blocks_per_sm() {
  constexpr int STAGES = q8_decode_stages<HD>();
  auto kernel = attn_decode_q8_kernel<HD, STAGES, false>;
  constexpr size_t smem = q8_decode_smem<HD, STAGES>();
  int n = 0;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kDecodeThreads, smem) != cudaSuccess) return 0;
  return n;
}

#define KVCM_FOR_Q8_HEAD_DIMS(X) X(32) X(64) X(96) X(128) X(160) X(192) X(224) X(256)

}  // namespace
}  // namespace kvcm

using namespace kvcm;

// Blocks of the kernel that an SM of the current device holds at once (0: it cannot say).
KVCM_API int kvcm_attention_decode_q8_blocks_per_sm(int hd) {
#define X(N) if (hd == N) return q8_blocks_per_sm<N>();
  KVCM_FOR_Q8_HEAD_DIMS(X)
#undef X
  return 0;
}

// num_parts > 0: that many partitions of part_size keys (a multiple of 128) cover [first visible key rounded down, context).
// More than 8 of them, or cluster_merge == 0, want scratch: seqs * nh * num_parts * (hd + 2) floats.
// num_parts == 0: `shares` blocks take equal shares of all requests' and heads' tiles of 128 keys, and a second kernel joins what
// was cut; scratch: shares * 16 * (hd + 2) floats, then seqs * nh * 2 ints.
KVCM_API int kvcm_attention_decode_q8_bf16(const void* q, long long q_stride, void* out, long long out_stride, const void* k_codes,
                                           const void* v_codes, const float* k_scale, const float* v_scale, int num_pages,
                                           const int* block_tables, int max_blocks, const int* seq_ctx_len, int seqs, int nh, int nkv, int hd,
                                           int block_size, float scale, int window, int part_size, int num_parts, int shares, float* scratch,
                                           int cluster_merge, float softcap, const float* sink, void* stream) {
  if (seqs <= 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || block_size <= 0 || block_size > q8::kMaxBlock || max_blocks <= 0 || num_pages <= 0 || num_parts < 0 ||
      seqs > 65535 || nh > 65535 || hd < 32 || hd > 256 || hd % 32)
    return KVCM_ERR_UNSUPPORTED;
  if (num_parts > 0 ? (part_size <= 0 || part_size % kQ8DTile) : (shares <= 0 || shares > (1 << 20))) return KVCM_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(q) | uintptr_t(q_stride * 2) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15) ||
      ((reinterpret_cast<uintptr_t>(out) | uintptr_t(out_stride * 2)) & 7))
    return KVCM_ERR_UNSUPPORTED;
  // pages are found by 32-bit counts of 16 bytes
  if ((unsigned long long)block_size * (hd / 16) * (unsigned long long)num_pages * nkv > 0xffffffffull) return KVCM_ERR_UNSUPPORTED;
  if (num_parts == 0 || num_parts > kDecodeClusterParts || num_parts < 2) cluster_merge = 0;
  if (num_parts != 1 && !cluster_merge && (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 15))) return KVCM_ERR_UNSUPPORTED;
  const int head_tiles = (nh / nkv + kDecodeHeads - 1) / kDecodeHeads;
  const size_t pieces = num_parts == 0 ? size_t(shares) * 2 * kDecodeHeads : size_t(seqs) * nh * num_parts;
  DecodeQ8Params p;
  p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.out_stride = out_stride;
  p.k_codes = (const uint8_t*)k_codes; p.v_codes = (const uint8_t*)v_codes; p.k_scale = k_scale; p.v_scale = v_scale;
  p.num_pages = num_pages; p.block_tables = block_tables; p.max_blocks = max_blocks; p.seq_ctx_len = seq_ctx_len;
  p.max_keys = q8::max_keys(max_blocks, block_size);
  p.seqs = seqs;
  p.part_o = scratch; p.part_ml = scratch ? scratch + pieces * hd : nullptr;
  p.part_first = scratch ? reinterpret_cast<int*>(scratch + pieces * (hd + 2)) : nullptr;
  p.nh = nh; p.nkv = nkv; p.block_size = block_size; p.window = window;
  p.part_size = part_size; p.num_parts = num_parts; p.cluster_merge = cluster_merge;
  p.scale_log2 = (softcap > 0.f ? softcap : scale) * 1.4426950408889634f;
  p.cap_pre = softcap > 0.f ? scale / softcap : 0.f;
  p.sink = sink;
  p.log2_block = -1;
  for (int b = 0; b < 31; ++b) if ((1 << b) == block_size) p.log2_block = b;
  int rc = KVCM_ERR_UNSUPPORTED;
#define X(N) if (hd == N) rc = softcap > 0.f ? launch_decode_q8<N, true>(p, shares, (cudaStream_t)stream) : launch_decode_q8<N, false>(p, shares, (cudaStream_t)stream);
  KVCM_FOR_Q8_HEAD_DIMS(X)
#undef X
  if (rc != 0 || num_parts == 1 || cluster_merge) return rc;
  if (num_parts == 0)
    return pdl_launch(attn_decode_shares_kernel, dim3(seqs, nkv * head_tiles), dim3(128), 0, (cudaStream_t)stream, (const float*)p.part_o,
                      (const float*)p.part_ml, (const int*)p.part_first, seq_ctx_len, p.max_keys, window, p.out, out_stride, nh, nkv, hd, kDecodeHeads, sink);
  return pdl_launch(attn_decode_merge_kernel, dim3(seqs, nh), dim3(hd < 64 ? 32 : 64), 0, (cudaStream_t)stream, (const float*)p.part_o,
                    (const float*)p.part_ml, p.out, out_stride, nh, hd, num_parts, p.sink);
}

KVCM_PACKED(kvcm_attention_decode_q8_bf16)
