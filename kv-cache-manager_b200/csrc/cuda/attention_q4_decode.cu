// Decode attention over a paged cache in 4 bits (layout and formulas: q4.cuh): one query row a request, bfloat16 rows.
//
// One block per piece of work (keys of one request, KV head x 4 or 8 query heads), four warps; a warp takes every fourth step of 32
// keys and needs no other warp until the end.  The products are transposed, so that the query heads are the columns of the
// products and the rows are keys (S^T = K Q^T) and then elements of the head (O^T = V^T P^T): a group of few heads wastes little.
//   S^T  in whole numbers, m16n8k32: a lane's codes of a key are hd/4 elements in a row (any order of the contraction is as good as
//        another if q is read in the same one) and enter as they are, four to a register for one shift and two ands a word; q enters
//        as 16-bit fixed point relative to its head's largest element, in two 8-bit halves that are two columns: four heads to a
//        product.  Exact but for q's rounding, 2^-16 of its largest element: half a bfloat16 step of elements 2^-8 as large, less
//        of the larger ones.  (zero sum(q) takes q as it is.)   q.k = scale (q.code) + zero sum(q)  follows in float32.
//   O^T  in float16, m16n8k16: an element of two neighbouring keys is one register (the words of the two keys, half by half), as
//        code - 8 (exact), and  sum p x = sum (p scale)(code - 8) + sum p (zero + 8 scale).  p scale enters in units of the power of
//        two in the head's largest weight that the warp has seen, so a weight is rounded by 2^-11 of itself at most (the largest key's not
//        at all: it is its scale), and by 2^-25 of that unit where it is smaller than 2^-14 of it.
//        (Units of the largest scale alone, whatever its key's probability, let one large value without weight take the others' bits,
//        a unit for all heads of a warp one that has weight in one head only, one that forgets how large the largest weight was by now
//        one that scores climb away from slowly.  A unit of the largest weight itself, which O would not have to follow, rounds the
//        largest key's weight too: a fifth more results off by a bfloat16 step.)
//   P goes from accumulators to operands by a transposing register move (movmatrix): no shared memory in between.
// The scores of the next step are formed under the softmax of this one.  Pages come by 16-byte asynchronous copies into a ring of
// steps per warp: no barriers between warps, pages of any size.
//
// Pieces of work: partitions of every request (of the grid), of which up to 8 are the blocks of a cluster that merges through
// distributed shared memory, or equal shares of all requests' tiles of 128 keys, for batches of ragged or many requests: a share
// begins and ends inside a request, the two pieces go through scratch memory, and a second kernel joins them.
//
// What bounds it, B200: instructions.  A step of 32 keys x 128 elements x 4 heads costs a warp some 550, of which products are 24; an
// SM's four schedulers are 63 % busy (waits for the products' own results in between) and memory 5.0 TB/s: 64 requests of 8,192
// keys, 32 heads on 8 of 128 elements, 571 MB: 113 us (88 at the rate of a copy; up to 127 on a GPU that has been at it for seconds).  64
// requests of 100 to 8,192 keys (106 MB): 41.4 us, of which the shares' starts and the second kernel are about 11.  27 requests of up
// to 1,024 keys behind a window, capped: 11.4 us; 8 of 1,500 keys 8.0 us; one of 148 keys 4.8 us: launch, lengths, table, q and keys
// behind one another.  One of 32,768 keys 38 us (5.5 at the rate of a copy): equal shares cut it into some 70 pieces a head, which eight
// blocks join one after another.
#include "decode_join.cuh"
#include "packed.cuh"
#include "pdl.cuh"
#include "q4.cuh"

namespace kvcm {

constexpr int kQ4Warps = 4;
constexpr int kQ4DecodeThreads = kDecodeThreads;
static_assert(kQ4DecodeThreads == 32 * kQ4Warps, "four warps");
constexpr int kQ4Step = 32;                        // keys of a warp's step
constexpr int kQ4Tile = kQ4Step * kQ4Warps;        // keys of a round of the block
constexpr int kQ4Heads = kDecodeHeads;
constexpr int kQ4TabMax = 512;                     // page-table entries of a partition kept in shared memory
constexpr int kQ4ClusterParts = kDecodeClusterParts;
constexpr float kQ4Lowest = 3.402823466e38f;
constexpr float kQ4Least = 1.17549435e-38f;        // 2^-126
// What it costs to start on a request and head, in tiles of 128 keys, for the shares: its table, its q, an empty ring.  (0, 2, 4, 6 and
// 8, ragged requests up to 8,192 keys, heads of 128: 64 of them 54, 45, 43, 41 and 42 us; 100 shorter ones 64, 48, 46, 44 and 45;
// 16 of them 32, 30, 30, 29 and 27.)
constexpr int kQ4Start = 6;
// Exponents (of float32) by which a weight may be above its unit before the unit is formed anew: 2^12 is far from float16's end, and
// a unit that is too small costs no bits.  Without it eight heads' units were formed anew every other step.
constexpr uint32_t kQ4UnitRoom = 12u << 23;

struct DecodeQ4Params {
  const bf16* q; long long q_stride;
  bf16* out; long long out_stride;
  const uint8_t* k_cache; const uint8_t* v_cache;
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
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// Elements of a value as float16, two keys a register: codes at bits 0..3 of the halves give 1024 + code, those at bits 4..7
// 1024 + 16 code; less 1032 and 1152 they are code - 8 and 16 (code - 8), whole numbers and exact.
__device__ __forceinline__ uint32_t low_codes(uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;\n" : "=r"(r) : "r"(v));
  asm("sub.f16x2 %0, %0, %1;\n" : "+r"(r) : "r"(0x64086408u));
  return r;
}
__device__ __forceinline__ uint32_t high_codes(uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;\n" : "=r"(r) : "r"(v));
  asm("sub.f16x2 %0, %0, %1;\n" : "+r"(r) : "r"(0x64806480u));
  return r;
}
// The largest power of two in a positive number, as a float's bits.
__device__ __forceinline__ uint32_t power_of_two(float x) { return __float_as_uint(x) & 0x7f800000u; }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// D(16x8) += A(16x32 or 16x16, row) * B(.. x8, col): codes times 8-bit halves of q, float16 weights.  (Not volatile: the compiler may
// order them among the unpacking of other operands.)
__device__ __forceinline__ void mma_codes(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four 8-bit numbers as a register.
__device__ __forceinline__ uint32_t bytes4(int a, int b, int c, int d) {
  return uint32_t(a & 255) | (uint32_t(b & 255) << 8) | (uint32_t(c & 255) << 16) | (uint32_t(d) << 24);
}
__device__ __forceinline__ void mma_half(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int HD, int STAGES> constexpr size_t q4_decode_core_smem() {
  const size_t ring = size_t(kQ4Warps) * STAGES * Q4Shape<HD>::kStageBytes;
  const size_t merge = (size_t(kQ4Warps + 1) * kQ4Heads * HD + size_t(2 * kQ4Warps + 2) * kQ4Heads) * sizeof(float);
  return ring > merge ? ring : merge;
}
template <int HD, int STAGES> constexpr size_t q4_decode_smem() { return q4_decode_core_smem<HD, STAGES>() + kQ4TabMax * sizeof(int); }

// A block's piece of work: keys [begin, end) of one request for eight query heads of a KV head.
struct Q4Segment {
  int seq, kvh, head0, heads_here, begin, end;
  int slot;                            // >= 0: where the partial result goes; < 0: the result itself
};

// HG: heads come in groups of four, one or two.  A lane of a warp has the sums of heads t4 and (second group) t4 + 4.
template <int HD, int STAGES, bool CAP, int HG>
__global__ void __launch_bounds__(kQ4DecodeThreads, HD > 128 ? 2 : HG == 1 ? 4 : 3) attn_decode_q4_kernel(DecodeQ4Params p) {
  typedef Q4Shape<HD> S;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  unsigned* stab = reinterpret_cast<unsigned*>(smem_raw + q4_decode_core_smem<HD, STAGES>());     // pages of the head, in units of 16 bytes
  __shared__ int found[2];
  const int G = p.nh / p.nkv, head_tiles = (G + 4 * HG - 1) / (4 * HG);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  float* mo = reinterpret_cast<float*>(smem_raw);                  // after the key loop: [warps][8][HD]
  float* mm = mo + kQ4Warps * kQ4Heads * HD;                       // [warps][8] maximum
  float* ml = mm + kQ4Warps * kQ4Heads;                            // [warps][8] sum
  float* bo = ml + kQ4Warps * kQ4Heads;                            // [8][HD] the block's result
  float* bm = bo + kQ4Heads * HD;                                  // [8]
  float* bl = bm + kQ4Heads;                                       // [8]
  const bool shares = p.num_parts == 0;

  // Everything is read behind the wait: a caller may have written a whole prompt by the kernel before this one, and the lengths by
  // one of the same step (step_tables, or a sum of its own), which nothing else makes visible here.
  pdl_launch_dependents();
  pdl_wait();
  auto length = [&](int s) { return min(p.seq_ctx_len[s], p.max_keys); };     // (a context ends with its table)
  auto first_key = [&](int ctx) { return ctx > 0 ? first_visible(ctx - 1, p.window, 0) : 0; };
  // a request's cost for each head: its tiles of keys behind the start
  auto cost_of = [&](int ctx) { return ctx > 0 ? kQ4Start + (ctx - first_key(ctx) / kQ4Step * kQ4Step + kQ4Tile - 1) / kQ4Tile : 0; };
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
    const int per = (p.seqs + kQ4DecodeThreads - 1) / kQ4DecodeThreads;
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
    for (int w = 0; w < kQ4Warps; ++w) {
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

  const size_t head_bytes = q4::page_bytes(p.block_size, HD);
  const unsigned head_units = unsigned(head_bytes / 16);
  const int pairs_at = p.block_size * (HD / 2);
  const int row_g = S::row(g), row_a = S::row(2 * t4), row_b = S::row(2 * t4 + 1);
  unsigned char* const ring = smem_raw + size_t(warp) * STAGES * S::kStageBytes;

  for (;;) {
    // ---- the next piece of work
    Q4Segment w;
    const int ctx = length(seq), lo = first_key(ctx), base = lo / kQ4Step * kQ4Step;
    w.seq = seq;
    w.slot = -1;
    int of_h;
    bool empty;
    if (!shares) {
      of_h = blockIdx.y;
      const int from = base + int(blockIdx.x) * p.part_size;
      w.begin = max(lo, from);
      w.end = int(blockIdx.x) + 1 == p.num_parts ? ctx : min(ctx, from + p.part_size);     // (the last one takes what is left)
      if (p.num_parts > 1 && !p.cluster_merge) w.slot = blockIdx.x;
    } else {
      of_h = unit_h;
      const int n = cost_of(ctx), take = int(min((long long)(n - at_cost), left));
      const int tile0 = max(0, at_cost - kQ4Start), tile1 = max(0, at_cost + take - kQ4Start);
      w.begin = max(lo, base + tile0 * kQ4Tile);
      w.end = min(ctx, base + tile1 * kQ4Tile);
      empty = tile1 <= tile0;                                      // the start alone: the next block takes it
      if (tile0 > 0 || tile1 < n - kQ4Start) w.slot = 2 * int(blockIdx.x) + (tile0 == 0 ? 1 : 0);
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
            do ++seq; while (length(seq) <= 0);             // (there is more, so there is such a request)
        }
      }
      if (empty) {
        if (left <= 0) return;
        continue;
      }
    }
    w.kvh = of_h / head_tiles;
    const int ht = of_h - w.kvh * head_tiles;
    w.head0 = w.kvh * G + ht * 4 * HG;
    w.heads_here = min(4 * HG, G - ht * 4 * HG);

    // heads t4, t4 + 4; sums over this lane's keys (the maximum starts finite: no difference to it is not-a-number)
    float m[2] = {-kQ4Lowest, -kQ4Lowest}, l[2] = {0.f, 0.f}, zacc[2] = {0.f, 0.f};
    float o[S::kTiles][4];
#pragma unroll
    for (int i = 0; i < S::kTiles; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float heaviest[2] = {kQ4Least, kQ4Least};                      // weight of a head so far; the power of two in it is their unit
    if (w.begin < w.end) {
      // ---- q as the second operand: column g of group h is half g % 2 of head 4 h + g / 2, elements in the order in which a lane's
      // codes lie (of a word's eight, bytes 0, 4, 1, 5 and 2, 6, 3, 7)
      uint32_t qb[HG][S::kKeyWords][2];
      float step[HG], qs[HG];                                      // of heads t4 (+ 4): what q's whole numbers count, sum of q; times scale
#pragma unroll
      for (int h = 0; h < HG; ++h) {
        const int head = 4 * h + (g >> 1);
        const bf16* row = p.q + size_t(w.seq) * p.q_stride + size_t(w.head0 + head) * HD;
        uint4 v[S::kKeyWords];
        float sum = 0.f, largest = 0.f;
        int bad = 0;
#pragma unroll
        for (int i = 0; i < S::kKeyWords; ++i) {
          const int word = (S::kKeyWords % 4 == 0) ? (i / 4) * 16 + t4 * 4 + (i & 3) : t4 * S::kKeyWords + i;
          v[i] = make_uint4(0u, 0u, 0u, 0u);
          if (head < w.heads_here) v[i] = *reinterpret_cast<const uint4*>(row + word * 8);
          const uint32_t e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float lo16 = __uint_as_float(e[j] << 16), hi16 = __uint_as_float(e[j] & 0xffff0000u);
            sum += lo16 + hi16;
            largest = fmaxf(largest, fmaxf(fabsf(lo16), fabsf(hi16)));
            bad |= !(fabsf(lo16) <= kQ4Lowest) || !(fabsf(hi16) <= kQ4Lowest);
          }
        }
#pragma unroll
        for (int off = 1; off <= 2; off *= 2) {
          sum += __shfl_xor_sync(0xffffffffu, sum, off);
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, off));
          bad |= __shfl_xor_sync(0xffffffffu, bad, off);
        }
        // whole numbers up to 127 * 256 in size; halves of -128 .. 127
        const float unit_q = fmaxf(largest * (1.f / 32512.f), 1.17549435e-38f), per = 1.f / unit_q;
#pragma unroll
        for (int i = 0; i < S::kKeyWords; ++i) {
          const uint32_t e[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
          int n[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            n[2 * j] = __float2int_rn(__uint_as_float(e[j] << 16) * per);
            n[2 * j + 1] = __float2int_rn(__uint_as_float(e[j] & 0xffff0000u) * per);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int high = (n[j] + 128) >> 8;
            n[j] = (g & 1) ? n[j] - high * 256 : high;
          }
          qb[h][i][0] = bytes4(n[0], n[4], n[1], n[5]);
          qb[h][i][1] = bytes4(n[2], n[6], n[3], n[7]);
        }
        const float unit_of_scores = CAP ? 1.f : p.scale_log2;
        const float mine = bad ? __int_as_float(0x7fffffff) : unit_q;      // an element that is not finite: no score is
        step[h] = __shfl_sync(0xffffffffu, mine, t4 * 8) * unit_of_scores;
        qs[h] = __shfl_sync(0xffffffffu, sum, t4 * 8) * unit_of_scores;
      }
      const int* table = p.block_tables + size_t(w.seq) * p.max_blocks;
      // rounds of 128 keys; as many at a time as the table slice has pages for
      const int first = w.begin / kQ4Step * kQ4Step;
      const int rounds_at_once = max(1, (kQ4TabMax - 1) * p.block_size / kQ4Tile);
      for (int at = first; at < w.end; at += rounds_at_once * kQ4Tile) {
        const int stop = min(w.end, at + rounds_at_once * kQ4Tile);
        const int tab0 = max(at, w.begin) / p.block_size, pages = (stop - 1) / p.block_size - tab0 + 1;
        if (at != first) __syncthreads();                          // the slice before is read
        for (int j = tid; j < pages; j += kQ4DecodeThreads)
          stab[j] = (unsigned(min(max(table[tab0 + j], 0), p.num_pages - 1)) * unsigned(p.nkv) + unsigned(w.kvh)) * head_units;
        __syncthreads();

        // the warp's steps of 32 keys: at + 32 (4 i + warp)
        const int steps = ((stop - at + kQ4Step - 1) / kQ4Step - warp + kQ4Warps - 1) / kQ4Warps;
        unsigned char* load_to = ring;
        int load_key = at + warp * kQ4Step, loads = steps;
        auto load_step = [&]() {
          if (loads > 0) {
            unsigned char* const pairs = load_to + 2 * S::kCodeBytes + lane * 4;
            const unsigned* const tab = stab - tab0;
            if (p.log2_block >= 0 && load_key >= w.begin && load_key + kQ4Step <= w.end) {      // the usual step
              const int lb = p.log2_block, in_page = p.block_size - 1;
#pragma unroll
              for (int c = 0; c < S::kChunks; ++c) {
                const int piece = c * 32 + lane, r = piece / S::kChunks, ch = piece - r * S::kChunks;
                const int key = load_key + r, to = S::at(r, ch);
                const unsigned u = tab[key >> lb] + unsigned((key & in_page) * S::kChunks + ch);
                cp_async16(load_to + to, p.k_cache + size_t(u) * 16);
                cp_async16(load_to + S::kCodeBytes + to, p.v_cache + size_t(u) * 16);
              }
              const int key = load_key + lane;
              const size_t u = size_t(tab[key >> lb]) * 16 + unsigned(pairs_at + (key & in_page) * 4);
              cp_async4(pairs, p.k_cache + u);
              cp_async4(pairs + kQ4Step * 4, p.v_cache + u);
            } else {                                               // pages of any size, keys outside the piece of work
#pragma unroll 1
              for (int piece = lane; piece < kQ4Step * S::kChunks; piece += 32) {
                const int r = piece / S::kChunks, ch = piece - r * S::kChunks, key = load_key + r;
                if (key < w.begin || key >= w.end) continue;
                const int pi = key / p.block_size, off = key - pi * p.block_size;
                const size_t u = size_t(tab[pi] + unsigned(off * S::kChunks + ch)) * 16;
                const int to = S::at(r, ch);
                cp_async16(load_to + to, p.k_cache + u);
                cp_async16(load_to + S::kCodeBytes + to, p.v_cache + u);
              }
              const int key = load_key + lane;
              if (key >= w.begin && key < w.end) {
                const int pi = key / p.block_size, off = key - pi * p.block_size;
                const size_t u = size_t(tab[pi]) * 16 + unsigned(pairs_at + off * 4);
                cp_async4(pairs, p.k_cache + u);
                cp_async4(pairs + kQ4Step * 4, p.v_cache + u);
              } else {                                             // zero, so that zero times it stays zero (codes are finite whatever they are)
                *reinterpret_cast<uint32_t*>(pairs) = 0u;
                *reinterpret_cast<uint32_t*>(pairs + kQ4Step * 4) = 0u;
              }
            }
            --loads;
            load_key += kQ4Tile;
            load_to = load_to + S::kStageBytes == ring + STAGES * S::kStageBytes ? ring : load_to + S::kStageBytes;
          }
          cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) load_step();

        // scores of a step in log2 units: x[16 keys][key g, key g + 8][head t4, t4 + 4]
        auto scores = [&](const unsigned char* st, float (&x)[2][2][HG]) {
          const uint32_t* kpair = reinterpret_cast<const uint32_t*>(st + 2 * S::kCodeBytes);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            uint32_t ka[S::kKeyWords], kb[S::kKeyWords];
            const int ra = mt * 16 + row_g, rb = ra + 8;
            if constexpr (S::kKeyWords % 4 == 0) {
#pragma unroll
              for (int j = 0; j < S::kKeyWords / 4; ++j) {
                const uint4 a = *reinterpret_cast<const uint4*>(st + S::at(ra, j * 4 + t4));
                const uint4 b = *reinterpret_cast<const uint4*>(st + S::at(rb, j * 4 + t4));
                ka[4 * j] = a.x; ka[4 * j + 1] = a.y; ka[4 * j + 2] = a.z; ka[4 * j + 3] = a.w;
                kb[4 * j] = b.x; kb[4 * j + 1] = b.y; kb[4 * j + 2] = b.z; kb[4 * j + 3] = b.w;
              }
            } else if constexpr (HD == 64) {
              const uint2 a = *reinterpret_cast<const uint2*>(st + S::at(ra, t4 >> 1) + (t4 & 1) * 8);
              const uint2 b = *reinterpret_cast<const uint2*>(st + S::at(rb, t4 >> 1) + (t4 & 1) * 8);
              ka[0] = a.x; ka[1] = a.y; kb[0] = b.x; kb[1] = b.y;
            } else {
#pragma unroll
              for (int j = 0; j < S::kKeyWords; ++j) {
                ka[j] = *reinterpret_cast<const uint32_t*>(st + S::at(ra, 0) + (t4 * S::kKeyWords + j) * 4);
                kb[j] = *reinterpret_cast<const uint32_t*>(st + S::at(rb, 0) + (t4 * S::kKeyWords + j) * 4);
              }
            }
            // sums start at 1.5 * 2^23 as a float's bits: a float again without a conversion (they stay below 2^22)
            int c[HG][4];
#pragma unroll
            for (int h = 0; h < HG; ++h) c[h][0] = c[h][1] = c[h][2] = c[h][3] = 0x4b400000;
#pragma unroll
            for (int j = 0; j < S::kKeyWords; ++j) {
              const uint32_t a0 = ka[j] & 0x0f0f0f0fu, a1 = kb[j] & 0x0f0f0f0fu, a2 = (ka[j] >> 4) & 0x0f0f0f0fu, a3 = (kb[j] >> 4) & 0x0f0f0f0fu;
#pragma unroll
              for (int h = 0; h < HG; ++h) mma_codes(c[h], a0, a1, a2, a3, qb[h][j][0], qb[h][j][1]);
            }
            const uint32_t pa = kpair[ra], pb = kpair[rb];
            const float sa = q4::scale_of(pa), sb = q4::scale_of(pb), za = q4::zero_of(pa), zb = q4::zero_of(pb);
#pragma unroll
            for (int h = 0; h < HG; ++h) {
              const float na = fmaf(256.f, __int_as_float(c[h][0]) - 12582912.f, __int_as_float(c[h][1]) - 12582912.f);
              const float nb = fmaf(256.f, __int_as_float(c[h][2]) - 12582912.f, __int_as_float(c[h][3]) - 12582912.f);
              x[mt][0][h] = fmaf(sa * step[h], na, za * qs[h]);      // (large keys and small queries, or the reverse, meet first)
              x[mt][1][h] = fmaf(sb * step[h], nb, zb * qs[h]);
              if constexpr (CAP) {
                x[mt][0][h] = fast_tanh(x[mt][0][h] * p.cap_pre) * p.scale_log2;
                x[mt][1][h] = fast_tanh(x[mt][1][h] * p.cap_pre) * p.scale_log2;
              }
            }
          }
        };
        // The scores of step i + 1 are formed while the softmax of step i, whose steps wait for one another, is under way.
        const unsigned char* st = ring;
        int key0 = at + warp * kQ4Step;
        float x[2][2][HG], ahead[2][2][HG];
        if (steps > 0) {
          cp_async_wait<STAGES - 2>();
          __syncwarp();
          scores(st, ahead);
        }
        for (int i = 0; i < steps; ++i) {
          load_step();
          cp_async_wait<STAGES - 2>();
          __syncwarp();
          const uint32_t* vpair = reinterpret_cast<const uint32_t*>(st + 2 * S::kCodeBytes) + kQ4Step;
          const unsigned char* const next = st + S::kStageBytes == ring + STAGES * S::kStageBytes ? ring : st + S::kStageBytes;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int h = 0; h < HG; ++h) x[mt][k][h] = ahead[mt][k][h];
          if (key0 < w.begin || key0 + kQ4Step > w.end) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int key = key0 + mt * 16 + row_g + k * 8;
#pragma unroll
                for (int h = 0; h < HG; ++h) x[mt][k][h] = key >= w.begin && key < w.end ? x[mt][k][h] : -INFINITY;
              }
          }
          scores(next, ahead);                                     // (behind the last step: of what lies there, and nobody reads it)
          // ---- running maximum
          float top[HG];
          bool moved = false;
#pragma unroll
          for (int h = 0; h < HG; ++h) {
            top[h] = fmaxf(fmaxf(x[0][0][h], x[0][1][h]), fmaxf(x[1][0][h], x[1][1][h]));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 4));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 8));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 16));
            moved |= top[h] > m[h];
          }
          auto rescale = [&](const float (&f)[HG]) {
#pragma unroll
            for (int k = 0; k < S::kTiles; ++k) {
              o[k][0] *= f[0]; o[k][2] *= f[0];
              if constexpr (HG == 2) { o[k][1] *= f[1]; o[k][3] *= f[1]; }
            }
          };
          if (__any_sync(0xffffffffu, moved)) {
            float grown[HG];
#pragma unroll
            for (int h = 0; h < HG; ++h) {
              const float m_new = fmaxf(m[h], top[h]);
              grown[h] = fast_exp2(m[h] - m_new);                  // (zero where nothing was seen yet)
              m[h] = m_new;
              l[h] *= grown[h];
              zacc[h] *= grown[h];
              // the weights so far have become `grown` of what they were, and so has the largest of them
              const uint32_t unit = power_of_two(heaviest[h]);
              heaviest[h] = fmaxf(heaviest[h] * grown[h], kQ4Least);
              if (grown[h] > 0.f) grown[h] *= __uint_as_float(0x3f800000u + (unit - power_of_two(heaviest[h])));     // (old unit / new unit)
            }
            rescale(grown);
          }
          // ---- weights p scale, and their unit
          float most_of[HG];
#pragma unroll
          for (int h = 0; h < HG; ++h) most_of[h] = 0.f;
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint32_t pa = vpair[mt * 16 + row_g], pb = vpair[mt * 16 + row_g + 8];
            const float sa = q4::scale_of(pa), za = fmaf(8.f, sa, q4::zero_of(pa));
            const float sb = q4::scale_of(pb), zb = fmaf(8.f, sb, q4::zero_of(pb));
#pragma unroll
            for (int h = 0; h < HG; ++h) {
              const float ea = fast_exp2(x[mt][0][h] - m[h]), eb = fast_exp2(x[mt][1][h] - m[h]);
              l[h] += ea + eb;
              zacc[h] = fmaf(ea, za, fmaf(eb, zb, zacc[h]));
              x[mt][0][h] = ea * sa;
              x[mt][1][h] = eb * sb;
              most_of[h] = fmaxf(most_of[h], fmaxf(x[mt][0][h], x[mt][1][h]));
            }
          }
          bool beyond = false;
#pragma unroll
          for (int h = 0; h < HG; ++h) beyond |= __float_as_uint(most_of[h]) >= power_of_two(heaviest[h]) + kQ4UnitRoom;
          if (__any_sync(0xffffffffu, beyond)) {
            float f[HG];
#pragma unroll
            for (int h = 0; h < HG; ++h) {
#pragma unroll
              for (int off = 4; off <= 16; off *= 2) most_of[h] = fmaxf(most_of[h], __shfl_xor_sync(0xffffffffu, most_of[h], off));
              // (up to 2^126: its reciprocal is a normal number)
              const float now = fmaxf(heaviest[h], fminf(most_of[h], 1.f / kQ4Least));
              const uint32_t apart = power_of_two(now) - power_of_two(heaviest[h]);
              f[h] = __uint_as_float(0x3f800000u - min(apart, 0x3f800000u));                   // old unit / new unit; zero below 2^-126
              heaviest[h] = now;
            }
            rescale(f);
          }
          float per_unit[HG];
#pragma unroll
          for (int h = 0; h < HG; ++h) per_unit[h] = __uint_as_float(0x7f000000u - power_of_two(heaviest[h]));
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            float wa[2] = {0.f, 0.f}, wb[2] = {0.f, 0.f};
#pragma unroll
            for (int h = 0; h < HG; ++h) {
              wa[h] = x[mt][0][h] * per_unit[h];
              wb[h] = x[mt][1][h] * per_unit[h];
            }
            // columns of O: 2 t4 is head t4, 2 t4 + 1 head t4 + 4 (of one group: nobody)
            const uint32_t b0 = transposed(pack_half(wa[0], wa[1])), b1 = transposed(pack_half(wb[0], wb[1]));
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
                for (int j = 0; j < S::kFull; ++j) v[k][j] = *reinterpret_cast<const uint32_t*>(vt + S::at(r, 0) + (g * S::kFull + j) * 4);
              }
            }
#pragma unroll
            for (int j = 0; j < S::kFull; ++j) {
              uint32_t ea = __byte_perm(v[0][j], v[1][j], 0x5410), oa = __byte_perm(v[0][j], v[1][j], 0x7632);    // even, odd elements
              uint32_t eb = __byte_perm(v[2][j], v[3][j], 0x5410), ob = __byte_perm(v[2][j], v[3][j], 0x7632);
#pragma unroll
              for (int k = 0; k < 4; k += 2) {
                const uint32_t a[4] = {low_codes(ea), low_codes(oa), low_codes(eb), low_codes(ob)};
                mma_half(o[4 * j + k], a, b0, b1);
                const uint32_t c[4] = {high_codes(ea), high_codes(oa), high_codes(eb), high_codes(ob)};
                mma_half(o[4 * j + k + 1], c, b0, b1);
                ea >>= 8; oa >>= 8; eb >>= 8; ob >>= 8;
              }
            }
            if constexpr (S::kHalf) {                              // the last four words: lane groups 2w and 2w + 1 take the halves of word w
              uint32_t u[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                u[k] = *reinterpret_cast<const uint32_t*>(vt + S::at(((k & 1) ? r1 : r0) + (k >> 1) * 8, 0) + (8 * S::kFull + (g >> 1)) * 4);
              const uint32_t pick = (g & 1) ? 0x7632 : 0x5410;
              uint32_t a_ = __byte_perm(u[0], u[1], pick), b_ = __byte_perm(u[2], u[3], pick);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const uint32_t a[4] = {low_codes(a_), high_codes(a_), low_codes(b_), high_codes(b_)};
                mma_half(o[4 * S::kFull + k], a, b0, b1);
                a_ >>= 8; b_ >>= 8;
              }
            }
          }
          __syncwarp();                                            // the step's place is loaded again next round
          key0 += kQ4Tile;
          st = next;
        }
        cp_async_wait<0>();
      }
    }
    __syncthreads();                                               // the rings give way to the merge

    // ---- the warp's partial result: lanes over keys joined, units taken out, the zeros' part added to every element
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int off = 4; off <= 16; off *= 2) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], off);
        zacc[h] += __shfl_xor_sync(0xffffffffu, zacc[h], off);
      }
    const float f_low[2] = {__uint_as_float(power_of_two(heaviest[0])), __uint_as_float(power_of_two(heaviest[1]))}, f_high[2] = {f_low[0] * 0.0625f, f_low[1] * 0.0625f};
    float* row0 = mo + (warp * kQ4Heads + t4) * HD;
    float* row1 = row0 + 4 * HD;
#pragma unroll
    for (int j = 0; j < S::kFull; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int d = 8 * (g * S::kFull + j) + 2 * k;
        const float (&f)[2] = (k & 1) ? f_high : f_low;
        const float (&c)[4] = o[4 * j + k];
        *reinterpret_cast<float2*>(row0 + d) = make_float2(fmaf(c[0], f[0], zacc[0]), fmaf(c[2], f[0], zacc[0]));
        if constexpr (HG == 2) *reinterpret_cast<float2*>(row1 + d) = make_float2(fmaf(c[1], f[1], zacc[1]), fmaf(c[3], f[1], zacc[1]));
      }
    if constexpr (S::kHalf) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = 8 * (8 * S::kFull + (g >> 1)) + 4 * k + (g & 1);
        const float (&c)[4] = o[4 * S::kFull + k];
        row0[d] = fmaf(c[0], f_low[0], zacc[0]); row0[d + 2] = fmaf(c[2], f_high[0], zacc[0]);
        if constexpr (HG == 2) { row1[d] = fmaf(c[1], f_low[1], zacc[1]); row1[d + 2] = fmaf(c[3], f_high[1], zacc[1]); }
      }
    }
    if (g == 0) {
      mm[warp * kQ4Heads + t4] = m[0]; mm[warp * kQ4Heads + t4 + 4] = m[1];
      ml[warp * kQ4Heads + t4] = l[0]; ml[warp * kQ4Heads + t4 + 4] = l[1];
    }
    __syncthreads();
    // ---- the four warps, four adjacent elements an item
    constexpr int Q = HD / 4;
    for (int it = tid; it < w.heads_here * Q; it += kQ4DecodeThreads) {
      const int r = it / Q, d = (it - r * Q) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kQ4Warps; ++k) top = fmaxf(top, mm[k * kQ4Heads + r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < kQ4Warps; ++k) {
        const float lk = ml[k * kQ4Heads + r];
        if (lk == 0.f) continue;                                   // a warp without keys
        const float f = fast_exp2(mm[k * kQ4Heads + r] - top);
        const float4 v = *reinterpret_cast<const float4*>(mo + (k * kQ4Heads + r) * HD + d);
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
        const size_t at = shares ? size_t(w.slot) * kQ4Heads + r : (size_t(w.seq) * p.nh + head) * p.num_parts + w.slot;
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

// Steps in flight.  Four blocks of three an SM for one group of heads at 128 registers a thread; two groups want 168, and then
// three blocks of four steps.  (The other way round: 64 requests of 8,192 keys, 8 KV heads of 128, 113.6 us and not 113.2, ragged 42.4
// and not 41.4, behind a window 10.5 and not 11.4; eight query heads on each of 4 KV heads of 64, 8 requests of 1,536 keys 8.6 us and not
// 8.0, but 64 of some 2,048 30 and not 33.)
template <int HD, int HG> constexpr int q4_decode_stages() { return HD > 128 || HG == 1 ? 3 : 4; }

// Query heads of a block: four where a KV head has no more, else eight.
inline int q4_tile_heads(int nh, int nkv) { return nh / nkv <= 4 ? 4 : 8; }

template <int HD, bool CAP, int HG>
int launch_decode_q4_as(const DecodeQ4Params& p, int shares, cudaStream_t s) {
  constexpr int STAGES = q4_decode_stages<HD, HG>();
  auto kernel = attn_decode_q4_kernel<HD, STAGES, CAP, HG>;
  constexpr size_t smem = q4_decode_smem<HD, STAGES>();
  static OncePerDevice once;
  if (smem > 48 * 1024) {
    const int rc = allow_shared_memory(once, kernel, smem);
    if (rc != 0) return rc;
  }
  const int tiles = (p.nh / p.nkv + 4 * HG - 1) / (4 * HG);
  const dim3 grid = p.num_parts == 0 ? dim3(shares) : dim3(p.num_parts, p.nkv * tiles, p.seqs);
  if (p.cluster_merge) return pdl_launch_cluster(kernel, grid, dim3(kQ4DecodeThreads), smem, s, p.num_parts, p);
  return pdl_launch(kernel, grid, dim3(kQ4DecodeThreads), smem, s, p);
}
template <int HD, bool CAP>
int launch_decode_q4(const DecodeQ4Params& p, int shares, cudaStream_t s) {
  return q4_tile_heads(p.nh, p.nkv) == 4 ? launch_decode_q4_as<HD, CAP, 1>(p, shares, s) : launch_decode_q4_as<HD, CAP, 2>(p, shares, s);
}

template <int HD, int HG> int q4_blocks_per_sm_of() {
  constexpr int STAGES = q4_decode_stages<HD, HG>();
  auto kernel = attn_decode_q4_kernel<HD, STAGES, false, HG>;
  constexpr size_t smem = q4_decode_smem<HD, STAGES>();
  int n = 0;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kQ4DecodeThreads, smem) != cudaSuccess) return 0;
  return n;
}
template <int HD> int q4_blocks_per_sm(int groups) { return groups == 1 ? q4_blocks_per_sm_of<HD, 1>() : q4_blocks_per_sm_of<HD, 2>(); }

#define KVCM_FOR_Q4_HEAD_DIMS(X) X(32) X(64) X(96) X(128) X(160) X(192) X(224) X(256)

}  // namespace kvcm

using namespace kvcm;

// 1 if the tensor-core kernels take this head size.
KVCM_API int kvcm_attention_q4_decode_supports(int hd) { return hd > 0 && hd <= 256 && hd % 32 == 0; }

// Blocks of the kernel that an SM of the current device holds at once (0: it cannot say), for heads in one or two groups of four.
KVCM_API int kvcm_attention_decode_q4_blocks_per_sm(int hd, int groups) {
#define X(N) if (hd == N) return q4_blocks_per_sm<N>(groups);
  KVCM_FOR_Q4_HEAD_DIMS(X)
#undef X
  return 0;
}

// num_parts > 0: that many partitions of part_size keys (a multiple of 128) cover [first visible key rounded down to 32, context).
// More than 8 of them, or cluster_merge == 0, want scratch: seqs * nh * num_parts * (hd + 2) floats.
// num_parts == 0: `shares` blocks take equal shares of all requests' and heads' tiles of 128 keys, and a second kernel joins what
// was cut; scratch: shares * 16 * (hd + 2) floats, then seqs * nh * 2 ints.
KVCM_API int kvcm_attention_decode_q4_bf16(const void* q, long long q_stride, void* out, long long out_stride, const void* k_cache,
                                           const void* v_cache, int num_pages, const int* block_tables, int max_blocks,
                                           const int* seq_ctx_len, int seqs, int nh, int nkv, int hd, int block_size, float scale,
                                           int window, int part_size, int num_parts, int shares, float* scratch, int cluster_merge,
                                           float softcap, const float* sink, void* stream) {
  if (seqs == 0) return 0;
  if (nkv <= 0 || nh <= 0 || nh % nkv || block_size <= 0 || block_size > q4::kMaxBlock || max_blocks <= 0 || num_pages <= 0 || num_parts < 0 || seqs > 65535 || nh > 65535 ||
      !kvcm_attention_q4_decode_supports(hd))
    return KVCM_ERR_UNSUPPORTED;
  if (num_parts > 0 ? (part_size <= 0 || part_size % kQ4Tile) : (shares <= 0 || shares > (1 << 20))) return KVCM_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(q) | uintptr_t(q_stride * 2) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) ||
      ((reinterpret_cast<uintptr_t>(out) | uintptr_t(out_stride * 2)) & 7))
    return KVCM_ERR_UNSUPPORTED;
  // pages are found by 32-bit counts of 16 bytes
  if (q4::page_bytes(block_size, hd) / 16 * (unsigned long long)num_pages * nkv > 0xffffffffull) return KVCM_ERR_UNSUPPORTED;
  if (num_parts == 0 || num_parts > kQ4ClusterParts || num_parts < 2) cluster_merge = 0;
  if (num_parts != 1 && !cluster_merge && (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 15))) return KVCM_ERR_UNSUPPORTED;
  const int tile_heads = q4_tile_heads(nh, nkv), head_tiles = (nh / nkv + tile_heads - 1) / tile_heads;
  const size_t pieces = num_parts == 0 ? size_t(shares) * 2 * kQ4Heads : size_t(seqs) * nh * num_parts;
  DecodeQ4Params p;
  p.q = (const bf16*)q; p.q_stride = q_stride; p.out = (bf16*)out; p.out_stride = out_stride;
  p.k_cache = (const uint8_t*)k_cache; p.v_cache = (const uint8_t*)v_cache; p.num_pages = num_pages;
  p.block_tables = block_tables; p.max_blocks = max_blocks; p.seq_ctx_len = seq_ctx_len;
  p.max_keys = q4::max_keys(max_blocks, block_size);
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
#define X(N) if (hd == N) rc = softcap > 0.f ? launch_decode_q4<N, true>(p, shares, (cudaStream_t)stream) : launch_decode_q4<N, false>(p, shares, (cudaStream_t)stream);
  KVCM_FOR_Q4_HEAD_DIMS(X)
#undef X
  if (rc != 0 || num_parts == 1 || cluster_merge) return rc;
  if (num_parts == 0)
    return pdl_launch(attn_decode_shares_kernel, dim3(seqs, nkv * head_tiles), dim3(128), 0, (cudaStream_t)stream, (const float*)p.part_o,
                      (const float*)p.part_ml, (const int*)p.part_first, seq_ctx_len, 0x7fffffff, 0, p.out, out_stride, nh, nkv, hd, tile_heads,
                      sink);
  return pdl_launch(attn_decode_merge_kernel, dim3(seqs, nh), dim3(hd < 64 ? 32 : 64), 0, (cudaStream_t)stream, (const float*)p.part_o,
                    (const float*)p.part_ml, p.out, out_stride, nh, hd, num_parts, p.sink);
}

KVCM_PACKED(kvcm_attention_decode_q4_bf16)
