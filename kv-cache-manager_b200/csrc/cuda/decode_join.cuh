// What becomes of the pieces of single rows' attention over a quantised cache (attention_q4_decode.cu, attention_q8_decode.cu): partitions joined
// inside a cluster, partitions or shares joined out of scratch memory by a second kernel.  A piece is the unnormalised sum over its
// keys, their maximum (log2 units) and the sum of their weights, for up to eight query heads of a KV head.
#pragma once
#include <cooperative_groups.h>

#include "attention_mma.cuh"
#include "pdl.cuh"

namespace kvcm {

constexpr int kDecodeThreads = 128;
constexpr int kDecodeHeads = 8;                    // most query heads of a block
constexpr int kDecodeClusterParts = 8;

// The partitions of a cluster: every block has its partial result in its own shared memory (bo [8][HD], bm maximum, bl sum; an
// empty partition has bl = 0, a bm below every score, and no bo that is read).  The outputs are dealt out over the blocks, four adjacent elements an item; each adds
// the partitions up in their order.
template <int HD, typename Params>
__device__ __forceinline__ void decode_cluster_tail(const Params& p, int seq, int head0, int heads_here, float* bo, float* bm, float* bl) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int P = p.num_parts;
  constexpr int Q = HD / 4;
  for (int it = int(cluster.block_rank()) * kDecodeThreads + threadIdx.x; it < heads_here * Q; it += P * kDecodeThreads) {
    const int r = it / Q, d = (it - r * Q) * 4;
    float m[kDecodeClusterParts], l[kDecodeClusterParts], top = -INFINITY;
    float4 o[kDecodeClusterParts];
#pragma unroll
    for (int i = 0; i < kDecodeClusterParts; ++i) {
      m[i] = -INFINITY; l[i] = 0.f; o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < P) {
        m[i] = *cluster.map_shared_rank(bm + r, i);
        l[i] = *cluster.map_shared_rank(bl + r, i);
        o[i] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(bo + r * HD + d, i));
      }
    }
#pragma unroll
    for (int i = 0; i < kDecodeClusterParts; ++i) top = fmaxf(top, m[i]);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kDecodeClusterParts; ++i) {
      if (l[i] == 0.f) continue;                                   // nothing there
      const float f = fast_exp2(m[i] - top);
      acc.x = fmaf(f, o[i].x, acc.x); acc.y = fmaf(f, o[i].y, acc.y); acc.z = fmaf(f, o[i].z, acc.z); acc.w = fmaf(f, o[i].w, acc.w);
      sum = fmaf(f, l[i], sum);
    }
    if (p.sink && sum != 0.f) sum += fast_exp2(p.sink[head0 + r] * 1.4426950408889634f - top);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    bf16* dst = p.out + size_t(seq) * p.out_stride + size_t(head0 + r) * HD + d;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
  cluster.sync();                                                  // nobody leaves while its memory is read
}

// More partitions than a cluster merges, out of scratch memory, in their order.
static __global__ void attn_decode_merge_kernel(const float* part_o, const float* part_ml, bf16* __restrict__ out, long long out_stride, int nh,
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
    if (sink && sum != 0.f) sum += exp2f(sink[head] * 1.4426950408889634f - top);
    out[size_t(seq) * out_stride + size_t(head) * hd + d] = __float2bfloat16_rn(sum == 0.f ? 0.f : acc / sum);
  }
}

// The pieces of a request and its four or eight heads that blocks part_first[0] .. part_first[1] have left, in their order: the first
// block's lies in its second place, the others' in their first.  A row whose window begins at `max_keys` or behind it has none.  Up to six are asked for at once, maxima, sums and outputs in one trip
// to memory (64 ragged requests in all 1.3 us less).  A long request has many: the weights of 128 of them at a time are formed
// side by side, so that what follows one another is additions.
constexpr int kDecodeJoinAtOnce = 128;
constexpr int kDecodeJoinFew = 6;
static __global__ void __launch_bounds__(128) attn_decode_shares_kernel(const float* part_o, const float* part_ml, const int* part_first,
                                                                    const int* __restrict__ seq_ctx_len, int max_keys, int window,
                                                                    bf16* __restrict__ out,
                                                                    long long out_stride, int nh, int nkv, int hd, int tile_heads,
                                                                    const float* __restrict__ sink) {
  __shared__ float weight[kDecodeJoinAtOnce][kDecodeHeads];
  __shared__ float tops[4][kDecodeHeads], all_top[kDecodeHeads], all_sum[kDecodeHeads];
  pdl_launch_dependents();
  pdl_wait();
  const int G = nh / nkv, head_tiles = (G + tile_heads - 1) / tile_heads, H = nkv * head_tiles;
  const int seq = blockIdx.x, h = blockIdx.y, kvh = h / head_tiles, ht = h - kvh * head_tiles;
  const int head0 = kvh * G + ht * tile_heads, heads_here = min(tile_heads, G - ht * tile_heads);
  const int tid = threadIdx.x, quads = hd / 4, items = heads_here * quads;
  const int ctx = seq_ctx_len[seq];
  if (ctx <= 0 || max_keys <= first_visible(ctx - 1, window, 0)) {        // no key
    for (int it = tid; it < items; it += 128) {
      const int r = it / quads, d = (it - r * quads) * 4;
      *reinterpret_cast<uint2*>(out + size_t(seq) * out_stride + size_t(head0 + r) * hd + d) = make_uint2(0u, 0u);
    }
    return;
  }
  const int first = part_first[(seq * H + h) * 2], pieces = part_first[(seq * H + h) * 2 + 1] - first + 1;
  if (pieces == 1) return;                                         // one block had it all
  auto at = [&](int i, int r) { return size_t(2 * (first + i) + (i == 0)) * kDecodeHeads + r; };
  if (pieces <= kDecodeJoinFew) {                                      // the usual request: all of them asked for at once
    for (int it = tid; it < items; it += 128) {
      const int r = it / quads, d = (it - r * quads) * 4;
      float2 ml[kDecodeJoinFew];
      float4 v[kDecodeJoinFew];
#pragma unroll
      for (int i = 0; i < kDecodeJoinFew; ++i) {
        ml[i] = make_float2(-INFINITY, 0.f);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < pieces) {
          ml[i] = *reinterpret_cast<const float2*>(part_ml + at(i, r) * 2);
          v[i] = *reinterpret_cast<const float4*>(part_o + at(i, r) * hd + d);
        }
      }
      float top = -INFINITY, sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kDecodeJoinFew; ++i) top = fmaxf(top, ml[i].x);
#pragma unroll
      for (int i = 0; i < kDecodeJoinFew; ++i) {
        if (ml[i].y == 0.f) continue;
        const float f = fast_exp2(ml[i].x - top);
        sum = fmaf(f, ml[i].y, sum);
        o.x = fmaf(f, v[i].x, o.x); o.y = fmaf(f, v[i].y, o.y); o.z = fmaf(f, v[i].z, o.z); o.w = fmaf(f, v[i].w, o.w);
      }
      if (sink && sum != 0.f) sum += fast_exp2(sink[head0 + r] * 1.4426950408889634f - top);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(out + size_t(seq) * out_stride + size_t(head0 + r) * hd + d) =
          make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
    return;
  }
  // the largest maximum of every head
  {
    const int r = tid & 7;
    float top = -INFINITY;
    if (r < heads_here)
      for (int i = tid >> 3; i < pieces; i += 16) top = fmaxf(top, part_ml[at(i, r) * 2]);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    if ((tid & 31) < 8) tops[tid >> 5][r] = top;
    __syncthreads();
    if (tid < 8) {
      all_top[tid] = fmaxf(fmaxf(tops[0][tid], tops[1][tid]), fmaxf(tops[2][tid], tops[3][tid]));
      all_sum[tid] = 0.f;
    }
    __syncthreads();
  }
  constexpr int kMost = kDecodeHeads * 256 / 4 / 128;                  // items of a thread
  float4 acc[kMost];
#pragma unroll
  for (int k = 0; k < kMost; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < pieces; i0 += kDecodeJoinAtOnce) {
    const int n = min(kDecodeJoinAtOnce, pieces - i0);
    for (int j = tid; j < n * kDecodeHeads; j += 128) {
      const int i = j >> 3, r = j & 7;
      float w = 0.f;
      if (r < heads_here) {
        const float l = part_ml[at(i0 + i, r) * 2 + 1];
        w = l == 0.f ? 0.f : fast_exp2(part_ml[at(i0 + i, r) * 2] - all_top[r]);
      }
      weight[i][r] = w;
    }
    __syncthreads();
    if (tid < heads_here) {                                        // (one thread a head: the sums keep their order)
      float sum = all_sum[tid];
      for (int i = 0; i < n; ++i) sum = fmaf(weight[i][tid], part_ml[at(i0 + i, tid) * 2 + 1], sum);
      all_sum[tid] = sum;
    }
#pragma unroll
    for (int k = 0; k < kMost; ++k) {
      const int it = tid + k * 128;
      if (it >= items) break;
      const int r = it / quads, d = (it - r * quads) * 4;
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float f = weight[i][r];
        const float4 v = *reinterpret_cast<const float4*>(part_o + at(i0 + i, r) * hd + d);
        acc[k].x = fmaf(f, v.x, acc[k].x); acc[k].y = fmaf(f, v.y, acc[k].y); acc[k].z = fmaf(f, v.z, acc[k].z); acc[k].w = fmaf(f, v.w, acc[k].w);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int it = tid + k * 128;
    if (it >= items) break;
    const int r = it / quads, d = (it - r * quads) * 4;
    float sum = all_sum[r];
    if (sink && sum != 0.f) sum += fast_exp2(sink[head0 + r] * 1.4426950408889634f - all_top[r]);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    *reinterpret_cast<uint2*>(out + size_t(seq) * out_stride + size_t(head0 + r) * hd + d) =
        make_uint2(pack_bf16(acc[k].x * inv, acc[k].y * inv), pack_bf16(acc[k].z * inv, acc[k].w * inv));
  }
}

}  // namespace kvcm
