// The integer arrays of a step from the requests' lengths, on the device: what BatchBuilder::build (csrc/core/batch.cpp) and the
// page allocator do on the host, for loops that stay on the GPU for several steps.
//
// Request i holds pages for its first start[i] positions and brings n[i] new rows (n may be 0):
//     q_start[i] = n[0] + .. + n[i-1]                       ctx_len[i] = start[i] + n[i]
//     pages held  h[i] = ceil(start[i] / B),  new pages  e[i] = ceil(ctx_len[i] / B) - h[i]
//     new page k of all (requests in order) = free_pages[count - 1 - k];   table[i][h[i] + j] = new page (e[0] + .. + e[i-1] + j)
//     row q_start[i] + r:  position start[i] + r, request i, slot table[i][position / B] * B + position % B
//     tiles: requests with n[i] > 1, in order: (i, 0), (i, tile_rows), ..
// Rows behind the last one get position -1, request 0 and slot -1, tiles behind the last one (-1, -1).
//
// One thread-block cluster: every block adds up all lengths itself (a few KB from L2) and then takes its share of rows, pages
// and tiles, each finding its request by bisection in shared memory, so no block waits for another's results; one cluster
// barrier stands between the last read of start and count and the first write, so that ctx_len may be start and free_left may
// be free_count (a step that is replayed from a graph advances itself).  Integer sums only: the results do not depend on order.
// What bounds it: three dependent trips to memory (lengths, table or stack, the store) and the launch; the bytes are a few KB to 1 MB.
// B200: 250 requests of one row 5.1 us, 64 portions of some 120 rows 7.1 us, of which the second launch is 0.6.
//
// Many kernels of a step read its integers before their dependency wait, as what a completed launch has written (pdl.cuh).  A kernel
// that is launched early behind this one would start when its blocks have ended, which completes nothing, so both this kernel
// and an empty one behind it are launched the ordinary way: the empty one starts when this one is complete, and whoever starts
// behind that, however early, finds the arrays.
#include <cooperative_groups.h>

#include "common.cuh"
#include "packed.cuh"
#include "pdl.cuh"

namespace kvcm {

constexpr int kTabThreads = 1024;
constexpr int kTabMaxBlocks = 8;
constexpr int kTabMaxSeqs = 8192;

enum TabError { kTabNegative = 1, kTabTooLong = 2, kTabRows = 3, kTabTiles = 4, kTabPages = 5, kTabStack = 6 };

struct TabParams {
  const int* start; const int* n;
  int* block_tables; int max_blocks;
  const int* free_pages; int stack;               // room of the stack
  const int* free_count;
  int* q_start; int* ctx_len; int* positions; int* row_seq; int* slots; int* tile_seq; int* tile_q0; int* free_left; int* status;
  int seqs, rows, tiles, block_size, tile_rows;
};

struct Triple { int rows, pages, tiles; };
__device__ __forceinline__ Triple operator+(Triple a, Triple b) { return {a.rows + b.rows, a.pages + b.pages, a.tiles + b.tiles}; }
__device__ __forceinline__ Triple shfl_up(Triple t, int o) {
  return {__shfl_up_sync(0xffffffffu, t.rows, o), __shfl_up_sync(0xffffffffu, t.pages, o), __shfl_up_sync(0xffffffffu, t.tiles, o)};
}

// The last i with first[i] <= x (first[0] = 0 <= x).
__device__ __forceinline__ int last_at_most(const int* first, int count, int x) {
  int a = 0, b = count;
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (first[mid] <= x) a = mid; else b = mid;
  }
  return a;
}

__global__ void __launch_bounds__(kTabThreads) step_tables_kernel(TabParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ int arrays[];
  int* s_start = arrays;                           // [seqs] each
  int* s_row = s_start + p.seqs;
  int* s_page = s_row + p.seqs;
  int* s_tile = s_page + p.seqs;
  __shared__ Triple warp_sum_of[32];
  __shared__ int first_bad;                        // (request << 2 | code) of the first request that cannot be
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = p.block_size;
  if (tid == 0) first_bad = 0x7fffffff;
  const int count = *p.free_count;
  __syncthreads();

  // ---- prefix sums over the requests; a thread has `per` neighbouring ones
  const int per = (p.seqs + kTabThreads - 1) / kTabThreads;
  const int i0 = min(tid * per, p.seqs), i1 = min(i0 + per, p.seqs);
  auto of = [&](int i, int start) {                // what request i adds; nothing where it is refused
    const int n = p.n[i];
    int code = 0;
    if (start < 0 || n < 0) code = kTabNegative;
    else if ((long long)start + n > (long long)p.max_blocks * B) code = kTabTooLong;
    else if (n > p.rows) code = kTabRows;
    if (code) {
      atomicMin(&first_bad, (i << 2) | code);
      return Triple{0, 0, 0};
    }
    return Triple{n, (start + n + B - 1) / B - (start + B - 1) / B, n > 1 ? (n + p.tile_rows - 1) / p.tile_rows : 0};
  };
  Triple mine{0, 0, 0};
  for (int i = i0; i < i1; ++i) {
    const int start = p.start[i];
    s_start[i] = start;
    const Triple t = of(i, start);
    s_row[i] = t.rows; s_page[i] = t.pages; s_tile[i] = t.tiles;
    mine = mine + t;
  }
  Triple up = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Triple t = shfl_up(up, o);
    if (lane >= o) up = up + t;
  }
  if (lane == 31) warp_sum_of[warp] = up;
  __syncthreads();
  if (warp == 0) {
    Triple t = warp_sum_of[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const Triple u = shfl_up(t, o);
      if (lane >= o) t = t + u;
    }
    warp_sum_of[lane] = t;                         // sums up to and with the warp
  }
  __syncthreads();
  Triple at{up.rows - mine.rows, up.pages - mine.pages, up.tiles - mine.tiles};
  if (warp > 0) at = at + warp_sum_of[warp - 1];
  for (int i = i0; i < i1; ++i) {
    const Triple t{s_row[i], s_page[i], s_tile[i]};
    s_row[i] = at.rows; s_page[i] = at.pages; s_tile[i] = at.tiles;
    at = at + t;
  }
  Triple total = warp_sum_of[31];
  int code = 0, detail = 0;
  if (first_bad != 0x7fffffff) {
    code = first_bad & 3;
    detail = first_bad >> 2;
    if (code == kTabRows) detail = p.n[detail];    // (the text speaks of rows)
  }
  else if (total.rows > p.rows) { code = kTabRows; detail = total.rows; }
  else if (total.tiles > p.tiles && p.tile_seq != nullptr) { code = kTabTiles; detail = total.tiles; }
  else if (count < 0 || count > p.stack) { code = kTabStack; detail = count; }
  else if (total.pages > count) { code = kTabPages; detail = total.pages - count; }
  if (code) total = Triple{0, 0, 0};               // the step is refused whole: no row, no page, no tile

  const int shares = gridDim.x * kTabThreads, share = blockIdx.x * kTabThreads + tid;
  if (gridDim.x > 1) cg::this_cluster().sync();    // everybody has read start and count (and, in this block, published its sums)
  else __syncthreads();

  for (int i = share; i < p.seqs; i += shares) {
    const int rows_i = (i + 1 < p.seqs ? s_row[i + 1] : total.rows) - s_row[i];
    p.q_start[i] = code ? 0 : s_row[i];
    p.ctx_len[i] = s_start[i] + (code ? 0 : rows_i);
  }
  for (int r = share; r < p.rows; r += shares) {
    int position = -1, seq = 0, slot = -1;
    if (r < total.rows) {
      seq = last_at_most(s_row, p.seqs, r);
      const int start = s_start[seq], held = (start + B - 1) / B;
      position = start + r - s_row[seq];
      const int pi = position / B;
      const int page = pi < held ? p.block_tables[size_t(seq) * p.max_blocks + pi] : p.free_pages[count - 1 - (s_page[seq] + pi - held)];
      slot = page * B + (position - pi * B);
    }
    p.positions[r] = position;
    p.row_seq[r] = seq;
    p.slots[r] = slot;
  }
  for (int k = share; k < total.pages; k += shares) {
    const int seq = last_at_most(s_page, p.seqs, k);
    p.block_tables[size_t(seq) * p.max_blocks + (s_start[seq] + B - 1) / B + k - s_page[seq]] = p.free_pages[count - 1 - k];
  }
  if (p.tile_seq != nullptr)
    for (int k = share; k < p.tiles; k += shares) {
      const bool real = k < total.tiles;
      const int seq = real ? last_at_most(s_tile, p.seqs, k) : -1;
      p.tile_seq[k] = seq;
      p.tile_q0[k] = real ? (k - s_tile[seq]) * p.tile_rows : -1;
    }
  if (share == 0) {
    *p.free_left = count - total.pages;
    p.status[0] = code; p.status[1] = detail; p.status[2] = total.rows; p.status[3] = total.tiles;
  }
}

__global__ void step_tables_done_kernel() {}

}  // namespace kvcm

using namespace kvcm;

// Arrays: seqs ints (start, n, q_start, ctx_len), rows ints (positions, row_seq, slots), tiles ints (tile_seq, tile_q0; both null:
// no tiles), block_tables [seqs, max_blocks], free_pages [stack], free_count [1], free_left [1], status [4] = (code, detail, rows,
// tiles).  ctx_len may be start and free_left free_count; nothing else overlaps.
KVCM_API int kvcm_step_tables(const int* start, const int* n, int* block_tables, int max_blocks, const int* free_pages, int stack,
                              const int* free_count, int* q_start, int* ctx_len, int* positions, int* row_seq, int* slots, int* tile_seq,
                              int* tile_q0, int* free_left, int* status, int seqs, int rows, int tiles, int block_size, int tile_rows,
                              void* stream) {
  if (seqs <= 0 || seqs > kTabMaxSeqs || rows < 0 || tiles < 0 || block_size <= 0 || tile_rows <= 0 || max_blocks <= 0 || stack < 0)
    return KVCM_ERR_UNSUPPORTED;
  // sums of int32: a request brings at most `rows` rows and max_blocks pages
  if ((long long)seqs * rows > 0x7fffffffll || (long long)seqs * max_blocks > 0x7fffffffll ||
      (long long)max_blocks * block_size > 0x7fffffffll - block_size)
    return KVCM_ERR_UNSUPPORTED;
  if ((tile_seq == nullptr) != (tile_q0 == nullptr)) return KVCM_ERR_UNSUPPORTED;
  const size_t smem = size_t(4) * seqs * sizeof(int);
  static OncePerDevice once;
  if (smem > 48 * 1024) {
    const int rc = allow_shared_memory(once, step_tables_kernel, size_t(4) * kTabMaxSeqs * sizeof(int));
    if (rc != 0) return rc;
  }
  TabParams p;
  p.start = start; p.n = n; p.block_tables = block_tables; p.max_blocks = max_blocks; p.free_pages = free_pages; p.stack = stack;
  p.free_count = free_count; p.q_start = q_start; p.ctx_len = ctx_len; p.positions = positions; p.row_seq = row_seq; p.slots = slots;
  p.tile_seq = tile_seq; p.tile_q0 = tile_q0; p.free_left = free_left; p.status = status;
  p.seqs = seqs; p.rows = rows; p.tiles = tiles; p.block_size = block_size; p.tile_rows = tile_rows;
  // one block for steps of few rows (no cluster barrier), up to eight for many
  int blocks = (rows + 2 * kTabThreads - 1) / (2 * kTabThreads);
  blocks = blocks < 1 ? 1 : blocks > kTabMaxBlocks ? kTabMaxBlocks : blocks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kTabThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  const int rc = static_cast<int>(cudaLaunchKernelEx(&cfg, step_tables_kernel, p));
  if (rc != 0) return rc;
  return pdl_launch_if(false, step_tables_done_kernel, dim3(1), dim3(32), 0, (cudaStream_t)stream);
}

KVCM_PACKED(kvcm_step_tables)
