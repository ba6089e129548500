// Pages that requests share, on the device: requests that begin as copies of others, requests that end, and pools whose pages in
// use move to the front.  The counterparts of what the page allocator and the prefix cache do on the host, for loops that stay on the
// GPU (step_tables.cu takes pages from the same stack of free ones).
//
// State: page tables [seqs, max_blocks], lengths [seqs], a stack of free pages (the first `count` entries, taken from the top), and
// for each page of the pool `shared` = requests that hold it beyond the first (0 for a page of one request, and for a free one).
//   fork     entry k: request children[k], empty so far, gets the length L of parents[k]; L / B whole pages are shared, the page
//            behind them, if L mod B > 0, is a new one from the stack and a copy in every pool (both requests write to theirs).
//            The k-th copied page takes the (k+1)-th page from the top.
//   release  every page of the named requests loses a holder; pages without one go onto the stack, the lowest number on top.
//   compact  pages 0 .. used - 1 are in use behind it:  the r-th used page >= used moves into the r-th free page < used.
//            Tables, `shared` and the pools follow, the stack is used .. pages - 1 with the lowest on top, and map[page] says where
//            each page went (-1: it was free).
// Each is one thread-block cluster that checks everything before it writes anything, so a call that cannot be leaves all as it
// was, with the reason in `status`.  Whole numbers and atomic sums only: the results do not depend on order.  Outputs may be the inputs
// (a step that is replayed from a graph goes on from the one before); where they are not, they start as copies.
// The pages' contents are moved by a second kernel, a warp a piece of 4 KB.
// What bounds them: the small ones launches and a dozen dependent trips to memory with cluster barriers between them, the copy memory.
// B200: 48 requests forked into 144 15 us, their 140 pages in 8 layers (70 MB moved) 11; 100 of 250 requests released 14, the plan of a
// compaction 20, its 1,100 pages in 8 layers (580 MB) 89, the rate of a copy.
#include <cooperative_groups.h>

#include "packed.cuh"
#include "pdl.cuh"

namespace kvcm {

namespace cg = cooperative_groups;

constexpr int kPgThreads = 1024;
constexpr int kPgMaxBlocks = 8;
constexpr int kPgMaxSeqs = 65536;
constexpr int kPgMaxEntries = 8192;
constexpr int kPgPools = 64;
constexpr int kPgPiece = 4096;                     // bytes that a warp copies at once

enum PageError { kPgRequest = 1, kPgTwice = 2, kPgHolds = 3, kPgLength = 4, kPgPage = 5, kPgMissing = 6, kPgStack = 7, kPgHeld = 8 };

struct PageState {
  const int* seq_len; const int* block_tables; const int* shared; const int* free_pages; const int* free_count;
  int seqs, max_blocks, pages, stack, block_size;
};

namespace {

__device__ __forceinline__ int warp_scan(int v) {                  // sums up to and with the lane
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
// The sum of the threads before this one; `total` of all.  `sums` [33] of shared memory.
__device__ __forceinline__ int block_scan(int v, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int up = warp_scan(v);
  __syncthreads();                                                 // sums may still be read from a call before
  if (lane == 31) sums[warp] = up;
  __syncthreads();
  if (warp == 0) {
    const int w = lane < int(blockDim.x >> 5) ? sums[lane] : 0;
    const int t = warp_scan(w);
    sums[lane] = t - w;
    if (lane == 31) sums[32] = t;
  }
  __syncthreads();
  total = sums[32];
  return sums[warp] + up - v;
}

// The blocks of the cluster: a barrier, and the first thing that was found wrong anywhere (the least code, and of it the least number).
struct Team {
  unsigned long long* wrong;                       // of this block: code << 32 | number
  int rank, blocks, share, shares;
  __device__ __forceinline__ Team(unsigned long long* w) : wrong(w) {
    blocks = gridDim.x;
    rank = blockIdx.x;
    share = rank * kPgThreads + threadIdx.x;
    shares = blocks * kPgThreads;
    if (threadIdx.x == 0) *wrong = ~0ull;
    __syncthreads();
  }
  __device__ __forceinline__ void say(int code, int number) { atomicMin(wrong, (unsigned long long)code << 32 | unsigned(number)); }
  __device__ __forceinline__ void sync() {
    if (blocks > 1) cg::this_cluster().sync(); else __syncthreads();
  }
  // (between two barriers, so that nobody changes it or leaves)
  __device__ __forceinline__ unsigned long long first_wrong() {
    if (blocks == 1) return *wrong;
    const int lane = threadIdx.x & 31;                             // (a lane a block: one trip)
    unsigned long long w = lane < blocks ? *cg::this_cluster().map_shared_rank(wrong, lane) : ~0ull;
#pragma unroll
    for (int o = 1; o < kPgMaxBlocks; o *= 2) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, w, o);
      w = other < w ? other : w;
    }
    return __shfl_sync(0xffffffffu, w, 0);
  }
  // The sum of a number of every block, and of the blocks before this one.
  __device__ __forceinline__ int sum(int* of_block, int& before) {
    if (blocks == 1) { before = 0; return *of_block; }
    const int lane = threadIdx.x & 31;
    const int up = warp_scan(lane < blocks ? *cg::this_cluster().map_shared_rank(of_block, lane) : 0);
    before = rank == 0 ? 0 : __shfl_sync(0xffffffffu, up, rank - 1);
    return __shfl_sync(0xffffffffu, up, 31);
  }
};

__device__ __forceinline__ int blocks_of(int length, int B) { return (length + B - 1) / B; }

}  // namespace

struct ForkParams {
  PageState in;
  const int* parents; const int* children; int entries;
  int* block_tables; int* seq_len; int* shared; int* free_left; int* moves; int* status;      // moves: count, sources [entries], targets [entries]
};

__global__ void __launch_bounds__(kPgThreads) fork_requests_kernel(ForkParams p) {
  extern __shared__ int arrays[];                  // [entries] ranks of new pages, [(seqs + 31) / 32] who is a child
  __shared__ unsigned long long wrong;
  __shared__ int sums[33];
  const PageState& s = p.in;
  const int B = s.block_size, K = p.entries, tid = threadIdx.x, lane = tid & 31;
  int* rank_of = arrays;
  unsigned* is_child = reinterpret_cast<unsigned*>(arrays + K);
  Team team(&wrong);
  for (int i = tid; i < (s.seqs + 31) / 32; i += kPgThreads) is_child[i] = 0u;
  const int count = *s.free_count;
  __syncthreads();
  // ---- entries, alike in every block: who they are, and the rank of the page that each takes
  const int per = (K + kPgThreads - 1) / kPgThreads, k0 = min(tid * per, K), k1 = min(k0 + per, K);
  int takes = 0;
  for (int k = k0; k < k1; ++k) {
    const int parent = p.parents[k], child = p.children[k];
    rank_of[k] = -1;
    if (parent < 0) continue;                      // nobody
    if (parent >= s.seqs || child < 0 || child >= s.seqs) { team.say(kPgRequest, k); continue; }
    if (atomicOr(&is_child[child >> 5], 1u << (child & 31)) >> (child & 31) & 1u) team.say(kPgTwice, child);
    if (s.seq_len[child] != 0 || child == parent) team.say(kPgHolds, child);
    const int L = s.seq_len[parent];
    if (L < 0 || L > s.max_blocks * (long long)B) { team.say(kPgLength, parent); continue; }
    rank_of[k] = L % B ? 1 : 0;
    takes += L % B ? 1 : 0;
  }
  int total;
  int at = block_scan(takes, sums, total);         // (its barriers also publish who is a child)
  for (int k = k0; k < k1; ++k)
    if (rank_of[k] >= 0) {
      const int parent = p.parents[k];
      if (is_child[parent >> 5] >> (parent & 31) & 1u) team.say(kPgHolds, parent);      // (its length is about to change)
      const int t = rank_of[k];
      rank_of[k] = at;                             // (of an entry that takes none: not used)
      at += t;
    }
  if (tid == 0 && (count < 0 || count > s.stack)) team.say(kPgStack, count);
  else if (tid == 0 && total > count) team.say(kPgMissing, total - count);
  __syncthreads();
  // ---- every page that is shared, copied or taken lies in the pool; a warp an entry
  const bool sane = count >= 0 && count <= s.stack && total <= count;
  for (int k = team.share >> 5; k < K; k += team.shares >> 5) {
    if (rank_of[k] < 0) continue;
    const int parent = p.parents[k], L = s.seq_len[parent], n = blocks_of(L, B);
    for (int j = lane; j < n; j += 32) {
      const int page = s.block_tables[size_t(parent) * s.max_blocks + j];
      if (page < 0 || page >= s.pages) team.say(kPgPage, page);
    }
    if (lane == 0 && sane && L % B) {
      const int page = s.free_pages[count - 1 - rank_of[k]];
      if (page < 0 || page >= s.pages) team.say(kPgPage, page);
    }
  }
  if (p.seq_len != s.seq_len)
    for (int i = team.share; i < s.seqs; i += team.shares) p.seq_len[i] = s.seq_len[i];
  if (p.shared != s.shared)
    for (int i = team.share; i < s.pages; i += team.shares) p.shared[i] = s.shared[i];
  team.sync();
  const unsigned long long bad = team.first_wrong();
  if (bad == ~0ull)
    for (int k = team.share >> 5; k < K; k += team.shares >> 5) {
      if (rank_of[k] < 0) continue;
      const int parent = p.parents[k], child = p.children[k], L = s.seq_len[parent], full = L / B;
      const int* from = s.block_tables + size_t(parent) * s.max_blocks;
      int* to = p.block_tables + size_t(child) * s.max_blocks;
      for (int j = lane; j < full; j += 32) {
        const int page = from[j];
        to[j] = page;
        atomicAdd(&p.shared[page], 1);
      }
      if (lane == 0) {
        if (L % B) {
          const int page = s.free_pages[count - 1 - rank_of[k]];
          to[full] = page;
          p.shared[page] = 0;
          p.moves[1 + rank_of[k]] = from[full];
          p.moves[1 + K + rank_of[k]] = page;
        }
        p.seq_len[child] = L;
      }
    }
  if (team.share == 0) {
    *p.free_left = bad == ~0ull ? count - total : count;
    p.moves[0] = bad == ~0ull ? total : 0;
    p.status[0] = bad == ~0ull ? 0 : int(bad >> 32);
    p.status[1] = bad == ~0ull ? 0 : int(unsigned(bad));
    p.status[2] = bad == ~0ull ? total : 0;
    p.status[3] = 0;
  }
  team.sync();                                     // nobody leaves while its shared memory is read
}

struct ReleaseParams {
  PageState in;
  const int* requests; int entries;
  int* seq_len; int* shared; int* free_pages; int* free_left; int* status;
};

__global__ void __launch_bounds__(kPgThreads) release_requests_kernel(ReleaseParams p) {
  extern __shared__ int arrays[];                  // [(seqs + 31) / 32] who ends
  __shared__ unsigned long long wrong;
  __shared__ int sums[33], freed_here;
  const PageState& s = p.in;
  const int B = s.block_size, K = p.entries, tid = threadIdx.x, lane = tid & 31;
  unsigned* ends = reinterpret_cast<unsigned*>(arrays);
  Team team(&wrong);
  for (int i = tid; i < (s.seqs + 31) / 32; i += kPgThreads) ends[i] = 0u;
  const int count = *s.free_count;
  __syncthreads();
  for (int k = tid; k < K; k += kPgThreads) {
    const int r = p.requests[k];
    if (r < 0) continue;                           // nobody
    if (r >= s.seqs) { team.say(kPgRequest, k); continue; }
    if (atomicOr(&ends[r >> 5], 1u << (r & 31)) >> (r & 31) & 1u) team.say(kPgTwice, r);
    if (s.seq_len[r] < 0 || s.seq_len[r] > s.max_blocks * (long long)B) team.say(kPgLength, r);
  }
  if (tid == 0 && (count < 0 || count > s.stack)) team.say(kPgStack, count);
  __syncthreads();
  const bool readable = wrong == ~0ull;            // (alike in every block: each has looked at all entries)
  __syncthreads();
  if (readable)
    for (int k = team.share >> 5; k < K; k += team.shares >> 5) {
      const int r = p.requests[k];
      if (r < 0) continue;
      const int n = blocks_of(s.seq_len[r], B);
      for (int j = lane; j < n; j += 32) {
        const int page = s.block_tables[size_t(r) * s.max_blocks + j];
        if (page < 0 || page >= s.pages) team.say(kPgPage, page);
      }
    }
  if (p.seq_len != s.seq_len)
    for (int i = team.share; i < s.seqs; i += team.shares) p.seq_len[i] = s.seq_len[i];
  if (p.shared != s.shared)
    for (int i = team.share; i < s.pages; i += team.shares) p.shared[i] = s.shared[i];
  team.sync();
  unsigned long long bad = team.first_wrong();
  team.sync();                                     // (what is found wrong from here on is told apart)
  auto holders = [&](int by) {
    for (int k = team.share >> 5; k < K; k += team.shares >> 5) {
      const int r = p.requests[k];
      if (r < 0) continue;
      const int n = blocks_of(s.seq_len[r], B);
      for (int j = lane; j < n; j += 32) atomicAdd(&p.shared[s.block_tables[size_t(r) * s.max_blocks + j]], by);
    }
  };
  int freed = 0;
  if (bad == ~0ull) {
    holders(-1);
    __threadfence();
    team.sync();
    // ---- pages without a holder, in order: each block has a range of pages, each thread a piece of it
    const int per = (s.pages + team.shares - 1) / team.shares;
    const int i0 = min(team.share * per, s.pages), i1 = min(i0 + per, s.pages);
    int mine = 0;
    for (int i = i0; i < i1; ++i) {
      const int h = __ldcg(&p.shared[i]);
      if (h < -1) team.say(kPgHeld, i);
      mine += h < 0;
    }
    int total;
    int at = block_scan(mine, sums, total);
    if (tid == 0) freed_here = total;
    team.sync();
    bad = team.first_wrong();
    int before;
    freed = team.sum(&freed_here, before);
    at += before;
    if (bad == ~0ull && freed > s.stack - count) bad = (unsigned long long)kPgStack << 32 | unsigned(count + freed);
    team.sync();                                   // everybody knows, and has read who holds what
    if (bad == ~0ull) {
      for (int i = i0; i < i1; ++i)
        if (__ldcg(&p.shared[i]) < 0) {
          p.free_pages[count + freed - 1 - at++] = i;
          p.shared[i] = 0;
        }
      for (int k = team.share; k < K; k += team.shares)
        if (p.requests[k] >= 0) p.seq_len[p.requests[k]] = 0;
    } else {
      holders(1);                                  // as it was
    }
  }
  if (team.share == 0) {
    *p.free_left = bad == ~0ull ? count + freed : count;
    p.status[0] = bad == ~0ull ? 0 : int(bad >> 32);
    p.status[1] = bad == ~0ull ? 0 : int(unsigned(bad));
    p.status[2] = bad == ~0ull ? freed : 0;
    p.status[3] = 0;
  }
  team.sync();
}

struct CompactParams {
  PageState in;
  int* block_tables; int* shared; int* free_pages; int* map; int* moves; int* status;       // moves: count, sources [pages], targets [pages]
};

__global__ void __launch_bounds__(kPgThreads) compact_pages_kernel(CompactParams p) {
  __shared__ unsigned long long wrong;
  __shared__ int sums[33], holes_here, movers_here;
  const PageState& s = p.in;
  const int B = s.block_size, N = s.pages, tid = threadIdx.x, lane = tid & 31;
  Team team(&wrong);
  const int count = *s.free_count, used = N - count;
  const bool sane = count >= 0 && count <= s.stack && count <= N;
  if (tid == 0 && !sane) team.say(kPgStack, count);
  for (int i = team.share; i < N; i += team.shares) p.map[i] = i;
  __threadfence();
  team.sync();
  if (sane)
    for (int i = team.share; i < count; i += team.shares) {
      const int page = s.free_pages[i];
      if (page < 0 || page >= N) team.say(kPgPage, page);
      else if (atomicExch(&p.map[page], -1) == -1) team.say(kPgTwice, page);
    }
  __threadfence();
  team.sync();
  // ---- free pages below `used` and used ones above, in order
  const int per = (N + team.shares - 1) / team.shares;
  const int i0 = min(team.share * per, N), i1 = min(i0 + per, N);
  int holes = 0, movers = 0;
  if (sane)
    for (int i = i0; i < i1; ++i) {
      const bool is_free = __ldcg(&p.map[i]) < 0;
      holes += is_free && i < used;
      movers += !is_free && i >= used;
    }
  int total;
  int hole_at = block_scan(holes, sums, total);
  if (tid == 0) holes_here = total;
  int mover_at = block_scan(movers, sums, total);
  if (tid == 0) movers_here = total;
  // ---- and every page of a request is in use
  for (int i = team.share >> 5; i < s.seqs; i += team.shares >> 5) {
    const int L = s.seq_len[i];
    if (L < 0 || L > s.max_blocks * (long long)B) {
      if (lane == 0) team.say(kPgLength, i);
      continue;
    }
    const int n = blocks_of(L, B);
    for (int j = lane; j < n; j += 32) {
      const int page = s.block_tables[size_t(i) * s.max_blocks + j];
      if (page < 0 || page >= N || __ldcg(&p.map[page]) < 0) team.say(kPgPage, page);
    }
  }
  team.sync();
  const unsigned long long bad = team.first_wrong();
  int before;
  team.sum(&holes_here, before);
  hole_at += before;
  const int moved = team.sum(&movers_here, before);
  mover_at += before;
  if (bad == ~0ull)
    for (int i = i0; i < i1; ++i) {
      const bool is_free = __ldcg(&p.map[i]) < 0;
      if (is_free && i < used) p.moves[1 + N + hole_at++] = i;
      if (!is_free && i >= used) p.moves[1 + mover_at++] = i;
    }
  __threadfence();
  team.sync();
  if (bad == ~0ull) {
    for (int m = team.share; m < moved; m += team.shares) {
      const int from = __ldcg(&p.moves[1 + m]), to = __ldcg(&p.moves[1 + N + m]);
      p.map[from] = to;
      p.shared[to] = s.shared[from];
    }
  }
  __threadfence();
  team.sync();
  for (int i = team.share; i < N; i += team.shares) {
    const int to = __ldcg(&p.map[i]);
    if (bad != ~0ull) {
      if (p.shared != s.shared) p.shared[i] = s.shared[i];
      p.map[i] = i;
    } else if (i >= used) {
      p.shared[i] = 0;                             // (those that moved have been read, before the barrier)
    } else if (to == i && p.shared != s.shared) {
      p.shared[i] = s.shared[i];
    }
  }
  if (bad == ~0ull) {
    for (int i = team.share; i < count; i += team.shares) p.free_pages[i] = N - 1 - i;
  } else if (p.free_pages != s.free_pages && sane) {
    for (int i = team.share; i < count; i += team.shares) p.free_pages[i] = s.free_pages[i];
  }
  // ---- tables: a warp a request
  if (bad == ~0ull || p.block_tables != s.block_tables)
    for (int i = team.share >> 5; i < s.seqs; i += team.shares >> 5) {
      const int n = bad == ~0ull ? blocks_of(s.seq_len[i], B) : 0;
      const int stop = p.block_tables != s.block_tables ? s.max_blocks : n;
      for (int j = lane; j < stop; j += 32) {
        const int page = s.block_tables[size_t(i) * s.max_blocks + j];
        p.block_tables[size_t(i) * s.max_blocks + j] = j < n ? __ldcg(&p.map[page]) : page;
      }
    }
  if (team.share == 0) {
    p.moves[0] = bad == ~0ull ? moved : 0;
    p.status[0] = bad == ~0ull ? 0 : int(bad >> 32);
    p.status[1] = bad == ~0ull ? 0 : int(unsigned(bad));
    p.status[2] = bad == ~0ull ? moved : 0;
    p.status[3] = 0;
  }
  team.sync();
}

struct PagePool { char* at; long long layer_stride, page_bytes; int layers, first; };       // first: pieces of the pools before, of one page
struct CopyParams {
  const int* from; const int* to; const int* count; int most, pages;
  int pools, pieces;                               // pieces of one page in all pools
  PagePool pool[kPgPools];
};

template <typename V> __device__ __forceinline__ void copy_piece(char* to, const char* from, int bytes, int lane) {
  constexpr int kAtOnce = kPgPiece / 32 / 16;
  const int n = bytes / int(sizeof(V));
  for (int i = lane; i < n; i += 32 * kAtOnce) {
    V v[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (i + 32 * k < n) v[k] = reinterpret_cast<const V*>(from)[i + 32 * k];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k)
      if (i + 32 * k < n) reinterpret_cast<V*>(to)[i + 32 * k] = v[k];
  }
}

// Pages from[i] -> to[i] in all pools, a warp a piece; pairs outside the pool are none.
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyParams p) {
  const int count = p.count ? min(*p.count, p.most) : p.most;
  const long long items = (long long)count * p.pieces;
  const int lane = threadIdx.x & 31;
  for (long long it = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (long long)gridDim.x * 8) {
    const int i = int(it / p.pieces), piece = int(it - (long long)i * p.pieces);
    const int from = p.from[i], to = p.to[i];
    if (from < 0 || to < 0 || from >= p.pages || to >= p.pages || from == to) continue;
    int k = 0;
    while (k + 1 < p.pools && p.pool[k + 1].first <= piece) ++k;
    const PagePool& pool = p.pool[k];
    const int per_page = int((pool.page_bytes + kPgPiece - 1) / kPgPiece), of_pool = piece - pool.first;
    const int layer = of_pool / per_page;
    const long long at = (long long)(of_pool - layer * per_page) * kPgPiece;
    const int bytes = int(min((long long)kPgPiece, pool.page_bytes - at));
    char* const base = pool.at + layer * pool.layer_stride + at;
    char* const dst = base + to * pool.page_bytes;
    const char* const src = base + from * pool.page_bytes;
    const unsigned long long places = reinterpret_cast<unsigned long long>(dst) | reinterpret_cast<unsigned long long>(src) | unsigned(bytes);
    if ((places & 15) == 0) copy_piece<uint4>(dst, src, bytes, lane);
    else if ((places & 3) == 0) copy_piece<uint32_t>(dst, src, bytes, lane);
    else copy_piece<unsigned char>(dst, src, bytes, lane);
  }
}

__global__ void pages_done_kernel() {}

namespace {

static_assert(kPgMaxEntries * 4 + kPgMaxSeqs / 8 <= 47 * 1024, "the entries' arrays fit a block without an opt-in");

template <typename Params>
int launch_cluster(void (*kernel)(Params), const Params& p, long long work, size_t smem, cudaStream_t s) {
  // one block for little work (no cluster barrier), up to eight for much: a request's pages are a warp's, a round of them three trips to memory
  long long blocks = (work + kPgThreads - 1) / kPgThreads;
  blocks = blocks < 1 ? 1 : blocks > kPgMaxBlocks ? kPgMaxBlocks : blocks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kPgThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(blocks);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kernel, p));
}

bool state_ok(const PageState& s) {
  return s.seqs > 0 && s.seqs <= kPgMaxSeqs && s.max_blocks > 0 && s.pages > 0 && s.pages < (1 << 30) && s.stack >= 0 && s.block_size > 0 &&
         (long long)s.max_blocks * s.block_size <= 0x7fffffffll - s.block_size && (long long)s.seqs * s.max_blocks <= 0x7fffffffll;
}

// `table`: for each pool its address, layers, bytes between layers, bytes of a page.
int launch_copy(const int* from, const int* to, const int* count, int most, int pages, const long long* table, int pools, cudaStream_t s) {
  if (pools < 0 || pools > kPgPools) return KVCM_ERR_UNSUPPORTED;
  CopyParams p = {};
  p.from = from; p.to = to; p.count = count; p.most = most; p.pages = pages; p.pools = pools;
  long long pieces = 0;
  for (int i = 0; i < pools; ++i) {
    PagePool& q = p.pool[i];
    q.at = reinterpret_cast<char*>(static_cast<uintptr_t>(table[4 * i]));
    q.layers = int(table[4 * i + 1]); q.layer_stride = table[4 * i + 2]; q.page_bytes = table[4 * i + 3];
    if (q.layers < 0 || q.page_bytes < 0) return KVCM_ERR_UNSUPPORTED;
    q.first = int(pieces);
    pieces += (long long)q.layers * ((q.page_bytes + kPgPiece - 1) / kPgPiece);
    if (pieces > 0x7fffffffll) return KVCM_ERR_UNSUPPORTED;
  }
  p.pieces = int(pieces);
  if (pieces > 0 && most > 0) {
    const long long blocks = ((long long)most * pieces + 7) / 8, room = 148 * 8;
    const int rc = pdl_launch_if(false, copy_pages_kernel, dim3(unsigned(blocks < room ? blocks : room)), dim3(256), 0, s, p);
    if (rc != 0) return rc;
  }
  // (kernels of a step read its integers and earlier tokens' keys ahead of their dependency wait, as what a completed launch has written)
  return pdl_launch_if(false, pages_done_kernel, dim3(1), dim3(32), 0, s);
}

}  // namespace
}  // namespace kvcm

using namespace kvcm;

// Arrays: see the kernels.  moves: 1 + 2 * entries ints of the call; status [4].  Outputs may be the inputs.
KVCM_API int kvcm_fork_requests(const int* parents, const int* children, int entries, const int* seq_len, int seqs, int* block_tables,
                                int max_blocks, const int* shared, int pages, const int* free_pages, int stack, const int* free_count,
                                int block_size, int* seq_len_out, int* shared_out, int* free_left, int* moves, int* status,
                                const long long* pool_table, int pools, void* stream) {
  ForkParams p;
  p.in = PageState{seq_len, block_tables, shared, free_pages, free_count, seqs, max_blocks, pages, stack, block_size};
  if (!state_ok(p.in) || entries < 0 || entries > kPgMaxEntries) return KVCM_ERR_UNSUPPORTED;
  p.parents = parents; p.children = children; p.entries = entries;
  p.block_tables = block_tables; p.seq_len = seq_len_out; p.shared = shared_out; p.free_left = free_left; p.moves = moves; p.status = status;
  const long long work = 32ll * entries + (seq_len_out != seq_len ? seqs : 0) + (shared_out != shared ? pages / 4 : 0);
  const int rc = launch_cluster(fork_requests_kernel, p, work, size_t(entries + (seqs + 31) / 32) * sizeof(int), (cudaStream_t)stream);
  if (rc != 0) return rc;
  return launch_copy(moves + 1, moves + 1 + entries, moves, entries, pages, pool_table, pools, (cudaStream_t)stream);
}

KVCM_API int kvcm_release_requests(const int* requests, int entries, const int* seq_len, int seqs, const int* block_tables, int max_blocks,
                                   const int* shared, int pages, int* free_pages, int stack, const int* free_count, int block_size,
                                   int* seq_len_out, int* shared_out, int* free_left, int* status, void* stream) {
  ReleaseParams p;
  p.in = PageState{seq_len, block_tables, shared, free_pages, free_count, seqs, max_blocks, pages, stack, block_size};
  if (!state_ok(p.in) || entries < 0 || entries > kPgMaxEntries) return KVCM_ERR_UNSUPPORTED;
  p.requests = requests; p.entries = entries; p.seq_len = seq_len_out; p.shared = shared_out; p.free_pages = free_pages;
  p.free_left = free_left; p.status = status;
  const long long work = 32ll * entries + pages / 4;
  const int rc = launch_cluster(release_requests_kernel, p, work, size_t((seqs + 31) / 32) * sizeof(int), (cudaStream_t)stream);
  if (rc != 0) return rc;
  return pdl_launch_if(false, pages_done_kernel, dim3(1), dim3(32), 0, (cudaStream_t)stream);
}

// map [pages]; moves: 1 + 2 * pages ints of the call.
KVCM_API int kvcm_compact_pages(const int* seq_len, int seqs, const int* block_tables, int max_blocks, const int* shared, int pages,
                                const int* free_pages, int stack, const int* free_count, int block_size, int* tables_out, int* shared_out,
                                int* free_out, int* map, int* moves, int* status, const long long* pool_table, int pools, void* stream) {
  CompactParams p;
  p.in = PageState{seq_len, block_tables, shared, free_pages, free_count, seqs, max_blocks, pages, stack, block_size};
  if (!state_ok(p.in)) return KVCM_ERR_UNSUPPORTED;
  p.block_tables = tables_out; p.shared = shared_out; p.free_pages = free_out; p.map = map; p.moves = moves; p.status = status;
  const long long work = 32ll * seqs + pages / 4;
  const int rc = launch_cluster(compact_pages_kernel, p, work, 0, (cudaStream_t)stream);
  if (rc != 0) return rc;
  return launch_copy(moves + 1, moves + 1 + pages, moves, pages / 2, pages, pool_table, pools, (cudaStream_t)stream);
}

KVCM_API int kvcm_copy_pages(const int* from, const int* to, int count, int pages, const long long* pool_table, int pools, void* stream) {
  if (count < 0 || pages <= 0) return KVCM_ERR_UNSUPPORTED;
  return launch_copy(from, to, nullptr, count, pages, pool_table, pools, (cudaStream_t)stream);
}

KVCM_PACKED(kvcm_fork_requests)
KVCM_PACKED(kvcm_release_requests)
KVCM_PACKED(kvcm_compact_pages)
KVCM_PACKED(kvcm_copy_pages)
