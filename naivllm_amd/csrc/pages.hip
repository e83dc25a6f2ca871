// Pages of a paged cache copied, forked and compacted, in every pool that one
// numbering serves (K and V of all layers, key weights) at once, for gfx950.
// No reference counterpart: its pages belong to one sequence each, and to its
// host's bookkeeping.
//
// A plan kernel of one workgroup reads the block tables and writes the list of
// pages to move; a second kernel copies them and writes the new tables.  The
// tables alone say which pages are in use (a bit per page in LDS), beside
// those that the caller holds, so there is no allocator's state on the device
// to keep, and the host waits for nothing.
//
// No page is a source and a target of one call: fork's targets are pages that
// no row keeps, while a source stays with its first child; compact's targets
// are free.

#include "common.h"

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kMaxPages = 1 << 19;            // two bits each in LDS: 128 KiB
constexpr int kMaxWords = kMaxPages / 32;
constexpr int kMaxRows = 4096;
constexpr int kMoveThreads = 256;
constexpr int kUnit = kMoveThreads * 16 * 2;  // bytes of a page that a workgroup copies at a time
constexpr int kMoveGroups = 2048;
constexpr int kPoolsPerLaunch = 128;          // pools in one kernel's arguments

struct Pools {
  nsv_pool pool[kPoolsPerLaunch];
  int first[kPoolsPerLaunch + 1];  // units of a page before the pool's
  int n, block_size, num_blocks;
};

// The moves of a call: *count of them (or most, where count is NULL).
struct Moves {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* keys;   // nullable: whole pages
  const int32_t* count;  // nullable
  int most;
};

__device__ __forceinline__ uint32_t scan_u32(uint32_t v) {  // inclusive, over a wave
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// exclusive prefix over the workgroup, and the whole sum
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* red, uint32_t& total) {
  const uint32_t in = scan_u32(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = in;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += red[w];
    all += red[w];
  }
  total = all;
  return before + in - v;
}

__device__ __forceinline__ void mark_held(const uint8_t* held, int pages, uint32_t* bits) {
  if (!held) return;
  for (int i = threadIdx.x; i < pages; i += kPlanThreads)
    if (held[i]) atomicOr(&bits[i >> 5], 1u << (i & 31));
}

// the pages of a word that exist
__device__ __forceinline__ uint32_t word_mask(int w, int pages) {
  const int left = pages - 32 * w;
  return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
struct ForkArgs {
  const int32_t* tables;  // [B, W]
  const int64_t* lens;
  const int32_t* parents;
  const uint8_t* held;    // nullable [num_blocks]
  int B, W;
  int32_t* out_tables;
  int64_t* out_lens;
  int32_t* lacking;
  // workspace
  int32_t* count;         // moves
  int32_t* src;
  int32_t* dst;
  int32_t* keys;          // [B] each
  int32_t* base;          // [B] a row's first place in `fresh`; -1: the row is empty; -2: it has its parent's pages
  int32_t* fresh;         // free pages, rising
};

// keys of row b's parent, and its whole pages among W columns
__device__ __forceinline__ int64_t parent_keys(const ForkArgs& a, int p) {
  const int64_t n = a.lens[p];
  return n > 0 ? n : 0;
}
__device__ __forceinline__ int whole_pages(int64_t keys, int block_size, int W) {
  const int64_t n = keys / block_size;
  return n < W ? (int)n : W;
}

__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(ForkArgs a, int pages, int block_size) {
  __shared__ uint32_t used[kMaxWords], red[kPlanWaves];
  __shared__ int32_t first[kMaxRows];
  __shared__ uint32_t need[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int words = (pages + 31) / 32;
  for (int i = tid; i < words; i += kPlanThreads) used[i] = 0;
  for (int b = tid; b < a.B; b += kPlanThreads) first[b] = a.B;
  __syncthreads();
  for (int b = tid; b < a.B; b += kPlanThreads) {
    const int p = a.parents[b];
    if (p >= 0 && p < a.B) atomicMin(&first[p], b);
  }
  mark_held(a.held, pages, used);
  __syncthreads();
  // a first child keeps its parent's pages; the others need one for each that is not whole
  for (int b = wave; b < a.B; b += kPlanWaves) {
    const int p = a.parents[b];
    const bool live = p >= 0 && p < a.B;
    const int32_t* row = a.tables + (int64_t)(live ? p : 0) * a.W;
    uint32_t n = 0;
    if (live && first[p] == b) {
      for (int j = lane; j < a.W; j += 64) {
        const int e = row[j];
        if (e >= 0 && e < pages) atomicOr(&used[e >> 5], 1u << (e & 31));
      }
    } else if (live) {
      for (int j = whole_pages(parent_keys(a, p), block_size, a.W) + lane; j < a.W; j += 64) {
        const int e = row[j];
        n += e >= 0 && e < pages;
      }
      n = (uint32_t)__shfl((int)scan_u32(n), 63);
    }
    if (lane == 0) need[b] = n;
  }
  __syncthreads();
  // free pages before each thread's words
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  uint32_t mine = 0, free_pages, wanted = 0;
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w < words) mine += __popc(~used[w] & word_mask(w, pages));
  }
  uint32_t rank = block_scan(mine, red, free_pages);
  // places of the rows' pages among the free ones, row by row
  const int rows = (a.B + kPlanThreads - 1) / kPlanThreads;
  for (int i = 0; i < rows; ++i)
    if (tid * rows + i < a.B) wanted += need[tid * rows + i];
  uint32_t all;
  uint32_t at = block_scan(wanted, red, all);
  for (int i = 0; i < rows; ++i) {
    const int b = tid * rows + i;
    if (b >= a.B) break;
    const int p = a.parents[b];
    const bool live = p >= 0 && p < a.B;
    const uint32_t n = need[b];
    a.base[b] = !live ? -1 : n == 0 ? -2 : at + n <= free_pages ? (int32_t)at : -1;
    at += n;
  }
  const uint32_t most = all < free_pages ? all : free_pages;
  for (int i = 0; i < per && rank < most; ++i) {
    const int w = tid * per + i;
    if (w >= words) break;
    for (uint32_t f = ~used[w] & word_mask(w, pages); f && rank < most; f &= f - 1) a.fresh[rank++] = 32 * w + __ffs((int)f) - 1;
  }
  if (tid == 0) *a.lacking = (int32_t)(all > free_pages ? all - free_pages : 0);
  __syncthreads();  // base and fresh, for the whole workgroup
  // pages to copy: a row's first new page, where its parent's was partly filled
  uint32_t copies = 0, many;
  for (int i = 0; i < rows; ++i) {
    const int b = tid * rows + i;
    if (b >= a.B || a.base[b] < 0) continue;
    const int64_t n = parent_keys(a, a.parents[b]);
    const int j = whole_pages(n, block_size, a.W);
    if (j >= a.W || n % block_size == 0) continue;
    const int e = a.tables[(int64_t)a.parents[b] * a.W + j];
    copies += e >= 0 && e < pages;
  }
  uint32_t to = block_scan(copies, red, many);
  for (int i = 0; i < rows; ++i) {
    const int b = tid * rows + i;
    if (b >= a.B || a.base[b] < 0) continue;
    const int64_t n = parent_keys(a, a.parents[b]);
    const int j = whole_pages(n, block_size, a.W);
    if (j >= a.W || n % block_size == 0) continue;
    const int e = a.tables[(int64_t)a.parents[b] * a.W + j];
    if (e < 0 || e >= pages) continue;
    a.src[to] = e;
    a.dst[to] = a.fresh[a.base[b]];
    a.keys[to++] = (int32_t)(n % block_size);
  }
  if (tid == 0) *a.count = (int32_t)many;
}

// A row of the new tables, by one wave.
__device__ __forceinline__ void fork_row(const ForkArgs& a, int b, int pages, int block_size) {
  const int lane = threadIdx.x & 63;
  const int base = a.base[b], p = a.parents[b];
  const int64_t keys = base == -1 ? 0 : parent_keys(a, p);
  const int whole = whole_pages(keys, block_size, a.W);
  int at = base;
  for (int j0 = 0; j0 < a.W; j0 += 64) {
    const int j = j0 + lane;
    int e = base != -1 && j < a.W ? a.tables[(int64_t)p * a.W + j] : -1;
    if (e >= pages || e < 0) e = -1;
    if (base >= 0) {
      const bool own = e >= 0 && j >= whole;
      const uint64_t owns = __ballot(own);
      if (own) e = a.fresh[at + __popcll(owns & ((1ull << lane) - 1))];
      at += __popcll(owns);
    }
    if (j < a.W) a.out_tables[(int64_t)b * a.W + j] = e;
  }
  if (lane == 0) a.out_lens[b] = keys;
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------
struct CompactArgs {
  const int32_t* tables;  // [B, W]
  const uint8_t* held;    // nullable [num_blocks]
  int64_t entries;        // B * W
  int32_t* out_tables;
  int32_t* new_ids;       // [num_blocks]
  int32_t* top;
  // workspace
  int32_t* count;         // moves
  int32_t* src;
  int32_t* dst;           // [num_blocks] each
};

// The i-th movable page from above goes to the i-th hole from below while that
// lies before it: a page moves iff more holes lie below it than movable pages
// above, a hole is filled iff more movable pages lie above it than holes below.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(CompactArgs a, int pages) {
  __shared__ uint32_t used[kMaxWords], keep[kMaxWords], red[kPlanWaves];
  __shared__ int top;
  const int tid = threadIdx.x;
  const int words = (pages + 31) / 32, per = (words + kPlanThreads - 1) / kPlanThreads;
  for (int i = tid; i < words; i += kPlanThreads) used[i] = keep[i] = 0;
  if (tid == 0) top = -1;
  __syncthreads();
  for (int64_t i = tid; i < a.entries; i += kPlanThreads) {
    const int e = a.tables[i];
    if (e >= 0 && e < pages) atomicOr(&used[e >> 5], 1u << (e & 31));
  }
  mark_held(a.held, pages, keep);
  __syncthreads();
  uint32_t mine = 0, empty = 0, movable, holes;
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w >= words) break;
    mine += __popc(used[w] & ~keep[w]);
    empty += __popc(~(used[w] | keep[w]) & word_mask(w, pages));
  }
  uint32_t before = block_scan(mine, red, movable);  // movable pages below
  uint32_t below = block_scan(empty, red, holes);    // holes below
  int high = -1;
  uint32_t moved = 0, moves;
  for (int i = 0; i < per; ++i) {
    const int w = tid * per + i;
    if (w >= words) break;
    const uint32_t u = used[w], k = keep[w];
    for (int bit = 0; bit < 32 && 32 * w + bit < pages; ++bit) {
      const int id = 32 * w + bit;
      const uint32_t m = 1u << bit;
      int at = id;  // where the page's content is afterwards
      if (u & m & ~k) {
        const uint32_t above = movable - before - 1;
        if (below > above) {
          a.src[above] = id;
          ++moved;
        } else {
          high = id;
        }
        ++before;
      } else if (k & m) {
        high = id;
      } else {
        at = -1;
        if (movable - before > below) {
          a.dst[below] = id;
          high = id;
        }
        ++below;
      }
      a.new_ids[id] = at;
    }
  }
  if (high >= 0) atomicMax(&top, high);
  block_scan(moved, red, moves);
  __syncthreads();  // the lists and new_ids, for the whole workgroup
  for (uint32_t i = tid; i < moves; i += kPlanThreads) a.new_ids[a.src[i]] = a.dst[i];
  if (tid == 0) {
    *a.count = (int32_t)moves;
    *a.top = top + 1;
  }
}

// ---------------------------------------------------------------------------
// moving
// ---------------------------------------------------------------------------

// Bytes [lo, hi) of a pool's page, copied from page src to page dst; of a page
// that is not whole, only those of its first `keys` keys.
__device__ __forceinline__ void copy_unit(const nsv_pool& pool, int block_size, int src, int dst, int keys, int64_t lo) {
  const int64_t seg = (int64_t)block_size * pool.key_bytes, page = seg * pool.segments;
  const int64_t hi = min(lo + (int64_t)kUnit, page), live = (int64_t)keys * pool.key_bytes;
  const char* from = (const char*)pool.base + (int64_t)src * page;
  char* to = (char*)pool.base + (int64_t)dst * page;
  const bool whole = keys >= block_size;
  const int tid = threadIdx.x;
  if (((page | (uintptr_t)pool.base) & 15) == 0 && (whole || (pool.segments == 1 && (live & 15) == 0))) {
    const int64_t end = whole ? hi : min(hi, live);
    u32x4 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = lo + 16 * (tid + i * kMoveThreads);
      if (at < end) v[i] = *reinterpret_cast<const u32x4*>(from + at);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = lo + 16 * (tid + i * kMoveThreads);
      if (at < end) *reinterpret_cast<u32x4*>(to + at) = v[i];
    }
  } else if (((pool.key_bytes | (uintptr_t)pool.base) & 3) == 0) {
    for (int64_t at = lo + 4 * tid; at < hi; at += 4 * kMoveThreads)
      if (at % seg < live) *reinterpret_cast<uint32_t*>(to + at) = *reinterpret_cast<const uint32_t*>(from + at);
  } else {
    for (int64_t at = lo + 2 * tid; at < hi; at += 2 * kMoveThreads)
      if (at % seg < live) *reinterpret_cast<uint16_t*>(to + at) = *reinterpret_cast<const uint16_t*>(from + at);
  }
}

__device__ __forceinline__ void move_pages(const Pools& p, const Moves& m) {
  const int units = p.first[p.n];
  const int64_t count = m.count ? min(*m.count, m.most) : m.most;
  for (int64_t at = blockIdx.x; at < count * units; at += gridDim.x) {
    const int64_t move = at / units;
    const int unit = (int)(at - move * units);
    int lo = 0, hi = p.n;  // the pool: first[lo] <= unit < first[lo + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.first[mid] <= unit) lo = mid;
      else hi = mid;
    }
    const int src = m.src[move], dst = m.dst[move];
    if (src < 0 || dst < 0 || src >= p.num_blocks || dst >= p.num_blocks || src == dst) continue;  // uniform
    const int keys = m.keys ? m.keys[move] : p.block_size;
    copy_unit(p.pool[lo], p.block_size, src, dst, keys, (int64_t)(unit - p.first[lo]) * kUnit);
  }
}

__global__ __launch_bounds__(kMoveThreads) void copy_pages_kernel(Pools p, Moves m) { move_pages(p, m); }

__global__ __launch_bounds__(kMoveThreads) void fork_move_kernel(Pools p, Moves m, ForkArgs a) {
  const int waves = gridDim.x * (kMoveThreads / 64);
  for (int b = blockIdx.x + gridDim.x * (threadIdx.x >> 6); b < a.B; b += waves) fork_row(a, b, p.num_blocks, p.block_size);
  move_pages(p, m);
}

__global__ __launch_bounds__(kMoveThreads) void compact_move_kernel(Pools p, Moves m, CompactArgs a) {
  for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * kMoveThreads) {
    const int e = a.tables[i];
    a.out_tables[i] = e >= 0 && e < p.num_blocks ? a.new_ids[e] : -1;
  }
  move_pages(p, m);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
size_t a256(size_t x) { return (x + 255) & ~(size_t)255; }

int check_pools(const nsv_pool* pools, int npools, int num_blocks, int block_size) {
  if (npools < 0 || (npools && !pools) || num_blocks <= 0 || block_size <= 0) return NSV_ERR_ARG;
  for (int i = 0; i < npools; ++i) {
    const nsv_pool& p = pools[i];
    if (!p.base || ((uintptr_t)p.base & 1) || p.segments <= 0 || p.key_bytes <= 0 || (p.key_bytes & 1)) return NSV_ERR_ARG;
    if ((int64_t)p.segments * p.key_bytes > (int64_t)(1 << 30) / block_size) return NSV_ERR_UNSUPPORTED;
  }
  return num_blocks > kMaxPages ? NSV_ERR_UNSUPPORTED : NSV_OK;
}

// the pools from `at` on that fit one launch
Pools take_pools(const nsv_pool* pools, int npools, int at, int num_blocks, int block_size) {
  Pools p{};
  p.n = npools - at < kPoolsPerLaunch ? npools - at : kPoolsPerLaunch;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  int64_t units = 0;
  for (int i = 0; i < p.n; ++i) {
    p.pool[i] = pools[at + i];
    p.first[i] = (int)units;
    const int64_t bytes = (int64_t)block_size * p.pool[i].segments * p.pool[i].key_bytes;
    units += (bytes + kUnit - 1) / kUnit;
  }
  p.first[p.n] = (int)units;
  return p;
}

int move_grid(const Pools& p, int64_t moves, int64_t tables) {
  const int64_t n = moves * p.first[p.n];
  const int64_t most = n > tables ? n : tables;
  return (int)(most < 1 ? 1 : most > kMoveGroups ? kMoveGroups : most);
}

struct ForkLayout {
  size_t count, src, dst, keys, base, fresh, total;
};
ForkLayout fork_layout(int B, int W, int num_blocks) {
  ForkLayout L;
  const int64_t fresh = (int64_t)B * W < num_blocks ? (int64_t)B * W : num_blocks;
  const size_t row = a256((size_t)B * 4);
  L.count = 0;
  L.src = 256;
  L.dst = L.src + row;
  L.keys = L.dst + row;
  L.base = L.keys + row;
  L.fresh = L.base + row;
  L.total = L.fresh + a256((size_t)fresh * 4);
  return L;
}

}  // namespace

extern "C" {

int nsv_copy_pages(const nsv_pool* pools, int npools, int num_blocks, int block_size, const int32_t* src, const int32_t* dst,
                   const int32_t* keys, int moves, void* stream) {
  const int bad = check_pools(pools, npools, num_blocks, block_size);
  if (bad) return bad;
  if (moves < 0) return NSV_ERR_ARG;
  if (moves == 0 || npools == 0) return NSV_OK;
  if (!src || !dst) return NSV_ERR_ARG;
  const Moves m{src, dst, keys, nullptr, moves};
  for (int at = 0; at < npools; at += kPoolsPerLaunch) {
    const Pools p = take_pools(pools, npools, at, num_blocks, block_size);
    hipLaunchKernelGGL(copy_pages_kernel, dim3(move_grid(p, moves, 1)), dim3(kMoveThreads), 0, (hipStream_t)stream, p, m);
    const int rc = nsv_launch_status();
    if (rc) return rc;
  }
  return NSV_OK;
}

size_t nsv_fork_pages_workspace_size(int B, int max_blocks, int num_blocks) {
  if (B <= 0 || B > kMaxRows || max_blocks <= 0 || num_blocks <= 0) return 0;
  return fork_layout(B, max_blocks, num_blocks).total;
}

int nsv_fork_pages(const nsv_pool* pools, int npools, int num_blocks, int block_size, const int32_t* block_tables,
                   const int64_t* context_lens, const int32_t* parents, const uint8_t* held, int B, int max_blocks,
                   int32_t* out_block_tables, int64_t* out_context_lens, int32_t* lacking, void* workspace,
                   size_t workspace_bytes, void* stream) {
  const int bad = check_pools(pools, npools, num_blocks, block_size);
  if (bad) return bad;
  if (B < 0 || max_blocks <= 0) return NSV_ERR_ARG;
  if (B > kMaxRows) return NSV_ERR_UNSUPPORTED;
  if (!lacking) return NSV_ERR_ARG;
  if (B > 0 && (!block_tables || !context_lens || !parents || !out_block_tables || !out_context_lens)) return NSV_ERR_ARG;
  // (a row of the new tables is written while others of the old are read)
  const int64_t entries = (int64_t)B * max_blocks;
  if (B > 0 && (out_block_tables < block_tables + entries && block_tables < out_block_tables + entries)) return NSV_ERR_ARG;
  if (B > 0 && (out_context_lens < context_lens + B && context_lens < out_context_lens + B)) return NSV_ERR_ARG;
  const ForkLayout L = fork_layout(B, max_blocks, num_blocks);
  if (!workspace || workspace_bytes < L.total) return NSV_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  ForkArgs a{};
  a.tables = block_tables;
  a.lens = context_lens;
  a.parents = parents;
  a.held = held;
  a.B = B;
  a.W = max_blocks;
  a.out_tables = out_block_tables;
  a.out_lens = out_context_lens;
  a.lacking = lacking;
  a.count = (int32_t*)(ws + L.count);
  a.src = (int32_t*)(ws + L.src);
  a.dst = (int32_t*)(ws + L.dst);
  a.keys = (int32_t*)(ws + L.keys);
  a.base = (int32_t*)(ws + L.base);
  a.fresh = (int32_t*)(ws + L.fresh);
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, num_blocks, block_size);
  int rc = nsv_launch_status();
  if (rc) return rc;
  const Moves m{a.src, a.dst, a.keys, a.count, B};
  for (int at = 0; at == 0 || at < npools; at += kPoolsPerLaunch) {
    const Pools p = take_pools(pools, npools, at, num_blocks, block_size);
    if (at == 0) hipLaunchKernelGGL(fork_move_kernel, dim3(move_grid(p, B, B)), dim3(kMoveThreads), 0, s, p, m, a);
    else hipLaunchKernelGGL(copy_pages_kernel, dim3(move_grid(p, B, 1)), dim3(kMoveThreads), 0, s, p, m);
    if ((rc = nsv_launch_status())) return rc;
  }
  return NSV_OK;
}

size_t nsv_compact_pages_workspace_size(int num_blocks) {
  if (num_blocks <= 0 || num_blocks > kMaxPages) return 0;
  return 256 + 2 * a256((size_t)num_blocks * 4);
}

int nsv_compact_pages(const nsv_pool* pools, int npools, int num_blocks, int block_size, const int32_t* block_tables,
                      const uint8_t* held, int B, int max_blocks, int32_t* out_block_tables, int32_t* new_ids, int32_t* top,
                      void* workspace, size_t workspace_bytes, void* stream) {
  const int bad = check_pools(pools, npools, num_blocks, block_size);
  if (bad) return bad;
  if (B < 0 || max_blocks <= 0 || !new_ids || !top) return NSV_ERR_ARG;
  if (B > 0 && (!block_tables || !out_block_tables)) return NSV_ERR_ARG;
  const int64_t entries = (int64_t)B * max_blocks;
  // (the same tables are written place by place, others may not overlap them)
  if (out_block_tables != block_tables && out_block_tables < block_tables + entries &&
      block_tables < out_block_tables + entries)
    return NSV_ERR_ARG;
  if (!workspace || workspace_bytes < nsv_compact_pages_workspace_size(num_blocks)) return NSV_ERR_WORKSPACE;
  char* ws = (char*)workspace;
  CompactArgs a{};
  a.tables = block_tables;
  a.held = held;
  a.entries = entries;
  a.out_tables = out_block_tables;
  a.new_ids = new_ids;
  a.top = top;
  a.count = (int32_t*)ws;
  a.src = (int32_t*)(ws + 256);
  a.dst = (int32_t*)(ws + 256 + a256((size_t)num_blocks * 4));
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, a, num_blocks);
  int rc = nsv_launch_status();
  if (rc) return rc;
  // (at most half of the pages move)
  const Moves m{a.src, a.dst, nullptr, a.count, num_blocks};
  for (int at = 0; at == 0 || at < npools; at += kPoolsPerLaunch) {
    const Pools p = take_pools(pools, npools, at, num_blocks, block_size);
    const int64_t moves = num_blocks / 2;
    if (at == 0)
      hipLaunchKernelGGL(compact_move_kernel, dim3(move_grid(p, moves, (entries + kMoveThreads - 1) / kMoveThreads)),
                         dim3(kMoveThreads), 0, s, p, m, a);
    else hipLaunchKernelGGL(copy_pages_kernel, dim3(move_grid(p, moves, 1)), dim3(kMoveThreads), 0, s, p, m);
    if ((rc = nsv_launch_status())) return rc;
  }
  return NSV_OK;
}

}  // extern "C"
