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
constexpr int kMaxPages = 1 << 18;            // two bits each in LDS, and two counts per 32: 128 KiB
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
  const int32_t* via;    // nullable: dst holds places of this list
};

// exclusive prefix over the workgroup, and the whole sum
template <typename T>
__device__ __forceinline__ T block_scan(T v, uint64_t* red, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T in = wave_scan(v);
  __syncthreads();
  if (lane == 63) red[wave] = in;
  __syncthreads();
  const uint64_t waves = lane < kPlanWaves ? red[lane] : 0ull, upto = wave_scan(waves);
  total = (T)lane_u64(upto, 63);
  return (T)lane_u64(upto - waves, wave) + in - v;
}

// the pages of a word that exist
__device__ __forceinline__ uint32_t word_mask(int w, int pages) {
  const int left = pages - 32 * w;
  return left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
}

// bits of the held pages, 64 of a wave at a time
__device__ __forceinline__ void mark_held(const uint8_t* held, int pages, uint32_t* bits) {
  if (!held) return;
  const int lane = threadIdx.x & 63;
#pragma unroll 4
  for (int first = threadIdx.x - lane; first < pages; first += kPlanThreads) {
    const uint64_t m = __ballot(held[min(first + lane, pages - 1)] != 0 && first + lane < pages);
    const uint32_t half = lane ? (uint32_t)(m >> 32) : (uint32_t)m;
    if (lane < 2 && half) atomicOr(&bits[(first >> 5) + lane], half);
  }
}

// the n-th set bit
__device__ __forceinline__ int nth_bit(uint32_t f, uint32_t n) {
  int at = 0;
#pragma unroll
  for (int h = 16; h; h >>= 1) {
    const uint32_t c = __popc(f & ((1u << h) - 1));
    if (n >= c) {
      n -= c;
      at += h;
      f >>= h;
    }
  }
  return at;
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
  int32_t* dst;           // (places of `fresh`)
  int32_t* keys;          // [B] each
  int32_t* base;          // [B] a row's first place in `fresh`; -1: the row is empty; -2: it has its parent's pages
  int32_t* fresh;         // free pages, rising
};

// How keys fill a row of W pages: whole pages, and the keys of the one behind
// them (0 where the row ends with them).
struct Filled {
  int whole, rest;
};
__device__ __forceinline__ Filled filled(int64_t keys, int block_size, int W) {
  const int64_t room = (int64_t)W * block_size;
  if (keys <= 0) return {0, 0};
  if (keys >= room) return {W, 0};
  if (room <= 0x7fffffff) {  // uniform (a 64-bit division is some 150 instructions)
    const uint32_t k = (uint32_t)keys, q = k / (uint32_t)block_size;
    return {(int)q, (int)(k - q * (uint32_t)block_size)};
  }
  return {(int)(keys / block_size), (int)(keys % block_size)};
}

// 4 rows 4.2 us, 64 rows of 128 pages 7.0: some ten barriers and three round trips
// to memory.  One workgroup, since places among the free pages follow from all
// rows before; a wave per row, four rows of loads at a time.
__global__ __launch_bounds__(kPlanThreads) void fork_plan_kernel(ForkArgs a, int pages, int block_size) {
  __shared__ uint32_t used[kMaxWords], before[kMaxWords];
  __shared__ uint64_t red[kPlanWaves];
  __shared__ int32_t first[kMaxRows], parent[kMaxRows], partly[kMaxRows], rest[kMaxRows];
  __shared__ uint32_t need[kMaxRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int words = (pages + 31) / 32;
  for (int b = tid; b < a.B; b += kPlanThreads) {
    const int p = a.parents[b];
    parent[b] = p >= 0 && p < a.B ? p : -1;
    first[b] = a.B;
  }
  for (int i = tid; i < words; i += kPlanThreads) used[i] = 0;
  __syncthreads();
  for (int b = tid; b < a.B; b += kPlanThreads)
    if (parent[b] >= 0) atomicMin(&first[parent[b]], b);
  mark_held(a.held, pages, used);
  __syncthreads();
  // a first child keeps its parent's pages; the others need one for each that
  // is not whole.  Four rows of a wave and 128 columns at a time, their loads
  // beside each other.
  constexpr int kAtOnce = 4;
  for (int b0 = wave; b0 < a.B; b0 += kAtOnce * kPlanWaves) {
    int64_t keys[kAtOnce];
    Filled fill[kAtOnce];
    int p[kAtOnce], src[kAtOnce];  // src: the partly filled page that a row copies
    uint32_t n[kAtOnce] = {};
    for (int j0 = 0; j0 < a.W; j0 += 128) {
      int e[kAtOnce][2];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int b = b0 + i * kPlanWaves;
        if (j0 == 0) {
          p[i] = b < a.B ? parent[b] : -1;
          src[i] = -1;
        }
        const int row = max(p[i], 0);
        if (j0 == 0) keys[i] = a.lens[row];
#pragma unroll
        for (int h = 0; h < 2; ++h) e[i][h] = a.tables[(int64_t)row * a.W + min(j0 + 64 * h + lane, a.W - 1)];
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (p[i] < 0) continue;  // uniform
        const bool keeps = first[p[i]] == b0 + i * kPlanWaves;
        if (j0 == 0) fill[i] = filled(keys[i], block_size, a.W);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = j0 + 64 * h + lane, id = e[i][h];
          if (j >= a.W || id < 0 || id >= pages) continue;
          if (keeps) atomicOr(&used[id >> 5], 1u << (id & 31));
          else n[i] += j >= fill[i].whole;
          if (!keeps && j == fill[i].whole && fill[i].rest) src[i] = id;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int b = b0 + i * kPlanWaves;
      if (b >= a.B) break;  // uniform
      const uint32_t all = lane_u32(wave_scan(n[i]), 63);
      const uint64_t has = __ballot(src[i] >= 0);
      const int one = has ? (int)lane_u32((uint32_t)src[i], __ffsll((long long)has) - 1) : -1;
      if (lane == 0) {
        need[b] = all;
        partly[b] = one;
        rest[b] = p[i] >= 0 ? fill[i].rest : 0;
      }
    }
  }
  __syncthreads();
  auto is_free = [&](int w) { return ~used[w] & word_mask(w, pages); };
  // the free pages before each word, and places of the rows' pages among them, row by row
  const int per = (words + kPlanThreads - 1) / kPlanThreads, w0 = tid * per, w1 = min(w0 + per, words);
  const int rows = (a.B + kPlanThreads - 1) / kPlanThreads, r0 = tid * rows, r1 = min(r0 + rows, a.B);
  uint64_t mine = 0, both;
  for (int w = w0; w < w1; ++w) mine += __popc(is_free(w));
  for (int b = r0; b < r1; ++b) mine += (uint64_t)need[b] << 32;
  const uint64_t places = block_scan(mine, red, both);
  const uint32_t free_pages = (uint32_t)both, all = (uint32_t)(both >> 32);
  uint32_t below = (uint32_t)places, at = (uint32_t)(places >> 32), copies = 0, many;
  for (int w = w0; w < w1; ++w) {
    before[w] = below;
    below += __popc(is_free(w));
  }
  const uint32_t start = at;
  for (int b = r0; b < r1; ++b) {
    at += need[b];
    copies += partly[b] >= 0 && at <= free_pages;
  }
  uint32_t to = block_scan(copies, red, many);
  at = start;
  for (int b = r0; b < r1; ++b) {
    const uint32_t n = need[b];
    const bool fits = at + n <= free_pages;
    a.base[b] = parent[b] < 0 ? -1 : n == 0 ? -2 : fits ? (int32_t)at : -1;
    if (partly[b] >= 0 && fits) {  // the row's first new page, of its parent's partly filled one
      a.src[to] = partly[b];
      a.dst[to] = (int32_t)at;
      a.keys[to++] = rest[b];
    }
    at += n;
  }
  const uint32_t most = all < free_pages ? all : free_pages;
  for (int id = tid; id < pages && before[id >> 5] < most; id += kPlanThreads) {  // (rising: none behind the last that is wanted)
    const uint32_t f = is_free(id >> 5), rank = before[id >> 5] + __popc(f & ((1u << (id & 31)) - 1));
    if (((f >> (id & 31)) & 1) && rank < most) a.fresh[rank] = id;
  }
  if (tid == 0) {
    *a.lacking = (int32_t)(all > free_pages ? all - free_pages : 0);
    *a.count = (int32_t)many;
  }
}

// A row of the new tables, by one wave.
__device__ __forceinline__ void fork_row(const ForkArgs& a, int b, int pages, int block_size) {
  const int lane = threadIdx.x & 63;
  const int base = a.base[b], p = a.parents[b];
  const int64_t keys = base == -1 ? 0 : a.lens[p] > 0 ? a.lens[p] : 0;
  const int whole = filled(keys, block_size, a.W).whole;
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
// 8 sequences of some 40 pages 4.0 us: six barriers and two round trips; a thread per
// page, its move worked out from the counts per word without a list of holes.
__global__ __launch_bounds__(kPlanThreads) void compact_plan_kernel(CompactArgs a, int pages) {
  __shared__ uint32_t used[kMaxWords], keep[kMaxWords], below_m[kMaxWords], below_h[kMaxWords];
  __shared__ uint64_t red[kPlanWaves];
  __shared__ int top, moves;
  const int tid = threadIdx.x;
  const int words = (pages + 31) / 32;
  for (int i = tid; i < words; i += kPlanThreads) used[i] = keep[i] = 0;
  if (tid == 0) {
    top = -1;
    moves = 0;
  }
  __syncthreads();
#pragma unroll 4
  for (int64_t i = tid; i < a.entries; i += kPlanThreads) {
    const int e = a.tables[i];
    if (e >= 0 && e < pages) atomicOr(&used[e >> 5], 1u << (e & 31));
  }
  mark_held(a.held, pages, keep);
  __syncthreads();
  // movable pages and holes before each word
  const int per = (words + kPlanThreads - 1) / kPlanThreads, w0 = tid * per, w1 = min(w0 + per, words);
  auto counts = [&](int w) {
    return ((uint64_t)__popc(used[w] & ~keep[w]) << 32) | __popc(~(used[w] | keep[w]) & word_mask(w, pages));
  };
  uint64_t mine = 0, all;
  for (int w = w0; w < w1; ++w) mine += counts(w);
  uint64_t below_w = block_scan(mine, red, all);
  for (int w = w0; w < w1; ++w) {
    below_m[w] = (uint32_t)(below_w >> 32);
    below_h[w] = (uint32_t)below_w;
    below_w += counts(w);
  }
  __syncthreads();
  const uint32_t movable = (uint32_t)(all >> 32);
  int high = -1, moved = 0;  // of the wave
  for (int id = tid; id < pages; id += kPlanThreads) {
    const int w = id >> 5;
    const uint32_t u = used[w], k = keep[w], bit = 1u << (id & 31), low = bit - 1;
    const uint32_t below = below_h[w] + __popc(~(u | k) & low);                 // holes
    const uint32_t above = movable - below_m[w] - __popc(u & ~k & (low | bit));  // movable pages
    int at = id;  // where the page's content is afterwards
    bool taken = true;  // whether the place is in use then
    if (u & bit & ~k) {
      if (below > above) {
        // hole number `above`: the last word with no more holes before it, then its bit
        int lo = 0, hi = w + 1;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (below_h[mid] <= above) lo = mid;
          else hi = mid;
        }
        at = 32 * lo + nth_bit(~(used[lo] | keep[lo]), above - below_h[lo]);
        a.src[above] = id;
        a.dst[above] = at;
        taken = false;
      }
    } else if (!(k & bit)) {
      at = -1;
      taken = above > below;
    }
    a.new_ids[id] = at;
    const uint64_t t = __ballot(taken);
    if (t) high = (id & ~63) + 63 - __clzll((long long)t);
    moved += __popcll(__ballot(at >= 0 && at != id));
  }
  if ((tid & 63) == 0) {
    if (high >= 0) atomicMax(&top, high);
    if (moved) atomicAdd(&moves, moved);
  }
  __syncthreads();
  if (tid == 0) {
    *a.count = moves;
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
    const int src = m.src[move], to = m.dst[move], dst = m.via ? m.via[to] : to;
    if (src < 0 || dst < 0 || src >= p.num_blocks || dst >= p.num_blocks || src == dst) continue;  // uniform
    const int keys = m.keys ? m.keys[move] : p.block_size;
    copy_unit(p.pool[lo], p.block_size, src, dst, keys, (int64_t)(unit - p.first[lo]) * kUnit);
  }
}

// Bound by memory where there is much to move: 41.7 MB compacted in 15.0 us, 5.6
// TB/s read and written; 22 MB of a fork in 6.3, 1.5 MB in 3.7.  A workgroup
// copies 8 KiB at a time, so few pages still spread over the chip.
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
  const Moves m{src, dst, keys, nullptr, moves, nullptr};
  for (int at = 0; at < npools; at += kPoolsPerLaunch) {
    const Pools p = take_pools(pools, npools, at, num_blocks, block_size);
    hipLaunchKernelGGL(copy_pages_kernel, dim3(move_grid(p, moves, 1)), dim3(kMoveThreads), 0, (hipStream_t)stream, p, m);
    const int rc = nsv_launch_status();
    if (rc) return rc;
  }
  return NSV_OK;
}

size_t nsv_fork_pages_workspace_size(int B, int max_blocks, int num_blocks) {
  if (B < 0 || B > kMaxRows || max_blocks <= 0 || num_blocks <= 0) return 0;
  return fork_layout(B, max_blocks, num_blocks).total;
}

int nsv_fork_pages(const nsv_pool* pools, int npools, int num_blocks, int block_size, const int32_t* block_tables,
                   const int64_t* context_lens, const int32_t* parents, const uint8_t* held, int B, int max_blocks,
                   int32_t* out_block_tables, int64_t* out_context_lens, int32_t* lacking, void* workspace,
                   size_t workspace_bytes, void* stream) {
  const int bad = check_pools(pools, npools, num_blocks, block_size);
  if (bad) return bad;
  if (B < 0 || max_blocks <= 0) return NSV_ERR_ARG;
  if (B > kMaxRows || (int64_t)B * max_blocks > 0x7fffffff) return NSV_ERR_UNSUPPORTED;  // (entries are counted in 32 bits)
  if (!lacking) return NSV_ERR_ARG;
  if (B > 0 && (!block_tables || !context_lens || !parents || !out_block_tables || !out_context_lens)) return NSV_ERR_ARG;
  // (a row of the new tables is written while others of the old are read)
  const int64_t entries = (int64_t)B * max_blocks;
  if (B > 0 && (out_block_tables < block_tables + entries && block_tables < out_block_tables + entries)) return NSV_ERR_ARG;
  if (B > 0 && (out_context_lens < context_lens + B && context_lens < out_context_lens + B)) return NSV_ERR_ARG;
  const ForkLayout L = fork_layout(B, max_blocks, num_blocks);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < L.total) return NSV_ERR_WORKSPACE;
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
  const Moves m{a.src, a.dst, a.keys, a.count, B, a.fresh};
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
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < nsv_compact_pages_workspace_size(num_blocks))
    return NSV_ERR_WORKSPACE;
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
  const Moves m{a.src, a.dst, nullptr, a.count, num_blocks, nullptr};
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
