// Eviction from a paged cache by accumulated attention weight, for gfx950.
//
// Of every (sequence, kv head) with more than `budget` keys, budget stay: the
// first `sinks`, the last `recent` and, of the rest, those with the most
// weight (of equal ones the lower position; NaN counts as -inf).  Their K, V
// and weight rows move to the front, in the order of their positions, of the
// sequence's own table or of another.
//
// Selection (evict_select_kernel), one workgroup of 16 waves per (sequence, kv
// head): the weights are read once into registers, four neighbours per load
// (beyond 32,768 keys, and of pages of fewer than four keys, they are read again
// in every pass: 131,072 keys of 8 heads 135 us), and compared as unsigned words of the same order, in which the
// keys that stay anyway are the largest.  The budget-th largest word comes from
// three passes over 11, 11 and 10 bits (four histograms, taken by a wave's lanes
// in turn: weights share few leading digits, and equal adds wait for one
// another); then each wave counts, per load, what lies above that word and
// what equals it, a scan over those counts gives every kept key its place, and
// keys and weights go there by way of LDS, so that they are written by full
// waves.  Bound by its passes' latency (two round trips, some 15 barriers) and
// above 10,000 keys by the histograms' adds and the words' comparisons.
//
// Moving (evict_move_kernel): every kept row read and written once.  Within a
// table rows move forward only: row i comes from kept[i] >= i.  A workgroup
// owns a column of one (sequence, kv head, K or V), all of the row or 64 or
// 128 bytes of it where there are few sequences, and takes its rows in
// ascending chunks, each read whole before it is written and the next one's
// reads under way: what a chunk overwrites no later chunk reads, and no other
// workgroup touches the column.  Between tables that share no page nothing can
// be overwritten, and the rows are dealt to many workgroups; so they are where
// few sequences have long rows to move, by way of staging rows.  A second table
// may also be a copy of the first, or keep some of its pages at their places:
// every workgroup compares the two, and such a sequence is moved as in place.
// Bound by the rows' bytes.
//
// Measured on MI355X: one sequence, 1,250 -> 512 keys of 8 heads, bf16, D 128,
// to pages apart: 9.0 us of selection, 3.5 of moving; 16 sequences of 16k-32k
// -> 2,048 keys in place: 23.5 and 56 (268 MB read and written, 4.8 TB/s; a large
// copy 4.8).  The selection took 36 of the latter with every page looked up
// before its weights and again at each kept key's place, kept keys written from
// where they were found, and one histogram per wave; 50 with the words made
// anew in each pass, 128 with one serial scan per pass.

#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelLoads = 8;     // loads of four weights that a thread holds: 32,768 keys in all
constexpr int kBins = 2048, kCopies = 4;
constexpr int kAgain = 4;        // loads in a round trip where the weights are read again
constexpr int kOutPages = 4096;  // entries of the destination's table held in LDS
constexpr int kMoveThreads = 512;
constexpr int kMoveUnroll = 8;   // 16-byte pieces per lane and chunk

struct EvictArgs {
  char* k;
  char* v;
  float* weights;                // [num_blocks][Hkv][block_size]
  const int32_t* block_tables;
  const int32_t* out_tables;
  const int64_t* context_lens;
  int64_t* lens;                 // [B]
  int32_t* kept;                 // [B][Hkv][budget]
  int Hkv, row_bytes, bs_log2, max_blocks, out_blocks, budget, sinks, recent;
  int vector;                    // four weights of a page in one load
  int apart;                     // out_tables is another table
  char* staged;                  // null, or [B][Hkv][2][budget] rows: K, V by way of it
};

__device__ __forceinline__ int clamp_len(const EvictArgs& a, int b) {
  const int64_t len = a.context_lens[b], cap = (int64_t)a.max_blocks << a.bs_log2;
  return (int)(len < 0 ? 0 : (len < cap ? len : cap));
}

// A weight as an unsigned word of the same order (-0 as 0, NaN as -inf).
__device__ __forceinline__ uint32_t ordered(float f) {
  uint32_t u = __float_as_uint(f);
  if (f != f) u = 0xff800000u;
  if (u == 0x80000000u) u = 0u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The wave's loads have returned (a barrier alone orders their issue).
__device__ __forceinline__ void loads_back() { __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ __forceinline__ int wave_scan(int v) {  // the sum over the lanes up to this one
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// HELD: every weight of a context fits the workgroup's registers, and so do
// their words.
template <bool HELD>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  constexpr int STEP = kSelThreads * 4;  // keys per load of the workgroup
  __shared__ __attribute__((aligned(16))) int hist[3][kBins][kCopies];  // one per pass
  __shared__ __attribute__((aligned(16))) int wave_sum[kSelWaves];
  __shared__ int out_page[HELD ? kOutPages : 1];
  __shared__ int digit, rest, share;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x - b * a.Hkv;
  const int n = clamp_len(a, b), got = min(n, a.budget);
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int32_t* bt = a.block_tables + (int64_t)b * a.max_blocks;
  const int32_t* ot = a.out_tables + (int64_t)b * a.out_blocks;
  const bool apart = a.apart != 0;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  auto at = [&](int page, int key) {  // the weight of a key there (of a hole: page 0's)
    return a.weights + ((((int64_t)max(page, 0) * a.Hkv + h) << a.bs_log2) + (key & bs_mask));
  };
  if (tid == 0 && h == 0) a.lens[b] = got;
  for (int i = got + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
  if (n <= a.budget && !apart) {  // uniform: nothing moves
    for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
    return;
  }

  // The weights of keys key[u] .. key[u] + 3 (multiples of 4), 0 in a hole, past
  // the context whatever: every page in one round trip, then every weight.  (Past
  // the context the last key's are loaded, of a hole page 0's: a load under a
  // condition would be waited for there.)
  auto fetch = [&](const auto& key, auto& x, auto count) {
    constexpr int U = decltype(count)::value;
    if (a.vector) {  // uniform: pages of four keys or more, on 16 bytes
      int page[U];
#pragma unroll
      for (int u = 0; u < U; ++u) page[u] = bt[min(key[u], n - 1) >> a.bs_log2];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const f32x4*>(at(page[u], min(key[u], (n - 1) & ~3)));
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = page[u] >= 0 ? x[u][j] : 0.f;
    } else {
      int page[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) page[u][j] = bt[min(key[u] + j, n - 1) >> a.bs_log2];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = *at(page[u][j], min(key[u] + j, n - 1));
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[u][j] = page[u][j] >= 0 ? x[u][j] : 0.f;
    }
  };
  // words of keys key .. key + 3: the largest for keys that stay anyway, 0 (less than every weight's) past the context
  auto words = [&](int key, f32x4 x) {
    u32x4 u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[j] = key + j < a.sinks || key + j >= n - a.recent ? 0xffffffffu : ordered(x[j]);
      u[j] = key + j < n ? u[j] : 0u;
    }
    return u;
  };
  const int loads = (n + STEP - 1) / STEP;
  f32x4 held[HELD ? kSelLoads : 1];
  u32x4 word[HELD ? kSelLoads : 1];
  uint32_t mapped = 0;  // HELD: bit e: load e has a page
  if constexpr (HELD) {  // every page in one round trip, then every weight (a.vector holds)
    int page[kSelLoads];
#pragma unroll
    for (int e = 0; e < kSelLoads; ++e)
      if (e < loads) page[e] = bt[min(e * STEP + tid * 4, n - 1) >> a.bs_log2];  // uniform
#pragma unroll
    for (int e = 0; e < kSelLoads; ++e)
      if (e < loads) {  // (past the context the last key's group, of a hole page 0: a load under a condition would be waited for)
        const int key = min(e * STEP + tid * 4, (n - 1) & ~3);
        held[e] = *reinterpret_cast<const f32x4*>(at(page[e], key));
        mapped |= page[e] >= 0 ? 1u << e : 0u;
      }
  }
  if constexpr (HELD) {
    const int pages = got > 0 ? ((got - 1) >> a.bs_log2) + 1 : 0;
    for (int i = tid; i < min(pages, kOutPages); i += kSelThreads) out_page[i] = ot[i];
  }
  for (int i = tid; i < 3 * kCopies * kBins / 4; i += kSelThreads)  // (while the weights are under way)
    reinterpret_cast<u32x4*>(&hist[0][0][0])[i] = u32x4{0u, 0u, 0u, 0u};
  if constexpr (HELD) {
#pragma unroll
    for (int e = 0; e < kSelLoads; ++e)
      if (e < loads) {
#pragma unroll
        for (int j = 0; j < 4; ++j) held[e][j] = (mapped >> e) & 1 ? held[e][j] : 0.f;
        word[e] = words(e * STEP + tid * 4, held[e]);
      }
  }
  auto each = [&](auto f) {  // f(e, first key, weights, words) for every load
    if constexpr (HELD) {
#pragma unroll
      for (int e = 0; e < kSelLoads; ++e)
        if (e < loads) {  // uniform
          // (nothing derived from these is kept from one use to the next: registers)
          int key = e * STEP + tid * 4;
          __asm__ volatile("" : "+v"(word[e]), "+v"(key));
          f(e, key, held[e], word[e]);
        }
    } else {
      for (int e0 = 0; e0 < loads; e0 += kAgain) {
        int key[kAgain];
        f32x4 x[kAgain];
#pragma unroll
        for (int u = 0; u < kAgain; ++u) key[u] = (e0 + u) * STEP + tid * 4;
        fetch(key, x, std::integral_constant<int, kAgain>{});
#pragma unroll
        for (int u = 0; u < kAgain; ++u)
          if (e0 + u < loads) f(e0 + u, key[u], x[u], words(key[u], x[u]));  // uniform
      }
    }
  };
  __syncthreads();

  // ---- the got-th largest word: its leading bits `prefix` down to bit `low`,
  // and how many of the words that share them stay (all of them, if low > 0)
  uint32_t prefix = 0;
  int want = n > a.budget ? got : 0, low = 0;
  if (n > a.budget) {  // uniform
    int above_bits = 32;  // leading bits not yet told apart end here
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bits = above_bits - shift;
      int* mine = hist[pass][0] + (lane & (kCopies - 1));
      const uint32_t head = pass == 0 ? 0u : prefix >> above_bits;
      each([&](int, int, f32x4, u32x4 u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (pass > 0 && (u[j] >> above_bits) != head) continue;
          atomicAdd(&mine[((u[j] >> shift) & ((1u << bits) - 1)) * kCopies], 1);
        }
      });
      __syncthreads();
      // two bins per thread, from the top: what lies above them
      const int top = kBins - 1 - 2 * tid;
      int c1 = 0, c0 = 0;
#pragma unroll
      for (int k = 0; k < kCopies; k += 4) {
        const int4 x = *reinterpret_cast<const int4*>(&hist[pass][top - 1][k]);
        const int4 y = *reinterpret_cast<const int4*>(&hist[pass][top][k]);
        c0 += x.x + x.y + x.z + x.w;
        c1 += y.x + y.y + y.z + y.w;
      }
      const int sum = wave_scan(c1 + c0);
      if (lane == 63) wave_sum[w] = sum;
      __syncthreads();
      int above = sum - c1 - c0;
#pragma unroll
      for (int ww = 0; ww < kSelWaves; ww += 4) {
        const int4 x = *reinterpret_cast<const int4*>(&wave_sum[ww]);
        above += (ww < w ? x.x : 0) + (ww + 1 < w ? x.y : 0) + (ww + 2 < w ? x.z : 0) + (ww + 3 < w ? x.w : 0);
      }
      if (above < want && above + c1 + c0 >= want) {  // one thread
        const bool first = above + c1 >= want;
        digit = first ? top : top - 1;
        rest = first ? want - above : want - above - c1;
        share = first ? c1 : c0;
      }
      __syncthreads();
      prefix |= (uint32_t)digit << shift;
      want = rest;
      above_bits = shift;
      if (want == share) {  // uniform: every word that shares them stays
        low = shift;
        break;
      }
    }
  }
  // (a context that is short enough: every weight's word is above 0, and stays)

  // ---- places: the kept keys before each wave's four-key groups of each load, by a scan over counts in LDS
  const uint32_t least = prefix, most = prefix | ((1u << low) - 1);  // (low < 32) words that tie: least .. most
  int* count_gt = &hist[0][0][0];  // [load][wave]
  int* count_eq = &hist[0][kBins / 2][0];
  // of a lane's four words: those above the tie, and from it up (<< 16)
  auto counts = [&](u32x4 u) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) c += (u[j] > most ? 1 : 0) + (u[j] >= least ? 1 << 16 : 0);
    return c;
  };
  // f(j, place) for those of a lane's keys that stay, after the wave's at_gt above the tie and at_eq tied ones
  auto emit = [&](u32x4 u, int at_gt, int at_eq, int before, auto f) {
    int g = at_gt + (before & 0xffff), q = at_eq + (before >> 16) - (before & 0xffff);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool gt = u[j] > most, eq = u[j] >= least && !gt;
      if (gt || (eq && q < want)) f(j, g + min(q, want));
      g += gt;
      q += eq;
    }
  };
  constexpr int GROUP = kBins / kSelWaves;  // loads whose counts fit at a time
  int base_gt = 0, base_eq = 0;
  int before[HELD ? kSelLoads : 1];  // the wave's counts of a load before this lane's keys
  for (int e0 = 0; e0 < loads; e0 += GROUP) {  // (one turn up to 524,288 keys)
    __syncthreads();
    each([&](int e, int, f32x4, u32x4 u) {
      if (e < e0 || e >= e0 + GROUP) return;  // uniform
      const int own = counts(u), upto = wave_scan(own);
      if constexpr (HELD) before[e] = upto - own;
      if (lane == 63) {
        count_gt[(e - e0) * kSelWaves + w] = upto & 0xffff;
        count_eq[(e - e0) * kSelWaves + w] = (upto >> 16) - (upto & 0xffff);
      }
    });
    __syncthreads();
    const int m = min(GROUP, loads - e0) * kSelWaves;
    if (w == 0) {  // exclusive scan of the counts, 64 at a time
      int run_gt = base_gt, run_eq = base_eq;
      for (int i0 = 0; i0 < m; i0 += 64) {
        const int i = i0 + lane;
        const int g = i < m ? count_gt[i] : 0, q = i < m ? count_eq[i] : 0;
        const int sg = wave_scan(g), sq = wave_scan(q);
        if (i < m) {
          count_gt[i] = run_gt + sg - g;
          count_eq[i] = run_eq + sq - q;
        }
        run_gt += __builtin_amdgcn_readlane(sg, 63);
        run_eq += __builtin_amdgcn_readlane(sq, 63);
      }
      if (lane == 0) {
        wave_sum[0] = run_gt;
        wave_sum[1] = run_eq;
      }
    }
    __syncthreads();
    base_gt = wave_sum[0];
    base_eq = wave_sum[1];
    if constexpr (!HELD) {
      each([&](int e, int key, f32x4, u32x4 u) {
        if (e < e0 || e >= e0 + GROUP) return;  // uniform
        const int c = (e - e0) * kSelWaves + w, own = counts(u);
        emit(u, count_gt[c], count_eq[c], wave_scan(own) - own, [&](int j, int i) { kept[i] = key + j; });
      });
    }
  }
  if constexpr (HELD) {
    // By way of LDS, kPlaces at a time, so that the lanes that write are all
    // busy: few of a load's keys stay.  (Every weight of the context is in
    // registers: places may be overwritten.)
    constexpr int kPlaces = 2 * kCopies * kBins / 2;  // (two histograms, two words a place)
    int2* list = reinterpret_cast<int2*>(&hist[1][0][0]);  // (key, or ~key where it has no page; weight)
    for (int i0 = 0; i0 < got; i0 += kPlaces) {
      each([&](int e, int key, f32x4 x, u32x4 u) {
        emit(u, count_gt[e * kSelWaves + w], count_eq[e * kSelWaves + w], before[e], [&](int j, int i) {
          if ((unsigned)(i - i0) < (unsigned)kPlaces)
            list[i - i0] = make_int2((mapped >> e) & 1 ? key + j : ~(key + j), __float_as_int(x[j]));
        });
      });
      __syncthreads();
      for (int i = i0 + tid; i < min(got, i0 + kPlaces); i += kSelThreads) {
        const int2 x = list[i - i0];
        kept[i] = x.x < 0 ? ~x.x : x.x;
        const int pi = i >> a.bs_log2;
        const int p = pi < kOutPages ? out_page[pi] : ot[pi];
        if (x.x >= 0 && p >= 0) *at(p, i) = __int_as_float(x.y);
      }
      if (i0 + kPlaces < got) __syncthreads();
    }
  }
  if constexpr (!HELD) {
    // the weights themselves, a chunk at a time: every read of a chunk before its first write
    __syncthreads();
    for (int i0 = 0; i0 < got; i0 += kSelThreads * kMoveUnroll) {
      int key[kMoveUnroll], from[kMoveUnroll], to[kMoveUnroll];
      float x[kMoveUnroll];
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u) key[u] = kept[min(i0 + u * kSelThreads + tid, got - 1)];
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u) {
        from[u] = bt[key[u] >> a.bs_log2];
        to[u] = ot[min(i0 + u * kSelThreads + tid, got - 1) >> a.bs_log2];
      }
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u) x[u] = *at(from[u], key[u]);
      loads_back();
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u) {
        const int i = i0 + u * kSelThreads + tid;
        if (i < got && from[u] >= 0 && to[u] >= 0) *at(to[u], i) = x[u];
      }
      __syncthreads();
    }
  }
}

// grid: (sequence, kv head, column) x (K, V) x rows (1 workgroup in place).
// TO_STAGED: kept rows to the staging rows; FROM_STAGED: those to the table;
// neither: at once.
enum Move { kAtOnce, kToStaged, kFromStaged };
template <Move MOVE>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a, int lanes_log2) {
  const int lanes = 1 << lanes_log2;               // 16-byte pieces per row and column
  const int rows = kMoveThreads >> lanes_log2;     // rows that a step of the workgroup takes
  const int columns = a.row_bytes / (16 * lanes);
  const int column = blockIdx.x % columns, rest = blockIdx.x / columns;
  const int h = rest % a.Hkv, b = rest / a.Hkv;
  const int n = clamp_len(a, b), got = min(n, a.budget);
  const bool apart = a.apart != 0;
  if (got == 0 || (n <= a.budget && !apart)) return;  // uniform: nothing moves
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int32_t* bt = a.block_tables + (int64_t)b * a.max_blocks;
  const int32_t* ot = a.out_tables + (int64_t)b * a.out_blocks;
  const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
  const int piece = (column * lanes + (threadIdx.x & (lanes - 1))) * 16;
  char* base = (blockIdx.y ? a.v : a.k) + (int64_t)h * a.row_bytes + piece;
  char* staged = a.staged + (((int64_t)b * a.Hkv + h) * 2 + blockIdx.y) * a.budget * a.row_bytes + piece;
  const int64_t stride = (int64_t)a.Hkv * a.row_bytes;
  const int r = threadIdx.x >> lanes_log2;
  const int chunk = rows * kMoveUnroll;
  struct Chunk {
    u32x4 x[kMoveUnroll];
    int to[kMoveUnroll];   // the page that a row goes to; -1: the row does not move (a hole, or past the last)
  };
  // (rows past the last read it again and those of a hole page 0, so that no
  // load is under a condition: it would be waited for there)
  auto read = [&](Chunk& c, int i0) {
    int key[kMoveUnroll], p[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) key[u] = kept[min(i0 + u * rows + r, got - 1)];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      p[u] = bt[key[u] >> a.bs_log2];
      c.to[u] = MOVE == kToStaged ? 0 : ot[min(i0 + u * rows + r, got - 1) >> a.bs_log2];
    }
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = min(i0 + u * rows + r, got - 1);
      if (i0 + u * rows + r >= got || p[u] < 0) c.to[u] = -1;
      const char* src = MOVE == kFromStaged ? staged + (int64_t)i * a.row_bytes
                                            : base + (((int64_t)max(p[u], 0) << a.bs_log2) + (key[u] & bs_mask)) * stride;
      c.x[u] = load16_stream(src);
    }
  };
  auto write = [&](const Chunk& c, int i0) {
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = i0 + u * rows + r;
      char* dst = MOVE == kToStaged ? staged + (int64_t)i * a.row_bytes
                                    : base + (((int64_t)c.to[u] << a.bs_log2) + (i & bs_mask)) * stride;
      if (c.to[u] >= 0) __builtin_nontemporal_store(c.x[u], reinterpret_cast<u32x4*>(dst));
    }
  };
  Chunk c;
  if (MOVE != kAtOnce) {
    for (int i0 = blockIdx.z * chunk; i0 < got; i0 += gridDim.z * chunk) {
      read(c, i0);
      write(c, i0);
    }
    return;
  }
  // (the next chunk's sources lie behind this chunk's destinations; the barrier
  // puts every read of a chunk before its first write)
  auto in_order = [&] {
    for (int i0 = 0; i0 < got; i0 += chunk) {
      Chunk next;
      loads_back();
      __syncthreads();
      if (i0 + chunk < got) read(next, i0 + chunk);
      write(c, i0);
      c = next;
    }
  };
  if (!apart) {
    read(c, 0);
    in_order();
    return;
  }
  const int first = blockIdx.z * chunk;
  if (first >= got) return;  // uniform
  const int pages = ((got - 1) >> a.bs_log2) + 1, mine = min((int)threadIdx.x, pages - 1);
  const int from = bt[mine], into = ot[mine];
  read(c, first);
  if (n > a.budget) {  // uniform
    // Another table may hold pages of this one at their places, in which rows
    // move as they do in place: one workgroup takes the column then.  (Its
    // entries are looked up beside the first chunk, and before any write.)
    int same = from >= 0 && from == into;
    for (int i = kMoveThreads + threadIdx.x; i < pages; i += kMoveThreads) same |= bt[i] >= 0 && bt[i] == ot[i];
    if (__syncthreads_or(same)) {  // uniform
      if (blockIdx.z == 0) in_order();
      return;
    }
  }
  write(c, first);
  for (int i0 = first + gridDim.z * chunk; i0 < got; i0 += gridDim.z * chunk) {
    read(c, i0);
    write(c, i0);
  }
}

// How the rows move: `lanes_log2` of a column; rows staged, or at once; grid z.
struct MovePlan {
  int lanes_log2, z;
  size_t staged;
};

MovePlan plan_move(int B, int Hkv, int row_bytes, int64_t cap, int budget, bool apart) {
  const int64_t most = std::min<int64_t>(cap, budget), units = (int64_t)B * Hkv * 2;
  MovePlan p{2, 1, 0};
  // a row's pieces to one workgroup where the (sequence, head, K or V)s fill the
  // chip (whole lines, one read of the page and position lists), or the rows
  // are dealt to several; else down to 64 bytes
  auto widen = [&](int64_t least) {
    while (p.lanes_log2 < 5 && row_bytes % (32 << p.lanes_log2) == 0 && units * (row_bytes / (32 << p.lanes_log2)) >= least)
      ++p.lanes_log2;
  };
  auto chunk = [&] { return (int64_t)(kMoveThreads >> p.lanes_log2) * kMoveUnroll; };
  widen(apart ? 0 : 256);
  // In place, few workgroups take many chunks one after another, each a chain
  // of three round trips: past two chunks by way of staging rows, which any
  // number of workgroups may fill and empty (twice the bytes, a third launch).
  // Whole calls, at once against staged: 12,000 -> 4,205 keys of 8 heads, 3
  // sequences of 128-byte rows 49 and 42 us, 1 of 256 bytes 46 and 34; 4,000 ->
  // 1,000 (one chunk) 18.1 and 19.8.  Not where the workgroups fill the chip.
  const int64_t columns = row_bytes / (16 << p.lanes_log2);
  if (!apart && budget < cap && units * columns < 256 && most > 2 * chunk()) {
    p.staged = (size_t)units * budget * row_bytes;
    widen(0);
  }
  if (apart || p.staged) p.z = (int)std::min<int64_t>((most + chunk() - 1) / chunk(), 64);
  return p;
}

int64_t evict_cap(int block_size, int max_blocks) { return (int64_t)max_blocks * block_size; }

int evict_args(int B, int Hkv, int D, int block_size, int max_blocks, int out_blocks, bool apart, int dtype, int budget,
               int sinks, int recent) {
  if (B < 0 || Hkv <= 0 || D <= 0 || max_blocks <= 0 || budget <= 0 || sinks < 0 || recent < 0) return NSV_ERR_ARG;
  if (dtype != NSV_F32 && dtype != NSV_BF16) return NSV_ERR_ARG;
  if ((int64_t)sinks + recent > budget || (apart && out_blocks <= 0)) return NSV_ERR_ARG;
  const int64_t row_bytes = (int64_t)D * (dtype == NSV_BF16 ? 2 : 4), cap = evict_cap(block_size, max_blocks);
  if (block_size <= 0 || (block_size & (block_size - 1)) || row_bytes % 64 || row_bytes > 65536) return NSV_ERR_UNSUPPORTED;
  if (cap > (int64_t)1 << 30 || (int64_t)B * Hkv * (row_bytes / 64) > 0x7fffffff) return NSV_ERR_UNSUPPORTED;
  if (apart && (int64_t)out_blocks * block_size < std::min<int64_t>(cap, budget)) return NSV_ERR_ARG;
  return NSV_OK;
}

}  // namespace

extern "C" {

size_t nsv_evict_workspace_size(int B, int Hkv, int D, int block_size, int max_blocks, int apart, int dtype, int budget) {
  if (evict_args(B, Hkv, D, block_size, max_blocks, max_blocks, false, dtype, budget, 0, 0) != NSV_OK) return 0;
  return plan_move(B, Hkv, D * (dtype == NSV_BF16 ? 2 : 4), evict_cap(block_size, max_blocks), budget, apart != 0).staged;
}

int nsv_evict_kv(void* k_cache, void* v_cache, float* key_weights, const int32_t* block_tables,
                 const int64_t* context_lens, const int32_t* out_block_tables, int64_t* lens, int32_t* kept, int B,
                 int Hkv, int D, int block_size, int max_blocks, int out_blocks, int dtype, int budget, int sinks,
                 int recent, void* workspace, size_t workspace_bytes, void* stream) {
  const bool apart = out_block_tables && (out_block_tables != block_tables || out_blocks != max_blocks);
  const int bad = evict_args(B, Hkv, D, block_size, max_blocks, out_blocks, out_block_tables != nullptr, dtype, budget, sinks,
                             recent);
  if (bad != NSV_OK) return bad;
  if (B == 0) return NSV_OK;
  if (!k_cache || !v_cache || !key_weights || !block_tables || !context_lens || !lens || !kept) return NSV_ERR_ARG;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)workspace) % 16) return NSV_ERR_ARG;
  const int row_bytes = D * (dtype == NSV_BF16 ? 2 : 4);
  const int64_t cap = evict_cap(block_size, max_blocks);
  const MovePlan p = plan_move(B, Hkv, row_bytes, cap, budget, apart);
  if (p.staged && (!workspace || workspace_bytes < p.staged)) return NSV_ERR_WORKSPACE;
  int bs_log2 = 0;
  while ((1 << bs_log2) < block_size) ++bs_log2;
  EvictArgs a{(char*)k_cache, (char*)v_cache, key_weights, block_tables, apart ? out_block_tables : block_tables,
              context_lens, lens, kept, Hkv, row_bytes, bs_log2, max_blocks, apart ? out_blocks : max_blocks,
              budget, sinks, recent, bs_log2 >= 2 && (uintptr_t)key_weights % 16 == 0, apart, (char*)workspace};
  hipStream_t s = (hipStream_t)stream;
  if (cap <= (int64_t)kSelThreads * 4 * kSelLoads && a.vector)
    hipLaunchKernelGGL(evict_select_kernel<true>, dim3(B * Hkv), dim3(kSelThreads), 0, s, a);
  else
    hipLaunchKernelGGL(evict_select_kernel<false>, dim3(B * Hkv), dim3(kSelThreads), 0, s, a);
  int rc = nsv_launch_status();
  if (rc) return rc;
  const dim3 grid(B * Hkv * (row_bytes / (16 << p.lanes_log2)), 2, p.z);
  if (p.staged) {
    hipLaunchKernelGGL(evict_move_kernel<kToStaged>, grid, dim3(kMoveThreads), 0, s, a, p.lanes_log2);
    rc = nsv_launch_status();
    if (rc) return rc;
    hipLaunchKernelGGL(evict_move_kernel<kFromStaged>, grid, dim3(kMoveThreads), 0, s, a, p.lanes_log2);
  } else {
    hipLaunchKernelGGL(evict_move_kernel<kAtOnce>, grid, dim3(kMoveThreads), 0, s, a, p.lanes_log2);
  }
  return nsv_launch_status();
}

}  // extern "C"
