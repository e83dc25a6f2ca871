// Eviction from a paged cache by accumulated attention weight, for gfx950.
//
// Of every (sequence, kv head) with more than `budget` keys, budget stay: the
// first `sinks`, the last `recent` and, of the rest, those with the most
// weight (of equal ones the lower position; NaN counts as -inf).  Their K, V
// and weight rows move to the front, in the order of their positions, of the
// sequence's own table or of another.
//
// Selection (evict_select_kernel), one workgroup per (sequence, kv head): the
// weights as unsigned words of the same order; the need-th largest found by
// four passes over 8 bits each (a histogram per wave, so that equal words
// cost few collisions); then one pass per wave over a run of its own counts
// what lies above that word and what equals it, and a second one writes the
// kept positions in order.  Bound by the latency of its passes over weights
// that stay in L2.
//
// Moving (evict_move_kernel): every kept row read and written once.  Within a
// table rows move forward only: row i comes from kept[i] >= i.  A workgroup
// owns one 64-byte column of one (sequence, kv head, K or V) and takes its
// rows in ascending chunks, each read whole before it is written, so what a
// chunk overwrites no later chunk reads, and no other workgroup touches the
// column.  Bound by the rows' bytes.

#include "common.h"

#include <algorithm>

namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;   // rows per lane and chunk

struct EvictArgs {
  char* k;
  char* v;
  float* weights;                // [num_blocks][Hkv][block_size]
  const int32_t* block_tables;
  const int32_t* out_tables;     // = block_tables: in place
  const int64_t* context_lens;
  int64_t* lens;                 // [B]
  int32_t* kept;                 // [B][Hkv][budget]
  int Hkv, row_bytes, bs_log2, max_blocks, out_blocks, budget, sinks, recent;
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

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ int hist[kSelWaves][256];
  __shared__ int above[256];
  __shared__ int wave_gt[kSelWaves], wave_eq[kSelWaves];
  __shared__ int digit, rest;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / a.Hkv, h = blockIdx.x - b * a.Hkv;
  const int n = clamp_len(a, b);
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int32_t* bt = a.block_tables + (int64_t)b * a.max_blocks;
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  auto place = [&](const int32_t* table, int key) -> int64_t {  // of a key's weight; -1: no page
    const int p = table[key >> a.bs_log2];
    return p < 0 ? -1 : ((((int64_t)p * a.Hkv + h) << a.bs_log2) + (key & bs_mask));
  };
  auto word = [&](int key) {
    const int64_t at = place(bt, key);
    return at < 0 ? 0u : ordered(a.weights[at]);
  };
  if (tid == 0 && h == 0) a.lens[b] = min(n, a.budget);
  const int got = min(n, a.budget);
  for (int i = got + tid; i < a.budget; i += kSelThreads) kept[i] = -1;
  if (n <= a.budget) {  // uniform: all of them stay
    for (int i = tid; i < n; i += kSelThreads) kept[i] = i;
  } else {
    const int lo = a.sinks, hi = n - a.recent;      // the keys that compete
    const int need = a.budget - a.sinks - a.recent; // how many of them stay
    uint32_t prefix = 0;                            // the leading bits of the need-th largest word
    int want = need;                                // which of the words with that prefix it is, from the top
    for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
      for (int i = tid; i < kSelWaves * 256; i += kSelThreads) (&hist[0][0])[i] = 0;
      __syncthreads();
      for (int key = lo + tid; key < hi; key += kSelThreads) {
        const uint32_t u = word(key);
        if (shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[w][(u >> shift) & 255], 1);
      }
      __syncthreads();
      if (tid < 256) {
        int s = 0;
        for (int ww = 0; ww < kSelWaves; ++ww) s += hist[ww][tid];
        above[tid] = s;
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, left = want;
        while (d > 0 && above[d] < left) left -= above[d--];
        digit = d;
        rest = left;
      }
      __syncthreads();
      prefix |= (uint32_t)digit << shift;
      want = rest;
      __syncthreads();
    }
    // words above `prefix` stay, and of those equal to it the first `want`
    const int per = ((hi - lo + kSelWaves - 1) / kSelWaves + 63) & ~63;  // a wave's run
    const int r0 = lo + w * per, r1 = min(hi, r0 + per);
    int gt = 0, eq = 0;
    if (need > 0) {
      for (int key = r0 + lane; key - lane < r1; key += 64) {
        const uint32_t u = key < r1 ? word(key) : 0u;
        gt += __popcll(__ballot(key < r1 && u > prefix));
        eq += __popcll(__ballot(key < r1 && u == prefix));
      }
    }
    if (lane == 0) {
      wave_gt[w] = gt;
      wave_eq[w] = eq;
    }
    __syncthreads();
    int at_gt = 0, at_eq = 0;
    for (int ww = 0; ww < w; ++ww) {
      at_gt += wave_gt[ww];
      at_eq += wave_eq[ww];
    }
    if (need > 0) {
      const uint64_t below = (1ull << lane) - 1;
      for (int key = r0 + lane; key - lane < r1; key += 64) {
        const uint32_t u = key < r1 ? word(key) : 0u;
        const bool is_gt = key < r1 && u > prefix, is_eq = key < r1 && u == prefix;
        const uint64_t bg = __ballot(is_gt), be = __ballot(is_eq);
        const int g = at_gt + __popcll(bg & below), e = at_eq + __popcll(be & below);
        if (is_gt || (is_eq && e < want)) kept[a.sinks + g + min(e, want)] = key;
        at_gt += __popcll(bg);
        at_eq += __popcll(be);
      }
    }
    for (int i = tid; i < a.sinks; i += kSelThreads) kept[i] = i;
    for (int i = tid; i < a.recent; i += kSelThreads) kept[a.budget - a.recent + i] = hi + i;
  }
  if (n <= a.budget && a.out_tables == a.block_tables) return;
  // the weights themselves, a chunk at a time: every read of a chunk before its first write
  __syncthreads();
  const int32_t* ot = a.out_tables + (int64_t)b * a.out_blocks;
  for (int i0 = 0; i0 < got; i0 += kSelThreads) {
    const int i = i0 + tid;
    float x = 0.f;
    bool on = false;
    if (i < got) {
      const int64_t at = place(bt, kept[i]);
      on = at >= 0;
      if (on) x = a.weights[at];
    }
    __syncthreads();
    if (on) {
      const int64_t to = place(ot, i);
      if (to >= 0) a.weights[to] = x;
    }
    __syncthreads();
  }
}

__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
  constexpr int ROWS = kMoveThreads / 4;  // rows a step of the workgroup takes: four lanes of 16 bytes each
  const int slices = a.row_bytes / 64;
  const int slice = blockIdx.x % slices, rest = blockIdx.x / slices;
  const int h = rest % a.Hkv, b = rest / a.Hkv;
  const int n = clamp_len(a, b), got = min(n, a.budget);
  if (n <= a.budget && a.out_tables == a.block_tables) return;  // uniform: nothing moves
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int32_t* bt = a.block_tables + (int64_t)b * a.max_blocks;
  const int32_t* ot = a.out_tables + (int64_t)b * a.out_blocks;
  const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
  char* base = (blockIdx.y ? a.v : a.k) + (int64_t)h * a.row_bytes + slice * 64 + (threadIdx.x & 3) * 16;
  const int64_t stride = (int64_t)a.Hkv * a.row_bytes;
  const int r = threadIdx.x >> 2;
  auto row = [&](const int32_t* table, int key) -> char* {
    const int p = table[key >> a.bs_log2];
    return p < 0 ? nullptr : base + (((int64_t)p << a.bs_log2) + (key & bs_mask)) * stride;
  };
  for (int i0 = 0; i0 < got; i0 += ROWS * kMoveUnroll) {
    u32x4 x[kMoveUnroll];
    bool on[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = i0 + u * ROWS + r;
      const char* src = i < got ? row(bt, kept[i]) : nullptr;
      on[u] = src != nullptr;
      x[u] = u32x4{0u, 0u, 0u, 0u};
      if (on[u]) x[u] = load16_stream(src);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = i0 + u * ROWS + r;
      char* dst = on[u] ? row(ot, i) : nullptr;
      if (dst) *reinterpret_cast<u32x4*>(dst) = x[u];
    }
    __syncthreads();
  }
}

}  // namespace

extern "C" {

int nsv_evict_kv(void* k_cache, void* v_cache, float* key_weights, const int32_t* block_tables,
                 const int64_t* context_lens, const int32_t* out_block_tables, int64_t* lens, int32_t* kept, int B,
                 int Hkv, int D, int block_size, int max_blocks, int out_blocks, int dtype, int budget, int sinks,
                 int recent, void* stream) {
  if (B < 0 || Hkv <= 0 || D <= 0 || max_blocks <= 0 || budget <= 0 || sinks < 0 || recent < 0) return NSV_ERR_ARG;
  if (dtype != NSV_F32 && dtype != NSV_BF16) return NSV_ERR_ARG;
  if ((int64_t)sinks + recent > budget || (out_block_tables && out_blocks <= 0)) return NSV_ERR_ARG;
  const int row_bytes = D * (dtype == NSV_BF16 ? 2 : 4);
  if (block_size <= 0 || (block_size & (block_size - 1)) || row_bytes % 64) return NSV_ERR_UNSUPPORTED;
  const int64_t cap = (int64_t)max_blocks * block_size;
  if (cap > (int64_t)1 << 30 || (int64_t)B * Hkv * (row_bytes / 64) > 0x7fffffff) return NSV_ERR_UNSUPPORTED;
  if (out_block_tables && (int64_t)out_blocks * block_size < std::min<int64_t>(cap, budget)) return NSV_ERR_ARG;
  if (B == 0) return NSV_OK;
  if (!k_cache || !v_cache || !key_weights || !block_tables || !context_lens || !lens || !kept) return NSV_ERR_ARG;
  if (((uintptr_t)k_cache | (uintptr_t)v_cache) % 16) return NSV_ERR_ARG;
  int bs_log2 = 0;
  while ((1 << bs_log2) < block_size) ++bs_log2;
  EvictArgs a{(char*)k_cache, (char*)v_cache, key_weights, block_tables, out_block_tables ? out_block_tables : block_tables,
              context_lens, lens, kept, Hkv, row_bytes, bs_log2, max_blocks, out_block_tables ? out_blocks : max_blocks,
              budget, sinks, recent};
  hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_select_kernel, dim3(B * Hkv), dim3(kSelThreads), 0, s, a);
  const int rc = nsv_launch_status();
  if (rc) return rc;
  hipLaunchKernelGGL(evict_move_kernel, dim3(B * Hkv * (row_bytes / 64), 2), dim3(kMoveThreads), 0, s, a);
  return nsv_launch_status();
}

}  // extern "C"
