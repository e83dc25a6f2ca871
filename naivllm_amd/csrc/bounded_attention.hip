// Paged attention of a few query rows per sequence (verify rows, decode
// steps) over a bounded cache, for gfx950:
//   * with a sliding window and a few first tokens that stay visible;
//   * with the attention weight of every key added to a paged table.
//
//   row r at position p sees key j  <=>  j <= p, j < context, its page is
//   mapped, and (with a window W) j > p - W or j < sinks
//   out_r = sum_j 2^(s_rj - m_r) v_j / l_r,  s_rj = scale log2(e) q_r . k_j
//   weight of (kv head, key j) = sum_r sum_(heads of the group) 2^(s_rj - m_r) / l_r
//
// What bounds it: the K/V bytes of the keys that some row of a sequence
// sees.  Those are one or two runs of keys (the first ones, the windows'
// union), numbered through as virtual keys; a workgroup takes a part of one
// (sequence, kv head) pair's virtual keys for up to 64 query rows (the pair's
// group heads x rows; further heads in workgroups of their own), so no byte
// is read for a key that no row sees.  Its four waves take tiles of keys in
// turn, each wave from its own LDS: K and V rows go from memory straight to
// LDS two tiles deep, with no barrier in the loop.
//
// Products: S^T = K Q^T puts a row's scores into four lanes (16-lane group g
// holds keys 4 g + i), which is the operand layout of O^T = V^T P^T, so
// weights move through no shuffle.  bf16: v_mfma_f32_16x16x32_bf16, V^T from
// the transposing LDS reads; fp32: v_mfma_f32_16x16x4_f32, whose terms are
// numbered so that 16-byte LDS reads feed them.  Maxima, sums and outputs are
// held in fp32.  For the second product a weight of P is the sum of two bf16
// numbers (16 bits; one bf16 number left the outputs up to 1.86e-3 from 64 bits,
// two leave the final rounding's 1.7e-3), in two products: 4% of the time at 36
// rows of a kv head over 4,096 keys (34.7 -> 36.3 us), nothing measurable at 2 rows
// or where 36 read 16k keys and more.
// The key weights are never rounded.
//
// Key weights need every row's final statistics, so they are a second pass:
// over the scores, which the first one stores where a call has few of them
// (up to 64 rows of a kv head and 32 MiB: 64 pairs, 2 rows, 1,250 keys 15 us
// against 26 from the keys again; 36 rows over 16k-32k keys, 604 MB of scores,
// 714 us against 490), or over K again, whose products are made anew.
//
// Measured on MI355X, us, bytes that it cannot do without per second: window
// 512 + 4 sinks, 1 row of 16/8 heads 7.6 (latency: the metadata's, the table's
// and the tiles' round trips); window 4,096, 8 sequences of 9 rows, 32/8 heads,
// 36.5 (3.7 TB/s; loads alone 33); fp32, 3 sequences, window 999, 9.3; key weights
// of 8 sequences of 1,250 keys, 1 row, 15.1 (2.7 TB/s); of 16 sequences of
// 16k-32k keys, 9 rows of 32/8 heads, 492: 322 for the attention (5.4 TB/s), 167
// for K again (5.2 TB/s).

#include "common.h"

#include <algorithm>
#include <type_traits>

namespace {

constexpr int kWaves = 4;         // waves per workgroup
constexpr int kMaxPages = 2048;   // block-table entries of a workgroup's keys held in LDS
constexpr int kMaxSplits = 64;
constexpr int kJoinedSplits = 8;  // the most that the kernel joins itself
constexpr int kCounters = 16384;  // words of the arrival counters
constexpr float kNegInf = -__builtin_inff();

// The word of a (pair, head subset): the first 256 have a 256-byte line each
// (device-scope atomics on one line wait for one another).
__device__ __forceinline__ int counter_slot(int unit) { return ((unit & 255) << 6) | (unit >> 8); }

enum Mode { kAttend, kAttendScores, kAttendFirst, kWeights };  // kAttendFirst: kWeights follows

struct RowArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* block_tables;
  const int64_t* context_lens;
  const int32_t* cu_seqlens_q;
  const int64_t* positions;
  float2* part_ml;    // [npairs * subsets][S][R]: (maximum, log2 domain; sum)
  float* part_o;      // [npairs * subsets][S][R][D], unnormalised
  unsigned* counters; // null, or splits of a (pair, head subset) done so far, 0 between calls (kAttend)
  float* scores;      // [npairs * subsets][R][score_keys], log2 domain, -inf where masked (kAttendScores)
  float* key_weights; // [num_blocks][Hkv][block_size]
  float scale_log2;
  int H, Hkv, G, subsets;  // query heads, kv heads, query heads of a kv head that a workgroup serves, how often
  int bs_log2, max_blocks, QL, R, S, npairs;  // R = G * QL
  int window, sinks;  // window 0: every key up to the row
  int score_keys;
  int weight_splits;  // kWeights: workgroups that a pair's keys are dealt to
  int first_subset;   // kWeights: the subset this launch adds
};

typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;

__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint2 lds_read_tr(const unsigned char* p) {
  const i16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p));
  return __builtin_bit_cast(uint2, v);
}

// over the four 16-lane groups' values of the same lane
__device__ __forceinline__ float groups_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// over the wave
template <typename F>
__device__ __forceinline__ int wave_reduce(int v, F f) {
  v = f(v, (int)dpp_u32<kDppXor1>((uint32_t)v));
  v = f(v, (int)dpp_u32<kDppXor2>((uint32_t)v));
  v = f(v, (int)dpp_u32<kDppHalfMirror>((uint32_t)v));
  v = f(v, (int)dpp_u32<kDppMirror>((uint32_t)v));
  auto r = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = f((int)r[0], (int)r[1]);
  r = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return uniform(f((int)r[0], (int)r[1]));
}

// The keys of a sequence that some row of the call sees, numbered 0 .. total
// - 1: the first `head` keys, then those from head + gap on.
struct Span {
  int total, head, gap;
  int pos_min, pos_max;  // of the sequence's rows that are no padding
  __device__ int key(int v) const { return v < head ? v : v + gap; }
};

// The position of the sequence's row `lane` (whatever behind the last of them:
// a load under a condition would be waited for there).
__device__ __forceinline__ int64_t row_position(const RowArgs& a, int q0, int qlen) {
  return a.positions[max(q0 + min((int)(threadIdx.x & 63), qlen - 1), 0)];  // (T > 0)
}

// (every lane of the wave; the sequence's rows are q0 .. q0 + qlen - 1, p64
// their positions, len its context length)
__device__ __forceinline__ Span make_span(const RowArgs& a, int64_t len, int qlen, int64_t p64, int& my_pos) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)a.max_blocks << a.bs_log2;
  const int ctx = uniform((int)(len < 0 ? 0 : (len < cap ? len : cap)));
  my_pos = lane >= qlen || p64 < 0 ? -1 : (int)(p64 < 0x3fffffff ? p64 : 0x3fffffff);
  Span s;
  s.pos_min = wave_reduce(my_pos < 0 ? 0x7fffffff : my_pos, [](int x, int y) { return min(x, y); });
  s.pos_max = wave_reduce(my_pos, [](int x, int y) { return max(x, y); });
  s.total = s.head = min(ctx, s.pos_max + 1);  // (no row at all: 0)
  s.gap = 0;
  if (a.window > 0 && s.pos_max >= 0) {
    const int first = max(0, s.pos_min - a.window + 1);  // of the windows' union
    const int head = min(a.sinks, s.total);
    if (first > head) {
      s.head = head;
      s.gap = first - head;
      s.total = head + max(0, s.total - first);
    }
  }
  return s;
}

// Keys per split: the span spread evenly over S splits, in whole turns of
// the workgroup's waves where that leaves none of them short.
template <int TK>
__device__ __forceinline__ int split_keys(int total, int S) {
  const int per = (total + S - 1) / S;
  return max((per + TK - 1) / TK * TK, TK * kWaves);
}

// A row's maximum and 1 / sum over its splits, for `rows` <= 64 rows from (pair,
// head subset) ps on, into LDS (a barrier follows): four neighbouring lanes per
// row, each with every fourth split, all of them loaded in one round trip (a
// wave per row and a lane per split took 14 us for 64 rows).  A row that sees
// nothing: 0 and 0.
template <int N>  // 4 N >= a.S
__device__ __forceinline__ void join_stats_of(const RowArgs& a, int ps, int rows, float2* stat) {
  const int j = threadIdx.x & 3, m = threadIdx.x >> 2;
  const int row = min(m, rows - 1), sub = row / a.R;  // (rows may run on into the pair's next subsets)
  const float2* src = a.part_ml + (int64_t)(ps + sub) * a.S * a.R + row - sub * a.R;
  float2 x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = src[(int64_t)min(4 * k + j, a.S - 1) * a.R];
  float M = kNegInf, L = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) M = fmaxf(M, x[k].x);  // (a split read twice changes nothing here)
  M = fmaxf(M, dpp_f32<kDppXor1>(M));
  M = fmaxf(M, dpp_f32<kDppXor2>(M));
  const float ref = M == kNegInf ? 0.f : M;
#pragma unroll
  for (int k = 0; k < N; ++k) L += 4 * k + j < a.S ? x[k].y * __builtin_amdgcn_exp2f(x[k].x - ref) : 0.f;
  L += dpp_f32<kDppXor1>(L);
  L += dpp_f32<kDppXor2>(L);
  if (j == 0 && m < rows) stat[m] = make_float2(ref, L == 0.f ? 0.f : 1.f / L);
}

__device__ __forceinline__ void join_stats(const RowArgs& a, int ps, int rows, float2* stat) {
  static_assert(kMaxSplits == 64, "four lanes take every split");
  if (a.S <= 4) join_stats_of<1>(a, ps, rows, stat);  // uniform
  else if (a.S <= 8) join_stats_of<2>(a, ps, rows, stat);
  else join_stats_of<16>(a, ps, rows, stat);
}

template <typename T, int DH>
struct Shape {
  static constexpr bool kBf16 = sizeof(T) == 2;
  static constexpr int TK = kBf16 ? 32 : 16;          // keys per tile
  static constexpr int ROWB = DH * (int)sizeof(T);    // bytes per row
  static constexpr int CPR = ROWB / 16;               // 16-byte chunks per row
  static constexpr int RPI = 64 / CPR;                // rows one load instruction fills
  static constexpr int J = TK / RPI;                  // load instructions per K (or V) tile
  static constexpr int TILEB = TK * ROWB;
  static constexpr int KT = TK / 16;                  // 16-key score tiles
  static constexpr int QV = DH / (kBf16 ? 32 : 16);   // 16-byte query pieces per lane
  // the slot of a row's chunk: the 16 rows (K) and the 8 or 4 rows (V) that
  // one read's lanes touch fall into different banks
  static __device__ __forceinline__ int kswz(int r) { return r & (CPR < 16 ? CPR - 1 : 15); }
  static __device__ __forceinline__ int vswz(int r) {
    if constexpr (!kBf16) return 0;  // (16 lanes read 256 consecutive bytes)
    else return CPR >= 16 ? (r & 7) << 1 : ((r >> 1) & 3) << 1;
  }
};

template <typename T, int MT, int DH, int MODE>
__global__ __launch_bounds__(kWaves * 64, 1) void row_attention_kernel(RowArgs a) {
  using S_ = Shape<T, DH>;
  constexpr bool BF16 = S_::kBf16;
  constexpr int TK = S_::TK, KT = S_::KT, J = S_::J, ROWB = S_::ROWB, CPR = S_::CPR, RPI = S_::RPI;
  constexpr int NT = kWaves * 64, MP = MT * 16;
  constexpr int DT = DH / 16;
  constexpr bool V = MODE != kWeights;
  constexpr int BUFS = 2;
  constexpr int WAVEB = BUFS * 2 * S_::TILEB;  // one wave's tiles; later its rows of O
  static_assert(WAVEB >= MP * DH * 4 || !V, "a wave's tiles hold its output rows");
  struct __attribute__((aligned(16))) Lds {
    unsigned char tiles[kWaves][V ? WAVEB : WAVEB / 2];
    int pages[kMaxPages];
    float2 ml[kWaves][MP];
    float2 row[MP];
    int holes, mapped;
  };
  __shared__ Lds lds;

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = uniform(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int pair = blockIdx.x % a.npairs;
  const int rest = blockIdx.x / a.npairs;
  const int sub = MODE == kWeights ? a.first_subset : rest % a.subsets;
  const int split = MODE == kWeights ? rest : rest / a.subsets;
  const int b = pair / a.Hkv, hk = pair - b * a.Hkv;
  const int head0 = hk * (a.G * a.subsets) + sub * a.G;  // first query head
  const int64_t len = a.context_lens[b];
  const int q0 = uniform(a.cu_seqlens_q[b]);
  const int qlen = min(uniform(a.cu_seqlens_q[b + 1]) - q0, a.QL);
  int my_pos;
  const Span sp = make_span(a, len, qlen, row_position(a, q0, qlen), my_pos);
  const int per = split_keys<TK>(sp.total, MODE == kWeights ? a.weight_splits : a.S);
  const int v0 = split * per;
  const int v1 = min(sp.total, v0 + per);
  const int64_t part = ((int64_t)(pair * a.subsets + sub) * a.S + split) * a.R;  // (unused by kWeights)
  const bool joins = MODE == kAttend && a.counters != nullptr;  // uniform: the last split to finish joins them all
  const int nsplit = max(1, (sp.total + per - 1) / per);        // those of this sequence
  if (v0 >= v1 && split > 0) {  // uniform: this sequence has fewer splits
    if (V && !joins && tid < a.R) a.part_ml[part + tid] = make_float2(kNegInf, 0.f);
    return;
  }

  // ---- query rows m = head * QL + t: the B operand of S^T, lane (g, c) holds row c
  u32x4 q[MT][S_::QV];
  int pos[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = mt * 16 + c;
    const int gh = m / a.QL, t = m - gh * a.QL;
    const int p = __shfl(my_pos, t & 63, 64);
    const bool live = m < a.R && t < qlen;
    pos[mt] = live ? p : -1;
    const T* src = (const T*)a.q + ((int64_t)(q0 + (live ? t : 0)) * a.H + head0 + (live ? gh : 0)) * DH + g * (16 / (int)sizeof(T));
#pragma unroll
    for (int j = 0; j < S_::QV; ++j) {
      u32x4 x = {0u, 0u, 0u, 0u};
      if (pos[mt] >= 0) x = *reinterpret_cast<const u32x4*>(src + j * (64 / (int)sizeof(T)));
      q[mt][j] = x;
    }
  }

  // ---- the block-table entries of a run of this split's keys, c0 .. c1 - 1, in
  // LDS: the head run's pages, then the window run's.  (Nothing else loads
  // pages: a load that the compiler knows of among those below would make it
  // wait for all of them.)  One run, unless pages are small and many.
  const int bs_mask = (1 << a.bs_log2) - 1;
  const int32_t* bt = a.block_tables + (int64_t)b * a.max_blocks;
  // (a run's two ends may lie inside pages, on both sides of the gap)
  const int run = (int)min((int64_t)1 << 30, ((int64_t)(kMaxPages - 4) << a.bs_log2) / TK * TK);
  int c0 = v0, c1 = v0;
  int pg_a, na, pg_b;
  bool holes;
  int spare;  // the cache row that an unmapped key reads: one of a key that the run has
  auto stage_pages = [&]() {  // the run's keys that count (0: none is mapped)
    const int headn = min(c1, sp.head);                      // end of the head run
    pg_a = c0 >> a.bs_log2;
    na = headn > c0 ? ((headn - 1) >> a.bs_log2) - pg_a + 1 : 0;
    const int win0 = max(c0, sp.head) + sp.gap, win1 = c1 + sp.gap;  // the window run's keys
    pg_b = win0 >> a.bs_log2;
    const int nb = c1 > sp.head && win1 > win0 ? ((win1 - 1) >> a.bs_log2) - pg_b + 1 : 0;
    if (tid == 0) {
      lds.holes = 0;
      lds.mapped = 0x7fffffff;
    }
    __syncthreads();
    for (int i = tid; i < na + nb; i += NT) {
      const int p = bt[i < na ? pg_a + i : pg_b + i - na];
      lds.pages[i] = p;
      if (p < 0) lds.holes = 1;
    }
    // (the query rows are waited for here, not behind the tiles loading ahead)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < S_::QV; ++j) __asm__ volatile("" ::"v"(q[mt][j]));
    __syncthreads();
    holes = uniform(lds.holes) != 0;
    spare = 0;
    if (!holes) return c1 - c0;  // uniform
    for (int i = tid; i < na + nb; i += NT)
      if (lds.pages[i] >= 0) atomicMin(&lds.mapped, i);
    __syncthreads();
    const int i = uniform(lds.mapped);
    if (i >= na + nb) return 0;
    const int key = i < na ? max((pg_a + i) << a.bs_log2, c0) : max((pg_b + i - na) << a.bs_log2, win0);
    spare = (lds.pages[i] << a.bs_log2) + (key & bs_mask);
    return c1 - c0;
  };
  auto page = [&](int key, bool head) { return lds.pages[(key >> a.bs_log2) - (head ? pg_a : pg_b - na)]; };

  // ---- K/V rows straight to LDS: instruction j fills rows j RPI .., the lane
  // picking the chunk that its slot holds; rows past the last key read it again
  const uint32_t row_bytes = (uint32_t)a.Hkv * ROWB;
  const char* kbase = (const char*)a.k + (int64_t)hk * ROWB;
  const char* vbase = (const char*)a.v + (int64_t)hk * ROWB;
  unsigned char* mine = lds.tiles[w];
  auto lds_at = [](const void* p) {
    return (uint32_t)uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
  };
#define NSV_LOAD_LDS(at, offset, src, policy)                                                       \
  __asm__ volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" policy ::"s"(at), \
                   "v"(src), "n"(offset)                                                            \
                   : "memory", "m0", "scc")
  auto ktile = [&](int buf) { return mine + buf * (V ? 2 : 1) * S_::TILEB; };
  auto vtile = [&](int buf) { return mine + (buf * 2 + 1) * S_::TILEB; };
  auto issue = [&](int buf, int tile) {
    const uint32_t kt = lds_at(ktile(buf)), vt = V ? lds_at(vtile(buf)) : 0u;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int r = j * RPI + lane / CPR, slot = lane % CPR;
      const int v = min(c0 + tile * TK + r, c1 - 1);
      const int key = sp.key(v);
      const int p = page(key, v < sp.head);
      const uint32_t row = p >= 0 ? (uint32_t)((p << a.bs_log2) + (key & bs_mask)) : (uint32_t)spare;
      const uint64_t off = (uint64_t)row * row_bytes;
      const char* ksrc = kbase + off + ((slot ^ S_::kswz(r)) << 4);
      if constexpr (MODE == kAttendFirst) NSV_LOAD_LDS(kt, j * 1024, ksrc, "");
      else NSV_LOAD_LDS(kt, j * 1024, ksrc, " nt");
      if constexpr (V) NSV_LOAD_LDS(vt, j * 1024, vbase + off + ((slot ^ S_::vswz(r)) << 4), " nt");
    }
  };
  auto landed = [&](bool ahead) {
    constexpr int N = J * (V ? 2 : 1);
    if (ahead) __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    else __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };

  // ---- running state
  constexpr int NACC = V ? DT : 1;
  f32x4 acc[MT][NACC];
  float m_run[MT], l_run[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m_run[mt] = kNegInf;
    l_run[mt] = 0.f;
#pragma unroll
    for (int d = 0; d < NACC; ++d) acc[mt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // kWeights: S = Q K^T instead, so that a lane holds one key (c) and rows
  // 16 mt + 4 g + i, which it adds up in registers; the rows' maxima, 1 / their
  // sums (+inf and 0: a row that sees nothing, whose weights are then 0) and
  // positions
  float row_m[MT][4], row_inv[MT][4];
  int row_pos[MT][4];
  if constexpr (MODE == kWeights) {
    join_stats(a, pair * a.subsets + sub, a.R, lds.row);
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = mt * 16 + g * 4 + i;
        const float2 x = m < a.R ? lds.row[m] : make_float2(0.f, 0.f);
        const int t = m - m / a.QL * a.QL;
        const int p = __shfl(my_pos, t & 63, 64);
        row_pos[mt][i] = m < a.R && t < qlen ? p : -1;
        row_inv[mt][i] = x.y;
        row_m[mt][i] = x.y == 0.f ? __builtin_inff() : x.x;
      }
  }

  // scores of a tile: element i of s[mt][u] is key 16 u + 4 g + i, row c
  f32x4 s[MT][KT];
  auto scores = [&](const unsigned char* kt) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < KT; ++u) s[mt][u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < KT; ++u) {
      const int r = u * 16 + c;
      u32x4 ka[S_::QV];
#pragma unroll
      for (int j = 0; j < S_::QV; ++j)
        ka[j] = *reinterpret_cast<const u32x4*>(kt + r * ROWB + (((j * 4 + g) ^ S_::kswz(r)) << 4));
#pragma unroll
      for (int j = 0; j < S_::QV; ++j)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const u32x4 x = V ? ka[j] : q[mt][j], y = V ? q[mt][j] : ka[j];
          if constexpr (BF16) {
            s[mt][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(x), as_bf16x8(y), s[mt][u], 0, 0, 0);
          } else {
            const f32x4 xf = __builtin_bit_cast(f32x4, x), yf = __builtin_bit_cast(f32x4, y);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[mt][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(xf[e], yf[e], s[mt][u], 0, 0, 0);
          }
        }
    }
    if constexpr (V) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int u = 0; u < KT; ++u) s[mt][u] *= a.scale_log2;
    }
  };
  auto mask = [&](int tile) {
    const int vt = c0 + tile * TK;
    const int k_first = sp.key(vt), k_last = sp.key(min(vt + TK, c1) - 1);
    // uniform: every key exists and every row sees it
    const bool all = vt + TK <= c1 && k_last <= sp.pos_min &&
                     (a.window == 0 || k_last < a.sinks || k_first > sp.pos_max - a.window);
    if (!all) {
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = vt + u * 16 + g * 4 + i;
          const int key = sp.key(v);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const bool on = v < c1 && key <= pos[mt] && (a.window == 0 || key > pos[mt] - a.window || key < a.sinks);
            s[mt][u][i] = on ? s[mt][u][i] : kNegInf;
          }
        }
    }
    if (holes) {  // uniform
      const int v = min(vt + (lane & (TK - 1)), c1 - 1);
      const uint64_t mapped = __ballot(page(sp.key(v), v < sp.head) >= 0);
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            s[mt][u][i] = (mapped >> (u * 16 + g * 4 + i)) & 1 ? s[mt][u][i] : kNegInf;
    }
  };
  auto attend = [&](const unsigned char* vt) {
    // bf16: the weights as the B operand (elements 0..3 keys 4 g + i, 4..7 keys
    // 16 + 4 g + i), each as the sum of two bf16 numbers
    u32x4 pB[MT], pL[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx = kNegInf;
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[mt][u][i]);
      const float m_new = fmaxf(m_run[mt], groups_max(mx));
      const float ref = m_new == kNegInf ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run[mt] - ref);  // (from -inf: 0)
      m_run[mt] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < KT; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[mt][u][i] = __builtin_amdgcn_exp2f(s[mt][u][i] - ref);
          sum += s[mt][u][i];
        }
      l_run[mt] = fmaf(l_run[mt], alpha, sum);
      if (__ballot(alpha != 1.f)) {
#pragma unroll
        for (int d = 0; d < NACC; ++d) acc[mt][d] *= alpha;
      }
      if constexpr (BF16) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = s[mt][e < 2 ? 0 : KT - 1][2 * (e & 1)], y = s[mt][e < 2 ? 0 : KT - 1][2 * (e & 1) + 1];
          pB[mt][e] = pack_bf16x2(x, y);
          pL[mt][e] = pack_bf16x2(x - __uint_as_float(pB[mt][e] << 16), y - __uint_as_float(pB[mt][e] & 0xffff0000u));
        }
      }
    }
    if constexpr (BF16) {
      // V^T: 16-lane group g reads rows 4 g .. (and 16 + 4 g ..), dims 16 dt .. + 15
      const int r = g * 4 + (c >> 2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const unsigned char* src = vt + r * ROWB + (((dt * 2 + ((c & 3) >> 1)) ^ S_::vswz(r)) << 4) + (c & 1) * 8;
        const uint2 lo = lds_read_tr(src), hi = lds_read_tr(src + 16 * ROWB);  // (vswz(r + 16) == vswz(r))
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(u32x4{lo.x, lo.y, hi.x, hi.y}),
                                                                as_bf16x8(pB[mt]), acc[mt][dt], 0, 0, 0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          acc[mt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(u32x4{lo.x, lo.y, hi.x, hi.y}),
                                                                as_bf16x8(pL[mt]), acc[mt][dt], 0, 0, 0);
      }
    } else {
      // step i takes keys 4 g + i: V[key][64 h + 4 c + e] feeds tile (h, e), whose row c is dim 64 h + 4 c + e
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < DH / 64; ++h) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(vt + (g * 4 + i) * ROWB + (h * 16 + c) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              acc[mt][h * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], s[mt][0][i], acc[mt][h * 4 + e], 0, 0, 0);
        }
    }
  };

  do {
    c0 = c1;
    c1 = min(v1, c0 + run);
    const int ntiles = (stage_pages() + TK - 1) / TK;
    // The call's new keys start from zero, to which the launches behind this one
    // add: another sequence may have the same page behind it (a prefix that one
    // sequence of the step computes and the next shares).
    if constexpr (MODE == kAttendScores || MODE == kAttendFirst) {
      if (sub == 0 && ntiles > 0 && sp.pos_min < c1) {  // uniform
        for (int v = max(c0, sp.pos_min) + tid; v < c1; v += NT) {
          const int p = page(v, true);
          if (p >= 0) a.key_weights[((int64_t)p * a.Hkv + hk) * (bs_mask + 1) + (v & bs_mask)] = 0.f;
        }
      }
    }
    // (kWeights from the last tile back: with K read without the streaming policy
    // by kAttendFirst, its end is still in the last-level cache.  36 rows over 4,
    // 8 and 16 sequences of 16k-32k keys: 142, 254 and 492 us -> 135, 241 and 485.)
    auto at = [&](int t) { return MODE == kWeights ? ntiles - 1 - t : t; };
    if (w < ntiles) issue(0, at(w));
    if (w + kWaves < ntiles) issue(1, at(w + kWaves));
    int buf = 0;
    for (int t = w; t < ntiles; t += kWaves) {
      landed(t + kWaves < ntiles);
      scores(ktile(buf));
      if constexpr (V) mask(t);
      if constexpr (MODE == kAttendScores) {
        const int vt = c0 + t * TK;
#pragma unroll
        for (int u = 0; u < KT; ++u)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            if (mt * 16 + c < a.R) {
              float* dst = a.scores + ((int64_t)(pair * a.subsets + sub) * a.R + mt * 16 + c) * a.score_keys + vt + u * 16 + g * 4;
              *reinterpret_cast<f32x4*>(dst) = s[mt][u];  // (score_keys is a whole number of tiles; c0 too)
            }
      }
      if constexpr (V) {
        attend(vtile(buf));
      } else {
        const int vt = c0 + at(t) * TK;
        // uniform: every row sees every key (a key past the run's last, or unmapped, is not written)
        const bool all = min(vt + TK, c1) - 1 <= sp.pos_min;
        float sum[KT];
#pragma unroll
        for (int u = 0; u < KT; ++u) {
          sum[u] = 0.f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float e = __builtin_amdgcn_exp2f(fmaf(s[mt][u][i], a.scale_log2, -row_m[mt][i]));
              const float y = fmaf(e, row_inv[mt][i], sum[u]);
              sum[u] = all || vt + u * 16 + c <= row_pos[mt][i] ? y : sum[u];
            }
          sum[u] = groups_sum(sum[u]);
        }
        const int v = vt + g * 16 + c;  // lane (g, c) of the first KT groups writes the key of tile g
        if (g < KT && v < c1) {
          const int p = page(v, true);
          if (p >= 0) {
            const float y = KT == 1 || g == 0 ? sum[0] : sum[KT - 1];
            unsafeAtomicAdd(a.key_weights + ((int64_t)p * a.Hkv + hk) * (bs_mask + 1) + (v & bs_mask), y);
          }
        }
      }
      if (t + 2 * kWaves < ntiles) {
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read: its buffer may be filled again
        issue(buf, at(t + 2 * kWaves));
      }
      buf ^= 1;
    }
    if (c1 < v1) __syncthreads();  // (uniform) the run's pages are read
  } while (c1 < v1);
  if constexpr (!V) return;

  auto store_row = [&](int m, int ch, f32x4 o) {  // a 16-byte piece of row m's output
    const int gh = m / a.QL, t = m - gh * a.QL;
    if (t >= qlen) return;
    T* dst = (T*)a.out + ((int64_t)(q0 + t) * a.H + head0 + gh) * DH + ch * 4;
    if constexpr (BF16) *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    else *reinterpret_cast<f32x4*>(dst) = o;
  };

  // ---- the waves' rows combined through LDS
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l_run[mt] = groups_sum(l_run[mt]);
    if (pos[mt] < 0) {  // padding: no key, whatever an unmasked tile gave it
      m_run[mt] = kNegInf;
      l_run[mt] = 0.f;
    }
    if (g == 0) lds.ml[w][mt * 16 + c] = make_float2(m_run[mt], l_run[mt]);
  }
  __syncthreads();
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int m = mt * 16 + c;
    float M = kNegInf, L = 0.f;
#pragma unroll
    for (int ww = 0; ww < kWaves; ++ww) M = fmaxf(M, lds.ml[ww][m].x);
    const float ref = M == kNegInf ? 0.f : M;
#pragma unroll
    for (int ww = 0; ww < kWaves; ++ww) L += lds.ml[ww][m].y * __builtin_amdgcn_exp2f(lds.ml[ww][m].x - ref);
    const float f = __builtin_amdgcn_exp2f(m_run[mt] - ref);
    if (w == 0 && g == 0) lds.row[m] = make_float2(L != L ? ref : M, L);  // (a sum that is NaN stays with its row)
    // (row m of a wave's O as DH floats; its 16-byte pieces rotated by the row, for the banks)
    float* dst = reinterpret_cast<float*>(mine) + m * DH;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      f32x4 x;
      int ch;
      if constexpr (BF16) {
        x = acc[mt][d];
        ch = d * 4 + g;  // dims 16 d + 4 g ..
      } else {
        const int h = d >> 2, i = d & 3;  // dims 64 h + 16 g + 4 i ..
        x = f32x4{acc[mt][h * 4][i], acc[mt][h * 4 + 1][i], acc[mt][h * 4 + 2][i], acc[mt][h * 4 + 3][i]};
        ch = h * 16 + g * 4 + i;
      }
      *reinterpret_cast<f32x4*>(dst + ((ch + m) & (DH / 4 - 1)) * 4) = f > 0.f ? x * f : f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }
  __syncthreads();
  const bool whole = a.S == 1 || (joins && nsplit == 1);  // uniform: nothing to join
  const __amdgpu_buffer_rsrc_t prs = block_rsrc(a.part_o + part * DH);
  for (int idx = tid; idx < a.R * (DH / 4); idx += NT) {
    const int m = idx / (DH / 4), ch = idx % (DH / 4);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ww = 0; ww < kWaves; ++ww)
      o += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds.tiles[ww]) + m * DH + ((ch + m) & (DH / 4 - 1)) * 4);
    const float2 ml = lds.row[m];
    if (whole) {
      if (a.key_weights && ch == 0) a.part_ml[part + m] = ml;  // (uniform) for the weights, however these are made
      store_row(m, ch, ml.y == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : o * (1.f / ml.y));
    } else if (joins) {
      store16_agent(prs, (unsigned)(m * DH + ch * 4) * 4u, o);
      if (ch == 0)
        __hip_atomic_store(reinterpret_cast<uint64_t*>(a.part_ml + part + m),
                           (uint64_t)__float_as_uint(ml.x) | ((uint64_t)__float_as_uint(ml.y) << 32), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    } else {
      if (ch == 0) a.part_ml[part + m] = ml;
      *reinterpret_cast<f32x4*>(a.part_o + (part + m) * DH + ch * 4) = o;
    }
  }
  if (whole || !joins) return;

  // ---- the splits joined by the last of them to finish.  As the verify
  // kernel's: partials are written through to the device's point of coherence
  // (sc1), every thread waits for its stores' acknowledgement before the barrier
  // ahead of the arrival's count, and the workgroup that counts last loads them
  // from there, after the count came back; no cache is written back or
  // invalidated.  Joined in split order, whichever comes last.
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  unsigned* counter = a.counters + counter_slot(pair * a.subsets + sub);
  if (tid == 0)
    lds.holes = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(nsplit - 1);
  __syncthreads();
  if (!uniform(lds.holes)) return;
  if (tid == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int64_t first = part - (int64_t)split * a.R;  // row 0 of split 0
  const __amdgpu_buffer_rsrc_t ors = block_rsrc(a.part_o + first * DH), mrs = block_rsrc(a.part_ml + first);
  auto join = [&](auto width) {
    constexpr int CW = decltype(width)::value;            // splits loaded in a round trip: all of them
    constexpr int IG = CW == 4 ? 3 : 2;                   // items of a thread at a time
    const int items = a.R * (DH / 4);
    for (int i0 = tid; i0 < items; i0 += IG * NT) {
      float2 ml[IG][CW];
      f32x4 o[IG][CW];
#pragma unroll
      for (int k = 0; k < CW; ++k) {
        const unsigned rows = (unsigned)(uniform(k < nsplit ? k : 0) * a.R);
#pragma unroll
        for (int i = 0; i < IG; ++i) {
          const int idx = min(i0 + i * NT, items - 1);
          ml[i][k] = load8_agent(mrs, (unsigned)(idx / (DH / 4)) * 8u, rows * 8u);
          o[i][k] = load16_agent(ors, (unsigned)idx * 16u, rows * (DH * 4u));
        }
      }
#pragma unroll
      for (int i = 0; i < IG; ++i) {
        const int idx = i0 + i * NT;
        if (idx >= items) break;
        float M = kNegInf, den = 0.f;
        f32x4 num = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < CW; ++k) M = fmaxf(M, k < nsplit ? ml[i][k].x : kNegInf);
        const float ref = M == kNegInf ? 0.f : M;
#pragma unroll
        for (int k = 0; k < CW; ++k) {
          const float wk = k < nsplit ? __builtin_amdgcn_exp2f(ml[i][k].x - ref) : 0.f;
          den = fmaf(ml[i][k].y, wk, den);
#pragma unroll
          for (int e = 0; e < 4; ++e) num[e] = fmaf(o[i][k][e], wk, num[e]);
        }
        store_row(idx / (DH / 4), idx % (DH / 4), den == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : num * (1.f / den));
      }
    }
  };
  if (nsplit <= 4) join(std::integral_constant<int, 4>{});  // uniform
  else join(std::integral_constant<int, kJoinedSplits>{});
}

// ---------------------------------------------------------------------------
// The splits joined, and the key weights from stored scores.
//
// Workgroups y < merges: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s of
// a (pair, head subset)'s rows, one after another; the splits of a row are
// dealt to `1 << sg_log2` groups of D / 4 lanes (a call of few pairs has up to
// 64 of them, 14 us one after another), whose parts are added in order.  A split
// without a key of the row (maximum -inf) holds no output.
//
// Workgroups behind them: 256 keys of a pair, one per thread, for all its
// rows, whose statistics they join themselves.  One thread adds to a place (of a
// key at or behind the sequence's first row: to the zero that the attention left
// there), by an atomic add, so that sequences which share a page lose nothing.
// ---------------------------------------------------------------------------
template <typename T, int DH>
__device__ __forceinline__ void merge_rows(const RowArgs& a, int ps, int block, int sg_log2) {
  constexpr int C4 = DH / 4, GROUPS = 256 / C4;
  __shared__ __attribute__((aligned(16))) f32x4 nums[GROUPS][C4];
  __shared__ float2 mls[GROUPS];
  const int grp = threadIdx.x / C4, ch = threadIdx.x % C4;
  const int sg = 1 << sg_log2, si = grp & (sg - 1);
  const int m = block * (GROUPS >> sg_log2) + (grp >> sg_log2);
  const int pair = ps / a.subsets, sub = ps - pair * a.subsets;
  const int b = pair / a.Hkv, hk = pair - b * a.Hkv;
  const int q0 = a.cu_seqlens_q[b], qlen = a.cu_seqlens_q[b + 1] - q0;
  const int gh = m / a.QL, t = m - gh * a.QL;
  const bool row = m < a.R && t < qlen;
  const int64_t base = (int64_t)ps * a.S * a.R + (row ? m : 0);
  constexpr int CH = kJoinedSplits;  // splits per round trip: what the attention kernel joins, joined alike, bit for bit
  float M = kNegInf, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = si; s0 < a.S; s0 += sg * CH) {
    float2 ml[CH];
    f32x4 o[CH];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int64_t r = base + (int64_t)min(s0 + k * sg, a.S - 1) * a.R;
      ml[k] = a.part_ml[r];
      o[k] = *reinterpret_cast<const f32x4*>(a.part_o + r * DH + ch * 4);
    }
    float Mn = M;
#pragma unroll
    for (int k = 0; k < CH; ++k) Mn = fmaxf(Mn, s0 + k * sg < a.S ? ml[k].x : kNegInf);
    const float ref = Mn == kNegInf ? 0.f : Mn;
    const float w0 = __builtin_amdgcn_exp2f(M - ref);  // (from -inf: 0)
    den *= w0;
    num *= w0;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const bool on = s0 + k * sg < a.S && ml[k].x > kNegInf;  // (else its output may hold anything)
      const float wk = on ? __builtin_amdgcn_exp2f(ml[k].x - ref) : 0.f;
      den = fmaf(on ? ml[k].y : 0.f, wk, den);
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = on ? fmaf(o[k][e], wk, num[e]) : num[e];
    }
    M = Mn;
  }
  if (sg > 1) {  // uniform
    nums[grp][ch] = num;
    if (ch == 0) mls[grp] = make_float2(M, den);
    __syncthreads();
    if (si != 0) return;
    for (int k = 1; k < sg; ++k) {
      const float2 x = mls[grp + k];
      if (!(x.x > kNegInf)) continue;
      const float Mn = fmaxf(M, x.x);
      const float w0 = __builtin_amdgcn_exp2f(M - Mn), w1 = __builtin_amdgcn_exp2f(x.x - Mn);
      den = fmaf(x.y, w1, den * w0);
      num = num * w0 + nums[grp + k][ch] * w1;
      M = Mn;
    }
  }
  if (!row) return;
  num = den == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : num * (1.f / den);
  T* dst = (T*)a.out + ((int64_t)(q0 + t) * a.H + hk * (a.G * a.subsets) + sub * a.G + gh) * DH + ch * 4;
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(num[0], num[1]), pack_bf16x2(num[2], num[3]));
  else *reinterpret_cast<f32x4*>(dst) = num;
}

constexpr int kMaxStoredRows = 64;

// CH: rows whose scores are loaded in a round trip.
template <int CH>
__device__ __forceinline__ void stored_weights(const RowArgs& a, int pair, int block) {
  __shared__ float2 stat[kMaxStoredRows];  // maximum and 1 / sum
  const int b = pair / a.Hkv, hk = pair - b * a.Hkv;
  const int64_t len = a.context_lens[b];
  if (block * 256 >= len) return;  // uniform
  // the scores, the page and the statistics, in one round trip beside the sequence's rows' positions
  const int key = block * 256 + threadIdx.x, rows = a.R * a.subsets;
  const float* src = a.scores + (int64_t)pair * rows * a.score_keys + min(key, a.score_keys - 1);
  float s[CH];
  auto read = [&](int m0) {
#pragma unroll
    for (int k = 0; k < CH; ++k) s[k] = src[(int64_t)min(m0 + k, rows - 1) * a.score_keys];
  };
  read(0);
  const int entry = min(key >> a.bs_log2, a.max_blocks - 1);
  const int p = a.block_tables[(int64_t)b * a.max_blocks + entry];
  const int q0 = uniform(a.cu_seqlens_q[b]);
  const int qlen = min(uniform(a.cu_seqlens_q[b + 1]) - q0, a.QL);
  const int64_t p64 = row_position(a, q0, qlen);
  join_stats(a, pair * a.subsets, rows, stat);
  int my_pos;
  const Span sp = make_span(a, len, qlen, p64, my_pos);
  __syncthreads();
  if (key >= sp.total || p < 0) return;
  float y = 0.f;
  for (int m0 = 0; m0 < rows; m0 += CH) {
    if (m0 > 0) read(m0);
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const float2 x = stat[min(m0 + k, rows - 1)];
      const bool on = m0 + k < rows && x.y != 0.f && s[k] != kNegInf;  // (a masked key of a row that is NaN stays out of it)
      y = on ? fmaf(__builtin_amdgcn_exp2f(s[k] - x.x), x.y, y) : y;
    }
  }
  unsafeAtomicAdd(a.key_weights + (((int64_t)p * a.Hkv + hk) << a.bs_log2) + (key & ((1 << a.bs_log2) - 1)), y);
}

template <typename T, int DH>
__global__ __launch_bounds__(256) void row_finish_kernel(RowArgs a, int merges, int sg_log2) {
  if ((int)blockIdx.y < merges) {
    const int pair = blockIdx.x / a.subsets;  // (x: pairs x subsets for these, the rest of the grid's rows use pairs)
    if (pair < a.npairs) merge_rows<T, DH>(a, blockIdx.x, blockIdx.y, sg_log2);
  } else if ((int)blockIdx.x < a.npairs) {
    if (a.R * a.subsets <= 4) stored_weights<4>(a, blockIdx.x, blockIdx.y - merges);  // uniform
    else stored_weights<32>(a, blockIdx.x, blockIdx.y - merges);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
constexpr int kStoredMiB = 32;
constexpr int kCus = 256;        // compute units of an MI355X
constexpr int kOverheadKeys = 256;

// Splits per pair: the rounds of resident workgroups that a count takes, each
// as long as its keys and a workgroup's start and end, which take as long as
// kOverheadKeys keys (64 to 1,024: no difference), and 128 keys more where the
// splits are too many for the kernel to join.  Whole rounds: 64 pairs of 4,108
// keys in 4 splits (256 workgroups) 35 us, 6 48, 8 47, 12 54; 64 pairs of 1,250
// keys 15 us in 4, 19 in 6 and 8; 24 pairs of 1,009 keys in fp32 9.5 us in 8
// splits, 10.5 in 16.
int choose_splits(int64_t units, int64_t keys, int tile, int resident) {
  const int64_t most = std::min<int64_t>(kMaxSplits, (keys + tile * kWaves - 1) / (tile * kWaves));
  int64_t best = 1, best_cost = INT64_MAX;
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t rounds = (units * s + resident - 1) / resident;
    const int64_t cost = rounds * ((keys + s - 1) / s + kOverheadKeys) + (s > kJoinedSplits ? 128 : 0);
    if (cost < best_cost) {
      best = s;
      best_cost = cost;
    }
  }
  return (int)best;
}

struct RowPlan {
  int G, subsets, R, MT, S;
  bool stored;     // key weights: from stored scores, else from the keys again
  int score_keys;
  size_t ml_bytes, o_bytes, score_bytes;
};

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int make_row_plan(int B, int H, int Hkv, int D, int block_size, int max_blocks, int max_q_len, int dtype, int window,
                  int sinks, bool weights, RowPlan* p) {
  if (B < 0 || H <= 0 || Hkv <= 0 || max_blocks <= 0 || max_q_len <= 0 || window < 0 || sinks < 0) return NSV_ERR_ARG;
  if (dtype != NSV_F32 && dtype != NSV_BF16) return NSV_ERR_ARG;
  if (H % Hkv || (D != 64 && D != 128) || max_q_len > 64) return NSV_ERR_UNSUPPORTED;
  if (block_size <= 0 || (block_size & (block_size - 1))) return NSV_ERR_UNSUPPORTED;
  const int64_t cap = (int64_t)max_blocks * block_size;
  if (cap > (int64_t)1 << 30) return NSV_ERR_UNSUPPORTED;
  const int group = H / Hkv;
  p->G = group;
  while (p->G * max_q_len > 64) {
    int g = p->G - 1;
    while (group % g) --g;
    p->G = g;
  }
  p->subsets = group / p->G;
  p->R = p->G * max_q_len;
  p->MT = (p->R + 15) / 16;
  const int64_t pairs = (int64_t)B * Hkv;
  // the most keys that some row of a sequence of consecutive rows sees
  int64_t keys = cap;
  if (window > 0) keys = std::min<int64_t>(cap, (int64_t)window + sinks + max_q_len - 1);
  const int tile = dtype == NSV_BF16 ? 32 : 16;
  p->S = choose_splits(pairs * p->subsets, keys, tile, D == 64 ? 2 * kCus : kCus);
  p->score_keys = (int)((cap + 31) / 32 * 32);
  p->score_bytes = weights ? (size_t)pairs * p->subsets * p->R * p->score_keys * sizeof(float) : 0;
  p->stored = weights && p->R * p->subsets <= kMaxStoredRows && p->score_bytes <= ((size_t)kStoredMiB << 20);
  if (!p->stored) p->score_bytes = 0;
  const size_t rows = (size_t)pairs * p->subsets * p->S * p->R;
  p->ml_bytes = align256(rows * sizeof(float2));
  p->o_bytes = p->S > 1 ? align256(rows * (size_t)D * sizeof(float)) : 0;
  if (pairs * p->subsets * p->S > 0x7fffffff) return NSV_ERR_UNSUPPORTED;
  return NSV_OK;
}

template <typename T, int DH, int MODE>
void launch_rows(const RowArgs& a, int MT, dim3 grid, hipStream_t s) {
  const dim3 block(kWaves * 64);
  switch (MT) {
    case 1: hipLaunchKernelGGL((row_attention_kernel<T, 1, DH, MODE>), grid, block, 0, s, a); break;
    case 2: hipLaunchKernelGGL((row_attention_kernel<T, 2, DH, MODE>), grid, block, 0, s, a); break;
    case 3: hipLaunchKernelGGL((row_attention_kernel<T, 3, DH, MODE>), grid, block, 0, s, a); break;
    default: hipLaunchKernelGGL((row_attention_kernel<T, 4, DH, MODE>), grid, block, 0, s, a); break;
  }
}

template <typename T, int DH>
int launch_call(RowArgs& a, const RowPlan& p, hipStream_t s) {
  const dim3 grid((unsigned)(a.npairs * p.subsets * p.S));
  if (p.stored) launch_rows<T, DH, kAttendScores>(a, p.MT, grid, s);
  else if (a.key_weights) launch_rows<T, DH, kAttendFirst>(a, p.MT, grid, s);
  else launch_rows<T, DH, kAttend>(a, p.MT, grid, s);
  int rc = nsv_launch_status();
  if (rc != NSV_OK) return rc;
  constexpr int groups = 256 / (DH / 4);
  int sg_log2 = 0;
  while ((1 << sg_log2) < groups && (kJoinedSplits << sg_log2) < p.S) ++sg_log2;  // a group takes eight splits in a round trip
  const int per = groups >> sg_log2;
  const int merges = p.S > 1 && !a.counters ? (p.R + per - 1) / per : 0, blocks = p.stored ? (p.score_keys + 255) / 256 : 0;
  if (merges + blocks > 0) {
    const dim3 fgrid(a.npairs * (merges ? p.subsets : 1), merges + blocks);
    hipLaunchKernelGGL((row_finish_kernel<T, DH>), fgrid, dim3(256), 0, s, a, merges, sg_log2);
    rc = nsv_launch_status();
    if (rc != NSV_OK) return rc;
  }
  if (!a.key_weights || p.stored) return NSV_OK;
  // (no V tiles: twice as many workgroups fit a compute unit, and no split leaves anything to join)
  a.weight_splits = choose_splits(a.npairs, (int64_t)a.max_blocks << a.bs_log2, sizeof(T) == 2 ? 32 : 16,
                                  2 * (DH == 64 ? 2 * kCus : kCus));
  for (a.first_subset = 0; a.first_subset < p.subsets; ++a.first_subset) {
    launch_rows<T, DH, kWeights>(a, p.MT, dim3((unsigned)(a.npairs * a.weight_splits)), s);
    rc = nsv_launch_status();
    if (rc != NSV_OK) return rc;
  }
  return NSV_OK;
}

int row_attention(void* out, const void* q, const void* k_cache, const void* v_cache, float* key_weights,
                  const int32_t* block_tables, const int64_t* context_lens, const int32_t* cu_seqlens_q,
                  const int64_t* positions, float scale, int B, int T, int H, int Hkv, int D, int block_size,
                  int max_blocks, int max_q_len, int dtype, int window, int sinks, bool weights, unsigned* counters,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0) return NSV_ERR_ARG;
  RowPlan p;
  const int rc = make_row_plan(B, H, Hkv, D, block_size, max_blocks, max_q_len, dtype, window, sinks, weights, &p);
  if (rc != NSV_OK) return rc;
  if (B == 0 || T == 0) return NSV_OK;
  if (!out || !q || !k_cache || !v_cache || !block_tables || !context_lens || !cu_seqlens_q || !positions ||
      (weights && !key_weights))
    return NSV_ERR_ARG;
  if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)counters) % 16) return NSV_ERR_ARG;
  if (!workspace || workspace_bytes < p.ml_bytes + p.o_bytes + p.score_bytes) return NSV_ERR_WORKSPACE;
  RowArgs a;
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.out = out;
  a.block_tables = block_tables;
  a.context_lens = context_lens;
  a.cu_seqlens_q = cu_seqlens_q;
  a.positions = positions;
  a.part_ml = (float2*)workspace;
  a.part_o = (float*)((char*)workspace + p.ml_bytes);
  a.scores = (float*)((char*)workspace + p.ml_bytes + p.o_bytes);
  a.counters = !weights && p.S <= kJoinedSplits && (int64_t)B * Hkv * p.subsets <= kCounters ? counters : nullptr;
  a.key_weights = weights ? key_weights : nullptr;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.H = H;
  a.Hkv = Hkv;
  a.G = p.G;
  a.subsets = p.subsets;
  a.bs_log2 = __builtin_ctz((unsigned)block_size);
  a.max_blocks = max_blocks;
  a.QL = max_q_len;
  a.R = p.R;
  a.S = p.S;
  a.npairs = B * Hkv;
  a.window = window;
  a.sinks = sinks;
  a.score_keys = p.score_keys;
  a.weight_splits = 1;
  a.first_subset = 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == NSV_BF16) return D == 128 ? launch_call<bf16_t, 128>(a, p, s) : launch_call<bf16_t, 64>(a, p, s);
  return D == 128 ? launch_call<float, 128>(a, p, s) : launch_call<float, 64>(a, p, s);
}

}  // namespace

extern "C" {

size_t nsv_window_attention_workspace_size(int B, int H, int Hkv, int D, int block_size, int max_blocks, int max_q_len,
                                           int dtype, int window, int sinks) {
  RowPlan p;
  if (window <= 0 || make_row_plan(B, H, Hkv, D, block_size, max_blocks, max_q_len, dtype, window, sinks, false, &p) != NSV_OK)
    return 0;
  return p.ml_bytes + p.o_bytes;
}

int nsv_window_attention(void* out, const void* q, const void* k_cache, const void* v_cache,
                         const int32_t* block_tables, const int64_t* context_lens, const int32_t* cu_seqlens_q,
                         const int64_t* positions, float scale, int B, int T, int H, int Hkv, int D, int block_size,
                         int max_blocks, int max_q_len, int dtype, int window, int sinks, void* counters,
                         void* workspace, size_t workspace_bytes, void* stream) {
  if (window <= 0) return NSV_ERR_ARG;
  return row_attention(out, q, k_cache, v_cache, nullptr, block_tables, context_lens, cu_seqlens_q, positions, scale, B,
                       T, H, Hkv, D, block_size, max_blocks, max_q_len, dtype, window, sinks, false, (unsigned*)counters, workspace,
                       workspace_bytes, stream);
}

size_t nsv_weights_attention_workspace_size(int B, int H, int Hkv, int D, int block_size, int max_blocks, int max_q_len,
                                            int dtype) {
  RowPlan p;
  if (make_row_plan(B, H, Hkv, D, block_size, max_blocks, max_q_len, dtype, 0, 0, true, &p) != NSV_OK) return 0;
  return p.ml_bytes + p.o_bytes + p.score_bytes;
}

int nsv_weights_attention(void* out, const void* q, const void* k_cache, const void* v_cache, float* key_weights,
                          const int32_t* block_tables, const int64_t* context_lens, const int32_t* cu_seqlens_q,
                          const int64_t* positions, float scale, int B, int T, int H, int Hkv, int D, int block_size,
                          int max_blocks, int max_q_len, int dtype, void* workspace, size_t workspace_bytes,
                          void* stream) {
  return row_attention(out, q, k_cache, v_cache, key_weights, block_tables, context_lens, cu_seqlens_q, positions, scale,
                       B, T, H, Hkv, D, block_size, max_blocks, max_q_len, dtype, 0, 0, true, nullptr, workspace,
                       workspace_bytes, stream);
}

}  // extern "C"
