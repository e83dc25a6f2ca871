// Sampling and acceptance of drafts under a temperature, top-k, top-p and
// min-p, for gfx950.  No reference counterpart (its sampler has a temperature
// only); the operators stand beside nsv_sample and nsv_accept_stochastic.
//
// Of a row x with maximum M and temperature T the weights are
// w = exp((x - M) / T) (1 where x = M, 0 where x = -inf), and its tokens are
// ordered by falling x, equal ones by rising index.  Each filter leaves a
// beginning of that order: top-k its first k; top-p the fewest whose sum
// reaches p times the sum that top-k left; min-p those with w >= min_p.  So
// what all of them leave is described by its last token: a value, and an index
// among the tokens of that value.  The sample of u is the first token whose
// running sum along the order exceeds u W, W the sum of what is left: one
// uniform number per row, and no noise of the vocabulary's size to draw and
// read.  T <= 1e-6, and rows with a NaN or without a value above -inf, leave
// the argmax alone (first maximum, NaN above all, torch's rule).
//
// filter_rows_kernel works one row out per workgroup.
//   bf16 (count_row): a row has few distinct values, so one pass counts the
//     tokens of each of the 65,536 in LDS (16 bits each), and everything else
//     comes from the counts: a value's tokens weigh count * w, one exponential
//     per value that occurs (some 3,000) instead of one per token.  The row
//     stays in registers, where the sampled token is found by its value and
//     its rank among the tokens of that value.
//   fp32 (filter_row): a value is found by radix descent over its
//     order-preserving bits: per level a histogram in LDS of the row's tokens
//     below the prefix so far, counts and weights, and a scan of its bins.
//     Weights are added up as 64-bit integers, w 2^s rounded, so sums do not
//     depend on the order of the additions; s leaves room for the vocabulary
//     (44 bits for 2^18 tokens), each weight off by 2^-45 of the largest, where
//     fp32 sums would move the sample of one row in a hundred.

#include "common.h"
#include "exp_f64.h"

namespace {

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kBins = 2048;
constexpr int kVec = 8;                          // elements a thread takes at a time
constexpr int kStep = kRowThreads * kVec;        // elements a workgroup takes at a time
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxSteps = kMaxVocab / kStep + 1; // (a row that starts off a 16-byte boundary)
constexpr int kMaxDrafts = 63;                   // K + 1 rows fit one 64-lane ballot
constexpr int kChunkThreads = 256;
constexpr int kChunk = kChunkThreads * kVec;     // of the residual passes

struct Part;
template <typename T> struct Elem;
template <> struct Elem<uint16_t> {  // bf16 bits
  __device__ static float get(uint16_t v) { return bf16_bits_to_f32(v); }
  __device__ static float unpack(const u32x4& w, int e) {
    return bf16_bits_to_f32((e & 1) ? (w[e >> 1] >> 16) : (w[e >> 1] & 0xffffu));
  }
};
template <> struct Elem<float> {
  __device__ static float get(float v) { return v; }
  __device__ static float unpack(const u32x4& w, int e) { return __uint_as_float(w[e]); }
};

// What the filters leave of a row: tokens of x > cut, and of x == cut up to
// the index `last`; top: the row's maximum; total: W; kept: how many.  kept 1
// is `token` alone, whatever the row holds.
struct RowCut {
  float top, cut;
  int32_t last, kept, token, pad;
  double total;
};

struct FilterArgs {
  const void* target;      // row r of sequence b at b * t_seq + r * t_row elements
  int64_t t_seq, t_row;
  const void* draft;       // nullable; row i of sequence b at (b * d_seq + i * d_row) * V
  int64_t d_seq, d_row;
  int B, K, V;             // K -1: the sampler (one row per sequence, one uniform)
  int shift;               // weights are held as integers, w 2^shift
  const float* temperature;
  const int32_t* top_k;    // nullable
  const float* top_p;      // nullable
  const float* min_p;      // nullable
  const float* uniforms;   // [B, K + 1]
  const int32_t* drafts;   // [B, K]
  const int32_t* num_drafts;
  const int32_t* mode;     // nullable; 0: sequence b has no draft rows
  RowCut* cuts;            // [B, 2K + 1]: target rows 0..K, then draft rows
  double* probs;           // [B, 2K + 1]: the probability of the row's draft
  Part* row_parts;         // [B, rows per sequence, split]
  int split;
  double* parts;           // [B, chunks, 2]: sums of the residual and of p_target
  int chunks;
  int32_t* tokens;         // sampler: row b's at b * out_stride
  int64_t out_stride;
  int32_t* kept;           // sampler, nullable
  int32_t* out_tokens;     // [B, K + 1]
  int32_t* out_len;
};

__device__ __forceinline__ bool is_greedy(float T) { return !(T > 1e-6f); }
// u of the sample's goal u W: what is no number in [0, 1] is taken to its end
__device__ __forceinline__ double unit(float u) { return fmin(fmax((double)u, 0.0), 1.0); }
// sequence b's drafts are decided by their probabilities
__device__ __forceinline__ bool by_rows(const FilterArgs& a, int b) {
  return a.draft && !(a.mode && a.mode[b] == 0) && !is_greedy(a.temperature[b]);
}
__device__ __forceinline__ int draft_count(const FilterArgs& a, int b) { return min(max(a.num_drafts[b], 0), a.K); }
__device__ __forceinline__ int64_t draft_at(const FilterArgs& a, int b, int i) {
  return ((int64_t)b * a.d_seq + (int64_t)i * a.d_row) * a.V;
}

// order-preserving bits, complemented: rising along the order of the tokens;
// -0 as +0
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k : ~(k | 0x80000000u));
}

__device__ __forceinline__ double weight_of(float x, float top, double inv_t, const double* tab) {
  return x == top ? 1.0 : nsv_exp_nonpos(((double)x - (double)top) * inv_t, tab);
}
// w 2^shift, rounded: added to 2^52 it lies in the low bits of the sum
__device__ __forceinline__ uint64_t fixed_weight(double w, double scale) {
  return (uint64_t)__double_as_longlong(fma(w, scale, 0x1p52)) & 0x000fffffffffffffull;
}

// elements base .. base + 7 of a row, those past its end -inf
template <typename T>
__device__ __forceinline__ void load_vec(const T* row, int64_t base, int V, float (&x)[kVec]) {
  constexpr int PER = 16 / sizeof(T);
  if (((uintptr_t)row & 15) == 0 && base + kVec <= V) {
    u32x4 w[kVec / PER];
#pragma unroll
    for (int l = 0; l < kVec / PER; ++l) w[l] = *reinterpret_cast<const u32x4*>(row + base + l * PER);
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = Elem<T>::unpack(w[e / PER], e % PER);
  } else {
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = base + e < V ? Elem<T>::get(row[base + e]) : -__builtin_inff();
  }
}

// f(index, x) of every element of a row, a workgroup's threads together
template <typename T, typename F>
__device__ __forceinline__ void each(const T* row, int V, F f) {
  for (int64_t lo = 0; lo < V; lo += kStep) {
    const int64_t base = lo + kVec * threadIdx.x;
    if (base >= V) continue;
    float x[kVec];
    load_vec<T>(row, base, V, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (base + e < V) f((int)(base + e), x[e]);
  }
}

// Inclusive scan over a wave's 64 lanes on the VALU: within rows of 16 by
// shifts of 1, 2, 4 and 8 lanes, then the last lane of row 0 and 2 to the row
// behind it, and of row 1 to rows 2 and 3 (what has no source adds 0).  A
// sixth of the shuffles' time, whose every step is a round trip through LDS.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp_or_zero(T v) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, ((uint64_t)hi << 32) | lo);
  }
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += dpp_or_zero<0x111, 0xf>(v);
  v += dpp_or_zero<0x112, 0xf>(v);
  v += dpp_or_zero<0x114, 0xf>(v);
  v += dpp_or_zero<0x118, 0xf>(v);
  v += dpp_or_zero<0x142, 0xa>(v);
  v += dpp_or_zero<0x143, 0xc>(v);
  return v;
}
// lane l's value (l uniform), and the lane's before a lane's own
__device__ __forceinline__ double lane_f64(double v, int l) {
  return __longlong_as_double((long long)lane_u64((uint64_t)__double_as_longlong(v), l));
}
template <typename T>
__device__ __forceinline__ T lane_before(T v) {
  return dpp_or_zero<0x138, 0xf>(v);  // the whole wave one lane up, 0 into the first
}

struct RowLds {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
  uint32_t found[kMaxSteps * kRowWaves];
  uint64_t red[kRowWaves];
  uint64_t red2[kRowWaves];
  double tab[256];
  int hit;
  uint64_t hit_mass, hit_before;
  uint32_t hit_count, hit_cbefore;
};

__device__ __forceinline__ uint64_t block_max(uint64_t v, RowLds& s) {
  v = wave_max_u64_dpp(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = s.red[0];
  for (int i = 1; i < kRowWaves; ++i) r = s.red[i] > r ? s.red[i] : r;
  return r;
}
__device__ __forceinline__ uint64_t block_sum(uint64_t v, RowLds& s) {
  v = wave_scan(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s.red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t r = 0;
  for (int i = 0; i < kRowWaves; ++i) r += s.red[i];
  return r;
}

// A place in the order: the tokens of one value, what lies before them, and
// the weight of each.
struct Spot {
  uint32_t key;            // order_bits of the value
  uint32_t before, count;  // tokens
  uint64_t mass;           // weights before
  uint64_t weight;
};
enum Seek { kByCount, kReach, kAbove, kBeyond };

// The last value with: tokens before it < goal (kByCount); weights before it
// < goal (kReach) or <= goal (kBeyond), and a weight of its own.
template <typename T>
__device__ Spot seek(Seek kind, double goal, const T* row, int V, float top, double inv_t, double scale, RowLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Spot at{0u, 0u, 0u, 0ull, 0ull};
  constexpr int kShift[3] = {21, 10, 0}, kWidth[3] = {11, 11, 10};
  for (int level = 0; level < 3; ++level) {
    const int sh = kShift[level], bits = kWidth[level];
    __syncthreads();
    for (int i = tid; i < kBins; i += kRowThreads) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
    if (tid == 0) s.hit = -1;
    __syncthreads();
    each<T>(row, V, [&](int, float x) {
      const uint32_t k = order_bits(x);
      if (level && (k >> (sh + bits)) != (at.key >> (sh + bits))) return;
      const uint32_t bin = (k >> sh) & ((1u << bits) - 1);
      atomicAdd(&s.count[bin], 1u);
      const uint64_t q = fixed_weight(weight_of(x, top, inv_t, s.tab), scale);
      if (q) atomicAdd(&s.mass[bin], (unsigned long long)q);
    });
    __syncthreads();
    const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
    const uint64_t m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
    const uint32_t c = wave_scan(c0 + c1);
    const uint64_t m = wave_scan(m0 + m1);
    if (lane == 63) {
      s.red[wave] = c;
      s.red2[wave] = m;
    }
    __syncthreads();
    uint32_t cb = at.before + c - c0 - c1;
    uint64_t mb = at.mass + m - m0 - m1;
    for (int i = 0; i < wave; ++i) {
      cb += (uint32_t)s.red[i];
      mb += s.red2[i];
    }
    auto fits = [&](uint32_t n, uint64_t w, uint32_t before, uint64_t mass) {
      if (kind == kByCount) return n > 0 && (double)before < goal;
      return w > 0 && (kind == kReach ? (double)mass < goal : (double)mass <= goal);
    };
    int best = -1;
    if (fits(c0, m0, cb, mb)) best = 2 * tid;
    if (fits(c1, m1, cb + c0, mb + m0)) best = 2 * tid + 1;
    if (best >= 0) atomicMax(&s.hit, best);
    __syncthreads();
    if (best >= 0 && best == s.hit) {
      const bool second = best & 1;
      s.hit_cbefore = cb + (second ? c0 : 0);
      s.hit_before = mb + (second ? m0 : 0);
      s.hit_count = second ? c1 : c0;
      s.hit_mass = second ? m1 : m0;
    }
    __syncthreads();
    at.key |= (uint32_t)max(s.hit, 0) << sh;
    at.before = s.hit_cbefore;
    at.mass = s.hit_before;
    at.count = s.hit_count;
    at.weight = s.hit_mass;
  }
  at.weight /= at.count;  // (equal values have equal weights)
  return at;
}

// index of the token with j of its value before it
template <typename T>
__device__ int index_of(float value, uint32_t j, const T* row, int V, RowLds& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int steps = (V + kStep - 1) / kStep;
  __syncthreads();
  for (int it = 0; it < steps; ++it) {
    const int64_t base = (int64_t)it * kStep + kVec * threadIdx.x;
    float x[kVec];
    int n = 0;
    if (base < V) {
      load_vec<T>(row, base, V, x);
      for (int e = 0; e < kVec; ++e) n += base + e < V && x[e] == value;
    }
    n = (int)wave_scan((uint32_t)n);
    if (lane == 63) s.found[it * kRowWaves + wave] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t left = j;
    int g = 0;
    while (g < steps * kRowWaves - 1 && left >= s.found[g]) left -= s.found[g++];
    s.hit = g;
    s.hit_count = left;
  }
  __syncthreads();
  const int g = s.hit;
  const uint32_t left = s.hit_count;
  if (wave == g % kRowWaves) {
    const int64_t base = (int64_t)(g / kRowWaves) * kStep + kVec * threadIdx.x;
    float x[kVec];
    uint32_t n = 0;
    if (base < V) {
      load_vec<T>(row, base, V, x);
      for (int e = 0; e < kVec; ++e) n += base + e < V && x[e] == value;
    }
    uint32_t before = wave_scan(n) - n;
    if (base < V)
      for (int e = 0; e < kVec; ++e)
        if (base + e < V && x[e] == value) {
          if (before == left) s.hit_cbefore = (uint32_t)(base + e);
          ++before;
        }
  }
  __syncthreads();
  return (int)s.hit_cbefore;
}

// What the filters leave of a row, and its sample of u where one is wanted.
template <typename T>
__device__ RowCut filter_row(const FilterArgs& a, int b, const T* row, bool sampled, float u, bool ends, RowLds& s) {
  const int V = a.V;
  const float T_ = a.temperature[b];
  RowCut out;
  // the argmax: NaN above all, equal values by the lower index
  uint64_t best = 0;
  each<T>(row, V, [&](int i, float x) {
    const uint32_t k = x != x ? 0xffffffffu : ~order_bits(x);
    const uint64_t key = ((uint64_t)k << 32) | (uint32_t)~i;
    best = key > best ? key : best;
  });
  best = block_max(best, s);
  const int first = (int)~(uint32_t)best;
  const bool nan = (uint32_t)(best >> 32) == 0xffffffffu;
  out.top = nan ? __builtin_nanf("") : order_value(~(uint32_t)(best >> 32));
  out.cut = out.top;
  out.last = out.token = first;
  out.kept = 1;
  out.pad = 0;
  out.total = 1.0;
  if (is_greedy(T_) || nan || out.top == -__builtin_inff()) return out;  // uniform

  const double inv_t = 1.0 / (double)T_, scale = (double)(1ull << a.shift);
  const float top = out.top;
  if (threadIdx.x < 256) s.tab[threadIdx.x] = kExp2Frac256[threadIdx.x];
  const int k = a.top_k ? a.top_k[b] : 0;
  const double p = a.top_p ? (double)a.top_p[b] : 1.0, m = a.min_p ? (double)a.min_p[b] : 0.0;
  out.kept = V;
  out.cut = -__builtin_inff();
  out.last = V - 1;
  __syncthreads();
  uint64_t total;
  if (k > 0 && k < V) {
    const Spot at = seek<T>(kByCount, (double)k, row, V, top, inv_t, scale, s);
    out.kept = k;
    out.cut = order_value(at.key);
    out.last = (uint32_t)k - at.before == at.count ? V - 1 : -(int)((uint32_t)k - at.before);  // (negative: to be looked up)
    total = at.mass + (uint64_t)((uint32_t)k - at.before) * at.weight;
  } else {
    uint64_t sum = 0;
    each<T>(row, V, [&](int, float x) { sum += fixed_weight(weight_of(x, top, inv_t, s.tab), scale); });
    total = block_sum(sum, s);
  }
  if (p < 1.0) {
    const double goal = fmax(p * (double)total, 0.5);  // (the first token stays)
    const Spot at = seek<T>(kReach, goal, row, V, top, inv_t, scale, s);
    const double need = ceil((goal - (double)at.mass) / (double)at.weight);
    const uint32_t n = (uint32_t)fmin(fmax(need, 1.0), (double)at.count);
    if ((int)(at.before + n) < out.kept) {
      out.kept = (int)(at.before + n);
      out.cut = order_value(at.key);
      out.last = n == at.count ? V - 1 : -(int)n;
      total = at.mass + (uint64_t)n * at.weight;
    }
  }
  if (m > 0.0) {
    uint64_t sum = 0, count = 0, low = 0;  // low: the furthest key along the order
    each<T>(row, V, [&](int, float x) {
      const double w = weight_of(x, top, inv_t, s.tab);
      if (x != top && !(w >= m)) return;
      sum += fixed_weight(w, scale);
      ++count;
      const uint64_t key = order_bits(x);
      low = key > low ? key : low;
    });
    count = block_sum(count, s);
    if ((int)count < out.kept) {
      out.kept = (int)count;
      out.last = V - 1;
      total = block_sum(sum, s);
      out.cut = order_value((uint32_t)block_max(low, s));
    }
  }
  out.total = (double)total / scale;
  if (sampled) {
    const double goal = unit(u) * (double)total;
    const Spot at = seek<T>(kBeyond, goal, row, V, top, inv_t, scale, s);
    double j = floor((goal - (double)at.mass) / (double)at.weight);
    j = fmin(fmax(j, 0.0), (double)(at.count - 1));
    j = fmin(j, (double)(out.kept - 1 - (int)at.before));
    out.token = index_of<T>(order_value(at.key), (uint32_t)j, row, V, s);
  }
  if (out.last < 0) out.last = ends ? index_of<T>(out.cut, (uint32_t)(-out.last - 1), row, V, s) : V - 1;
  return out;
}


// ---------------------------------------------------------------------------
// bf16 rows by counts
// ---------------------------------------------------------------------------
constexpr int kGroups = 512;   // of 128 values each, along the order of the tokens: 64 words of two counts
constexpr int kAhead = 4;      // vectors a thread loads ahead of those it counts
constexpr int kSafeSteps = 7;  // steps whose 57,344 tokens fit a 16-bit count beside ..
constexpr uint32_t kFull = 65536 - kSafeSteps * kStep;  // .. fewer than these
constexpr int kMaxHeavy = kRowWaves + kMaxVocab / kFull + 1;
constexpr int kMaxParts = 32;  // of a row, counted by a workgroup each ..
constexpr int kMaxSplit = 8;  // .. for speed this many

struct CountLds {
  uint32_t bin[32768];         // counts of values 2i (low half) and 2i + 1
  uint32_t occurs[kGroups / 32];
  // groups that occur, along the order
  double mass[kGroups];        // weights of a group, first of its first value's
  double before[kGroups];      // weights before a group
  uint32_t count[kGroups];
  uint32_t cbefore[kGroups];
  uint32_t ref[kGroups];       // group << 16 | bits of its first value that occurs
  uint32_t found[kMaxSteps * kRowWaves];
  double tab[256];
  uint32_t heavy[kMaxHeavy], heavy_count[kMaxHeavy];  // counts beside the bins
  uint32_t part_occurs[kMaxParts * kGroups / 32];
  int heavies;
  uint32_t slots;              // tokens counted
  int nan, index;
  // what wave 0 decides
  float top, cut;
  int kept, rank, cut_rank;    // rank -1: no token is looked up; cut_rank -1: no index is
  uint32_t value, cut_value;   // bits
  double total;
};

// A row as vectors of 8 elements on 16 bytes: vector g holds elements 8 g -
// skew .. + 7; what lies outside the row counts as -inf.
struct Row {
  const uint16_t* at;
  int V, skew, vecs;
  __device__ Row(const uint16_t* row, int V_) : at(row), V(V_), skew((int)(((uintptr_t)row & 15) >> 1)) {
    vecs = (V + skew + 7) / 8;
  }
  __device__ __forceinline__ u32x4 load(int g) const {
    const int64_t e0 = (int64_t)8 * g - skew;
    if (e0 >= 0 && e0 + 8 <= V) return *reinterpret_cast<const u32x4*>(at + e0);
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t a = e0 + 2 * i, b = a + 1;
      const uint32_t lo = a >= 0 && a < V ? at[a] : 0xff80u, hi = b >= 0 && b < V ? at[b] : 0xff80u;
      v[i] = lo | (hi << 16);
    }
    return v;
  }
};

// f(step, vector, whether there is one) of the vectors lo .. hi - 1, a
// workgroup's threads together, kAhead of them loaded ahead.  The loop stays
// rolled: a row kept in registers (one unrolled body per vector) saved its
// second reading, and cost more in instructions fetched once.
template <typename F>
__device__ __forceinline__ void each_vec(const Row& row, int lo, int hi, F f) {
  const int steps = (hi - lo + kRowThreads - 1) / kRowThreads;
  u32x4 v[kAhead];
  int g = lo + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) v[j] = row.load(min(g + j * kRowThreads, hi - 1));
#pragma unroll 1
  for (int it = 0; it < steps; it += kAhead) {
    u32x4 w[kAhead];
    if (it + kAhead < steps) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) w[j] = row.load(min(g + (kAhead + j) * kRowThreads, hi - 1));
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (it + j < steps) f(it + j, v[j], g + j * kRowThreads < hi);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) v[j] = w[j];
    g += kAhead * kRowThreads;
  }
}

__device__ __forceinline__ void count_value(uint32_t* bin, uint32_t bits) {
  atomicAdd(&bin[bits >> 1], 1u << ((bits & 1) << 4));
}

// The tokens of a vector counted.  A value that many of a wave's lanes hold
// (a mask's) would be 64 additions to one address one after another: the
// wave's first such value is added up beside the bins.
__device__ __forceinline__ void count_vec(uint32_t* bin, const u32x4& v, uint32_t& heavy, uint32_t& many) {
  const uint32_t some = (uint32_t)__builtin_amdgcn_readfirstlane((int)(v[0] & 0xffffu));
  if (__popcll(__ballot((v[0] & 0xffffu) == some)) >= 16 && (heavy == some || heavy == ~0u)) {  // uniform
    heavy = some;
    u32x4 w = v;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {  // (rarely run: small)
      const uint32_t lo = w[0] & 0xffffu, hi = w[0] >> 16;
      many += __popcll(__ballot(lo == some)) + __popcll(__ballot(hi == some));
      if (lo != some) count_value(bin, lo);
      if (hi != some) count_value(bin, hi);
      w = u32x4{w[1], w[2], w[3], w[0]};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) count_value(bin, (e & 1) ? v[e >> 1] >> 16 : v[e >> 1] & 0xffffu);
}

__device__ __forceinline__ void clear_bins(uint32_t* bin) {
  for (int i = threadIdx.x; i < 32768 / 4; i += kRowThreads) reinterpret_cast<u32x4*>(bin)[i] = u32x4{0u, 0u, 0u, 0u};
}

// Counts that another kSafeSteps might carry over 16 bits, beside the bins.
__device__ __forceinline__ void flush_full(CountLds& s) {
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < 32768; i += kRowThreads) {
    uint32_t w = s.bin[i];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t c = (w >> (16 * half)) & 0xffffu;
      if (c < kFull) continue;
      const int at = atomicAdd(&s.heavies, 1);
      s.heavy[at] = 2 * i + half;
      s.heavy_count[at] = c;
      w -= c << (16 * half);
    }
    s.bin[i] = w;
  }
  __syncthreads();
}

// a lane's word of a group
__device__ __forceinline__ uint32_t word_of(int g) {
  const int lane = threadIdx.x & 63;
  return g >= kGroups / 2 ? 64 * g + lane : 64 * (kGroups / 2 - 1 - g) + 63 - lane;
}
__device__ __forceinline__ int group_of(uint32_t value) {
  return value & 0x8000u ? (int)(value >> 7) : kGroups / 2 - 1 - (int)(value >> 7);
}

// Which of a wave's 32 groups have values, as bits; f(group, a lane's word) of
// each that has.
template <typename F>
__device__ __forceinline__ uint32_t own_groups(const uint32_t* bin, F f) {
  const int wave = threadIdx.x >> 6;
  uint32_t has = 0;
#pragma unroll 1
  for (int i = 0; i < 32; i += 8) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = bin[word_of(32 * wave + i + j)];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (__ballot(w[j] != 0)) {  // uniform
        has |= 1u << (i + j);
        f(32 * wave + i + j, w[j]);
      }
  }
  return has;
}

// The n-th group that occurs; lanes 0..15 hold the words of bits in `occurs`
// and their running counts in `upto`.
__device__ __forceinline__ int nth_group(int n, uint32_t occurs, uint32_t upto) {
  const int lane = threadIdx.x & 63;
  const int l = __ffsll((long long)__ballot(upto > (uint32_t)n)) - 1;
  const uint32_t word = lane_u32(occurs, l), skip = n - (lane_u32(upto, l) - __popc(word));
  const bool me = lane < 32 && ((word >> lane) & 1) && __popc(word & ((1u << (lane & 31)) - 1)) == skip;
  return 32 * l + __ffsll((long long)__ballot(me)) - 1;
}

__device__ __forceinline__ uint32_t heavy_of(const CountLds& s, int heavies, uint32_t value) {
  uint32_t c = 0;
  for (int i = 0; i < heavies; ++i)
    if (s.heavy[i] == value) c += s.heavy_count[i];
  return c;
}

// The two values of a lane in a group, in order, and their counts; -0 counts as +0.
struct Pair {
  uint32_t v1, v2, c1, c2;
};
__device__ __forceinline__ Pair pair_of(const CountLds& s, int heavies, int g) {
  const bool neg = g >= kGroups / 2;
  const uint32_t w = word_of(g), both = s.bin[w], lo = both & 0xffffu, hi = both >> 16;
  Pair p{2 * w + !neg, 2 * w + neg, neg ? lo : hi, neg ? hi : lo};
  if (heavies) {  // uniform
    p.c1 += heavy_of(s, heavies, p.v1);
    p.c2 += heavy_of(s, heavies, p.v2);
  }
  if (w == 0x4000u) p.c1 = 0;
  if (w == 0) p.c2 += (s.bin[0x4000] & 0xffffu) + heavy_of(s, heavies, 0x8000u);
  return p;
}

// weights of a pair's values against the value `top` (0 where a value does not
// occur), without a branch: the two chains run beside each other
__device__ __forceinline__ void pair_weights(const Pair& p, float top, double inv_t, const double* tab, double& w1, double& w2) {
  const float x1 = bf16_bits_to_f32(p.c1 ? p.v1 : 0xff80u), x2 = bf16_bits_to_f32(p.c2 ? p.v2 : 0xff80u);
  const double e1 = nsv_exp_nonpos(((double)x1 - (double)top) * inv_t, tab);
  const double e2 = nsv_exp_nonpos(((double)x2 - (double)top) * inv_t, tab);
  w1 = x1 == top ? 1.0 : e1;
  w2 = x2 == top ? 1.0 : e2;
}

struct Place {
  uint32_t value;          // bits
  uint32_t before, count;  // tokens
  double mass, weight;     // weights before; of one token
};

// As seek, from the counts of `groups` groups, by one wave.  kAbove: the last
// value of weight >= goal.
__device__ __forceinline__ Place seek_counts(int kind, double goal, const CountLds& s, int groups, int heavies, float top,
                                             double inv_t) {
  const int lane = threadIdx.x & 63;
  int at_group = -1;
#pragma unroll 1
  for (int i = (groups - 1) >> 6; i >= 0 && at_group < 0; --i) {
    const int mine = min(64 * i + lane, groups - 1);
    bool fits;
    if (kind == kByCount) fits = (double)s.cbefore[mine] < goal;
    else if (kind == kAbove) fits = weight_of(bf16_bits_to_f32(s.ref[mine] & 0xffffu), top, inv_t, s.tab) >= goal;
    else fits = s.mass[mine] > 0.0 && (kind == kReach ? s.before[mine] < goal : s.before[mine] <= goal);
    const uint64_t yes = __ballot(fits && s.count[mine] > 0 && 64 * i + lane < groups);  // (a group of -0 alone is empty)
    if (yes) at_group = 64 * i + 63 - __clzll((long long)yes);
  }
  at_group = max(at_group, 0);
  const Pair p = pair_of(s, heavies, (int)(s.ref[at_group] >> 16));
  double w1, w2;
  pair_weights(p, top, inv_t, s.tab, w1, w2);
  const double m1 = p.c1 * w1, m = m1 + p.c2 * w2;
  const double before = lane_before(wave_scan(m)) + s.before[at_group];
  const uint32_t cbefore = s.cbefore[at_group] + wave_scan(p.c1 + p.c2) - p.c1 - p.c2;
  auto fits = [&](uint32_t c, double w, uint32_t cb, double mb) {
    if (kind == kByCount) return c && (double)cb < goal;
    if (kind == kAbove) return c && w >= goal;
    return c && w > 0.0 && (kind == kReach ? mb < goal : mb <= goal);
  };
  const uint64_t y1 = __ballot(fits(p.c1, w1, cbefore, before)), y2 = __ballot(fits(p.c2, w2, cbefore + p.c1, before + m1));
  const int l1 = y1 ? 63 - __clzll((long long)y1) : -1, l2 = y2 ? 63 - __clzll((long long)y2) : -1;
  const bool second = l2 >= l1;
  const int l = max(max(l1, l2), 0);
  Place at;
  at.value = lane_u32(second ? p.v2 : p.v1, l);
  at.count = lane_u32(second ? p.c2 : p.c1, l);
  at.before = lane_u32(second ? cbefore + p.c1 : cbefore, l);
  at.mass = lane_f64(second ? before + m1 : before, l);
  at.weight = lane_f64(second ? w2 : w1, l);
  return at;
}

// how many of a vector's tokens have the value (`both`: twice its bits, under
// `mask`), and whether any has
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t matches(const u32x4& v, uint32_t both, uint32_t mask) {
  u16x2 n = {0, 0};  // others
#pragma unroll
  for (int i = 0; i < 4; ++i)
    n += __builtin_elementwise_min(__builtin_bit_cast(u16x2, (v[i] & mask) ^ both), (u16x2){1, 1});
  return 8u - n[0] - n[1];
}
__device__ __forceinline__ bool has_value(const u32x4& v, uint32_t both, uint32_t mask) {
  u16x2 d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] = __builtin_bit_cast(u16x2, (v[i] & mask) ^ both);
  const u16x2 m = __builtin_elementwise_min(__builtin_elementwise_min(d[0], d[1]), __builtin_elementwise_min(d[2], d[3]));
  return m[0] == 0 || m[1] == 0;
}

// s.index = the index of the token of bits `value` with `rank` of them before
// it among the vectors lo .. hi - 1
__device__ __forceinline__ void find_token(const Row& row, int lo, int hi, uint32_t value, uint32_t rank, CountLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t mask = value ? ~0u : 0x7fff7fffu, both = value | (value << 16);  // (+0: -0 too)
  each_vec(row, lo, hi, [&](int it, const u32x4& v, bool in) {
    uint32_t all = 0;
    if (__ballot(in && has_value(v, both, mask))) {
      const uint32_t n = in ? matches(v, both, mask) : 0u;
#pragma unroll
      for (int b = 0; b < 4; ++b) all += __popcll(__ballot((n >> b) & 1)) << b;
    }
    if (lane == 0) s.found[it * kRowWaves + wave] = all;
  });
  __syncthreads();
  // the (step, wave) that holds it: every wave looks, one goes on
  const int entries = (hi - lo + kRowThreads - 1) / kRowThreads * kRowWaves, per = (entries + 63) / 64;
  uint32_t mine = 0;
#pragma unroll 1
  for (int i = 0; i < per; ++i)
    if (lane * per + i < entries) mine += s.found[lane * per + i];
  const uint32_t upto = wave_scan(mine);
  const uint64_t yes = __ballot(upto > rank);
  const int l = yes ? __ffsll((long long)yes) - 1 : 63;
  uint32_t left = rank - lane_u32(upto - mine, l);
  int at = l * per;
#pragma unroll 1
  while (at < min(entries, (l + 1) * per) - 1 && left >= s.found[at]) left -= s.found[at++];
  at = __builtin_amdgcn_readfirstlane(min(at, entries - 1));
  if (wave == at % kRowWaves) {  // uniform
    const int g = lo + at / kRowWaves * kRowThreads + tid;
    u32x4 v{};
    if (g < hi) v = row.load(g);
    const uint32_t n = g < hi ? matches(v, both, mask) : 0u;
    const uint32_t before = wave_scan(n) - n;
    if (n && left >= before && left < before + n) {
      uint32_t k = before;
      int e = 0;
      for (; e < 7; ++e) {
        const bool hit = ((v[0] ^ both) & mask & 0xffffu) == 0;
        if (hit && k == left) break;
        k += hit;
        if (e & 1) v = u32x4{v[1], v[2], v[3], v[0]};
        else v[0] >>= 16;
      }
      s.index = 8 * g - row.skew + e;
    }
  }
  __syncthreads();
}

struct Settings {
  float T, p, least, u;
  int k;
  bool sampled, ends;
  double inv_t;
};
// (as vector loads: scalar ones would be waited for with the LDS writes)
__device__ __forceinline__ Settings settings_of(const FilterArgs& a, int b, bool sampled, int64_t at_u, bool ends) {
  int vb = b;
  int64_t vu = at_u;
  asm volatile("" : "+v"(vb), "+v"(vu));
  Settings f;
  f.T = a.temperature[vb];
  f.k = a.top_k ? a.top_k[vb] : 0;
  f.p = a.top_p ? a.top_p[vb] : 1.f;
  f.least = a.min_p ? a.min_p[vb] : 0.f;
  f.u = a.uniforms[vu];
  f.sampled = sampled;
  f.ends = ends;
  return f;
}

// Counts and weights of the groups that occur, the waves in turn; their number.
__device__ __forceinline__ int weigh_groups(double inv_t, int heavies, CountLds& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t occurs = lane < kGroups / 32 ? s.occurs[lane] : 0u;
  // (-0 counts with +0, the last value of the positive ones)
  if (lane == kGroups / 64 - 1 && (s.occurs[kGroups / 64] & 1)) occurs |= 1u << 31;
  const uint32_t upto = wave_scan((uint32_t)__popc(occurs));
  const int groups = (int)lane_u32(upto, 63);
  uint32_t slots = 0;
#pragma unroll 1
  for (int n = wave; n < groups; n += kRowWaves) {
    const int g = nth_group(n, occurs, upto);
    const Pair q = pair_of(s, heavies, g);
    if ((q.c1 && (q.v1 & 0x7fffu) > 0x7f80u) || (q.c2 && (q.v2 & 0x7fffu) > 0x7f80u)) s.nan = 1;
    const uint64_t y1 = __ballot(q.c1 > 0), y2 = __ballot(q.c2 > 0);
    const int l1 = y1 ? __ffsll((long long)y1) - 1 : 64, l2 = y2 ? __ffsll((long long)y2) - 1 : 64;
    const uint32_t ref = lane_u32(l1 <= l2 ? q.v1 : q.v2, min(min(l1, l2), 63));
    double w1, w2;
    pair_weights(q, bf16_bits_to_f32(ref), inv_t, s.tab, w1, w2);
    const double m = wave_sum_dpp(q.c1 * w1 + q.c2 * w2);
    const uint32_t all = lane_u32(wave_scan(q.c1 + q.c2), 63);
    slots += all;
    if (lane == 0) {
      s.count[n] = all;
      s.mass[n] = m;
      s.ref[n] = ((uint32_t)g << 16) | ref;
    }
  }
  if (lane == 0) atomicAdd(&s.slots, slots);
  return groups;
}

// What the filters leave, from the weighed groups, by one wave: into s.
__device__ __forceinline__ void decide(const Settings& f, int V, int groups, int heavies, CountLds& s) {
  const int lane = threadIdx.x & 63;
  const uint32_t top_bits = s.ref[0] & 0xffffu;  // the maximum: the first value
  const float top = bf16_bits_to_f32(top_bits);
  uint32_t cut = top_bits, value = top_bits;
  int kept = 1, rank = 0, cut_rank = -1;
  double total = 1.0;
  if (!is_greedy(f.T) && top != -__builtin_inff()) {  // uniform
    // weights and tokens before each group
    total = 0.0;
    uint32_t n = 0;
#pragma unroll 1
    for (int i = 0; i < groups; i += 64) {
      const int g = min(i + lane, groups - 1);
      const bool in = i + lane < groups;
      const double m = in ? s.mass[g] * weight_of(bf16_bits_to_f32(s.ref[g] & 0xffffu), top, f.inv_t, s.tab) : 0.0;
      const uint32_t c = in ? s.count[g] : 0u;
      const double fu = wave_scan(m);
      const uint32_t nu = wave_scan(c);
      if (in) {
        s.mass[g] = m;
        s.before[g] = total + lane_before(fu);
        s.cbefore[g] = n + nu - c;
      }
      total += lane_f64(fu, 63);
      n += lane_u32(nu, 63);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup", "local");  // (this wave's own)
    kept = V;
    cut = 0xff80u;
#pragma unroll 1
    for (int kind = 0; kind < 4; ++kind) {
      double goal = 0.0;
      if (kind == kByCount) {
        if (f.k <= 0 || f.k >= V) continue;
        goal = (double)f.k;
      } else if (kind == kReach) {
        if (!(f.p < 1.f)) continue;
        goal = fmax((double)f.p * total, 0x1p-1000);  // (the first token stays)
      } else if (kind == kAbove) {
        if (!(f.least > 0.f)) continue;
        goal = fmin((double)f.least, 1.0);
      } else {
        if (!f.sampled || kept == 1) continue;
        goal = unit(f.u) * total;
      }
      const Place at = seek_counts(kind, goal, s, groups, heavies, top, f.inv_t);
      if (kind == kBeyond) {
        const double j = fmin(floor((goal - at.mass) / at.weight), (double)min((int)at.count, kept - (int)at.before) - 1.0);
        value = at.value;
        rank = (int)fmax(j, 0.0);
        continue;
      }
      uint32_t stay = at.count;  // tokens of the value that do
      if (kind == kByCount) stay = (uint32_t)f.k - at.before;
      if (kind == kReach) stay = (uint32_t)fmin(fmax(ceil((goal - at.mass) / at.weight), 1.0), (double)at.count);
      if ((int)(at.before + stay) >= kept) continue;
      kept = (int)(at.before + stay);
      cut = at.value;
      cut_rank = stay < at.count ? (int)stay - 1 : -1;
      total = at.mass + stay * at.weight;
    }
    if (!f.sampled && kept > 1) rank = -1;
    // (a cut among tokens of weight 0 cuts nothing; a lone token is looked up as the sample)
    if (!f.ends || kept == 1 || cut == 0xff80u) cut_rank = -1;
  }
  if (lane == 0) {
    s.top = top;
    s.cut = bf16_bits_to_f32(cut);
    s.cut_value = cut;
    s.kept = kept;
    s.total = total;
    s.value = value;
    s.rank = rank;
    s.cut_rank = cut_rank;
  }
}

// The first NaN of a row that has one.
__device__ __forceinline__ RowCut nan_row(const Row& row, CountLds& s) {
  if (threadIdx.x == 0) s.index = row.V;
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < row.V; i += kRowThreads)
    if ((row.at[i] & 0x7fffu) > 0x7f80u) atomicMin(&s.index, i);
  __syncthreads();
  return RowCut{__builtin_nanf(""), __builtin_nanf(""), s.index, 1, s.index, 0, 1.0};
}

// find(value, rank) -> s.index, for what decide() wants looked up
template <typename F>
__device__ __forceinline__ RowCut look_up(int V, const CountLds& s, F find) {
  RowCut out{s.top, s.cut, V - 1, s.kept, 0, 0, s.total};
  const int rank = s.rank, cut_rank = s.cut_rank;
  const uint32_t value = s.value, cut_value = s.cut_value;
  if (out.top == -__builtin_inff()) {  // uniform: nothing above it, the first token
    out.last = 0;
    return out;
  }
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const int r = which ? cut_rank : rank;
    if (r < 0) continue;  // uniform
    find(which ? cut_value : value, (uint32_t)r);
    if (which) out.last = s.index;
    else out.token = s.index;
  }
  if (out.kept == 1) out.last = out.token;
  return out;
}

// filter_row for bf16, by one workgroup.
__device__ __forceinline__ RowCut count_row(const Row& row, Settings f, CountLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  clear_bins(s.bin);
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) {
    s.nan = s.heavies = 0;
    s.slots = 0;
  }
  lds_barrier();
  f.inv_t = is_greedy(f.T) ? 1.0 : 1.0 / (double)f.T;
  // A bin runs over only where one value has more than 65,535 tokens: the
  // counts then miss some, and are taken again with the full ones put aside
  // in between.
  int groups = 0, heavies = 0;
#pragma unroll 1
  for (int careful = 0; careful < 2; ++careful) {
    uint32_t heavy = ~0u, many = 0;
    const int whole = (row.vecs + kRowThreads - 1) / kRowThreads * kRowThreads;
    const int run = careful ? kSafeSteps * kRowThreads : whole;
#pragma unroll 1
    for (int lo = 0; lo < row.vecs; lo += run) {
      each_vec(row, lo, min(lo + run, row.vecs), [&](int, const u32x4& v, bool in) {
        if (in) count_vec(s.bin, v, heavy, many);
      });
      if (careful) flush_full(s);
    }
    // (a wave's lanes count alike, but those without a last vector)
    heavy = (uint32_t)__builtin_amdgcn_readfirstlane((int)heavy);
    many = (uint32_t)__builtin_amdgcn_readfirstlane((int)many);
    if (lane == 0 && many) {
      const int at = atomicAdd(&s.heavies, 1);
      s.heavy[at] = heavy;
      s.heavy_count[at] = many;
    }
    __syncthreads();
    heavies = s.heavies;
    uint32_t has = own_groups(s.bin, [](int, uint32_t) {});
    for (int i = 0; i < heavies; ++i) {
      const int g = group_of(s.heavy[i]);
      if (g >> 5 == wave) has |= 1u << (g & 31);
    }
    if (lane == 0) s.occurs[wave] = has;
    __syncthreads();
    groups = weigh_groups(f.inv_t, heavies, s);
    __syncthreads();
    if (s.slots == 8u * (uint32_t)row.vecs) break;  // uniform
    __syncthreads();
    clear_bins(s.bin);
    if (tid == 0) {
      s.heavies = 0;
      s.slots = 0;
    }
    __syncthreads();
  }
  if (s.nan) return nan_row(row, s);  // uniform
  if (wave == 0) decide(f, row.V, groups, heavies, s);
  __syncthreads();
  return look_up(row.V, s, [&](uint32_t value, uint32_t rank) { find_token(row, 0, row.vecs, value, rank, s); });
}

// A row in parts, each counted by a workgroup of its own (at most kSafeSteps
// steps, so that 16 bits hold every count): which groups occur, and the words
// of those that do.
struct Part {
  uint32_t occurs[kGroups / 32];
  uint32_t word[kGroups * 64];
};

__device__ __forceinline__ int part_vecs(const Row& row, int parts) { return (row.vecs + parts - 1) / parts; }

__device__ __forceinline__ void count_part(const Row& row, int part, int parts, uint32_t* bin, Part* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int per = part_vecs(row, parts), lo = part * per, hi = min(lo + per, row.vecs);
  clear_bins(bin);
  lds_barrier();
  uint32_t heavy = ~0u, many = 0;
  if (lo < hi)
    each_vec(row, lo, hi, [&](int, const u32x4& v, bool in) {
      if (in) count_vec(bin, v, heavy, many);
    });
  heavy = (uint32_t)__builtin_amdgcn_readfirstlane((int)heavy);
  many = (uint32_t)__builtin_amdgcn_readfirstlane((int)many);
  if (lane == 0 && many) atomicAdd(&bin[heavy >> 1], many << ((heavy & 1) << 4));
  __syncthreads();
  const uint32_t has = own_groups(bin, [&](int g, uint32_t w) { out->word[64 * g + lane] = w; });
  if (lane == 0) out->occurs[wave] = has;
}

// filter_row for bf16, from the counts of a row's parts.
__device__ __forceinline__ RowCut merge_row(const Row& row, Settings f, const Part* in, int parts, CountLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid < kGroups / 32 * parts) s.part_occurs[tid] = in[tid / (kGroups / 32)].occurs[tid % (kGroups / 32)];
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) {
    s.nan = s.heavies = 0;
    s.slots = 0;
    s.bin[0x4000] = 0;  // (read with the word of +0, whether its own group occurs or not)
  }
  __syncthreads();
  uint32_t occurs = 0;
  if (lane < kGroups / 32) {
#pragma unroll 8
    for (int c = 0; c < parts; ++c) occurs |= s.part_occurs[c * (kGroups / 32) + lane];
  }
  if (wave == 0 && lane < kGroups / 32) s.occurs[lane] = occurs;
  if (lane == kGroups / 64 - 1 && (lane_u32(occurs, kGroups / 64) & 1)) occurs |= 1u << 31;  // (+0's group where there is -0)
  const uint32_t upto = wave_scan((uint32_t)__popc(occurs));
  const int groups = (int)lane_u32(upto, 63);
#pragma unroll 1
  for (int n = wave; n < groups; n += kRowWaves) {
    const int g = nth_group(n, occurs, upto);
    // parts that have it (the word of one that has not is whatever the memory held)
    const uint64_t have = __ballot(lane < parts && ((s.part_occurs[min(lane, parts - 1) * (kGroups / 32) + (g >> 5)] >> (g & 31)) & 1));
    uint32_t lo = 0, hi = 0;
#pragma unroll 1
    for (int c0 = 0; c0 < parts; c0 += 8) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = in[min(c0 + j, parts - 1)].word[64 * g + lane];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool has = (have >> (c0 + j)) & 1;
        lo += has ? w[j] & 0xffffu : 0u;
        hi += has ? w[j] >> 16 : 0u;
      }
    }
    const int64_t word = g >= kGroups / 2 ? 64 * g + lane : 64 * (kGroups / 2 - 1 - g) + 63 - lane;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t& c = half ? hi : lo;
      if (c < 65536) continue;  // (rows of one value mostly)
      const int at = atomicAdd(&s.heavies, 1);
      s.heavy[at] = 2 * (uint32_t)word + half;
      s.heavy_count[at] = c;
      c = 0;
    }
    s.bin[word] = lo | (hi << 16);
  }
  f.inv_t = is_greedy(f.T) ? 1.0 : 1.0 / (double)f.T;
  __syncthreads();
  const int heavies = s.heavies;
  weigh_groups(f.inv_t, heavies, s);
  __syncthreads();
  if (s.nan) return nan_row(row, s);  // uniform
  if (wave == 0) decide(f, row.V, groups, heavies, s);
  __syncthreads();
  return look_up(row.V, s, [&](uint32_t value, uint32_t rank) {
    // the part that holds the token, by its counts of the value
    uint32_t c = 0;
    auto count = [&](uint32_t v) {
      const int g = group_of(v);
      if (lane >= parts || !((s.part_occurs[lane * (kGroups / 32) + (g >> 5)] >> (g & 31)) & 1)) return;
      const uint32_t w = v >> 1, at = g >= kGroups / 2 ? w & 63 : 63 - (w & 63);
      const uint32_t both = in[lane].word[64 * g + at];
      c += (v & 1) ? both >> 16 : both & 0xffffu;
    };
    count(value);
    if (value == 0) count(0x8000u);
    const uint32_t upto_c = wave_scan(c);
    const int part = max(__ffsll((long long)__ballot(upto_c > rank)) - 1, 0);
    const int per = part_vecs(row, parts), lo = part * per;
    find_token(row, lo, min(lo + per, row.vecs), value, rank - lane_u32(upto_c - c, part), s);
  });
}

// probability of token i of logit x
__device__ __forceinline__ double prob_of(const RowCut& c, float x, int i, double inv_t, const double* tab) {
  if (c.kept == 1) return i == c.token ? 1.0 : 0.0;
  const bool in = x > c.cut || (x == c.cut && i <= c.last);
  return in ? weight_of(x, c.top, inv_t, tab) / c.total : 0.0;
}

// The row of workgroup (r, b): where it lies, and what is wanted of it.
struct Job {
  int64_t at;       // elements, from `target` or `draft`
  int64_t u;        // its number among the uniforms
  bool active, is_draft, sampled, ends;
  int draft;        // the draft that its probability is wanted of; -1: none
};
__device__ __forceinline__ Job job_of(const FilterArgs& a, int r, int b) {
  if (a.K < 0) return Job{(int64_t)b * a.t_seq, b, true, false, true, false, -1};
  const int kb = draft_count(a, b);
  const bool rows = by_rows(a, b), is_draft = r > a.K;
  const int i = is_draft ? r - a.K - 1 : r;
  Job j;
  j.at = is_draft ? draft_at(a, b, i) : (int64_t)b * a.t_seq + (int64_t)i * a.t_row;
  j.u = (int64_t)b * (a.K + 1) + (rows ? a.K : i);
  j.active = is_draft ? rows && i < kb : i <= kb;
  j.is_draft = is_draft;
  j.sampled = !rows || i == kb;
  j.ends = !j.sampled;
  j.draft = rows && i < kb ? i : -1;
  return j;
}

template <typename T>
__device__ __forceinline__ void put_row(const FilterArgs& a, int r, int b, const Job& j, const T* row, const RowCut& c) {
  if (threadIdx.x != 0) return;
  if (a.K < 0) {
    a.tokens[(int64_t)b * a.out_stride] = c.token;
    if (a.kept) a.kept[b] = c.kept;
    return;
  }
  const int64_t at = (int64_t)b * (2 * a.K + 1) + r;
  a.cuts[at] = c;
  if (j.draft >= 0) {
    const int32_t d = a.drafts[(int64_t)b * a.K + j.draft];
    const bool in = d >= 0 && d < a.V;  // a token outside the vocabulary has probability 0
    const double inv_t = 1.0 / (double)a.temperature[b];
    a.probs[at] = in ? prob_of(c, Elem<T>::get(row[d]), d, inv_t, kExp2Frac256) : 0.0;
  }
}

// grid (rows per sequence, B): target rows, then draft rows
__global__ __launch_bounds__(kRowThreads) void filter_rows_f32_kernel(FilterArgs a) {
  __shared__ RowLds s;
  const int r = blockIdx.x, b = blockIdx.y;
  const Job j = job_of(a, r, b);
  if (!j.active) return;  // uniform
  const float* row = (const float*)(j.is_draft ? a.draft : a.target) + j.at;
  put_row(a, r, b, j, row, filter_row<float>(a, b, row, j.sampled, a.uniforms[j.u], j.ends, s));
}

__global__ __launch_bounds__(kRowThreads) void filter_rows_bf16_kernel(FilterArgs a) {
  __shared__ CountLds s;
  const int r = blockIdx.x, b = blockIdx.y;
  const Job j = job_of(a, r, b);
  if (!j.active) return;  // uniform
  const uint16_t* row = (const uint16_t*)(j.is_draft ? a.draft : a.target) + j.at;
  put_row(a, r, b, j, row, count_row(Row(row, a.V), settings_of(a, b, j.sampled, j.u, j.ends), s));
}

// grid (parts, rows per sequence, B)
__global__ __launch_bounds__(kRowThreads) void filter_parts_kernel(FilterArgs a) {
  __shared__ uint32_t bin[32768];
  const int r = blockIdx.y, b = blockIdx.z;
  const Job j = job_of(a, r, b);
  if (!j.active) return;  // uniform
  const uint16_t* row = (const uint16_t*)(j.is_draft ? a.draft : a.target) + j.at;
  count_part(Row(row, a.V), blockIdx.x, gridDim.x, bin, a.row_parts + ((int64_t)b * gridDim.y + r) * gridDim.x + blockIdx.x);
}
// grid (rows per sequence, B)
__global__ __launch_bounds__(kRowThreads) void filter_merge_kernel(FilterArgs a) {
  __shared__ CountLds s;
  const int r = blockIdx.x, b = blockIdx.y;
  const Job j = job_of(a, r, b);
  if (!j.active) return;  // uniform
  const uint16_t* row = (const uint16_t*)(j.is_draft ? a.draft : a.target) + j.at;
  const Part* in = a.row_parts + ((int64_t)b * gridDim.x + r) * a.split;
  put_row(a, r, b, j, row, merge_row(Row(row, a.V), settings_of(a, b, j.sampled, j.u, j.ends), in, a.split, s));
}

// drafts accepted before the first refused (a whole wave)
__device__ __forceinline__ int accepted_by_rows(const FilterArgs& a, int b, int kb) {
  const int i = threadIdx.x & 63;
  bool refused = false;
  if (i < kb) {
    const double pt = a.probs[(int64_t)b * (2 * a.K + 1) + i], pd = a.probs[(int64_t)b * (2 * a.K + 1) + a.K + 1 + i];
    refused = !((double)a.uniforms[(int64_t)b * (a.K + 1) + i] * pd < pt);
  }
  const uint64_t no = __ballot(refused);
  return no ? __ffsll((long long)no) - 1 : kb;
}

// a thread's residuals max(p_target - p_draft, 0) and p_target of a chunk
template <typename T>
__device__ __forceinline__ void residuals(const FilterArgs& a, int b, int r, int ch, const double* tab, double (&left)[kVec],
                                          double (&pt)[kVec]) {
  const T* t = (const T*)a.target + (int64_t)b * a.t_seq + (int64_t)r * a.t_row;
  const T* d = (const T*)a.draft + draft_at(a, b, r);
  const RowCut ct = a.cuts[(int64_t)b * (2 * a.K + 1) + r], cd = a.cuts[(int64_t)b * (2 * a.K + 1) + a.K + 1 + r];
  const double inv_t = 1.0 / (double)a.temperature[b];
  const int64_t base = (int64_t)ch * kChunk + kVec * threadIdx.x;
  float xt[kVec], xd[kVec];
  if (base < a.V) {
    load_vec<T>(t, base, a.V, xt);
    load_vec<T>(d, base, a.V, xd);
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    left[e] = pt[e] = 0.0;
    if (base + e >= a.V) continue;
    pt[e] = prob_of(ct, xt[e], (int)(base + e), inv_t, tab);
    if (pt[e] > 0.0) left[e] = fmax(pt[e] - prob_of(cd, xd[e], (int)(base + e), inv_t, tab), 0.0);
  }
}

// grid (chunks, B): chunk sums of the refused row's residuals
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void filter_residual_kernel(FilterArgs a) {
  __shared__ double tab[256], red[2 * kChunkThreads / 64];
  const int b = blockIdx.y, ch = blockIdx.x;
  if (!by_rows(a, b)) return;  // uniform
  const int kb = draft_count(a, b), n = accepted_by_rows(a, b, kb);
  if (n == kb) return;  // uniform: every draft stays
  tab[threadIdx.x] = kExp2Frac256[threadIdx.x];
  __syncthreads();
  double left[kVec], pt[kVec], sl = 0.0, sp = 0.0;
  residuals<T>(a, b, n, ch, tab, left, pt);
  for (int e = 0; e < kVec; ++e) {
    sl += left[e];
    sp += pt[e];
  }
  sl = wave_sum_dpp(sl);
  sp = wave_sum_dpp(sp);
  if ((threadIdx.x & 63) == 0) {
    red[2 * (threadIdx.x >> 6)] = sl;
    red[2 * (threadIdx.x >> 6) + 1] = sp;
  }
  __syncthreads();
  if (threadIdx.x < 2) {
    double r = 0.0;
    for (int w = 0; w < kChunkThreads / 64; ++w) r += red[2 * w + threadIdx.x];
    a.parts[((int64_t)b * a.chunks + ch) * 2 + threadIdx.x] = r;
  }
}

// grid B: the sequence's tokens
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void filter_finish_kernel(FilterArgs a) {
  __shared__ double tab[256], red[kChunkThreads / 64], goal_s, before_s;
  __shared__ int which, use_pt, token;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int K = a.K, kb = draft_count(a, b);
  const RowCut* cuts = a.cuts + (int64_t)b * (2 * K + 1);
  int32_t* out = a.out_tokens + (int64_t)b * (K + 1);
  const int32_t d = lane < kb ? a.drafts[(int64_t)b * K + lane] : -1;
  if (!by_rows(a, b)) {  // uniform: every row was sampled
    if (wave) return;
    const int32_t t = lane <= kb ? cuts[lane].token : 0;
    const uint64_t no = __ballot(lane < kb && t != d);
    const int n = no ? __ffsll((long long)no) - 1 : kb;
    if (lane <= n) out[lane] = t;
    if (lane == 0) a.out_len[b] = n + 1;
    return;
  }
  const int n = accepted_by_rows(a, b, kb);
  if (wave == 0 && lane < n) out[lane] = d;
  if (tid == 0) a.out_len[b] = n + 1;
  if (n == kb) {  // uniform: the bonus token
    if (tid == 0) out[n] = cuts[n].token;
    return;
  }
  tab[tid] = kExp2Frac256[tid];
  // the chunk that holds the token: the last with any weight whose sums before it do not exceed the goal
  const double* parts = a.parts + (int64_t)b * a.chunks * 2;
  if (wave == 0) {
    double sl = 0.0;
    for (int c = lane; c < a.chunks; c += 64) sl += parts[2 * c];
    const int col = wave_sum_dpp(sl) > 0.0 ? 0 : 1;  // no residual: the target row itself
    double total = 0.0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
      const double v = wave_scan(c0 + lane < a.chunks ? parts[2 * (c0 + lane) + col] : 0.0);
      total += __shfl(v, 63);
    }
    const double goal = unit(a.uniforms[(int64_t)b * (K + 1) + K]) * total;
    double run = 0.0, before = 0.0;
    int at = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
      const double mine = c0 + lane < a.chunks ? parts[2 * (c0 + lane) + col] : 0.0;
      const double v = wave_scan(mine);
      double prev = __shfl_up(v, 1);
      if (lane == 0) prev = 0.0;
      const uint64_t yes = __ballot(mine > 0.0 && run + prev <= goal);
      if (yes) {
        const int l = 63 - __clzll((long long)yes);
        at = c0 + l;
        before = run + __shfl(prev, l);
      }
      run += __shfl(v, 63);
    }
    if (lane == 0) {
      which = at;
      use_pt = col;
      goal_s = goal;
      before_s = before;
      token = -1;
    }
  }
  __syncthreads();
  double left[kVec], pt[kVec];
  residuals<T>(a, b, n, which, tab, left, pt);
  double mine = 0.0;
  for (int e = 0; e < kVec; ++e) {
    if (use_pt) left[e] = pt[e];
    mine += left[e];
  }
  const double v = wave_scan(mine);
  double run = __shfl_up(v, 1);
  if (lane == 0) run = 0.0;
  if (lane == 63) red[wave] = v;
  __syncthreads();
  double before = before_s;
  for (int w = 0; w < wave; ++w) before += red[w];
  run += before;
  // the last element with any weight whose sums before it do not exceed the goal
  int best = -1;
  for (int e = 0; e < kVec; ++e) {
    if (left[e] > 0.0 && run <= goal_s) best = which * kChunk + kVec * tid + e;
    run += left[e];
  }
  if (best >= 0) atomicMax(&token, best);
  __syncthreads();
  if (tid == 0) out[n] = token;
}

bool bad_rows(int B, int V, int dtype) { return B < 0 || V <= 0 || (dtype != NSV_F32 && dtype != NSV_BF16); }

// weights as integers: V of them, each at most 2^shift, stay below 2^62
int weight_shift(int V) {
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  const int s = 62 - bits;
  return s > 50 ? 50 : s;
}

size_t a256(size_t x) { return (x + 255) & ~(size_t)255; }
int residual_chunks(int V) { return (V + kChunk - 1) / kChunk; }

// Workgroups that count a bf16 row, each a part of it; 1: one workgroup does
// the whole row.  Up to 256 workgroups share few rows (one row of 151,936
// TIME1), as long as the parts' counts stay under 64 MiB.
int row_split(int rows, int V, int dtype) {
  if (dtype != NSV_BF16 || rows <= 0) return 1;
  const int least = (V + 7 + kSafeSteps * kStep - 1) / (kSafeSteps * kStep);
  int n = kMaxSplit;
  while (n > 1 && (rows * n > 256 || V < n * kStep)) n >>= 1;
  if (n < least) n = least;
  return n > 1 && rows * n <= 512 && n <= kMaxParts ? n : 1;
}
size_t parts_bytes(int rows, int V, int dtype) {
  const int n = row_split(rows, V, dtype);
  return n > 1 ? (size_t)rows * n * sizeof(Part) : 0;
}

struct Layout {
  size_t cuts, probs, parts, row_parts, total;
};
Layout layout(int B, int K, int V, int dtype, bool draft_rows) {
  Layout L;
  const size_t rows = (size_t)B * (2 * (size_t)K + 1);
  L.cuts = 0;
  L.probs = a256(rows * sizeof(RowCut));
  L.parts = L.probs + a256(rows * sizeof(double));
  L.row_parts = L.parts + a256((size_t)B * residual_chunks(V) * 2 * sizeof(double));
  L.total = L.row_parts + parts_bytes(B * (draft_rows ? 2 * K + 1 : K + 1), V, dtype);
  return L;
}

int launch_rows(FilterArgs& a, int rows, int dtype, char* row_parts, hipStream_t s) {
  a.split = row_split(rows * a.B, a.V, dtype);
  a.row_parts = (Part*)row_parts;
  const dim3 grid(rows, a.B), block(kRowThreads);
  if (dtype == NSV_F32) {
    hipLaunchKernelGGL(filter_rows_f32_kernel, grid, block, 0, s, a);
  } else if (a.split == 1) {
    hipLaunchKernelGGL(filter_rows_bf16_kernel, grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL(filter_parts_kernel, dim3(a.split, rows, a.B), block, 0, s, a);
    const int rc = nsv_launch_status();
    if (rc) return rc;
    hipLaunchKernelGGL(filter_merge_kernel, grid, block, 0, s, a);
  }
  return nsv_launch_status();
}

}  // namespace

extern "C" {

size_t nsv_sample_filtered_workspace_size(int B, int V, int dtype) {
  if (bad_rows(B, V, dtype) || V > kMaxVocab || B > 65535) return 0;
  return parts_bytes(B, V, dtype);
}

int nsv_sample_filtered(const void* logits, int64_t row_stride, const float* temperature, const int32_t* top_k,
                        const float* top_p, const float* min_p, const float* uniforms, int B, int V, int dtype,
                        int32_t* out_tokens, int64_t out_stride, int32_t* kept, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (bad_rows(B, V, dtype) || row_stride < V || out_stride < 1) return NSV_ERR_ARG;
  if (V > kMaxVocab || B > 65535) return NSV_ERR_UNSUPPORTED;
  if (B == 0) return NSV_OK;
  if (!logits || !temperature || !uniforms || !out_tokens) return NSV_ERR_ARG;
  const size_t need = parts_bytes(B, V, dtype);
  if (need && (!workspace || workspace_bytes < need)) return NSV_ERR_WORKSPACE;
  FilterArgs a{};
  a.target = logits;
  a.t_seq = row_stride;
  a.B = B;
  a.K = -1;
  a.V = V;
  a.shift = weight_shift(V);
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniforms = uniforms;
  a.tokens = out_tokens;
  a.out_stride = out_stride;
  a.kept = kept;
  return launch_rows(a, 1, dtype, (char*)workspace, (hipStream_t)stream);
}

size_t nsv_accept_filtered_workspace_size(int B, int K, int V, int dtype) {
  if (bad_rows(B, V, dtype) || K < 0 || K > kMaxDrafts || V > kMaxVocab || B > 65535) return 0;
  const size_t x = layout(B, K, V, dtype, false).total, y = layout(B, K, V, dtype, true).total;
  return x > y ? x : y;  // (with draft rows or without)
}

int nsv_accept_filtered(const void* target_logits, int64_t target_seq_stride, const void* draft_logits,
                        int64_t draft_seq_stride, int64_t draft_row_stride, const int32_t* draft_mode,
                        const int32_t* drafts, const int32_t* num_drafts, const float* temperature, const int32_t* top_k,
                        const float* top_p, const float* min_p, const float* uniforms, int B, int K, int V, int dtype,
                        int32_t* out_tokens, int32_t* out_len, void* workspace, size_t workspace_bytes, void* stream) {
  if (bad_rows(B, V, dtype) || K < 0 || K > kMaxDrafts || target_seq_stride < K + 1) return NSV_ERR_ARG;
  if (draft_logits && (draft_row_stride < 1 || draft_seq_stride < 0)) return NSV_ERR_ARG;
  if (draft_mode && !draft_logits) return NSV_ERR_ARG;
  if (V > kMaxVocab || B > 65535) return NSV_ERR_UNSUPPORTED;
  if (B == 0) return NSV_OK;
  if (!target_logits || (!drafts && K > 0) || !num_drafts || !temperature || !uniforms || !out_tokens || !out_len)
    return NSV_ERR_ARG;
  const Layout L = layout(B, K, V, dtype, K > 0 && draft_logits);
  if (!workspace || workspace_bytes < nsv_accept_filtered_workspace_size(B, K, V, dtype)) return NSV_ERR_WORKSPACE;
  FilterArgs a{};
  a.target = target_logits;
  a.t_seq = target_seq_stride * V;
  a.t_row = V;
  a.draft = K > 0 ? draft_logits : nullptr;
  a.d_seq = draft_seq_stride;
  a.d_row = draft_row_stride;
  a.B = B;
  a.K = K;
  a.V = V;
  a.shift = weight_shift(V);
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.uniforms = uniforms;
  a.drafts = drafts;
  a.num_drafts = num_drafts;
  a.mode = draft_mode;
  a.cuts = (RowCut*)((char*)workspace + L.cuts);
  a.probs = (double*)((char*)workspace + L.probs);
  a.parts = (double*)((char*)workspace + L.parts);
  a.chunks = residual_chunks(V);
  a.out_tokens = out_tokens;
  a.out_len = out_len;
  hipStream_t s = (hipStream_t)stream;
  int rc = launch_rows(a, a.draft ? 2 * K + 1 : K + 1, dtype, (char*)workspace + L.row_parts, s);
  if (rc) return rc;
  if (a.draft) {
    const dim3 grid(a.chunks, B);
    if (dtype == NSV_BF16) hipLaunchKernelGGL(filter_residual_kernel<uint16_t>, grid, dim3(kChunkThreads), 0, s, a);
    else hipLaunchKernelGGL(filter_residual_kernel<float>, grid, dim3(kChunkThreads), 0, s, a);
    if ((rc = nsv_launch_status())) return rc;
  }
  if (dtype == NSV_BF16) hipLaunchKernelGGL(filter_finish_kernel<uint16_t>, dim3(B), dim3(kChunkThreads), 0, s, a);
  else hipLaunchKernelGGL(filter_finish_kernel<float>, dim3(B), dim3(kChunkThreads), 0, s, a);
  return nsv_launch_status();
}

}  // extern "C"
