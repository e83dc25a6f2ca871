// Rows under a temperature, top-k, top-p and min-p (filter.h): what the filters
// leave of each, and its sample, for gfx950.
//
// Two kernels.  The first cuts a row into parts, a workgroup each, and leaves
// what a part holds of each value, or of each narrow range of values; the
// second, a workgroup per row, adds the parts up, finds the cuts and the
// sample's value along the order, and the sample's index in the row.
//   bf16: a row has few distinct values, so the first kernel counts the tokens
//     of each of the 65,536 in LDS (16 bits each), and everything else comes
//     from the counts: a value's tokens weigh count * w, one exponential per
//     value that occurs (some 3,000) instead of one per token.  The sampled
//     token is found by its value and its rank among the tokens of that value,
//     in the part that holds it.
//   fp32: 8,192 bins of equal leading bits, counts and weights.  Weights are
//     added up as 64-bit integers, w 2^s rounded, so sums do not depend on the
//     order of the additions; s leaves room for the vocabulary (44 bits for
//     2^18 tokens, 42 for 2^20), each weight off by 2^-(s+1) of its bin's largest
//     at most and a sum of V by V 2^-(s+1), 2^-27.8 at 151,936 tokens, where fp32
//     sums would move the sample of one row in a hundred.  The second kernel
//     lists the tokens of the few bins that matter and looks at those.  A row
//     with a NaN or more than 4,096 tokens to list goes by radix descent over its
//     order-preserving bits, three passes over the row per cut by one workgroup.
//     Many equal values do that, and so do rows of ordinary spread that are long
//     or lie away from 0, since a bin is as wide as its values are large (1/8 at
//     2, 1/2 at 10, 4 at 100).  One row of N(m, 2.2) under top-p 0.9, for m of 0,
//     5 and 100: 37, 39 and 278 us of 50,001 tokens, 63, 359 and 756 of 151,936,
//     91, 610 and 1,273 of 262,144; without a filter 34, 34 and 441 of 151,936.

#include "filter.h"

#include <type_traits>

using namespace nsv_filter;

namespace {

constexpr int kBins = 2048;
constexpr int kMaxSteps = kMaxVocab / kStep + 1; // (a row that starts off a 16-byte boundary)

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

// ---------------------------------------------------------------------------
// radix descent
// ---------------------------------------------------------------------------
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
  int only;                // seek_list's, of one token: its place in the list
};
enum { kByCount, kReach, kAbove, kBeyond };

// The last value with: tokens before it < goal (kByCount); weights before it
// < goal (kReach) or <= goal (kBeyond), and a weight of its own; kBeyond: with
// fewer than `limit` tokens before it too (what lies behind the kept ones has
// all their weights before it, which a goal of u = 1 does not exclude).
template <typename T>
__device__ __forceinline__ Spot seek(int kind, double goal, uint32_t limit, const T* row, int V, float top, double inv_t,
                                     double scale, RowLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Spot at{0u, 0u, 0u, 0ull, 0ull, 0};
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
      return w > 0 && (kind == kReach ? (double)mass < goal : (double)mass <= goal && before < limit);
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
__device__ __forceinline__ int index_of(float value, uint32_t j, const T* row, int V, RowLds& s) {
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

// ---------------------------------------------------------------------------
// rows in parts
// ---------------------------------------------------------------------------
constexpr int kFewParts = 8;   // workgroups that a row is cut over, at most ..
constexpr int kMaxParts = 32;  // .. and parts
constexpr int kSlab = 1024;    // parts of a launch: what they leave takes 128 MiB at most

// A row as 16-byte vectors of N elements: vector g holds elements N g - skew ..
// + N - 1; what lies outside the row counts as -inf.
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  const T* at;
  int V, skew, vecs;
  __device__ __forceinline__ Row(const T* row, int V_) : at(row), V(V_), skew((int)(((uintptr_t)row & 15) / sizeof(T))) {
    vecs = (V + skew + N - 1) / N;
  }
  __device__ __forceinline__ u32x4 load(int g) const {
    const int64_t e0 = (int64_t)N * g - skew;
    if (e0 >= 0 && e0 + N <= V) return *reinterpret_cast<const u32x4*>(at + e0);
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) {
        const int64_t a = e0 + 2 * i, b = a + 1;
        const uint32_t lo = a >= 0 && a < V ? at[a] : 0xff80u, hi = b >= 0 && b < V ? at[b] : 0xff80u;
        v[i] = lo | (hi << 16);
      } else {
        const int64_t a = e0 + i;
        v[i] = a >= 0 && a < V ? __float_as_uint(at[a]) : 0xff800000u;
      }
    }
    return v;
  }
};
// f(step, vector, whether there is one) of the vectors lo .. hi - 1, a
// workgroup's threads together, AHEAD of them loaded ahead (a step is 16 KiB,
// and a compute unit takes some ten of them in the time of one's way from
// memory).  The loop stays rolled: a row kept in registers (one unrolled body
// per vector) saved its second reading, and cost more in instructions fetched
// once.
template <int AHEAD, typename T, typename F>
__device__ __forceinline__ void each_vec(const Row<T>& row, int lo, int hi, F f) {
  const int steps = (hi - lo + kRowThreads - 1) / kRowThreads;
  u32x4 v[AHEAD];
  int g = lo + threadIdx.x;
#pragma unroll
  for (int j = 0; j < AHEAD; ++j) v[j] = row.load(min(g + j * kRowThreads, hi - 1));
#pragma unroll 1
  for (int it = 0; it < steps; it += AHEAD) {
    u32x4 w[AHEAD] = {};
    if (it + AHEAD < steps) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) w[j] = row.load(min(g + (AHEAD + j) * kRowThreads, hi - 1));
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (it + j < steps) f(it + j, v[j], g + j * kRowThreads < hi);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v[j] = w[j];
    g += AHEAD * kRowThreads;
  }
}

// The same of an fp32 row, in no order: f(its first element, vector, whether
// there is one).  Vectors that the row fills in part are taken by themselves,
// behind the others, not by a second path of every load.
template <int AHEAD, typename F>
__device__ __forceinline__ void each_vec32(const Row<float>& row, int lo, int hi, F f) {
  const int tid = threadIdx.x;
  const int a = max(lo, row.skew ? 1 : 0), b = min(hi, (row.V + row.skew) / 4);  // whole ones
  const u32x4* at = reinterpret_cast<const u32x4*>(row.at - row.skew);
  if (a < b) {  // uniform
    const int steps = (b - a + kRowThreads - 1) / kRowThreads;
    u32x4 v[AHEAD];
    int g = a + tid;
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) v[j] = at[min(g + j * kRowThreads, b - 1)];
#pragma unroll 1
    for (int it = 0; it < steps; it += AHEAD) {
      u32x4 w[AHEAD] = {};
      if (it + AHEAD < steps) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) w[j] = at[min(g + (AHEAD + j) * kRowThreads, b - 1)];
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (it + j < steps) f(4 * (g + j * kRowThreads) - row.skew, v[j], g + j * kRowThreads < b);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) v[j] = w[j];
      g += AHEAD * kRowThreads;
    }
  }
  const bool front = lo == 0 && row.skew, back = hi == row.vecs && (row.V + row.skew) % 4 && row.vecs - 1 >= a;
  if ((front || back) && tid < 64) {  // uniform
    const bool in = (tid == 0 && front) || (tid == 1 && back);
    const int g = tid == 0 ? 0 : row.vecs - 1;
    u32x4 v{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
    if (in) v = row.load(g);
    f(4 * g - row.skew, v, in);
  }
}

// What the filters of a row are, and what is wanted of it.
struct Settings {
  float T, p, least, u;
  int k;
  bool has_k, has_p, has_least, sampled, ends;
  double inv_t;
};
// (as vector loads: scalar ones would be waited for with the LDS writes)
__device__ __forceinline__ Settings settings_of(const FilterArgs& a, int b, bool sampled, int64_t at_u, bool ends) {
  int vb = b;
  int64_t vu = at_u;
  asm volatile("" : "+v"(vb), "+v"(vu));
  // (no load in a branch: each would be waited for before the next is issued)
  const int32_t* k = a.top_k ? a.top_k : (const int32_t*)a.temperature;
  const float* p = a.top_p ? a.top_p : a.temperature;
  const float* least = a.min_p ? a.min_p : a.temperature;
  Settings f;
  f.T = a.temperature[vb];
  f.k = k[vb];
  f.p = p[vb];
  f.least = least[vb];
  f.u = a.uniforms[vu];
  f.has_k = a.top_k != nullptr;
  f.has_p = a.top_p != nullptr;
  f.has_least = a.min_p != nullptr;
  f.sampled = sampled;
  f.ends = ends;
  return f;
}

// .. as they count, in scalar registers
__device__ __forceinline__ void make_uniform(Settings& f) {
  auto one = [](float x) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(x))); };
  f.T = one(f.T);
  f.p = f.has_p ? one(f.p) : 1.f;
  f.least = f.has_least ? one(f.least) : 0.f;
  f.u = one(f.u);
  f.k = f.has_k ? __builtin_amdgcn_readfirstlane(f.k) : 0;
}

// What the filters leave of a row, and its sample of u where one is wanted, by
// radix descent.
__device__ __forceinline__ RowCut radix_row(const float* row, int V, int shift, const Settings& f, RowLds& s) {
  RowCut out;
  // the argmax: NaN above all, equal values by the lower index
  uint64_t best = 0;
  each<float>(row, V, [&](int i, float x) {
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
  if (is_greedy(f.T) || nan || out.top == -__builtin_inff()) return out;  // uniform

  const double inv_t = 1.0 / (double)f.T, scale = (double)(1ull << shift);
  const float top = out.top;
  if (threadIdx.x < 256) s.tab[threadIdx.x] = kExp2Frac256[threadIdx.x];
  out.kept = V;
  out.cut = -__builtin_inff();
  out.last = V - 1;
  __syncthreads();
  uint64_t total = 0;
  each<float>(row, V, [&](int, float x) { total += fixed_weight(weight_of(x, top, inv_t, s.tab), scale); });
  total = block_sum(total, s);
  uint32_t value = 0, rank = 0;
  int cut_rank = -1;
#pragma unroll 1
  for (int kind = 0; kind < 4; ++kind) {
    double goal = 0.0;
    if (kind == kByCount) {
      if (f.k <= 0 || f.k >= V) continue;
      goal = (double)f.k;
    } else if (kind == kReach) {
      if (!(f.p < 1.f)) continue;
      goal = fmax((double)f.p * (double)total, 0.5);  // (the first token stays)
    } else if (kind == kAbove) {
      if (!(f.least > 0.f)) continue;
      uint64_t sum = 0, count = 0, low = 0;  // low: the furthest key along the order
      each<float>(row, V, [&](int, float x) {
        const double w = weight_of(x, top, inv_t, s.tab);
        if (x != top && !(w >= (double)f.least)) return;
        sum += fixed_weight(w, scale);
        ++count;
        const uint64_t key = order_bits(x);
        low = key > low ? key : low;
      });
      count = block_sum(count, s);
      if ((int)count >= out.kept) continue;
      out.kept = (int)count;
      cut_rank = -1;
      total = block_sum(sum, s);
      out.cut = order_value((uint32_t)block_max(low, s));
      continue;
    } else {
      if (!f.sampled) continue;
      goal = unit(f.u) * (double)total;
    }
    const Spot at = seek<float>(kind, goal, (uint32_t)out.kept, row, V, top, inv_t, scale, s);
    if (kind == kBeyond) {
      const double j = fmin(floor((goal - (double)at.mass) / (double)at.weight),
                            (double)min((int)at.count, out.kept - (int)at.before) - 1.0);
      value = at.key;
      rank = (uint32_t)fmax(j, 0.0);
      continue;
    }
    uint32_t stay = (uint32_t)f.k - at.before;
    if (kind == kReach) {
      const double need = ceil((goal - (double)at.mass) / (double)at.weight);
      stay = (uint32_t)fmin(fmax(need, 1.0), (double)at.count);
    }
    if ((int)(at.before + stay) >= out.kept) continue;
    out.kept = (int)(at.before + stay);
    out.cut = order_value(at.key);
    cut_rank = stay < at.count ? (int)stay - 1 : -1;
    total = at.mass + (uint64_t)stay * at.weight;
  }
  out.total = (double)total / scale;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if (which ? !f.ends || cut_rank < 0 : !f.sampled) continue;  // uniform
    const int at = index_of<float>(which ? out.cut : order_value(value), which ? (uint32_t)cut_rank : rank, row, V, s);
    if (which) out.last = at;
    else out.token = at;
  }
  return out;
}

// ---------------------------------------------------------------------------
// bf16 rows by counts
// ---------------------------------------------------------------------------
constexpr int kGroups = 512;   // of 128 values each, along the order of the tokens: 64 words of two counts
constexpr int kSafeSteps = 7;  // steps of a workgroup whose 57,344 tokens fit a 16-bit count
constexpr int kMaxHeavy = kMaxVocab / 65536 + 1;

struct CountLds {
  uint32_t bin[32768];         // counts of values 2i (low half) and 2i + 1
  // groups that occur, along the order
  double mass[kGroups];        // weights of a group, first of its first value's
  double before[kGroups];      // weights before a group
  uint32_t count[kGroups];
  uint32_t cbefore[kGroups];
  uint32_t ref[kGroups];       // group << 16 | bits of its first value that occurs
  uint16_t gid[kGroups];       // the groups themselves
  uint32_t found[kMaxSteps * kRowWaves];
  double tab[256];
  uint32_t heavy[kMaxHeavy], heavy_count[kMaxHeavy];  // counts beside the bins
  uint32_t part_occurs[kMaxParts * kGroups / 32];
  int heavies;
  int nan, index;
  // what wave 0 decides
  float top, cut;
  int kept, rank, cut_rank;    // rank -1: no token is looked up; cut_rank -1: no index is
  uint32_t value, cut_value;   // bits
  double total;
};

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

// a lane's word of a group
__device__ __forceinline__ uint32_t word_of(int g) {
  const int lane = threadIdx.x & 63;
  return g >= kGroups / 2 ? 64 * g + lane : 64 * (kGroups / 2 - 1 - g) + 63 - lane;
}
__device__ __forceinline__ int group_of(uint32_t value) {
  return value & 0x8000u ? (int)(value >> 7) : kGroups / 2 - 1 - (int)(value >> 7);
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
__device__ __forceinline__ Place seek_counts(int kind, double goal, uint32_t limit, const CountLds& s, int groups, int heavies,
                                             float top, double inv_t) {
  const int lane = threadIdx.x & 63;
  int at_group = -1;
#pragma unroll 1
  for (int i = (groups - 1) >> 6; i >= 0 && at_group < 0; --i) {
    const int mine = min(64 * i + lane, groups - 1);
    bool fits;
    if (kind == kByCount) fits = (double)s.cbefore[mine] < goal;
    else if (kind == kAbove) fits = weight_of(bf16_bits_to_f32(s.ref[mine] & 0xffffu), top, inv_t, s.tab) >= goal;
    else fits = s.mass[mine] > 0.0 && (kind == kReach ? s.before[mine] < goal : s.before[mine] <= goal && s.cbefore[mine] < limit);
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
    return c && w > 0.0 && (kind == kReach ? mb < goal : mb <= goal && cb < limit);
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
__device__ __forceinline__ void find_token(const Row<uint16_t>& row, int lo, int hi, uint32_t value, uint32_t rank, CountLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t mask = value ? ~0u : 0x7fff7fffu, both = value | (value << 16);  // (+0: -0 too)
  each_vec<kSafeSteps>(row, lo, hi, [&](int it, const u32x4& v, bool in) {
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

// Counts and weights of the groups that occur (s.gid), the waves in turn.
__device__ __forceinline__ void weigh_groups(double inv_t, int groups, int heavies, CountLds& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 1
  for (int n = wave; n < groups; n += kRowWaves) {
    const int g = __builtin_amdgcn_readfirstlane(s.gid[n]);
    const Pair q = pair_of(s, heavies, g);
    if (g == 0 || g == kGroups - 1) {  // uniform: infinities and NaNs
      if ((q.c1 && (q.v1 & 0x7fffu) > 0x7f80u) || (q.c2 && (q.v2 & 0x7fffu) > 0x7f80u)) s.nan = 1;
    }
    const uint64_t y1 = __ballot(q.c1 > 0), y2 = __ballot(q.c2 > 0);
    const int l1 = y1 ? __ffsll((long long)y1) - 1 : 64, l2 = y2 ? __ffsll((long long)y2) - 1 : 64;
    const uint32_t ref = lane_u32(l1 <= l2 ? q.v1 : q.v2, min(min(l1, l2), 63));
    double w1, w2;
    pair_weights(q, bf16_bits_to_f32(ref), inv_t, s.tab, w1, w2);
    const double m = wave_sum_dpp(q.c1 * w1 + q.c2 * w2);
    const uint32_t all = lane_u32(wave_scan(q.c1 + q.c2), 63);
    if (lane == 0) {
      s.count[n] = all;
      s.mass[n] = m;
      s.ref[n] = ((uint32_t)g << 16) | ref;
    }
  }
}

// What the filters leave, from the weighed groups, by one wave: into s.
__device__ __forceinline__ void decide(const Settings& f, int V, int groups, int heavies, CountLds& s) {
  const int lane = threadIdx.x & 63;
  // the maximum: the first value (group 255 is there for -0 and empty where
  // 256, which brought it, holds other values alone)
  const uint32_t top_bits = s.ref[s.count[0] ? 0 : min(1, groups - 1)] & 0xffffu;
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
      const Place at = seek_counts(kind, goal, (uint32_t)kept, s, groups, heavies, top, f.inv_t);
      if (kind == kBeyond) {
        value = at.value;
        if (at.count > 1) {
          const double j = fmin(floor((goal - at.mass) / at.weight), (double)min((int)at.count, kept - (int)at.before) - 1.0);
          rank = (int)fmax(j, 0.0);
        }
        continue;
      }
      uint32_t stay = at.count;  // tokens of the value that do
      if (kind == kByCount) stay = (uint32_t)f.k - at.before;
      if (kind == kReach && at.count > 1) stay = (uint32_t)fmin(fmax(ceil((goal - at.mass) / at.weight), 1.0), (double)at.count);
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
__device__ __forceinline__ RowCut nan_row(const Row<uint16_t>& row, CountLds& s) {
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

// What a part of a row holds (at most kSafeSteps steps of a workgroup, so that
// 16 bits hold every count): which groups occur, and the words of those that do.
struct Part {
  uint32_t occurs[kGroups / 32];
  uint32_t word[32768];
};

// A part's counts out of LDS, which is clear for the next one.  A wave takes
// 2,048 words, four a lane at a time: the 16 lanes of a group write it whole or
// not at all.
__device__ __forceinline__ void put_part(uint32_t* bin, Part* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t has = 0;  // of groups in the order of their words
  u32x4 w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const u32x4*>(bin + 2048 * wave + 256 * i + 4 * lane);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint64_t any = __ballot((w[i][0] | w[i][1] | w[i][2] | w[i][3]) != 0);
    if (!any) continue;  // uniform
    const int at = 2048 * wave + 256 * i + 4 * lane;
    if ((any >> (lane & 48)) & 0xffffu) {
      *reinterpret_cast<u32x4*>(out->word + at) = w[i];
      *reinterpret_cast<u32x4*>(bin + at) = u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) has |= ((any >> (16 * g)) & 0xffffu ? 1u : 0u) << (4 * i + g);
  }
  // (positive values: the order is that of falling words)
  if (lane == 0) out->occurs[wave < 8 ? 7 - wave : wave] = wave < 8 ? __brev(has) : has;
}

// Parts first .. last - 1 of `steps` steps each, counted by one workgroup one
// after another; the next one's first vectors are on their way meanwhile.
__device__ __forceinline__ void count_parts(const Row<uint16_t>& row, int first, int last, int steps, uint32_t* bin, Part* out) {
  const int lane = threadIdx.x & 63;
  const int lo = first * steps * kRowThreads, hi = min(last * steps * kRowThreads, row.vecs);
  clear_bins(bin);
  lds_barrier();
  uint32_t heavy = ~0u, many = 0;
  int left = steps;
  each_vec<4>(row, lo, hi, [&](int it, const u32x4& v, bool in) {
    if (in) count_vec(bin, v, heavy, many);
    if (--left && (it + 1) * kRowThreads < hi - lo) return;  // uniform
    // (a wave's lanes count alike, but those without a last vector)
    const uint32_t h = (uint32_t)__builtin_amdgcn_readfirstlane((int)heavy), m = (uint32_t)__builtin_amdgcn_readfirstlane((int)many);
    if (lane == 0 && m) atomicAdd(&bin[h >> 1], m << ((h & 1) << 4));
    lds_barrier();
    put_part(bin, out);
    lds_barrier();
    ++out;
    left = steps;
    heavy = ~0u;
    many = 0;
  });
}

// A bf16 row from the counts of its parts.
__device__ __forceinline__ RowCut merge_row(const Row<uint16_t>& row, Settings f, const Part* in, int parts, int steps, CountLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid < kGroups / 32 * parts) s.part_occurs[tid] = in[tid / (kGroups / 32)].occurs[tid % (kGroups / 32)];
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) {
    s.nan = s.heavies = 0;
    s.bin[0x4000] = 0;  // (read with the word of +0, whether its own group occurs or not)
  }
  __syncthreads();
  uint32_t occurs = 0;
  if (lane < kGroups / 32) {
#pragma unroll 8
    for (int c = 0; c < parts; ++c) occurs |= s.part_occurs[c * (kGroups / 32) + lane];
  }
  if (lane == kGroups / 64 - 1 && (lane_u32(occurs, kGroups / 64) & 1)) occurs |= 1u << 31;  // (-0 counts with +0, the last positive value)
  const uint32_t upto = wave_scan((uint32_t)__popc(occurs));
  const int groups = (int)lane_u32(upto, 63);
  {  // a thread per group: its place among those that occur
    const int l = (tid >> 5) & 15;
    const uint32_t word = (uint32_t)__shfl((int)occurs, l), before = (uint32_t)__shfl((int)upto, l) - __popc(word);
    if (tid < kGroups && ((word >> (tid & 31)) & 1)) s.gid[before + __popc(word & ((1u << (tid & 31)) - 1))] = (uint16_t)tid;
  }
  __syncthreads();
  // the words of a wave's groups, those of three groups in eight parts on their way at once
  constexpr int kAtOnce = 3, kBatch = 8;
  const int last = max(groups - 1, 0);
#pragma unroll 1
  for (int n0 = wave; n0 < groups; n0 += kAtOnce * kRowWaves) {
    const uint32_t gids = s.gid[min(n0 + min(lane, kAtOnce - 1) * kRowWaves, last)];
    uint32_t lo[kAtOnce] = {}, hi[kAtOnce] = {};
#pragma unroll 1
    for (int c0 = 0; c0 < parts; c0 += kBatch) {
      uint32_t w[kAtOnce][kBatch];
      uint64_t have[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int g = (int)lane_u32(gids, i);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) w[i][j] = in[min(c0 + j, parts - 1)].word[word_of(g)];
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int g = (int)lane_u32(gids, i), c = c0 + min(lane, kBatch - 1);
        have[i] = __ballot(c < parts && ((s.part_occurs[min(c, parts - 1) * (kGroups / 32) + (g >> 5)] >> (g & 31)) & 1));
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          // (the word of a group that a part has not is whatever the memory held)
          const uint32_t word = (have[i] >> j) & 1 ? w[i][j] : 0u;
          lo[i] += word & 0xffffu;
          hi[i] += word >> 16;
        }
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (n0 + i * kRowWaves >= groups) break;  // uniform
      const uint32_t word = word_of((int)lane_u32(gids, i));
      if (__ballot((lo[i] | hi[i]) >= 65536)) {  // (rows of one value mostly)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t& c = half ? hi[i] : lo[i];
          if (c < 65536) continue;
          const int at = atomicAdd(&s.heavies, 1);
          s.heavy[at] = 2 * word + half;
          s.heavy_count[at] = c;
          c = 0;
        }
      }
      s.bin[word] = lo[i] | (hi[i] << 16);
    }
  }
  make_uniform(f);
  f.inv_t = is_greedy(f.T) ? 1.0 : 1.0 / (double)f.T;
  __syncthreads();
  const int heavies = s.heavies;
  weigh_groups(f.inv_t, groups, heavies, s);
  __syncthreads();
  if (s.nan) return nan_row(row, s);  // uniform
  if (wave == 0) decide(f, row.V, groups, heavies, s);
  __syncthreads();
  return look_up(row.V, s, [&](uint32_t value, uint32_t rank) {
    // the part that holds the token, by its counts of the value
    uint32_t c = 0;
    auto count = [&](uint32_t v) {
      const int at = group_of(v);
      if (lane >= parts || !((s.part_occurs[lane * (kGroups / 32) + (at >> 5)] >> (at & 31)) & 1)) return;
      const uint32_t both = in[lane].word[v >> 1];
      c += (v & 1) ? both >> 16 : both & 0xffffu;
    };
    count(value);
    if (value == 0) count(0x8000u);
    const uint32_t upto_c = wave_scan(c);
    const int part = max(__ffsll((long long)__ballot(upto_c > rank)) - 1, 0);
    const int lo = part * steps * kRowThreads;
    find_token(row, lo, min(lo + steps * kRowThreads, row.vecs), value, rank - lane_u32(upto_c - c, part), s);
  });
}

// ---------------------------------------------------------------------------
// fp32 rows by bins
// ---------------------------------------------------------------------------
constexpr int kBinShift = 19;           // a bin: the tokens of equal leading 13 bits of their order
constexpr int kBins32 = 1 << (32 - kBinShift);
constexpr int kBinGroups = kBins32 / 64;
constexpr int kList = 4096;             // tokens looked at one by one
constexpr int kSubBins = 1024;
constexpr int kHead = kBinGroups / 32 + 4;

// What one workgroup added up of a row: its maximum, and the bins of the
// groups of 64 that occur: tokens above -inf, and their weights as integers of
// 2^-shift, of the bin's largest possible value (of the maximum in its own bin,
// which at a low temperature lies far above what the others weigh).
struct BinPart {
  uint32_t occurs[kBinGroups / 32];
  float top;
  uint32_t nan, pad[2];        // (kHead words up to here)
  uint32_t count[kBins32];
  unsigned long long mass[kBins32];
};

struct BinLds {
  uint32_t count[kBins32];
  unsigned long long mass[kBins32];
  double tab[256];
  float red[kRowWaves];
  int nan;
};

__device__ __forceinline__ uint32_t bin_of(float x) { return order_bits(x) >> kBinShift; }
__device__ __forceinline__ float bin_edge(uint32_t bin) { return order_value(bin << kBinShift); }

__device__ __forceinline__ void bin_part(const Row<float>& row, int part, int steps, float T, int shift, BinLds& s, BinPart* out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = part * steps * kRowThreads, hi = min(lo + steps * kRowThreads, row.vecs);
  for (int i = tid; i < kBins32 / 4; i += kRowThreads) reinterpret_cast<u32x4*>(s.count)[i] = u32x4{0u, 0u, 0u, 0u};
  for (int i = tid; i < kBins32 / 2; i += kRowThreads) reinterpret_cast<u32x4*>(s.mass)[i] = u32x4{0u, 0u, 0u, 0u};
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) s.nan = 0;
  float top = -__builtin_inff();
  bool nan = false;
  each_vec32<2>(row, lo, hi, [&](int, const u32x4& v, bool) {  // (a vector past the end is the last one again)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(v[e]);
      top = fmaxf(top, x);
      nan |= x != x;
    }
  });
  top = wave_max_dpp(top);
  if (lane == 0) s.red[wave] = top;
  __syncthreads();
  if (nan) s.nan = 1;
  top = s.red[0];
  for (int i = 1; i < kRowWaves; ++i) top = fmaxf(top, s.red[i]);
  __syncthreads();
  if (tid == 0) {
    out->top = top;
    out->nan = s.nan;
  }
  if (s.nan || top == -__builtin_inff()) {  // uniform
    if (tid < kBinGroups / 32) out->occurs[tid] = 0;
    return;
  }
  const double inv_t = is_greedy(T) ? 1.0 : 1.0 / (double)T, scale = (double)(1ull << shift);
  const uint32_t top_bin = bin_of(top);
  auto weigh = [&](float x, uint32_t bin) {
    return fixed_weight(weight_of(x, bin == top_bin ? top : bin_edge(bin), inv_t, s.tab), scale);
  };
  uint32_t heavy = 0xff800000u, many = 0;  // (-inf: none)
  each_vec32<2>(row, lo, hi, [&](int, const u32x4& v, bool in) {
    if (!in) return;
    // a value that many of a wave's lanes hold (a mask's) is added up beside the bins
    const uint32_t some = (uint32_t)__builtin_amdgcn_readfirstlane((int)v[0]);
    const bool crowd = some != 0xff800000u && __popcll(__ballot(v[0] == some)) >= 16 && (many == 0 || heavy == some);
    if (crowd) heavy = some;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(v[e]);
      const bool aside = crowd && v[e] == some;
      if (crowd) many += __popcll(__ballot(aside));
      if (x == -__builtin_inff() || aside) continue;
      const uint32_t bin = bin_of(x);
      atomicAdd(&s.count[bin], 1u);
      const uint64_t q = weigh(x, bin);
      if (q) atomicAdd(&s.mass[bin], (unsigned long long)q);
    }
  });
  heavy = (uint32_t)__builtin_amdgcn_readfirstlane((int)heavy);
  many = (uint32_t)__builtin_amdgcn_readfirstlane((int)many);
  if (many && lane == 0) {
    const float x = __uint_as_float(heavy);
    const uint32_t bin = bin_of(x);
    atomicAdd(&s.count[bin], many);
    atomicAdd(&s.mass[bin], (unsigned long long)many * weigh(x, bin));
  }
  __syncthreads();
  // the groups that occur: 8 each wave
  uint32_t has = 0;
#pragma unroll
  for (int i = 0; i < kBinGroups / kRowWaves; ++i) {
    const int at = (wave * (kBinGroups / kRowWaves) + i) * 64 + lane;
    const uint32_t c = s.count[at];
    if (!__ballot(c > 0)) continue;  // uniform
    has |= 1u << i;
    out->count[at] = c;
    out->mass[at] = s.mass[at];
  }
  static_assert(kBinGroups / kRowWaves == 8, "a byte of bits per wave");
  if (lane == 0) reinterpret_cast<uint8_t*>(out->occurs)[wave] = (uint8_t)has;
}

struct Bin {
  uint32_t bin;
  uint32_t before, count;  // tokens
  double mass, weight;     // weights before; of its tokens
};

struct ListLds {
  uint32_t count[kBins32];     // tokens of a bin; at the end the indices of equal tokens
  double weight[kBins32];      // their weights
  // groups that occur, along the order
  double gweight[kBinGroups], gbefore[kBinGroups];
  uint32_t gcount[kBinGroups], gcbefore[kBinGroups], gid[kBinGroups];
  uint32_t head[kMaxParts * kHead];  // of the parts
  double part_scale[kMaxParts];
  Bin at;                      // what wave 0 found
  Bin range_bin[4];            // by kind: the bin of a range of one bin
  int one_bin[4];
  float high[4], low[4];       // ranges of values to list
  int ranges;
  uint64_t list[kList];        // order bits << 32 | index
  uint32_t sub_count[kSubBins], sub_at[kSubBins];
  unsigned long long sub_mass[kSubBins];
  double tab[256];
  uint32_t red[kRowWaves];
  uint64_t red2[kRowWaves];
  int nan, listed, hit, index, equals;
  uint32_t hit_count, hit_before;
  uint64_t hit_mass, hit_mass_before;
};
union RowLds32 {
  ListLds bins;
  RowLds radix;
};

// The last bin with: tokens before it < goal (kByCount); weights before it <
// goal (kReach) or <= goal (kBeyond, and tokens before it < limit), and a weight
// of its own; a largest possible weight >= goal (kAbove).  By one wave.
__device__ __forceinline__ Bin seek_bin(int kind, double goal, uint32_t limit, const ListLds& s, int groups, float top, double inv_t) {
  const int lane = threadIdx.x & 63;
  int n = -1;
#pragma unroll 1
  for (int i = (groups - 1) >> 6; i >= 0 && n < 0; --i) {
    const int mine = min(64 * i + lane, groups - 1);
    bool fits;
    if (kind == kByCount) fits = (double)s.gcbefore[mine] < goal;
    // (a group's first bin may be empty: whether another of it is heavy enough shows below)
    else if (kind == kAbove) fits = weight_of(fminf(bin_edge(64 * s.gid[mine]), top), top, inv_t, s.tab) >= goal;
    else if (kind == kReach) fits = s.gweight[mine] > 0.0 && s.gbefore[mine] < goal;
    else fits = s.gweight[mine] > 0.0 && s.gbefore[mine] <= goal && s.gcbefore[mine] < limit;
    const uint64_t yes = __ballot(fits && 64 * i + lane < groups);
    if (yes) n = 64 * i + 63 - __clzll((long long)yes);
  }
  n = max(n, 0);
  Bin at{};
#pragma unroll 1
  for (;; --n) {  // (to a group before, where the bins that are heavy enough are empty, or those with a weight past the limit)
    const uint32_t bin = 64 * s.gid[n] + lane, c = s.count[bin];
    const double w = s.weight[bin];
    const double before = s.gbefore[n] + lane_before(wave_scan(w));
    const uint32_t cbefore = s.gcbefore[n] + wave_scan(c) - c;
    bool fits = c > 0;
    if (kind == kByCount) fits = fits && (double)cbefore < goal;
    else if (kind == kAbove) fits = fits && weight_of(fminf(bin_edge(bin), top), top, inv_t, s.tab) >= goal;
    else fits = fits && w > 0.0 && (kind == kReach ? before < goal : before <= goal && cbefore < limit);
    const uint64_t yes = __ballot(fits);
    if (!yes && n > 0) continue;
    const int l = yes ? 63 - __clzll((long long)yes) : 0;
    at.bin = lane_u32(bin, l);
    at.before = lane_u32(cbefore, l);
    at.count = lane_u32(c, l);
    at.mass = lane_f64(before, l);
    at.weight = lane_f64(w, l);
    return at;
  }
}

// .. for the whole workgroup: a range of one bin is that bin (kBeyond's begins
// with a bin that holds kept tokens: its goal is below the weights before the cut's)
__device__ __forceinline__ Bin find_bin(int kind, double goal, uint32_t limit, int groups, float top, double inv_t, ListLds& s) {
  if (__builtin_amdgcn_readfirstlane(s.one_bin[kind])) return s.range_bin[kind];
  if (threadIdx.x < 64) {
    const Bin at = seek_bin(kind, goal, limit, s, groups, top, inv_t);
    if (threadIdx.x == 0) s.at = at;
  }
  __syncthreads();
  return s.at;
}

// As seek, among the listed tokens of a bin.  mass, weight: integers of
// 2^-shift of the bin's reference value.  The first value always fits: the bin
// itself does, also where its tokens weigh nothing beside its reference (the
// bin's weight can come from the maximum of a part, weighed by that).
__device__ __forceinline__ Spot seek_list(int kind, double goal, uint32_t limit, uint32_t bin, float ref, double inv_t, double scale,
                                          ListLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Spot at{bin << kBinShift, 0u, 0u, 0ull, 0ull, -1};
#pragma unroll 1
  for (int level = 0; level < 2; ++level) {
    const int sh = level ? 0 : 9, bits = level ? 9 : 10;
    __syncthreads();
    s.sub_count[tid] = 0;
    s.sub_mass[tid] = 0;
    if (tid == 0) s.hit = -1;
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < s.listed; i += kRowThreads) {
      const uint32_t k = (uint32_t)(s.list[i] >> 32);
      if ((k >> (sh + bits)) != (at.key >> (sh + bits))) continue;
      const uint32_t sub = (k >> sh) & ((1u << bits) - 1);
      atomicAdd(&s.sub_count[sub], 1u);
      s.sub_at[sub] = i;
      const uint64_t q = fixed_weight(weight_of(order_value(k), ref, inv_t, s.tab), scale);
      if (q) atomicAdd(&s.sub_mass[sub], (unsigned long long)q);
    }
    __syncthreads();
    const uint32_t c = s.sub_count[tid], cu = wave_scan(c);
    const uint64_t m = s.sub_mass[tid], mu = wave_scan(m);
    if (lane == 63) {
      s.red[wave] = cu;
      s.red2[wave] = mu;
    }
    __syncthreads();
    const uint32_t cw = lane < kRowWaves ? s.red[lane] : 0u;
    const uint64_t mw = lane < kRowWaves ? s.red2[lane] : 0ull;
    const uint32_t cb = at.before + cu - c + lane_u32(wave_scan(cw) - cw, wave);
    const uint64_t mb = at.mass + mu - m + lane_u64(wave_scan(mw) - mw, wave);
    bool fits = c > 0;
    if (kind == kByCount) fits = fits && (double)cb < goal;
    else fits = fits && (cb == at.before || (m > 0 && (kind == kReach ? (double)mb < goal : (double)mb <= goal && cb < limit)));
    if (fits) atomicMax(&s.hit, tid);
    __syncthreads();
    if (tid == max(s.hit, 0)) {
      s.hit_count = c;
      s.hit_before = cb;
      s.hit_mass = m;
      s.hit_mass_before = mb;
    }
    __syncthreads();
    at.key |= (uint32_t)max(s.hit, 0) << sh;
    at.before = s.hit_before;
    at.mass = s.hit_mass_before;
    at.count = s.hit_count;
    at.weight = s.hit_mass;
    if (at.count == 1) {  // uniform: that token itself (fp32 values are apart as a rule)
      at.only = s.sub_at[max(s.hit, 0)];
      at.key = (uint32_t)(s.list[at.only] >> 32);
      break;
    }
  }
  // (equal values have equal weights, whole numbers below 2^51: the quotient of their sum is off by less than a half)
  if (at.count > 1) at.weight = (uint64_t)rint((double)at.weight / (double)at.count);
  return at;
}

// index of the listed token of the value with `rank` of them before it (the
// bins are overwritten)
__device__ __forceinline__ int index_in_list(uint32_t key, uint32_t rank, ListLds& s) {
  __syncthreads();
  if (threadIdx.x == 0) s.equals = s.index = 0;
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < s.listed; i += kRowThreads)
    if ((uint32_t)(s.list[i] >> 32) == key) s.count[atomicAdd(&s.equals, 1)] = (uint32_t)s.list[i];
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < s.equals; i += kRowThreads) {
    const uint32_t mine = s.count[i];
    uint32_t before = 0;
    for (int j = 0; j < s.equals; ++j) before += s.count[j] < mine;
    if (before == rank) s.index = (int)mine;
  }
  __syncthreads();
  return s.index;
}

// A row from its parts' bins.  Which bins the cuts and the sample lie in
// follows from the sums, but for the weights inside the bin of the cut before:
// so from the least and the most it may leave a range of bins is taken, the
// tokens of all ranges are listed in one pass over the row, and the values
// found among them.
__device__ __forceinline__ RowCut list_row(const Row<float>& row, Settings f, const BinPart* in, int parts, int shift, ListLds& s,
                                           bool& fits) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = row.V;
  constexpr int kWords = kBinGroups / 32;
  fits = true;
  if (tid < kHead * parts) s.head[tid] = reinterpret_cast<const uint32_t*>(&in[tid / kHead])[tid % kHead];
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) s.listed = 0;
  __syncthreads();
  make_uniform(f);
  const float my_top = lane < parts ? __uint_as_float(s.head[lane * kHead + kWords]) : -__builtin_inff();
  const float top = wave_max_dpp(my_top);
  const bool nan = __ballot(lane < parts && s.head[min(lane, parts - 1) * kHead + kWords + 1]) != 0;
  const bool greedy = is_greedy(f.T);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)f.T, scale = (double)(1ull << shift), per = 1.0 / scale;
  if (tid < parts) s.part_scale[tid] = weight_of(my_top, top, inv_t, s.tab) * per;
  RowCut out{top, top, V - 1, 1, 0, 0, 1.0};
  if (nan) {  // uniform
    fits = false;
    return out;
  }
  if (top == -__builtin_inff()) {  // uniform: nothing above it, the first token
    out.last = 0;
    return out;
  }
  // the parts' bins added up: those of a part's maximum by that, the others as integers
  uint32_t occurs = 0;
  if (lane < kWords) {
#pragma unroll 8
    for (int c = 0; c < parts; ++c) occurs |= s.head[c * kHead + lane];
  }
  __syncthreads();  // part_scale
  const uint32_t upto = wave_scan((uint32_t)__popc(occurs));
  const int groups = (int)lane_u32(upto, 63);
#pragma unroll 1
  for (int n = wave; n < groups; n += kRowWaves) {
    const int g = nth_group(n, occurs, upto);
    const uint64_t have = __ballot(lane < parts && ((s.head[min(lane, parts - 1) * kHead + (g >> 5)] >> (g & 31)) & 1));
    const uint32_t bin = 64 * g + lane;
    uint32_t count = 0;
    uint64_t mass = 0;
    double weight = 0.0;
#pragma unroll 1
    for (int c0 = 0; c0 < parts; c0 += 8) {
      uint32_t pc[8];
      unsigned long long pm[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const BinPart& p = in[min(c0 + j, parts - 1)];
        pc[j] = p.count[bin];
        pm[j] = p.mass[bin];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!((have >> (c0 + j)) & 1)) continue;  // uniform (what a part has not is whatever the memory held)
        const uint32_t tb = bin_of(__uint_as_float(lane_u32(__float_as_uint(my_top), c0 + j)));
        count += pc[j];
        if ((tb >> 6) == (uint32_t)g && bin == tb) weight += (double)pm[j] * s.part_scale[c0 + j];
        else mass += pm[j];
      }
    }
    weight += (double)mass * (weight_of(fminf(bin_edge(bin), top), top, inv_t, s.tab) * per);
    s.count[bin] = count;
    s.weight[bin] = weight;
    const double all = wave_sum_dpp(weight);
    const uint32_t many = lane_u32(wave_scan(count), 63);
    if (lane == 0) {
      s.gweight[n] = all;
      s.gcount[n] = many;
      s.gid[n] = g;
    }
  }
  __syncthreads();
  double total = 0.0;
  uint32_t tokens = 0;  // above -inf
  if (wave == 0) {
#pragma unroll 1
    for (int i = 0; i < groups; i += 64) {
      const int n = min(i + lane, groups - 1);
      const bool here = i + lane < groups;
      const double w = here ? s.gweight[n] : 0.0, wu = wave_scan(w);
      const uint32_t c = here ? s.gcount[n] : 0u, cu = wave_scan(c);
      if (here) {
        s.gbefore[n] = total + lane_before(wu);
        s.gcbefore[n] = tokens + cu - c;
      }
      total += lane_f64(wu, 63);
      tokens += lane_u32(cu, 63);
    }
  }
  __syncthreads();
  total = s.gbefore[groups - 1] + s.gweight[groups - 1];
  tokens = s.gcbefore[groups - 1] + s.gcount[groups - 1];

  // ranges of bins, from the least and the most that each cut may leave
  // (A cut leaves the weights before its bin and those of listed tokens: the same
  // integers that the bin's sum is of, but where it holds a part's maximum and so
  // was weighed by that.  At most kList of them, off by 2^-(shift+1) both times:
  // 2^-30 with the least shift, 42, of a W of 1 at least.)
  const double tiny = 0x1p-1000, slack = 0x1p-30;
  const bool by_count = !greedy && f.k > 0 && f.k < V && (uint32_t)f.k < tokens, reach = !greedy && f.p < 1.f,
             above = !greedy && f.least > 0.f, draws = !greedy && f.sampled;
  if (wave == 0) {
    double least = total, most = total;
    int ranges = 0;
    uint32_t hull_first = kBins32, hull_last = 0, hull_before = 0, hull_upto = 0;  // bins, tokens
#pragma unroll 1
    for (int kind = 0; kind < 5; ++kind) {  // (4: the maximum's bin)
      if (!(kind == kByCount ? by_count : kind == kReach ? reach : kind == kAbove ? above : kind == kBeyond ? draws : greedy)) continue;
      double g0 = 0.0, g1 = 0.0;
      if (kind == kByCount) g0 = g1 = (double)f.k;
      if (kind == kAbove) g0 = g1 = fmin((double)f.least, 1.0);
      if (kind == kReach) {
        g0 = fmax((double)f.p * least * (1.0 - slack), tiny);
        g1 = fmax((double)f.p * most * (1.0 + slack), tiny);
      }
      if (kind == kBeyond) {
        g0 = unit(f.u) * least * (1.0 - slack);
        g1 = unit(f.u) * most * (1.0 + slack);
      }
      uint32_t first = bin_of(top), last = first;
      uint32_t before = 0, upto_last = 0;
      if (kind < 4) {
        const Bin x = seek_bin(kind, g0, V, s, groups, top, inv_t);
        first = x.bin;
        before = x.before;
        upto_last = x.before + x.count;
        double m0 = x.mass, m1 = x.mass + x.weight;
        // (the bin reaches over both goals as a rule)
        if (kind == kReach ? m1 < g1 : kind == kBeyond && m1 <= g1) {
          const Bin y = seek_bin(kind, g1, V, s, groups, top, inv_t);
          last = y.bin;
          upto_last = y.before + y.count;
          m1 = y.mass + y.weight;
        } else {
          last = first;
        }
        if (lane == 0) {
          s.one_bin[kind] = first == last;
          s.range_bin[kind] = x;
        }
        if (kind == kAbove) {
          m0 = fmin(m0, least);
          m1 = fmin(m1, most);
        }
        least = m0;
        most = m1;
      }
      if (first < hull_first) {
        hull_first = first;
        hull_before = before;
      }
      hull_last = max(hull_last, last);
      hull_upto = max(hull_upto, upto_last);
      const float h = bin_edge(first);
      if (lane == 0) {
        s.high[ranges] = h == h ? h : __builtin_inff();  // (infinity's bin begins with NaNs)
        s.low[ranges] = order_value(((last + 1) << kBinShift) - 1);
      }
      ++ranges;
    }
    // Ranges with few tokens between them are one: a row of 50,001 is listed in
    // 9,500 cycles instead of 18,000 (comparisons, not memory, bound it).
    if (ranges > 1 && hull_upto - hull_before <= kList / 2) {
      const float h = bin_edge(hull_first);
      if (lane == 0) {
        s.high[0] = h == h ? h : __builtin_inff();
        s.low[0] = order_value(((hull_last + 1) << kBinShift) - 1);
      }
      ranges = 1;
    }
    if (lane == 0) s.ranges = ranges;
  }
  __syncthreads();
  const int ranges = __builtin_amdgcn_readfirstlane(s.ranges);
  auto bound = [&](const float* at, int i) {
    return i < ranges ? __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(at[i]))) : __builtin_nanf("");
  };
  const float h0 = bound(s.high, 0), h1 = bound(s.high, 1), h2 = bound(s.high, 2), h3 = bound(s.high, 3);
  const float l0 = bound(s.low, 0), l1 = bound(s.low, 1), l2 = bound(s.low, 2), l3 = bound(s.low, 3);
  auto list = [&](auto several) {
    each_vec32<4>(row, 0, row.vecs, [&](int e0, const u32x4& v, bool here) {
      const uint64_t some = __ballot(here);
      uint64_t in[4];  // of each element: the lanes whose is in a range (comparisons all, and no branch)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __uint_as_float(v[e]);
        in[e] = __ballot(x <= h0) & __ballot(x >= l0);
        if constexpr (several)
          in[e] |= (__ballot(x <= h1) & __ballot(x >= l1)) | (__ballot(x <= h2) & __ballot(x >= l2)) | (__ballot(x <= h3) & __ballot(x >= l3));
        in[e] &= some;
      }
      const int n = __popcll(in[0]) + __popcll(in[1]) + __popcll(in[2]) + __popcll(in[3]);
      if (!n) return;  // uniform
      int base = 0;
      if (lane == 0) base = atomicAdd(&s.listed, n);
      base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (__builtin_amdgcn_inverse_ballot_w64(in[e])) {
          const int at = base + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], 0));
          if (at < kList) s.list[at] = ((uint64_t)order_bits(__uint_as_float(v[e])) << 32) | (uint32_t)(e0 + e);
        }
        base += __popcll(in[e]);
      }
    });
  };
  if (ranges > 1) list(std::true_type{});
  else if (ranges) list(std::false_type{});
  __syncthreads();
  if (s.listed > kList) {  // uniform
    fits = false;
    return out;
  }
  // the cuts, one after another, among the listed tokens
  uint32_t cut_key = order_bits(top), token_key = cut_key, token_rank = 0;
  int cut_rank = -1, only = -1;
  bool cuts = false;  // cut_key is a value that stays in part at least
  double W = greedy ? 1.0 : total;
  int kept = greedy ? 1 : V;
  if (greedy) cuts = true;
  if (!greedy && f.k > 0 && f.k < V) kept = f.k;
  out.cut = greedy ? top : -__builtin_inff();
  auto ref_of = [&](uint32_t bin) { return fminf(bin_edge(bin), top); };
  if (by_count) {
    const Bin at = find_bin(kByCount, (double)f.k, V, groups, top, inv_t, s);
    const Spot x = seek_list(kByCount, (double)((uint32_t)f.k - at.before), V, at.bin, ref_of(at.bin), inv_t, scale, s);
    const uint32_t n = (uint32_t)f.k - at.before - x.before;
    W = at.mass + (double)(x.mass + n * x.weight) * (weight_of(ref_of(at.bin), top, inv_t, s.tab) * per);
    cut_key = x.key;
    cut_rank = n < x.count ? (int)n - 1 : -1;
    cuts = true;
  }
  if (reach) {
    const double goal = fmax((double)f.p * W, tiny);
    const Bin at = find_bin(kReach, goal, V, groups, top, inv_t, s);
    const double unit_w = weight_of(ref_of(at.bin), top, inv_t, s.tab) * per;
    const double inside = fmax((goal - at.mass) / unit_w, 0.5);
    const Spot x = seek_list(kReach, inside, V, at.bin, ref_of(at.bin), inv_t, scale, s);
    uint32_t n = 1;
    if (x.count > 1) {  // uniform
      const double need = ceil((inside - (double)x.mass) / (double)x.weight);
      n = (uint32_t)fmin(fmax(need, 1.0), (double)x.count);
    }
    if ((int)(at.before + x.before + n) < kept) {
      kept = (int)(at.before + x.before + n);
      W = at.mass + (double)(x.mass + n * x.weight) * unit_w;
      cut_key = x.key;
      cut_rank = n < x.count ? (int)n - 1 : -1;
      cuts = true;
    }
  }
  if (above) {
    const double goal = fmin((double)f.least, 1.0);
    const Bin at = find_bin(kAbove, goal, V, groups, top, inv_t, s);
    const float ref = ref_of(at.bin);
    // the bin's tokens that are heavy enough: how many, their weights, the lightest
    __syncthreads();
    if (tid == 0) {
      s.hit_count = 0;
      s.hit_mass = 0;
      s.hit_before = 0;
    }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < s.listed; i += kRowThreads) {
      const uint32_t k = (uint32_t)(s.list[i] >> 32);
      const float x = order_value(k);
      if (k >> kBinShift != at.bin || !(weight_of(x, top, inv_t, s.tab) >= goal)) continue;
      atomicAdd(&s.hit_count, 1u);
      atomicMax(&s.hit_before, k);
      atomicAdd((unsigned long long*)&s.hit_mass, (unsigned long long)fixed_weight(weight_of(x, ref, inv_t, s.tab), scale));
    }
    __syncthreads();
    const uint32_t n = s.hit_count;
    if ((int)(at.before + n) < kept) {
      kept = (int)(at.before + n);
      W = at.mass + (double)s.hit_mass * (weight_of(ref, top, inv_t, s.tab) * per);
      // (none: what lies before the bin, whose largest possible value none of its tokens has)
      cut_key = n ? s.hit_before : at.bin << kBinShift;
      cut_rank = -1;
      cuts = true;
    }
  }
  if (f.sampled && kept > 1) {
    const double goal = unit(f.u) * W;
    const Bin at = find_bin(kBeyond, goal, (uint32_t)kept, groups, top, inv_t, s);
    const double unit_w = weight_of(ref_of(at.bin), top, inv_t, s.tab) * per;
    const double inside = fmax((goal - at.mass) / unit_w, 0.0);
    const Spot x = seek_list(kBeyond, inside, (uint32_t)kept - at.before, at.bin, ref_of(at.bin), inv_t, scale, s);
    token_key = x.key;
    if (x.count > 1) {  // uniform
      const double j = fmin(floor((inside - (double)x.mass) / (double)x.weight),
                            (double)min((int)x.count, kept - (int)(at.before + x.before)) - 1.0);
      token_rank = (uint32_t)fmax(j, 0.0);
    }
    only = x.only;
  }
  out.kept = kept;
  out.total = W;
  if (cuts) out.cut = order_value(cut_key);
  if (only >= 0) out.token = (int)(uint32_t)s.list[only];
  else if (kept == 1 || f.sampled) out.token = index_in_list(token_key, token_rank, s);
  if (kept == 1 && only < 0 && s.equals == 0) {  // uniform: alone because of a bin behind its own, which was not listed
    if (tid == 0) s.index = V;
    __syncthreads();
    each<float>(row.at, V, [&](int i, float x) {
      if (x == top) atomicMin(&s.index, i);
    });
    __syncthreads();
    out.token = s.index;
  }
  if (kept == 1) out.last = out.token;
  else if (f.ends && cut_rank >= 0) out.last = index_in_list(cut_key, (uint32_t)cut_rank, s);
  return out;
}


// ---------------------------------------------------------------------------
// kernels
// ---------------------------------------------------------------------------

// Row r of sequence b: where it lies, and what is wanted of it.
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

// Parts of a row (one more than another's, maybe, where it starts off a 16-byte boundary).
template <typename T>
__device__ __forceinline__ int part_count(const Row<T>& row, int steps) {
  return (row.vecs + steps * kRowThreads - 1) / (steps * kRowThreads);
}

// What a launch's n-th row is.
template <typename T>
struct Work {
  int r, b;
  Job j;
  const T* row;
  __device__ __forceinline__ Work(const FilterArgs& a, int n) {
    b = (a.row0 + n) / a.rows;
    r = a.row0 + n - b * a.rows;
    j = job_of(a, r, b);
    row = (const T*)(j.is_draft ? a.draft : a.target) + j.at;
  }
};

// grid (workgroups of a row, rows).  Counting: 151,936 tokens in 7 workgroups
// 5.8 us, 256 such rows (77.8 MB) by a workgroup each 20.4 us, 3.7 TB/s.  Bound
// by the LDS: 8,192 additions at random words are 1,200 cycles, 0.6 of them bank
// conflicts.  Up to 8 workgroups a row, because one CU takes in some 50 GB/s
// however many loads are under way; not more, because the row's second
// workgroup reads what each leaves.
__global__ __launch_bounds__(kRowThreads) void filter_count_kernel(FilterArgs a) {
  __shared__ uint32_t bin[32768];
  const Work<uint16_t> w(a, blockIdx.y);
  if (!w.j.active) return;  // uniform
  const Row<uint16_t> row(w.row, a.V);
  const int first = blockIdx.x * a.share, last = min(first + a.share, part_count(row, a.steps));
  if (first < last) count_parts(row, first, last, a.steps, bin, (Part*)a.row_parts + (int64_t)blockIdx.y * a.split + first);
}
// grid (parts, rows).  21 rows of 50,001 (4.2 MB) 7.9 us, 45 such rows 11.2: the
// maximum, then an exponential and two LDS additions per token, the bins cleared
// before and put away behind (2,000 to 4,500 cycles each); its waves wait for
// 0.56 of their cycles.
__global__ __launch_bounds__(kRowThreads) void filter_bin_kernel(FilterArgs a) {
  __shared__ BinLds s;
  const Work<float> w(a, blockIdx.y);
  if (!w.j.active) return;  // uniform
  const Row<float> row(w.row, a.V);
  if ((int)blockIdx.x < part_count(row, a.steps))
    bin_part(row, blockIdx.x, a.steps, a.temperature[w.b], a.shift, s,
             (BinPart*)a.row_parts + (int64_t)blockIdx.y * a.split + blockIdx.x);
}
// grid rows.  1 row of 151,936 11.7 us, 88 rows 15.3, 256 rows 17.6: a chain of
// dependent steps in one workgroup (parts read and added 8,500 cycles, groups
// weighed 6,000, cuts and sample by one wave 4,800, its index 5,700 in a part of 3
// steps and 11,900 in one of 7, at 5.4 TB/s over the chip).  One workgroup a row,
// since the steps are too short to hand over.
__global__ __launch_bounds__(kRowThreads) void filter_merge_kernel(FilterArgs a) {
  __shared__ CountLds s;
  const Work<uint16_t> w(a, blockIdx.x);
  if (!w.j.active) return;  // uniform
  const Part* in = (const Part*)a.row_parts + (int64_t)blockIdx.x * a.split;
  const Row<uint16_t> row(w.row, a.V);
  put_row(a, w.r, w.b, w.j, w.row, merge_row(row, settings_of(a, w.b, w.j.sampled, w.j.u, w.j.ends), in,
                                             part_count(row, a.steps), a.steps, s));
}
// grid rows.  21 rows of 50,001 24.0 us, 45 rows 33.8, as long as the row with
// the most filters takes: parts added 10,500 cycles, a bin found 2,500, the row
// listed 9,500 (18,000 with several ranges), each cut and the sample 4,500.
__global__ __launch_bounds__(kRowThreads) void filter_list_kernel(FilterArgs a) {
  __shared__ RowLds32 s;
  const Work<float> w(a, blockIdx.x);
  if (!w.j.active) return;  // uniform
  const BinPart* in = (const BinPart*)a.row_parts + (int64_t)blockIdx.x * a.split;
  const Row<float> row(w.row, a.V);
  bool fits;
  RowCut c = list_row(row, settings_of(a, w.b, w.j.sampled, w.j.u, w.j.ends), in, part_count(row, a.steps), a.shift, s.bins, fits);
  // (worked out anew: kept over all that, it would be spilled)
  int n = blockIdx.x;
  asm volatile("" : "+s"(n));
  const Work<float> again(a, n);
  if (!fits) {  // uniform
    Settings f = settings_of(a, again.b, again.j.sampled, again.j.u, again.j.ends);
    make_uniform(f);
    __syncthreads();
    c = radix_row(again.row, a.V, a.shift, f, s.radix);
  }
  put_row(a, again.r, again.b, again.j, again.row, c);
}

// How rows are cut: `split` parts of `steps` steps of a workgroup each, `share`
// of them counted by one workgroup one after another.  As many workgroups a row
// as the rows leave of 256, 8 at most (the second kernel reads every part), and
// in bf16 so many parts that 16 bits count one.  Flat bf16 rows of 151,936, read
// again and again, in us per call: 32 rows 21.3, 64 23.3, 65 24.7, 85 25.6, 86
// 27.3, 128 29.5, 129 33.6, 255 37.5.  Just behind a step up compute units are
// without work (129 rows take 129 of them); choosing by the steps in turn was
// not measured.
struct Cut {
  int steps, split, share;
};
Cut cut_rows(int rows, int V, int dtype) {
  const int step = dtype == NSV_BF16 ? kStep : kStep / 2;
  const int whole = (V + (dtype == NSV_BF16 ? 7 : 3) + step - 1) / step;  // steps of a row
  int groups = rows >= 256 ? 1 : 256 / rows;
  if (groups > kFewParts) groups = kFewParts;
  Cut c;
  c.share = dtype == NSV_BF16 ? (whole + groups * kSafeSteps - 1) / (groups * kSafeSteps) : 1;
  c.steps = (whole + groups * c.share - 1) / (groups * c.share);
  c.split = (whole + c.steps - 1) / c.steps;
  return c;
}
size_t part_bytes(int dtype) { return dtype == NSV_BF16 ? sizeof(Part) : sizeof(BinPart); }
static_assert(sizeof(Part) % 16 == 0 && sizeof(BinPart) % 16 == 0 && kMaxVocab / (kSafeSteps * kStep) + 1 + kFewParts < kMaxParts &&
              kHead * kMaxParts <= kRowThreads, "parts");

}  // namespace

namespace nsv_filter {

size_t rows_bytes(int rows, int V, int dtype) {
  if (rows <= 0) return 0;
  const int n = cut_rows(rows, V, dtype).split, most = kSlab / n;
  return (size_t)(rows < most ? rows : most) * n * part_bytes(dtype);
}

int launch_rows(FilterArgs& a, int dtype, void* workspace, hipStream_t s) {
  const int total = a.rows * a.B;
  const Cut c = cut_rows(total, a.V, dtype);
  a.split = c.split;
  a.steps = c.steps;
  a.share = c.share;
  a.row_parts = workspace;
  const int most = kSlab / c.split;
  for (a.row0 = 0; a.row0 < total; a.row0 += most) {
    const int rows = total - a.row0 < most ? total - a.row0 : most;
    const dim3 parts((c.split + c.share - 1) / c.share, rows), block(kRowThreads);
    if (dtype == NSV_BF16) hipLaunchKernelGGL(filter_count_kernel, parts, block, 0, s, a);
    else hipLaunchKernelGGL(filter_bin_kernel, dim3(c.split, rows), block, 0, s, a);
    int rc = nsv_launch_status();
    if (rc) return rc;
    if (dtype == NSV_BF16) hipLaunchKernelGGL(filter_merge_kernel, dim3(rows), block, 0, s, a);
    else hipLaunchKernelGGL(filter_list_kernel, dim3(rows), block, 0, s, a);
    if ((rc = nsv_launch_status())) return rc;
  }
  return NSV_OK;
}

}  // namespace nsv_filter
