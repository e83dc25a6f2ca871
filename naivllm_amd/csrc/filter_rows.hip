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
//     2^18 tokens), each weight off by 2^-45 of the largest, where fp32 sums
//     would move the sample of one row in a hundred.  The second kernel lists
//     the tokens of the few bins that matter and looks at those.  A row whose
//     list is too long (many equal values) or that holds a NaN goes by radix
//     descent over its order-preserving bits, a pass over the row per level.

#include "filter.h"

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
// rows in parts
// ---------------------------------------------------------------------------
constexpr int kAhead = 4;      // vectors a thread loads ahead of those it works on
constexpr int kMaxParts = 32;  // of a row, by a workgroup each ..
constexpr int kMaxSplit = 8;   // .. and this many at most where one would do
constexpr int kSlab = 1024;    // parts of a launch: their counts take 128 MiB at most

// A row as 16-byte vectors of N elements: vector g holds elements N g - skew ..
// + N - 1; what lies outside the row counts as -inf.
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);
  const T* at;
  int V, skew, vecs;
  __device__ Row(const T* row, int V_) : at(row), V(V_), skew((int)(((uintptr_t)row & 15) / sizeof(T))) {
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
template <typename T>
__device__ __forceinline__ int part_vecs(const Row<T>& row, int parts) { return (row.vecs + parts - 1) / parts; }

// f(step, vector, whether there is one) of the vectors lo .. hi - 1, a
// workgroup's threads together, kAhead of them loaded ahead.  The loop stays
// rolled: a row kept in registers (one unrolled body per vector) saved its
// second reading, and cost more in instructions fetched once.
template <typename T, typename F>
__device__ __forceinline__ void each_vec(const Row<T>& row, int lo, int hi, F f) {
  const int steps = (hi - lo + kRowThreads - 1) / kRowThreads;
  u32x4 v[kAhead];
  int g = lo + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) v[j] = row.load(min(g + j * kRowThreads, hi - 1));
#pragma unroll 1
  for (int it = 0; it < steps; it += kAhead) {
    u32x4 w[kAhead] = {};
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

// What the filters of a row are, and what is wanted of it.
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

// .. for scalar registers and uniform branches
__device__ __forceinline__ void make_uniform(Settings& f) {
  auto one = [](float x) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(x))); };
  f.T = one(f.T);
  f.p = one(f.p);
  f.least = one(f.least);
  f.u = one(f.u);
  f.k = __builtin_amdgcn_readfirstlane(f.k);
}

// ---------------------------------------------------------------------------
// bf16 rows by counts
// ---------------------------------------------------------------------------
constexpr int kGroups = 512;   // of 128 values each, along the order of the tokens: 64 words of two counts
constexpr int kSafeSteps = 7;  // steps of a workgroup whose 57,344 tokens fit a 16-bit count
constexpr int kMaxHeavy = kMaxVocab / 65536 + 1;

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
__device__ __forceinline__ void find_token(const Row<uint16_t>& row, int lo, int hi, uint32_t value, uint32_t rank, CountLds& s) {
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

// Counts and weights of the groups that occur, the waves in turn; their number.
__device__ __forceinline__ int weigh_groups(double inv_t, int heavies, CountLds& s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t occurs = lane < kGroups / 32 ? s.occurs[lane] : 0u;
  // (-0 counts with +0, the last value of the positive ones)
  if (lane == kGroups / 64 - 1 && (s.occurs[kGroups / 64] & 1)) occurs |= 1u << 31;
  const uint32_t upto = wave_scan((uint32_t)__popc(occurs));
  const int groups = (int)lane_u32(upto, 63);
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
    if (lane == 0) {
      s.count[n] = all;
      s.mass[n] = m;
      s.ref[n] = ((uint32_t)g << 16) | ref;
    }
  }
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

// What one workgroup counted of a row (at most kSafeSteps steps, so that 16
// bits hold every count): which groups occur, and the words of those that do.
struct Part {
  uint32_t occurs[kGroups / 32];
  uint32_t word[kGroups * 64];
};

__device__ __forceinline__ void count_part(const Row<uint16_t>& row, int part, int parts, uint32_t* bin, Part* out) {
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
__device__ __forceinline__ RowCut merge_row(const Row<uint16_t>& row, Settings f, const Part* in, int parts, CountLds& s) {
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
  make_uniform(f);
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


// ---------------------------------------------------------------------------
// fp32 rows by bins
// ---------------------------------------------------------------------------
constexpr int kBinShift = 19;           // a bin: the tokens of equal leading 13 bits of their order
constexpr int kBins32 = 1 << (32 - kBinShift);
constexpr int kBinGroups = kBins32 / 64;
constexpr int kList = 4096;             // tokens looked at one by one
constexpr int kSubBins = 1024;

// What one workgroup added up of a row: its maximum, and the bins of the
// groups of 64 that occur: tokens above -inf, and their weights as integers of
// 2^-shift, of the bin's largest possible value (of the maximum in its own bin,
// which at a low temperature lies far above what the others weigh).
struct BinPart {
  uint32_t occurs[kBinGroups / 32];
  float top;
  uint32_t nan, pad[2];
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

__device__ __forceinline__ void bin_part(const Row<float>& row, int part, int parts, float T, int shift, BinLds& s, BinPart* out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = part_vecs(row, parts), lo = part * per, hi = min(lo + per, row.vecs);
  for (int i = tid; i < kBins32 / 4; i += kRowThreads) reinterpret_cast<u32x4*>(s.count)[i] = u32x4{0u, 0u, 0u, 0u};
  for (int i = tid; i < kBins32 / 2; i += kRowThreads) reinterpret_cast<u32x4*>(s.mass)[i] = u32x4{0u, 0u, 0u, 0u};
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) s.nan = 0;
  float top = -__builtin_inff();
  bool nan = false;
  if (lo < hi)
    each_vec(row, lo, hi, [&](int, const u32x4& v, bool) {  // (a vector past the end is the last one again)
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
  each_vec(row, lo, hi, [&](int, const u32x4& v, bool in) {
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

struct ListLds {
  uint32_t count[kBins32];     // tokens of a bin; at the end the indices of equal tokens
  double weight[kBins32];      // their weights
  // groups that occur, along the order
  double gweight[kBinGroups], gbefore[kBinGroups];
  uint32_t gcount[kBinGroups], gcbefore[kBinGroups], gid[kBinGroups];
  uint32_t part_occurs[kMaxParts * kBinGroups / 32];
  float part_top[kMaxParts];
  double part_scale[kMaxParts];
  uint64_t list[kList];        // order bits << 32 | index
  uint32_t sub_count[kSubBins];
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

struct Bin {
  uint32_t bin;
  uint32_t before, count;  // tokens
  double mass, weight;     // weights before; of its tokens
};

// The last bin with: tokens before it < goal (kByCount); weights before it <
// goal (kReach) or <= goal (kBeyond), and a weight of its own; a largest
// possible weight >= goal (kAbove).  By every wave alike.
__device__ __forceinline__ Bin seek_bin(int kind, double goal, const ListLds& s, int groups, float top, double inv_t) {
  const int lane = threadIdx.x & 63;
  int n = -1;
#pragma unroll 1
  for (int i = (groups - 1) >> 6; i >= 0 && n < 0; --i) {
    const int mine = min(64 * i + lane, groups - 1);
    bool fits;
    if (kind == kByCount) fits = (double)s.gcbefore[mine] < goal;
    // (a group's first bin may be empty: whether another of it is heavy enough shows below)
    else if (kind == kAbove) fits = weight_of(fminf(bin_edge(64 * s.gid[mine]), top), top, inv_t, s.tab) >= goal;
    else fits = s.gweight[mine] > 0.0 && (kind == kReach ? s.gbefore[mine] < goal : s.gbefore[mine] <= goal);
    const uint64_t yes = __ballot(fits && 64 * i + lane < groups);
    if (yes) n = 64 * i + 63 - __clzll((long long)yes);
  }
  n = max(n, 0);
  Bin at{};
#pragma unroll 1
  for (;; --n) {  // (kAbove: to a group before, where the bins that are heavy enough are empty)
    const uint32_t bin = 64 * s.gid[n] + lane, c = s.count[bin];
    const double w = s.weight[bin];
    const double before = s.gbefore[n] + lane_before(wave_scan(w));
    const uint32_t cbefore = s.gcbefore[n] + wave_scan(c) - c;
    bool fits = c > 0;
    if (kind == kByCount) fits = fits && (double)cbefore < goal;
    else if (kind == kAbove) fits = fits && weight_of(fminf(bin_edge(bin), top), top, inv_t, s.tab) >= goal;
    else fits = fits && w > 0.0 && (kind == kReach ? before < goal : before <= goal);
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

// As seek, among the listed tokens of a bin.  mass, weight: integers of
// 2^-shift of the bin's reference value.
__device__ __forceinline__ Spot seek_list(int kind, double goal, uint32_t bin, float ref, double inv_t, double scale, ListLds& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Spot at{bin << kBinShift, 0u, 0u, 0ull, 0ull};
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
    uint32_t cb = at.before + cu - c;
    uint64_t mb = at.mass + mu - m;
    for (int i = 0; i < wave; ++i) {
      cb += s.red[i];
      mb += s.red2[i];
    }
    bool fits = c > 0;
    if (kind == kByCount) fits = fits && (double)cb < goal;
    else fits = fits && m > 0 && (kind == kReach ? (double)mb < goal : (double)mb <= goal);
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
  }
  at.weight /= max(at.count, 1u);  // (equal values have equal weights)
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
  if (tid < kWords * parts) s.part_occurs[tid] = in[tid / kWords].occurs[tid % kWords];
  if (tid < parts) s.part_top[tid] = in[tid].top;
  if (tid < 256) s.tab[tid] = kExp2Frac256[tid];
  if (tid == 0) s.nan = s.listed = 0;
  __syncthreads();
  if (tid < parts && in[tid].nan) s.nan = 1;
  make_uniform(f);
  float top = -__builtin_inff();
  for (int c = 0; c < parts; ++c) top = fmaxf(top, s.part_top[c]);
  const bool greedy = is_greedy(f.T);
  const double inv_t = greedy ? 1.0 : 1.0 / (double)f.T, scale = (double)(1ull << shift);
  if (tid < parts) s.part_scale[tid] = weight_of(s.part_top[tid], top, inv_t, s.tab) / scale;
  __syncthreads();
  RowCut out{top, top, V - 1, 1, 0, 0, 1.0};
  if (s.nan) {  // uniform
    fits = false;
    return out;
  }
  if (top == -__builtin_inff()) {  // uniform: nothing above it, the first token
    out.last = 0;
    return out;
  }
  // the parts' bins added up: those of a part's maximum by that, the others as integers
  uint32_t occurs = 0;
  if (lane < kWords)
    for (int c = 0; c < parts; ++c) occurs |= s.part_occurs[c * kWords + lane];
  const uint32_t upto = wave_scan((uint32_t)__popc(occurs));
  const int groups = (int)lane_u32(upto, 63);
#pragma unroll 1
  for (int n = wave; n < groups; n += kRowWaves) {
    const int g = nth_group(n, occurs, upto);
    const uint64_t have = __ballot(lane < parts && ((s.part_occurs[min(lane, parts - 1) * kWords + (g >> 5)] >> (g & 31)) & 1));
    const uint32_t bin = 64 * g + lane;
    uint32_t count = 0;
    uint64_t mass = 0;
    double weight = 0.0;
#pragma unroll 1
    for (int c0 = 0; c0 < parts; c0 += 4) {
      uint32_t pc[4];
      unsigned long long pm[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const BinPart& p = in[min(c0 + j, parts - 1)];
        pc[j] = p.count[bin];
        pm[j] = p.mass[bin];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!((have >> (c0 + j)) & 1)) continue;  // uniform (what a part has not is whatever the memory held)
        const uint32_t tb = bin_of(s.part_top[c0 + j]);
        count += pc[j];
        if ((tb >> 6) == (uint32_t)g && bin == tb) weight += (double)pm[j] * s.part_scale[c0 + j];
        else mass += pm[j];
      }
    }
    weight += (double)mass * (weight_of(fminf(bin_edge(bin), top), top, inv_t, s.tab) / scale);
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

  // ranges of bins, from the least and the most that each cut may leave (all waves alike)
  const double tiny = 0x1p-1000, slack = 0x1p-30;  // (the sums' own error is below 2^-40)
  const bool by_count = !greedy && f.k > 0 && f.k < V && (uint32_t)f.k < tokens, reach = !greedy && f.p < 1.f,
             above = !greedy && f.least > 0.f;
  float hi[4], lo[4];
  int ranges = 0;
  auto take = [&](uint32_t first, uint32_t last) {
    const float h = bin_edge(first), l = order_value(((last + 1) << kBinShift) - 1);
    hi[0] = ranges == 0 ? h : hi[0];
    lo[0] = ranges == 0 ? l : lo[0];
    hi[1] = ranges == 1 ? h : hi[1];
    lo[1] = ranges == 1 ? l : lo[1];
    hi[2] = ranges == 2 ? h : hi[2];
    lo[2] = ranges == 2 ? l : lo[2];
    hi[3] = ranges == 3 ? h : hi[3];
    lo[3] = ranges == 3 ? l : lo[3];
    ++ranges;
  };
  double least = total, most = total;
  if (greedy) take(bin_of(top), bin_of(top));
  if (by_count) {
    const Bin at = seek_bin(kByCount, (double)f.k, s, groups, top, inv_t);
    take(at.bin, at.bin);
    least = at.mass;
    most = at.mass + at.weight;
  }
  if (reach) {
    const Bin x = seek_bin(kReach, fmax((double)f.p * least * (1.0 - slack), tiny), s, groups, top, inv_t);
    const Bin y = seek_bin(kReach, fmax((double)f.p * most * (1.0 + slack), tiny), s, groups, top, inv_t);
    take(x.bin, y.bin);
    least = x.mass;
    most = y.mass + y.weight;
  }
  if (above) {
    const Bin at = seek_bin(kAbove, fmin((double)f.least, 1.0), s, groups, top, inv_t);
    take(at.bin, at.bin);
    least = fmin(least, at.mass);
    most = fmin(most, at.mass + at.weight);
  }
  if (f.sampled && !greedy) {
    const Bin x = seek_bin(kBeyond, unit(f.u) * least * (1.0 - slack), s, groups, top, inv_t);
    const Bin y = seek_bin(kBeyond, unit(f.u) * most * (1.0 + slack), s, groups, top, inv_t);
    take(x.bin, y.bin);
  }
  // (bin_edge of the bins of infinity and of NaN is a NaN)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i >= ranges) hi[i] = lo[i] = __builtin_nanf("");
    else if (hi[i] != hi[i]) hi[i] = __builtin_inff();
  }
  if (ranges) each_vec(row, 0, row.vecs, [&](int it, const u32x4& v, bool here) {
    if (!here) return;
    const int64_t e0 = (int64_t)4 * (it * kRowThreads + tid) - row.skew;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(v[e]);
      bool is = x <= hi[0] && x >= lo[0];
      if (ranges > 1) is = is || (x <= hi[1] && x >= lo[1]);
      if (ranges > 2) is = is || (x <= hi[2] && x >= lo[2]);
      if (ranges > 3) is = is || (x <= hi[3] && x >= lo[3]);
      if (!is || x == -__builtin_inff()) continue;
      const int at = atomicAdd(&s.listed, 1);
      if (at < kList) s.list[at] = ((uint64_t)order_bits(x) << 32) | (uint32_t)(e0 + e);
    }
  });
  __syncthreads();
  if (s.listed > kList) {  // uniform
    fits = false;
    return out;
  }
  // the cuts, one after another, among the listed tokens
  uint32_t cut_key = order_bits(top), token_key = cut_key, token_rank = 0;
  int cut_rank = -1;
  bool cuts = false;  // cut_key is a value that stays in part at least
  double W = greedy ? 1.0 : total;
  int kept = greedy ? 1 : V;
  if (greedy) cuts = true;
  if (!greedy && f.k > 0 && f.k < V) kept = f.k;
  out.cut = greedy ? top : -__builtin_inff();
  auto ref_of = [&](uint32_t bin) { return fminf(bin_edge(bin), top); };
  if (by_count) {
    const Bin at = seek_bin(kByCount, (double)f.k, s, groups, top, inv_t);
    const Spot x = seek_list(kByCount, (double)((uint32_t)f.k - at.before), at.bin, ref_of(at.bin), inv_t, scale, s);
    const uint32_t n = (uint32_t)f.k - at.before - x.before;
    W = at.mass + (double)(x.mass + n * x.weight) * (weight_of(ref_of(at.bin), top, inv_t, s.tab) / scale);
    cut_key = x.key;
    cut_rank = n < x.count ? (int)n - 1 : -1;
    cuts = true;
  }
  if (reach) {
    const double goal = fmax((double)f.p * W, tiny);
    const Bin at = seek_bin(kReach, goal, s, groups, top, inv_t);
    const double unit_w = weight_of(ref_of(at.bin), top, inv_t, s.tab) / scale;
    const double inside = fmax((goal - at.mass) / unit_w, 0.5);
    const Spot x = seek_list(kReach, inside, at.bin, ref_of(at.bin), inv_t, scale, s);
    const double need = ceil((inside - (double)x.mass) / (double)x.weight);
    const uint32_t n = (uint32_t)fmin(fmax(need, 1.0), (double)x.count);
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
    const Bin at = seek_bin(kAbove, goal, s, groups, top, inv_t);
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
      W = at.mass + (double)s.hit_mass * (weight_of(ref, top, inv_t, s.tab) / scale);
      // (none: what lies before the bin, whose largest possible value none of its tokens has)
      cut_key = n ? s.hit_before : at.bin << kBinShift;
      cut_rank = -1;
      cuts = true;
    }
  }
  if (f.sampled && kept > 1) {
    const double goal = unit(f.u) * W;
    const Bin at = seek_bin(kBeyond, goal, s, groups, top, inv_t);
    const double unit_w = weight_of(ref_of(at.bin), top, inv_t, s.tab) / scale;
    const double inside = fmax((goal - at.mass) / unit_w, 0.0);
    const Spot x = seek_list(kBeyond, inside, at.bin, ref_of(at.bin), inv_t, scale, s);
    const double j = fmin(floor((inside - (double)x.mass) / (double)x.weight),
                          (double)min((int)x.count, kept - (int)(at.before + x.before)) - 1.0);
    token_key = x.key;
    token_rank = (uint32_t)fmax(j, 0.0);
  }
  out.kept = kept;
  out.total = W;
  if (cuts) out.cut = order_value(cut_key);
  if (kept == 1 || f.sampled) out.token = index_in_list(token_key, token_rank, s);
  if (kept == 1 && s.equals == 0) {  // uniform: alone because of a bin behind its own, which was not listed
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

// What a launch's n-th row is.
template <typename T>
struct Work {
  int r, b;
  Job j;
  const T* row;
  __device__ Work(const FilterArgs& a, int n) {
    b = (a.row0 + n) / a.rows;
    r = a.row0 + n - b * a.rows;
    j = job_of(a, r, b);
    row = (const T*)(j.is_draft ? a.draft : a.target) + j.at;
  }
};

// grid (parts, rows)
__global__ __launch_bounds__(kRowThreads) void filter_count_kernel(FilterArgs a) {
  __shared__ uint32_t bin[32768];
  const Work<uint16_t> w(a, blockIdx.y);
  if (!w.j.active) return;  // uniform
  count_part(Row<uint16_t>(w.row, a.V), blockIdx.x, a.split, bin, (Part*)a.row_parts + (int64_t)blockIdx.y * a.split + blockIdx.x);
}
__global__ __launch_bounds__(kRowThreads) void filter_bin_kernel(FilterArgs a) {
  __shared__ BinLds s;
  const Work<float> w(a, blockIdx.y);
  if (!w.j.active) return;  // uniform
  bin_part(Row<float>(w.row, a.V), blockIdx.x, a.split, a.temperature[w.b], a.shift, s,
           (BinPart*)a.row_parts + (int64_t)blockIdx.y * a.split + blockIdx.x);
}
// grid rows
__global__ __launch_bounds__(kRowThreads) void filter_merge_kernel(FilterArgs a) {
  __shared__ CountLds s;
  const Work<uint16_t> w(a, blockIdx.x);
  if (!w.j.active) return;  // uniform
  const Part* in = (const Part*)a.row_parts + (int64_t)blockIdx.x * a.split;
  put_row(a, w.r, w.b, w.j, w.row,
          merge_row(Row<uint16_t>(w.row, a.V), settings_of(a, w.b, w.j.sampled, w.j.u, w.j.ends), in, a.split, s));
}
__global__ __launch_bounds__(kRowThreads) void filter_list_kernel(FilterArgs a) {
  __shared__ RowLds32 s;
  const Work<float> w(a, blockIdx.x);
  if (!w.j.active) return;  // uniform
  const BinPart* in = (const BinPart*)a.row_parts + (int64_t)blockIdx.x * a.split;
  bool fits;
  RowCut c = list_row(Row<float>(w.row, a.V), settings_of(a, w.b, w.j.sampled, w.j.u, w.j.ends), in, a.split, a.shift, s.bins, fits);
  if (!fits) {  // uniform
    __syncthreads();
    c = filter_row<float>(a, w.b, w.row, w.j.sampled, a.uniforms[w.j.u], w.j.ends, s.radix);
  }
  put_row(a, w.r, w.b, w.j, w.row, c);
}

// Parts of a row, a workgroup each: more where the rows alone leave compute
// units idle, as long as each takes a step of a workgroup, and in bf16 so many
// that 16 bits hold a part's counts.
int row_split(int rows, int V, int dtype) {
  const int step = dtype == NSV_BF16 ? kStep : kStep / 2;
  int n = kMaxSplit;
  while (n > 1 && (rows * n > 256 || V < n * step)) n >>= 1;
  const int least = dtype == NSV_BF16 ? (V + 7 + kSafeSteps * kStep - 1) / (kSafeSteps * kStep) : 1;
  return n < least ? least : n;
}
size_t part_bytes(int dtype) { return dtype == NSV_BF16 ? sizeof(Part) : sizeof(BinPart); }
static_assert(sizeof(Part) % 16 == 0 && sizeof(BinPart) % 16 == 0 && (kMaxVocab + 7) / (kSafeSteps * kStep) < kMaxParts, "parts");

}  // namespace

namespace nsv_filter {

size_t rows_bytes(int rows, int V, int dtype) {
  if (rows <= 0) return 0;
  const int n = row_split(rows, V, dtype), most = kSlab / n;
  return (size_t)(rows < most ? rows : most) * n * part_bytes(dtype);
}

int launch_rows(FilterArgs& a, int dtype, void* workspace, hipStream_t s) {
  const int total = a.rows * a.B;
  a.split = row_split(total, a.V, dtype);
  a.row_parts = workspace;
  const int most = kSlab / a.split;
  for (a.row0 = 0; a.row0 < total; a.row0 += most) {
    const int rows = total - a.row0 < most ? total - a.row0 : most;
    const dim3 parts(a.split, rows), block(kRowThreads);
    if (dtype == NSV_BF16) hipLaunchKernelGGL(filter_count_kernel, parts, block, 0, s, a);
    else hipLaunchKernelGGL(filter_bin_kernel, parts, block, 0, s, a);
    int rc = nsv_launch_status();
    if (rc) return rc;
    if (dtype == NSV_BF16) hipLaunchKernelGGL(filter_merge_kernel, dim3(rows), block, 0, s, a);
    else hipLaunchKernelGGL(filter_list_kernel, dim3(rows), block, 0, s, a);
    if ((rc = nsv_launch_status())) return rc;
  }
  return NSV_OK;
}

}  // namespace nsv_filter
