// What the kernels of filtered sampling and acceptance share (filter_rows.hip,
// filter_accept.hip).
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
#pragma once

#include "common.h"
#include "exp_f64.h"

namespace nsv_filter {

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kVec = 8;                          // elements a thread takes at a time
constexpr int kStep = kRowThreads * kVec;        // elements a workgroup takes at a time
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxDrafts = 63;                   // K + 1 rows fit one 64-lane ballot

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
  int rows;                // per sequence: target rows, then draft rows
  int row0;                // a launch's first row, of all B * rows
  void* row_parts;         // [rows of a launch, split]
  int split, steps, share; // parts of a row, workgroup steps of a part, parts of a workgroup
  double* parts;           // [B, chunks, 2]: sums of the residual and of p_target
  int chunks;
  int32_t* tokens;         // sampler: row b's at b * out_stride
  int64_t out_stride;
  int32_t* kept;           // sampler, nullable
  int32_t* out_tokens;     // [B, K + 1]
  int32_t* out_len;
};

__device__ __forceinline__ bool is_greedy(float T) { return !(T > 1e-6f); }
// u of the sample's goal u W: what is no number in [0, 1] is taken to its end (1,
// which no running sum exceeds: the last token kept that has a weight)
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

// lane l's value (l uniform), and the lane's before a lane's own
__device__ __forceinline__ double lane_f64(double v, int l) {
  return __longlong_as_double((long long)lane_u64((uint64_t)__double_as_longlong(v), l));
}
template <typename T>
__device__ __forceinline__ T lane_before(T v) {
  return dpp_or_zero<0x138, 0xf>(v);  // the whole wave one lane up, 0 into the first
}

// probability of token i of logit x
__device__ __forceinline__ double prob_of(const RowCut& c, float x, int i, double inv_t, const double* tab) {
  if (c.kept == 1) return i == c.token ? 1.0 : 0.0;
  const bool in = x > c.cut || (x == c.cut && i <= c.last);
  return in ? weight_of(x, c.top, inv_t, tab) / c.total : 0.0;
}

// filter_rows.hip: the rows of every sequence (a.rows each) worked out, into
// a.tokens or a.cuts and a.probs, and the workspace that takes (16 bytes).
size_t rows_bytes(int rows, int V, int dtype);
int launch_rows(FilterArgs& a, int dtype, void* workspace, hipStream_t s);

inline size_t a256(size_t x) { return (x + 255) & ~(size_t)255; }
inline bool off_by(const void* at, int bytes) { return ((uintptr_t)at & (bytes - 1)) != 0; }
inline int elem_bytes(int dtype) { return dtype == NSV_BF16 ? 2 : 4; }
inline bool bad_rows(int B, int V, int dtype) { return B < 0 || V <= 0 || (dtype != NSV_F32 && dtype != NSV_BF16); }
// weights as integers: V of them, each at most 2^shift, stay below 2^62
inline int weight_shift(int V) {
  int bits = 0;
  while ((1 << bits) < V) ++bits;
  const int s = 62 - bits;
  return s > 50 ? 50 : s;
}

}  // namespace nsv_filter
