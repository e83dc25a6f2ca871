// Acceptance of drafts under the filters of filter.h, and the C entries of
// both operators.  No reference counterpart (its acceptance has a temperature
// only); the operators stand beside nsv_sample and nsv_accept_stochastic.
//
// A sequence with draft rows keeps draft d if u p_draft(d) < p_target(d), which
// the row kernels leave for every draft; at the first that it does not, a
// kernel adds up max(p_target - p_draft, 0) over that row, a workgroup per
// chunk, and the last one finds the chunk, then the index, that u' of the sum
// falls into.  Few tokens pass the filters as a rule, and only of those is an
// exponential taken.  Sums are 64-bit floating point in a fixed order.

#include "filter.h"

using namespace nsv_filter;

namespace {

constexpr int kChunkThreads = 256;
constexpr int kChunk = kChunkThreads * kVec;     // of the residual passes
constexpr int kMaxChunks = kMaxVocab / kChunk;

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

// grid (chunks, B): chunk sums of the refused row's residuals.  8 sequences of
// 151,936 (4.9 MB of target and draft rows) 5.2 us, 3 of 50,001 fp32 5.5: three
// dependent loads (counts, cuts, rows) and a sum; 2,048 tokens a workgroup so that
// one sequence still spreads over 75.
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

// grid B: the sequence's tokens.  6.3 us with draft rows (the chunk found by one
// wave, then its 2,048 residuals once more), 4.0 without: a chain of loads.
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void filter_finish_kernel(FilterArgs a) {
  __shared__ double tab[256], parts[2 * kMaxChunks], red[kChunkThreads / 64], goal_s, before_s;
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
  // (on their way beside what says whether they are needed; a refused draft's
  // chunks are there, else they are whatever the memory held)
  for (int i = tid; i < 2 * a.chunks; i += kChunkThreads) parts[i] = a.parts[(int64_t)b * a.chunks * 2 + i];
  const int n = accepted_by_rows(a, b, kb);
  if (wave == 0 && lane < n) out[lane] = d;
  if (tid == 0) a.out_len[b] = n + 1;
  if (n == kb) {  // uniform: the bonus token
    if (tid == 0) out[n] = cuts[n].token;
    return;
  }
  tab[tid] = kExp2Frac256[tid];
  __syncthreads();
  // the chunk that holds the token: the last with any weight whose sums before it do not exceed the goal
  if (wave == 0) {
    double sl = 0.0;
    for (int c = lane; c < a.chunks; c += 64) sl += parts[2 * c];
    const int col = wave_sum_dpp(sl) > 0.0 ? 0 : 1;  // no residual: the target row itself
    double total = 0.0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
      const double v = wave_scan(c0 + lane < a.chunks ? parts[2 * (c0 + lane) + col] : 0.0);
      total += lane_f64(v, 63);
    }
    const double goal = unit(a.uniforms[(int64_t)b * (K + 1) + K]) * total;
    double run = 0.0, before = 0.0;
    int at = 0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
      const double mine = c0 + lane < a.chunks ? parts[2 * (c0 + lane) + col] : 0.0;
      const double v = wave_scan(mine);
      const double prev = lane_before(v);
      const uint64_t yes = __ballot(mine > 0.0 && run + prev <= goal);
      if (yes) {
        const int l = 63 - __clzll((long long)yes);
        at = c0 + l;
        before = run + lane_f64(prev, l);
      }
      run += lane_f64(v, 63);
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
  double run = lane_before(v);
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

int residual_chunks(int V) { return (V + kChunk - 1) / kChunk; }

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
  L.total = L.row_parts + rows_bytes(B * (draft_rows ? 2 * K + 1 : K + 1), V, dtype);
  return L;
}

}  // namespace

extern "C" {

size_t nsv_sample_filtered_workspace_size(int B, int V, int dtype) {
  if (bad_rows(B, V, dtype) || V > kMaxVocab || B > 65535) return 0;
  return rows_bytes(B, V, dtype);
}

int nsv_sample_filtered(const void* logits, int64_t row_stride, const float* temperature, const int32_t* top_k,
                        const float* top_p, const float* min_p, const float* uniforms, int B, int V, int dtype,
                        int32_t* out_tokens, int64_t out_stride, int32_t* kept, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (bad_rows(B, V, dtype) || row_stride < V || out_stride < 1) return NSV_ERR_ARG;
  if (V > kMaxVocab || B > 65535) return NSV_ERR_UNSUPPORTED;
  if (B == 0) return NSV_OK;
  if (!logits || !temperature || !uniforms || !out_tokens || off_by(logits, elem_bytes(dtype))) return NSV_ERR_ARG;
  const size_t need = rows_bytes(B, V, dtype);
  if (!workspace || off_by(workspace, 16) || workspace_bytes < need) return NSV_ERR_WORKSPACE;
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
  a.rows = 1;
  return launch_rows(a, dtype, workspace, (hipStream_t)stream);
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
  if (!target_logits || (!drafts && K > 0) || !num_drafts || !temperature || !uniforms || !out_tokens || !out_len ||
      off_by(target_logits, elem_bytes(dtype)) || off_by(draft_logits, elem_bytes(dtype)))
    return NSV_ERR_ARG;
  const Layout L = layout(B, K, V, dtype, K > 0 && draft_logits);
  if (!workspace || off_by(workspace, 16) || workspace_bytes < nsv_accept_filtered_workspace_size(B, K, V, dtype))
    return NSV_ERR_WORKSPACE;
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
  a.rows = a.draft ? 2 * K + 1 : K + 1;
  int rc = launch_rows(a, dtype, (char*)workspace + L.row_parts, s);
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
