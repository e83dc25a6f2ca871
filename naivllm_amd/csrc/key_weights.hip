// Attention weights of a prompt's rows, summed per key, for gfx950 (bf16):
//
//   weight of (kv head, key j) = sum_(rows r at or behind j) sum_(heads of the
//   group) 2^(s_rj - m_r) / l_r,   s_rj = scale log2(e) q_r . k_j
//
// with the statistics (m_r, 1 / l_r) that nsv_prefill_window_attention leaves.
//
// What bounds it: one matrix product of 2 D flops per (row, key) pair, an
// exponential (quarter rate) and two fused multiply-adds, at the diagonal a
// select: at 8,192 rows the vector units are busy for 57% of the SIMDs' cycles
// and the matrix cores for 37%, and the two overlap little.  The keys stay, the
// rows stream: a wave holds 64 keys in registers as the A operand of S^T = K Q^T
// (v_mfma_f32_32x32x16_bf16), so a lane's 32 scores of a 32-row tile are added
// into 32 registers of its own and the sum over the lanes is taken once, at the
// end.  A workgroup's four waves
// (256 keys) read the row tiles from one LDS copy, loaded straight from memory
// three deep.  The (head, row tile) list of a key block is cut into parts so
// that the grid fills the chip; a second kernel adds the parts in their order
// (no atomics between them: the sums do not depend on which part ends first).
//
// Measured on MI355X: 8,192 rows of 32/8 heads 316 us at 2.0 GHz (870 TFLOP/s of
// the one product; without the sums 163, without the products 267, where the
// vector operations' issue alone takes about 200: the rest is the operands' reads
// and the waits for tiles), 1,206 rows of 16/8 heads 13.6 + 3.8.  Not better:
// both squares of 32 keys multiplied in turn (spills), 32 rows' operands read a
// half ahead, units ordered by their rows for the L2, one workgroup per compute
// unit (522).

#include "common.h"

#include <algorithm>
#include <array>
#include <new>
#include <type_traits>
#include <vector>

namespace {

constexpr int kBlockKeys = 256;   // keys per workgroup: 64 per wave
constexpr int kRows = 64;         // rows per tile
constexpr int kUnitWords = 8;     // int32 words of a unit record
constexpr int kSumWords = 6;      // and of a sum record
constexpr int kStages = 3;        // row tiles in LDS
// rounds of the chip that the parts make: 8,192 rows of 32/8 heads 392 us with one,
// 325 with two, 320 with four (1,206 rows of 16/8: no difference)
constexpr int64_t kRounds = 4;

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct KeyWeightsArgs {
  const bf16_t* q;
  const bf16_t* k;
  const float2* stats;          // [rows][H]
  const int32_t* block_tables;
  const int32_t* units;         // [n][kUnitWords]: sequence, first key, keys, row of q of the sequence's first, rows,
                                // position of that row, first (head, row tile), end
  float* part;                  // [units][Hkv][kBlockKeys]
  float* key_weights;           // [num_blocks][Hkv][block_size]
  float scale_log2;
  int H, Hkv, bs_log2, max_blocks;
};

__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

template <int DH>
__global__ __launch_bounds__(256, 2) void key_weights_kernel(KeyWeightsArgs a) {
  constexpr int CPR = DH / 8, ROWB = DH * 2, KS = DH / 16;
  constexpr int RPI = 64 / CPR;
  constexpr int J = kRows / RPI / 4;       // row loads per wave and tile
  struct __attribute__((aligned(16))) Lds {
    unsigned char q[kStages][kRows * ROWB];
    float stat[kStages][2][kRows];         // maximum, 1 / sum
  };
  __shared__ Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, h = lane >> 5;
  const int hk = blockIdx.x % a.Hkv, unit = blockIdx.x / a.Hkv;
  const int32_t* rec = a.units + (int64_t)unit * kUnitWords;
  const int seq = rec[0], key0 = rec[1], nkeys = rec[2], row0 = rec[3], nrows = rec[4], pos0 = rec[5];
  const int t_begin = rec[6], t_end = rec[7];
  const int G = a.H / a.Hkv;
  const int first = max(0, key0 - pos0);              // the first row that sees a key of the block
  const int tiles = (nrows - first + kRows - 1) / kRows;  // per head

  // the step's own keys start from zero, to which key_sum_kernel adds: another
  // sequence may have the same page behind it (a prefix that one sequence of the
  // step computes and the next shares)
  if (t_begin == 0 && tid < nkeys && key0 + tid >= pos0) {  // (one unit per block of keys begins at 0)
    const int key = key0 + tid, entry = key >> a.bs_log2;
    const int p = entry < a.max_blocks ? a.block_tables[(int64_t)seq * a.max_blocks + entry] : -1;
    if (p >= 0) a.key_weights[(((int64_t)p * a.Hkv + hk) << a.bs_log2) + (key & ((1 << a.bs_log2) - 1))] = 0.f;
  }

  // the keys: lane (h, col) holds key 32 t + col, dims 16 ks + 8 h ..; a key that is not there reads the block's last
  const int wkey = key0 + w * 64;
  u32x4 ka[2][KS];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int key = min(wkey + t * 32 + col, key0 + nkeys - 1);
    const int entry = min(key >> a.bs_log2, a.max_blocks - 1);  // (keys past the table do not exist: nothing is written)
    const int p = max(a.block_tables[(int64_t)seq * a.max_blocks + entry], 0);
    const bf16_t* src = a.k + ((((int64_t)p << a.bs_log2) + (key & ((1 << a.bs_log2) - 1))) * a.Hkv + hk) * DH + h * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[t][ks] = *reinterpret_cast<const u32x4*>(src + ks * 16);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) __asm__ volatile("" ::"v"(ka[t][ks]));

  auto lds_at = [](const void* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
  };
  // Row tiles straight to LDS (16-byte chunk X of row r at slot X ^ r, for the
  // banks of the operand reads); rows past the last read it again, and count
  // nothing.
  auto issue = [&](int buf, int t) {
    const int g = t / tiles, r0 = first + (t - g * tiles) * kRows;
    const int head = hk * G + g;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int rr = (w * J + j) * RPI, r = rr + lane / CPR, slot = lane % CPR;
      const bf16_t* src = a.q + ((int64_t)(row0 + min(r0 + r, nrows - 1)) * a.H + head) * DH + ((slot ^ (r & (CPR - 1))) << 3);
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_at(&lds.q[buf][rr * ROWB])), "v"(src)
                       : "memory", "m0");
    }
    // (every wave loads the tile's statistics, so that each waits for as many loads)
    const float* st = (const float*)(a.stats + (int64_t)(row0 + min(r0 + lane, nrows - 1)) * a.H + head);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_at(&lds.stat[buf][e][0])), "v"(st + e)
                       : "memory", "m0");
  };

  f32x16 sum[2], s[2];  // s[t]: scores of a half of 32 rows and of the wave's keys 32 t ..
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) sum[t][i] = 0.f;

  // 32 rows and 32 keys at a time: while the products of one such square are
  // made, the exponentials of the one before it are (a quarter-rate operation
  // each, so together longer than the products: what the loop is bound by).
  u32x4 qb[KS];
  auto read = [&](int buf, int half) {
    const int r = half * 32 + col;
    const unsigned char* src = lds.q[buf] + r * ROWB;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qb[ks] = *reinterpret_cast<const u32x4*>(src + (((ks * 2 + h) ^ (r & (CPR - 1))) << 4));
  };
  struct Rows {   // this lane's row of a half
    float nb, inv;
    int pos;
    bool full;    // uniform: every row sees every key of the wave
  };
  auto row_of = [&](int buf, int half, int r0) {
    const int r = half * 32 + col;
    Rows x;
    x.inv = r0 + r < nrows ? lds.stat[buf][1][r] : 0.f;
    x.nb = x.inv == 0.f ? -__builtin_inff() : -lds.stat[buf][0][r];  // (a row that sees nothing: weights 0)
    x.pos = pos0 + r0 + r;
    x.full = pos0 + r0 + half * 32 >= wkey + 63;
    return x;
  };
  auto weight = [&](float score, const Rows& x, float before) {
    return fmaf(__builtin_amdgcn_exp2f(fmaf(score, a.scale_log2, x.nb)), x.inv, before);
  };
  auto add_masked = [&](int t, const Rows& x) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int key = wkey + t * 32 + (i >> 2) * 8 + h * 4 + (i & 3);
      const float y = weight(s[t][i], x, sum[t][i]);
      sum[t][i] = key <= x.pos ? y : sum[t][i];
    }
  };
  // the products of square t, and meanwhile square 1 - t (of rows x) added
  auto square = [&](auto slot, const Rows& x) {
    constexpr int t = decltype(slot)::value;
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // (in three stages, so that nothing waits for the operation before it: an
    // element's argument, its exponential and its addition fall beside three
    // products in turn)
    constexpr int PER = 16 / KS;
    auto argument = [&](int i) { s[1 - t][i] = fmaf(s[1 - t][i], a.scale_log2, x.nb); };
#pragma unroll
    for (int i = 0; i < 2 * PER; ++i) argument(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(ka[t][ks]), as_bf16x8(qb[ks]), ks == 0 ? zero : s[t], 0, 0, 0);
#pragma unroll
      for (int i = ks * PER; i < (ks + 1) * PER; ++i) {
        s[1 - t][i] = __builtin_amdgcn_exp2f(s[1 - t][i]);
        if (i + 2 * PER < 16) argument(i + 2 * PER);
        if (i >= PER) sum[1 - t][i - PER] = fmaf(s[1 - t][i - PER], x.inv, sum[1 - t][i - PER]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 16 - PER; i < 16; ++i) sum[1 - t][i] = fmaf(s[1 - t][i], x.inv, sum[1 - t][i]);
  };
  auto multiply = [&](int t) {
    const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(ka[t][ks]), as_bf16x8(qb[ks]), ks == 0 ? zero : s[t], 0, 0, 0);
  };
  bool open = false;  // uniform: square 1 of the half before is multiplied and not yet added
  Rows last;
  auto step = [&](int buf, int half, int r0) {
    read(buf, half);
    const Rows x = row_of(buf, half, r0);
    if (open && last.full) {  // uniform
      square(std::integral_constant<int, 0>{}, last);
    } else {
      if (open) add_masked(1, last);
      multiply(0);
    }
    if (x.full) {  // uniform
      square(std::integral_constant<int, 1>{}, x);
    } else {
      multiply(1);
      add_masked(0, x);
    }
    last = x;
    open = true;
  };

  if (t_begin < t_end) issue(0, t_begin);
  if (t_begin + 1 < t_end) issue(1, t_begin + 1);
  int buf = 0;
  for (int tt = t_begin; tt < t_end; ++tt) {
    // the tile landed, one after it still in flight; behind the barrier it is
    // whole, and the buffer of the tile before it is free
    if (tt + 1 < t_end) __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(J + 2) : "memory");
    else __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (tt + 2 < t_end) issue(buf + 2 >= kStages ? buf + 2 - kStages : buf + 2, tt + 2);
    const int g = tt / tiles, r0 = first + (tt - g * tiles) * kRows;
    if (pos0 + r0 + kRows - 1 >= wkey) {  // uniform: some row sees one of this wave's keys
      step(buf, 0, r0);
      step(buf, 1, r0);
    }
    buf = buf + 1 == kStages ? 0 : buf + 1;
  }
  if (open) add_masked(1, last);

  // over the 32 rows of a half-wave, in a fixed order; lane col 0 of each half holds the keys' sums
  float* dst = a.part + ((int64_t)unit * a.Hkv + hk) * kBlockKeys + w * 64;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = sum[t][i];
      v += dpp_f32<kDppXor1>(v);
      v += dpp_f32<kDppXor2>(v);
      v += dpp_f32<kDppHalfMirror>(v);
      v += dpp_f32<kDppMirror>(v);
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
      sum[t][i] = v;
    }
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    float v = sum[t][0];
#pragma unroll
    for (int i = 1; i < 16; ++i) v = (col & 15) == i ? sum[t][i] : v;
    if (col < 16) dst[t * 32 + (col >> 2) * 8 + h * 4 + (col & 3)] = v;
  }
}

// The parts of a key block added in order, and that to the paged table, where
// the keys of the step itself (those at or behind its first row) are zero by
// now.  One workgroup per (block, kv head).
struct KeySumArgs {
  const float* part;
  const int32_t* sums;  // [n][kSumWords]: sequence, first key, keys, first unit, units, position of the first row
  const int32_t* block_tables;
  float* key_weights;   // [num_blocks][Hkv][block_size]
  int Hkv, bs_log2, max_blocks;
};

__global__ __launch_bounds__(kBlockKeys) void key_sum_kernel(KeySumArgs a) {
  const int32_t* rec = a.sums + (int64_t)blockIdx.x * kSumWords;
  const int seq = rec[0], key0 = rec[1], nkeys = rec[2], unit = rec[3], units = rec[4];
  const int hk = blockIdx.y, key = key0 + threadIdx.x;
  if ((int)threadIdx.x >= nkeys || (key >> a.bs_log2) >= a.max_blocks) return;
  const int p = a.block_tables[(int64_t)seq * a.max_blocks + (key >> a.bs_log2)];
  const float* src = a.part + ((int64_t)unit * a.Hkv + hk) * kBlockKeys + threadIdx.x;
  float y = 0.f;
#pragma unroll 8
  for (int u = 0; u < units; ++u) y += src[(int64_t)u * a.Hkv * kBlockKeys];
  if (p < 0) return;
  // (an atomic add: sequences may share a page)
  unsafeAtomicAdd(a.key_weights + (((int64_t)p * a.Hkv + hk) << a.bs_log2) + (key & ((1 << a.bs_log2) - 1)), y);
}

struct KeyTiling {
  std::vector<std::array<int32_t, kUnitWords>> units;
  std::vector<std::array<int32_t, kSumWords>> sums;
};

KeyTiling make_key_units(const int64_t* ql, const int64_t* kl, int n, int H, int Hkv, int cus) {
  const int64_t G = H / Hkv;
  auto tiles_of = [&](int b, int64_t key0) {
    const int64_t first = std::max<int64_t>(0, key0 - (kl[b] - ql[b]));
    return G * ((ql[b] - first + kRows - 1) / kRows);
  };
  // tiles per part: the fewest (at least two) with which the workgroups, of
  // which two fit a compute unit, make at most kRounds full rounds of the chip (a
  // round of a few of them more would take as long as a full one)
  auto units_of = [&](int64_t target) {
    int64_t units = 0;
    for (int b = 0; b < n; ++b)
      for (int64_t k = 0; k < kl[b]; k += kBlockKeys) units += (tiles_of(b, k) + target - 1) / target;
    return units * Hkv;
  };
  int64_t target = 2, above = 2;  // (above: a block's most tiles, a part per block)
  for (int b = 0; b < n; ++b) above = std::max(above, tiles_of(b, 0));
  while (target < above) {
    const int64_t mid = (target + above) / 2;
    if (units_of(mid) > kRounds * 2 * (int64_t)cus) target = mid + 1;
    else above = mid;
  }
  KeyTiling t;
  int64_t row0 = 0;
  for (int b = 0; b < n; ++b) {
    const int64_t pos0 = kl[b] - ql[b];
    for (int64_t k = 0; k < kl[b]; k += kBlockKeys) {
      const int64_t keys = std::min<int64_t>(kBlockKeys, kl[b] - k), nt = tiles_of(b, k);
      const int64_t parts = std::max<int64_t>(1, (nt + target - 1) / target), per = (nt + parts - 1) / parts;
      const int64_t unit = (int64_t)t.units.size();
      for (int64_t i = 0; i < nt; i += per)
        t.units.push_back({b, (int32_t)k, (int32_t)keys, (int32_t)row0, (int32_t)ql[b], (int32_t)pos0, (int32_t)i,
                           (int32_t)std::min(nt, i + per)});
      t.sums.push_back({b, (int32_t)k, (int32_t)keys, (int32_t)unit, (int32_t)(t.units.size() - unit), (int32_t)pos0});
    }
    row0 += ql[b];
  }
  return t;
}

}  // namespace

extern "C" {

int nsv_key_weights_units(const int64_t* seqlens_q, const int64_t* seqlens_k, int n, int H, int Hkv, int cus,
                          int32_t* out, int64_t capacity, int32_t* counts) {
  if (n < 0 || H <= 0 || Hkv <= 0 || H % Hkv || cus <= 0 || capacity < 0 || !counts) return NSV_ERR_ARG;
  if (n > 0 && (!seqlens_q || !seqlens_k || !out)) return NSV_ERR_ARG;
  int64_t rows = 0;
  for (int b = 0; b < n; ++b) {
    if (seqlens_q[b] <= 0 || seqlens_q[b] > seqlens_k[b] || seqlens_k[b] > ((int64_t)1 << 30)) return NSV_ERR_ARG;
    rows += seqlens_q[b];
  }
  if (rows > 0x7fffffff) return NSV_ERR_UNSUPPORTED;
  try {
    const KeyTiling t = make_key_units(seqlens_q, seqlens_k, n, H, Hkv, cus);
    counts[0] = (int32_t)t.units.size();
    counts[1] = (int32_t)t.sums.size();
    if ((int64_t)t.units.size() * kUnitWords + (int64_t)t.sums.size() * kSumWords > capacity) return NSV_ERR_WORKSPACE;
    for (const auto& x : t.units) out = std::copy(x.begin(), x.end(), out);
    for (const auto& x : t.sums) out = std::copy(x.begin(), x.end(), out);
  } catch (const std::bad_alloc&) {
    return NSV_ERR_WORKSPACE;
  }
  return NSV_OK;
}

int nsv_prefill_key_weights(const void* q, const void* k_cache, float* key_weights, const float* stats,
                            const int32_t* block_tables, const int32_t* units, int nunits, const int32_t* sums, int nsums,
                            float scale, int H, int Hkv, int D, int block_size, int max_blocks, void* partials,
                            void* stream) {
  if (nunits < 0 || nsums < 0 || H <= 0 || Hkv <= 0 || max_blocks <= 0) return NSV_ERR_ARG;
  if (H % Hkv || (D != 64 && D != 128) || block_size <= 0 || (block_size & (block_size - 1))) return NSV_ERR_UNSUPPORTED;
  if ((int64_t)max_blocks * block_size > ((int64_t)1 << 30) || (int64_t)nunits * Hkv > 0x7fffffff || Hkv > 65535)
    return NSV_ERR_UNSUPPORTED;
  if (nunits == 0 || nsums == 0) return NSV_OK;
  if (!q || !k_cache || !key_weights || !stats || !block_tables || !units || !sums) return NSV_ERR_ARG;
  if (((uintptr_t)q | (uintptr_t)k_cache) % 16) return NSV_ERR_ARG;
  if (!partials) return NSV_ERR_WORKSPACE;
  int bs_log2 = 0;
  while ((1 << bs_log2) < block_size) ++bs_log2;
  KeyWeightsArgs a{(const bf16_t*)q, (const bf16_t*)k_cache, (const float2*)stats, block_tables, units, (float*)partials,
                   key_weights, scale * 1.44269504088896340736f, H, Hkv, bs_log2, max_blocks};
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)((int64_t)nunits * Hkv));
  if (D == 128) hipLaunchKernelGGL(key_weights_kernel<128>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(key_weights_kernel<64>, grid, dim3(256), 0, s, a);
  const int rc = nsv_launch_status();
  if (rc) return rc;
  KeySumArgs m{(const float*)partials, sums, block_tables, key_weights, Hkv, bs_log2, max_blocks};
  hipLaunchKernelGGL(key_sum_kernel, dim3(nsums, Hkv), dim3(kBlockKeys), 0, s, m);
  return nsv_launch_status();
}

}  // extern "C"
