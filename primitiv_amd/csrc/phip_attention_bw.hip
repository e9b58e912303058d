// Gradients of attention.  With P = exp(scale q k^T - stats) (stats: the log of the sum of exponentials that the forward
// call left), dP = gy v^T, delta = the sum of gy * y over a row and dS = P * (dP - delta):
//   gv += P^T gy,   gq += scale dS k,   gk += scale dS^T q.
//
// Two kernels, one that walks over the keys for 32 queries per wavefront (gq, and delta on the way) and one that walks
// over the queries for 32 keys per wavefront (gk, gv).  P and dP are computed in both, which is 7 products instead of 5,
// and in exchange every gradient is summed in registers in a fixed order and written once: no atomics, no fp32 copy of
// gq in memory, the same bits on every run.  The heads that share a key head are rows of one problem (as in the forward
// kernel), so their contributions to gk and gv meet in the same registers.
//
// Bound like the forward kernel by the matrix and the vector pipe in turn: 2 x 8192 tokens, 32/8 heads of 128, bf16, causal:
// gq 1.65 ms (3 products, 1000 TFLOP/s), gk and gv 2.5 ms (4 products, 880 TFLOP/s).
#include <algorithm>
#include <type_traits>

#include "phip_attention.h"

namespace phip {
namespace attention {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

template <typename T>
struct BwArgs {
  const T *q, *k, *v, *y, *gy;
  const float *stats;
  float2 *values;               // scratch: per row stats as a power of two, and delta; written by the first kernel
  T *gq, *gk, *gv;
  Shape s;
  SequenceView seq;
  uint32_t tiles;               // tiles of a whole sample
  uint32_t vec;                 // rows of the gradients are aligned to four elements
  uint32_t acc_q, acc_k, acc_v; // add into what is there (otherwise overwrite)
};

template <typename T, int DP>
__device__ inline void emit_row(T *row, const f32x16 (&x)[DP / 32], float f, bool valid, uint32_t acc, uint32_t d, bool vec,
                                int lane) {
  if (acc && !valid) return;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d0 = 32 * db + 8 * i4 + 4 * (lane >> 5);
      float four[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) four[e] = valid ? x[db][4 * i4 + e] * f : 0.f;
      if (d0 >= (int)d) continue;
      if (acc) store4<T, true>(row + d0, four, (int)d - d0, vec);
      else store4<T, false>(row + d0, four, (int)d - d0, vec);
    }
}

// exp(score - stats) as a power of two, raised by kRaise; a row without keys has stats = -inf and must give 0.
template <typename T>
__device__ inline float row_base(float stats) { return stats == -INFINITY ? INFINITY : stats * kLog2e - kRaise<T>; }

// dS in fp16.  It is a probability, of thousands of keys perhaps, times a difference of any size: 2^-40 and 2^20 are ordinary
// values, and fp16 has neither.  So a wavefront scales its dS by a power of two before it is rounded, and its sums with it:
// the first block puts the largest between 2^13 and 2^14, and a block that goes beyond fp16 scales everything down to that
// again.  What is below 2^-27 of the largest so far loses bits; nothing overflows.  Eight maxima and a multiplication per 16
// values (queries: part of the multiply-add), the rest is rare: a training step with heads of 64 takes 3 to 4 % longer than
// with dS rounded as it is (16 heads, 8192 tokens: 860 against 832 us), with heads of 128 no longer.
template <typename T>
constexpr bool kRanged = __is_same(T, f16_t);
struct Range {
  float scale = 1.f;   // the same in all lanes
  bool known = false;  // some dS was not 0 yet
};

// m: the largest |x| of the lane's 16 values.  Returns what x and the sums were multiplied by.
template <int N>
__device__ inline float fit(Range &range, f32x16 &x, f32x16 (&sums)[N], float m) {
  if (range.known && !__any(m > 0x1.ffp15f)) return 1.f;
  if (!__any(m > 0.f)) return 1.f;
  float by = 1.f;
  // In steps of 16 to between 2^14 and 2^18, then down in steps of 2.  Up by 2^64 at most: what follows may be as large as fp16
  // operands allow (a raised probability of 2^15 times two sums of 128 products of 2^32: 2^55) and must not exceed fp32 before
  // it is seen here; if nothing larger follows, the gradients are below fp16 anyway.  Infinite values stay what they are.
#pragma unroll 1
  for (int i = 0; i < 16 && !__any(m * by >= 0x1p14f); ++i) by *= 0x1p4f;
#pragma unroll 1
  for (int i = 0; i < 32 && __any(m * by >= 0x1p18f); ++i) by *= 0x1p-4f;
#pragma unroll 1
  for (int i = 0; i < 4 && __any(m * by >= 0x1p14f); ++i) by *= 0.5f;
  range.known = true;
  range.scale *= by;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] *= by;
#pragma unroll
  for (int db = 0; db < N; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[db][i] *= by;
  return by;
}
template <int N>
__device__ inline void settle(f32x16 (&sums)[N], float f) {
#pragma unroll
  for (int db = 0; db < N; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) sums[db][i] *= f;
}

// A block of the kernels over the keys: p, the scores, becomes dS (of fp16 scaled by the range, and `rest` with it); pp (FIX)
// the probabilities.  Keys from lim on are hidden (first: the lane's first key).
template <typename T, bool FIX, int N>
__device__ inline void differences(f32x16 &p, f32x16 &pp, const f32x16 &dp, f32x16 (&sums)[N], float &rest, Range &range,
                                   float scale_log2, float base, float delta, bool masked, int first, int lim) {
  const float scaled_delta = kRanged<T> ? delta * range.scale : delta;
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float e = exp2_fast(fmaf(p[i], scale_log2, -base));
    const float x = e * (kRanged<T> ? fmaf(dp[i], range.scale, -scaled_delta) : dp[i] - delta);
    const bool hidden = masked && first + block_row(i) >= lim;
    if constexpr (FIX) pp[i] = hidden ? 0.f : e;
    p[i] = hidden ? 0.f : x;
    if constexpr (kRanged<T>) m = fmaxf(m, fabsf(p[i]));
    else rest += p[i];
  }
  if constexpr (kRanged<T>) {
    rest *= fit(range, p, sums, m);
#pragma unroll
    for (int i = 0; i < 16; ++i) rest += p[i];
  }
}

template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;

// gq and delta: the loop of the forward kernel with P recomputed instead of the running softmax.
//
// delta comes from y as it was stored.  In 16-bit storage its rounding is an error e of delta that adds -e P k to gq, and with
// few keys per row that shows.  FIX adds up P k as well, one more product on the fragments at hand, and takes e, which is minus
// the sum of a row of dS, back out.  Root mean square error of gq in units of that of rounding gq alone, and time of a training
// step on 32 Ki tokens (causal, bf16, 16 heads of 64 / 16 over 4 of 128; fp16 alike):
//   keys           8     16     32         64          128         512         1023
//   error without  1.82  1.72   1.65       1.59        1.54        1.52        1.50
//   error with     1.41  1.42   1.43       1.43        1.42        1.42        1.42
//   us without           1008 / 684  592 / 475  359 / 526  346 / 474  439 / 614  575 / 897
//   us with              1190 / 893  674 / 552  390 / 632  344 / 608  459 / 785  618 / 1152
// With heads of 128 the sums of P k cost the second workgroup per CU, so FIX is taken up to 64 keys, where it takes a tenth of
// the error.
constexpr uint64_t kFixKeys = 64;

template <typename T, int DP, bool DMA, bool FIX>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && DMA && !(FIX && DP == 128) ? 2 : 1) void queries_kernel(const BwArgs<T> a) {
  constexpr int KT = kKeys<T>, BM = 32 * kWaves;
  typedef Tile<T, DP> L;
  typedef TileLoader<T, DP, KT, kThreads, DMA> Loader;
  constexpr uint32_t kTile = (uint32_t)Loader::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char *)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shape &sh = a.s;
  const uint32_t head = blockIdx.x % sh.hk, slot = blockIdx.x / sh.hk;
  const Place at = find_place(a.seq, slot, a.tiles, BM, sh.g, false, sh.causal != 0);
  const SequenceEntry &e = at.e;
  const bool behind = e.sample == kNoSequence;
  const uint32_t token0 = behind ? a.seq.q_total : e.q_start;
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tq - a.seq.q_total : a.seq.packed ? e.q_len : a.seq.tq;
  if ((uint64_t)at.t * BM >= (uint64_t)tokens * sh.g) return;
  const int lq = behind ? 0 : (int)e.q_len, lk = (int)e.k_len, g = (int)sh.g;
  const int r0 = (int)at.t * BM, rows = lq * g;

  const uint32_t r = (uint32_t)(r0 + 32 * wave + (lane & 31)), tok = r / sh.g;
  const bool exists = tok < tokens, valid = exists && (int)tok < lq;
  const size_t row = ((sample * a.seq.tq + token0 + (exists ? tok : 0)) * sh.hq + head * sh.g + (r - tok * sh.g));
  const int lim = !valid ? 0 : sh.causal ? min(lk, max(0, (int)tok + lk - lq + 1)) : lk;

  auto seen_by = [&](int rr) { return sh.causal ? min(lk, max(0, rr / g + lk - lq + 1)) : lk; };
  const int last = min(rows, r0 + BM) - 1, wg_keys = last < r0 ? 0 : seen_by(last);
  const int w_first = r0 + 32 * wave, w_last = min(rows - 1, w_first + 31);
  const int w_keys = w_last < w_first ? 0 : seen_by(w_last), w_all = w_last < w_first ? 0 : seen_by(w_first);

  Frag<T> qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
  load_row<T>(qf, a.q + row * sh.d, valid, sh, lane);
  load_row<T>(gf, a.gy + row * sh.d, valid, sh, lane);
  {
    Frag<T> yf[DP / 16];
    load_row<T>(yf, a.y + row * sh.d, valid, sh, lane);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(element(gf[c], j), element(yf[c], j), delta);
  }
  delta = halves_sum(delta);
  const float base = valid ? row_base<T>(a.stats[row]) : INFINITY;

  // The sum of a row of dS is 0 but for the rounding of y in delta: what comes out instead is the correction of delta that
  // the other kernel uses (gradients of keys in fp16: error 1.5 -> 1.4 times that of rounding the result alone).
  float rest = 0.f;
  Range range;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
  [[maybe_unused]] f32x16 pk[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) pk[db] = f32x16{};
  const uint32_t stride = sh.hk * sh.d;
  const T *kp = a.k + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const T *vp = a.v + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  Loader lk_, lv_;
  lk_.init(1, stride, 0, tid);
  lv_ = lk_;
  auto fetch = [&](int t) {
    const uint32_t stage = lds0 + (uint32_t)(t & 1) * 2 * kTile;
    const size_t off = (size_t)t * KT * stride;
    lk_.fetch(kp + off, lk - t * KT, 0, 1, 1u << 22, stride, 0, (int)sh.d, stage, tid);
    lv_.fetch(vp + off, lk - t * KT, 0, 1, 1u << 22, stride, 0, (int)sh.d, stage + kTile, tid);
  };
  const int n = (wg_keys + KT - 1) / KT;
  if (n > 0) fetch(0);
  for (int t = 0; t < n; ++t) {
    const uint32_t stage = lds0 + (uint32_t)(t & 1) * 2 * kTile;
    if constexpr (DMA) {
      wait_loads<0>();
      if (!sh.whole) {  // the parts of the tiles that this thread cleans may be another wavefront's
        __syncthreads();
        Loader::clean(stage, (int)sh.d, tid);
        Loader::clean(stage + kTile, (int)sh.d, tid);
      }
    } else {
      lk_.put(stage, tid);
      lv_.put(stage + kTile, tid);
    }
    __syncthreads();
    if (t + 1 < n) fetch(t + 1);
    if (t * KT >= w_keys) continue;
    const bool masked = (t + 1) * KT > w_all;
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      __builtin_amdgcn_sched_barrier(0);
      f32x16 p = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) mma(p, L::row_frag(stage + row_at, kb, c), qf[c]);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) mma(dp, L::row_frag(stage + kTile + row_at, kb, c), gf[c]);
      __builtin_amdgcn_sched_barrier(0);
      [[maybe_unused]] f32x16 pp;
      differences<T, FIX>(p, pp, dp, acc, rest, range, sh.scale_log2, base, delta, masked,
                          t * KT + 32 * kb + 4 * (lane >> 5), lim);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> ds = as_operand(p, c, (Frag<T> *)nullptr);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
          const Frag<T> kt = L::col_frag(stage + col_at, 2 * kb + c, db);
          mma(acc[db], kt, ds);
          if constexpr (FIX) mma(pk[db], kt, as_operand(pp, c, (Frag<T> *)nullptr));
        }
      }
    }
  }
  rest = halves_sum(rest);
  if constexpr (kRanged<T>) {
    const float f = kLower<T> / range.scale;
    rest *= f;
    settle(acc, f);
    if constexpr (FIX) settle(pk, kLower<T>);
  }
  if (valid && lane < 32) a.values[row] = {base, delta + rest};
  if constexpr (FIX) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = fmaf(-rest, pk[db][i], acc[db][i]);
  }
  if (exists) emit_row<T, DP>(a.gq + row * sh.d, acc, sh.scale, valid, a.acc_q, sh.d, a.vec != 0, lane);
}

// What 32 rows (their q at LDS address q_at, gy `to_g` further on, values at `in`) add to the gradients of the wavefront's 32
// keys.  hidden: rows before it do not see the lane's key; live: the lane has a key (what the others compute is dropped, and
// must not count for the range).
template <typename T, int DP>
__device__ inline void keys_block(f32x16 (&gk)[DP / 32], f32x16 (&gv)[DP / 32], const Frag<T> (&kf)[DP / 16],
                                  const Frag<T> (&vf)[DP / 16], uint32_t q_at, uint32_t to_g, uint32_t in, bool masked,
                                  int hidden, bool live, Range &range, float scale_log2, uint32_t row_at, uint32_t col_at,
                                  int lane) {
  typedef Tile<T, DP> L;
  const uint32_t g_at = q_at + to_g;
  in += (uint32_t)(4 * (lane >> 5) * 8);
  hidden -= 4 * (lane >> 5);
  __builtin_amdgcn_sched_barrier(0);
  f32x16 p = f32x16{};
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) mma(p, L::row_frag(q_at + row_at, 0, c), kf[c]);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i2 = 0; i2 < 8; ++i2) {
    const f32x4 pair = *lds_ptr<f32x4>(in + (uint32_t)(block_row(2 * i2) * 8));  // two rows: base, delta, base, delta
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * i2 + e;
      p[i] = exp2_fast(fmaf(p[i], scale_log2, -pair[2 * e]));
      if (masked && block_row(i) < hidden) p[i] = 0.f;
    }
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const Frag<T> pf = as_operand(p, c, (Frag<T> *)nullptr);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) mma(gv[db], L::col_frag(g_at + col_at, c, db), pf);
  }
  __builtin_amdgcn_sched_barrier(0);
  f32x16 dp = f32x16{};
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) mma(dp, L::row_frag(g_at + row_at, 0, c), vf[c]);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i2 = 0; i2 < 8; ++i2) {
    const f32x4 pair = *lds_ptr<f32x4>(in + (uint32_t)(block_row(2 * i2) * 8));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = 2 * i2 + e;
      if constexpr (kRanged<T>) dp[i] = p[i] * range.scale * (dp[i] - pair[2 * e + 1]);  // finite, as fp16 operands are
      else dp[i] = p[i] == 0.f ? 0.f : p[i] * (dp[i] - pair[2 * e + 1]);
    }
  }
  if constexpr (kRanged<T>) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(dp[i]));
    fit(range, dp, gk, live ? m : 0.f);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const Frag<T> ds = as_operand(dp, c, (Frag<T> *)nullptr);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) mma(gk[db], L::col_frag(q_at + col_at, c, db), ds);
  }
}

// gk and gv: a workgroup takes 128 keys, 32 per wavefront, and walks over the rows (queries of the group) that see any of
// them in tiles of QT.  16-bit heads of 128 take 255 registers, 128 of them the sums, and the order of keys_block (P, its
// product, dP, its product, nothing moved across) is what fits: with two workgroups per CU 2.5 ms instead of 4.6 with one,
// and a spilled fragment, read back in the loop, would wait for the tiles on their way (3.4 ms).
template <typename T>
constexpr int kRows = sizeof(T) == 2 ? 64 : 32;

template <typename T, int DP, bool DMA>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 && DMA ? 2 : 1) void keys_kernel(const BwArgs<T> a) {
  constexpr int QT = kRows<T>, BN = 32 * kWaves;
  typedef Tile<T, DP> L;
  typedef TileLoader<T, DP, QT, kThreads, DMA> Loader;
  constexpr uint32_t kTile = (uint32_t)Loader::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char *)lds;
  const uint32_t values0 = lds0 + 4 * kTile;  // per stage: QT rows' values

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shape &sh = a.s;
  const uint32_t head = blockIdx.x % sh.hk, slot = blockIdx.x / sh.hk;
  const Place at = find_place(a.seq, slot, a.tiles, BN, 1, true, false);
  const SequenceEntry &e = at.e;
  const bool behind = e.sample == kNoSequence;
  const uint32_t token0 = behind ? a.seq.k_total : e.k_start;
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tk - a.seq.k_total : a.seq.packed ? e.k_len : a.seq.tk;
  if ((uint64_t)at.t * BN >= (uint64_t)tokens) return;
  const int lq = (int)e.q_len, lk = behind ? 0 : (int)e.k_len, g = (int)sh.g;
  const int k0 = (int)at.t * BN, key = k0 + 32 * wave + (lane & 31);
  const bool exists = key < (int)tokens, valid = exists && key < lk;
  const size_t row = ((sample * a.seq.tk + token0 + (exists ? (uint32_t)key : 0)) * sh.hk + head);

  // rows that see any key of the workgroup / the lane's key / any key and all keys of the wavefront: from `*_first` on
  const int rows = k0 < lk ? lq * g : 0;
  auto first_row = [&](int kk) { return sh.causal ? min(max(0, kk - (lk - lq)), lq) * g : 0; };
  const int wg_first = first_row(k0) / QT * QT, w_k0 = k0 + 32 * wave;
  const int w_first = w_k0 < lk ? first_row(w_k0) : rows, w_all = first_row(w_k0 + 31), my_first = first_row(key);

  Frag<T> kf[DP / 16], vf[DP / 16];
  load_row<T>(kf, a.k + row * sh.d, valid, sh, lane);
  load_row<T>(vf, a.v + row * sh.d, valid, sh, lane);
  f32x16 gk[DP / 32], gv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) gk[db] = gv[db] = f32x16{};

  const size_t q_row0 = (sample * a.seq.tq + e.q_start) * sh.hq + head * sh.g;
  const T *qp = a.q + q_row0 * sh.d, *gp = a.gy + q_row0 * sh.d;
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  Loader lq_, lg_;
  lq_.init(sh.g, sh.hq * sh.d, sh.d, tid);
  lg_ = lq_;
  RowWalk walk((uint32_t)wg_first, sh);
  float value = 0.f;
  Range range;
  // the tile of rows from r on, where the walk stands, into a stage; the values of a row side by side
  auto fetch = [&](int r, int stage_no) {
    const uint32_t stage = lds0 + (uint32_t)stage_no * 2 * kTile;
    const size_t off = (size_t)walk.t0 * sh.hq * sh.d;
    const int left = min(QT, rows - r);
    lq_.fetch(qp + off, left, walk.in0, sh.g, sh.inv_g, sh.hq * sh.d, sh.d, (int)sh.d, stage, tid);
    lg_.fetch(gp + off, left, walk.in0, sh.g, sh.inv_g, sh.hq * sh.d, sh.d, (int)sh.d, stage + kTile, tid);
    // rows past the end get zeros, which with their zeros for q and gy add nothing
    int lane_id = tid;
    asm volatile("" : "+v"(lane_id));
    const bool in = (lane_id >> 1) < left;
    const float *p = reinterpret_cast<const float *>(a.values + q_row0 + (size_t)walk.t0 * sh.hq);
    const uint32_t rr = walk.in0 + ((uint32_t)lane_id >> 1), t = (rr * sh.inv_g) >> 22;
    const uint32_t at_value = 2 * (t * sh.hq + (rr - t * sh.g)) + (lane_id & 1);
    if (wave < 2 * QT / 64) {
      if constexpr (DMA)
        lds_dma_b32(buffer_words(p, 0x7fffffffu), values0 + (uint32_t)((stage_no * 2 * QT + wave * 64) * 4), in ? at_value * 4 : kOutOfRange);
      else
        value = in ? p[at_value] : 0.f;
    }
    walk.advance(QT);
  };
  if (wg_first < rows) fetch(wg_first, 0);
  int s = 0;
  for (int r = wg_first; r < rows; r += QT, s ^= 1) {
    const uint32_t stage = lds0 + (uint32_t)s * 2 * kTile;
    const uint32_t values = values0 + (uint32_t)(s * 2 * QT * 4);
    if constexpr (DMA) {
      wait_loads<0>();
      if (!sh.whole) {  // the parts of the tiles that this thread cleans may be another wavefront's
        __syncthreads();
        Loader::clean(stage, (int)sh.d, tid);
        Loader::clean(stage + kTile, (int)sh.d, tid);
      }
    } else {
      if (tid < 2 * QT) *lds_ptr<float>(values + (uint32_t)tid * 4) = value;
      lq_.put(stage, tid);
      lg_.put(stage + kTile, tid);
    }
    __syncthreads();
    if (r + QT < rows) fetch(r + QT, s ^ 1);
    if (r + QT <= w_first) continue;  // none of these rows sees a key of the wavefront
    const bool masked = r < w_all;
#pragma unroll 1
    for (int qb = 0; qb < QT / 32; ++qb) {
      keys_block<T, DP>(gk, gv, kf, vf, stage + (uint32_t)(qb * 32 * L::kPitch), kTile, values + (uint32_t)(qb * 32 * 8), masked,
                        min(QT, my_first - r) - 32 * qb, valid, range, sh.scale_log2, row_at, col_at, lane);
    }
  }
  if constexpr (kRanged<T>) {
    settle(gk, kLower<T> / range.scale);
    settle(gv, kLower<T>);
  }
  if (!exists) return;
  // the two gradients may be one tensor (the same tensor as keys and values): one after the other, by the same lane
  emit_row<T, DP>(a.gk + row * sh.d, gk, sh.scale, valid, a.acc_k, sh.d, a.vec != 0, lane);
  emit_row<T, DP>(a.gv + row * sh.d, gv, 1.f, valid, a.acc_v, sh.d, a.vec != 0, lane);
}

// The same two for few tiles (short sequences, few heads): a workgroup of W wavefronts takes 32 queries (32 keys) and its
// wavefronts walk over blocks of 32 keys (rows) of their own, through rings of LDS tiles of their own; their sums meet in
// LDS at the end, in a fixed order.  With W = 1 a workgroup is one wavefront, for sequences so short that there is nothing
// to divide.
template <typename T, int DP, int W>
constexpr int kFewLds = W * std::max(2 * kStages<T, DP> * 32 * Tile<T, DP>::kPitch + 2 * kStages<T, DP> * 32 * 4, DP * 33 * 4);

// Adds the wavefronts' blocks (rows of the result across) through LDS and writes the 32 rows, four elements per thread at
// a time.  row(r): where row r goes, null where it does not exist; of these the first `filled` have a gradient.
template <typename T, int DP, int W, typename Row>
__device__ inline void emit_sum(const f32x16 (&x)[DP / 32], unsigned char *lds, float f, uint32_t acc, uint32_t d, bool vec,
                                Row row, int filled) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if constexpr (W == 1) {
    T *p = row(lane & 31);
    if (p != nullptr) emit_row<T, DP>(p, x, f, (lane & 31) < filled, acc, d, vec, lane);
    return;
  }
  constexpr int kPer = DP * 33;
  float *const area = reinterpret_cast<float *>(lds);
  __syncthreads();
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) area[wave * kPer + (32 * db + block_row(i) + 4 * (lane >> 5)) * 33 + (lane & 31)] = x[db][i];
  __syncthreads();
#pragma unroll
  for (uint32_t i = tid; i < 32 * (DP / 4); i += 64 * W) {
    const int r = (int)(i / (DP / 4));
    const uint32_t dd = i % (DP / 4) * 4;
    T *p = row(r);
    const bool valid = r < filled;
    if (p == nullptr || dd >= d || (acc && !valid)) continue;
    float four[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += area[w * kPer + (dd + e) * 33 + r];
      four[e] = valid ? sum * f : 0.f;
    }
    if (acc) store4<T, true>(p + dd, four, (int)(d - dd), vec);
    else store4<T, false>(p + dd, four, (int)(d - dd), vec);
  }
}

template <typename T, int DP, bool DMA, int W, bool FIX>
__global__ __launch_bounds__(64 * W, 1) void few_queries_kernel(const BwArgs<T> a) {
  constexpr int BM = 32, S = DMA ? kStages<T, DP> : 1;
  typedef Tile<T, DP> L;
  typedef TileLoader<T, DP, 32, 64, DMA> Loader;
  constexpr uint32_t kTile = (uint32_t)Loader::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char *)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shape &sh = a.s;
  const uint32_t head = blockIdx.x % sh.hk, slot = blockIdx.x / sh.hk;
  const Place at = find_place(a.seq, slot, a.tiles, BM, sh.g, false, sh.causal != 0);
  const SequenceEntry &e = at.e;
  const bool behind = e.sample == kNoSequence;
  const uint32_t token0 = behind ? a.seq.q_total : e.q_start;
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tq - a.seq.q_total : a.seq.packed ? e.q_len : a.seq.tq;
  if ((uint64_t)at.t * BM >= (uint64_t)tokens * sh.g) return;
  const int lq = behind ? 0 : (int)e.q_len, lk = (int)e.k_len, g = (int)sh.g;
  const int r0 = (int)at.t * BM, rows = lq * g;
  // the lane's row; keys that it, any row and all rows of the tile see
  const int exist = min((int)(tokens * sh.g) - r0, BM), filled = min(rows - r0, BM);
  auto seen_by = [&](int rr) { return sh.causal ? min(lk, max(0, rr / g + lk - lq + 1)) : lk; };
  const bool valid = (lane & 31) < filled;
  const int lim = valid ? seen_by(r0 + (lane & 31)) : 0;
  const int keys = filled <= 0 ? 0 : seen_by(r0 + filled - 1), all = filled <= 0 ? 0 : seen_by(r0);
  const RowWalk walk((uint32_t)r0, sh);
  const size_t row_0 = (sample * a.seq.tq + token0) * sh.hq + head * sh.g;
  const size_t row = row_0 + walk.at(valid ? lane & 31 : 0, sh.hq);

  const uint32_t stride = sh.hk * sh.d;
  const T *kp = a.k + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const T *vp = a.v + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const uint32_t ring = lds0 + (uint32_t)wave * (2 * S * kTile);
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  constexpr int kStep = 32 * W;
  Loader lk_, lv_;
  lk_.init(1, stride, 0, lane);
  lv_ = lk_;
  auto fetch = [&](int key, int s) {
    const size_t off = (size_t)min(key, keys) * stride;
    lk_.fetch(kp + off, keys - key, 0, 1, 1u << 22, stride, 0, (int)sh.d, ring + (uint32_t)s * 2 * kTile, lane);
    lv_.fetch(vp + off, keys - key, 0, 1, 1u << 22, stride, 0, (int)sh.d, ring + (uint32_t)s * 2 * kTile + kTile, lane);
  };
  Frag<T> qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
  load_row<T>(qf, a.q + row * sh.d, valid, sh, lane);
  load_row<T>(gf, a.gy + row * sh.d, valid, sh, lane);
  {
    Frag<T> yf[DP / 16];
    load_row<T>(yf, a.y + row * sh.d, valid, sh, lane);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = fmaf(element(gf[c], j), element(yf[c], j), delta);
  }
  int key = 32 * wave;
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(key + s * kStep, s);

  delta = halves_sum(delta);
  const float base = valid ? row_base<T>(a.stats[row]) : INFINITY;

  arrived(qf);
  arrived(gf);
  float rest = 0.f;  // corrects delta, as in queries_kernel
  Range range;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
  [[maybe_unused]] f32x16 pk[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) pk[db] = f32x16{};
  for (int s = 0; key < keys; key += kStep, s = s + 1 == S ? 0 : s + 1) {
    const uint32_t stage = ring + (uint32_t)s * 2 * kTile;
    if constexpr (DMA) {
      wait_loads<(S - 1) * 2 * Loader::kInstr>();
      if (!sh.whole) {
        Loader::clean(stage, (int)sh.d, lane);
        Loader::clean(stage + kTile, (int)sh.d, lane);
      }
    } else {
      lk_.put(stage, lane);
      lv_.put(stage + kTile, lane);
      fetch(key + kStep, 0);
    }
    f32x16 p = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) mma(p, L::row_frag(stage + row_at, 0, c), qf[c]);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) mma(dp, L::row_frag(stage + kTile + row_at, 0, c), gf[c]);
    const bool masked = key + 32 > all;
    [[maybe_unused]] f32x16 pp;
    differences<T, FIX>(p, pp, dp, acc, rest, range, sh.scale_log2, base, delta, masked, key + 4 * (lane >> 5), lim);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Frag<T> ds = as_operand(p, c, (Frag<T> *)nullptr);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        const Frag<T> kt = L::col_frag(stage + col_at, c, db);
        mma(acc[db], kt, ds);
        if constexpr (FIX) mma(pk[db], kt, as_operand(pp, c, (Frag<T> *)nullptr));
      }
    }
    if constexpr (DMA) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile's reads are done before its place is filled again
      fetch(key + S * kStep, s);
    }
  }
  wait_loads<0>();
  rest = halves_sum(rest);
  if constexpr (kRanged<T>) {
    const float f = kLower<T> / range.scale;
    rest *= f;
    settle(acc, f);
    if constexpr (FIX) settle(pk, kLower<T>);
  }
  if constexpr (W > 1) {
    __shared__ float rests[W][32];
    if (lane < 32) rests[wave][lane] = rest;
    __syncthreads();
    rest = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) rest += rests[w][lane & 31];
  }
  if (valid && tid < 32) a.values[row] = {base, delta + rest};
  if constexpr (FIX) {
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] = fmaf(-rest, pk[db][i], acc[db][i]);
  }
  emit_sum<T, DP, W>(acc, lds, sh.scale, a.acc_q, sh.d, a.vec != 0,
                     [&](int i) { return i < exist ? a.gq + (row_0 + walk.at((uint32_t)i, sh.hq)) * sh.d : (T *)nullptr; },
                     filled);
}

template <typename T, int DP, bool DMA, int W>
__global__ __launch_bounds__(64 * W, 1) void few_keys_kernel(const BwArgs<T> a) {
  constexpr int BN = 32, S = DMA ? kStages<T, DP> : 1;
  typedef Tile<T, DP> L;
  typedef TileLoader<T, DP, 32, 64, DMA> Loader;
  constexpr uint32_t kTile = (uint32_t)Loader::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char *)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shape &sh = a.s;
  const uint32_t head = blockIdx.x % sh.hk, slot = blockIdx.x / sh.hk;
  const Place at = find_place(a.seq, slot, a.tiles, BN, 1, true, false);
  const SequenceEntry &e = at.e;
  const bool behind = e.sample == kNoSequence;
  const uint32_t token0 = behind ? a.seq.k_total : e.k_start;
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tk - a.seq.k_total : a.seq.packed ? e.k_len : a.seq.tk;
  if ((uint64_t)at.t * BN >= (uint64_t)tokens) return;
  const int lq = (int)e.q_len, lk = behind ? 0 : (int)e.k_len, g = (int)sh.g;
  const int k0 = (int)at.t * BN, key = k0 + (lane & 31), exist = min((int)tokens - k0, BN);
  const bool valid = key < lk;
  const size_t row_0 = (sample * a.seq.tk + token0 + (uint32_t)k0) * sh.hk + head;  // keys lie hk rows apart
  const size_t row = row_0 + (valid ? (size_t)(lane & 31) * sh.hk : 0);
  const int rows = k0 < lk ? lq * g : 0;
  auto first_row = [&](int kk) { return sh.causal ? min(max(0, kk - (lk - lq)), lq) * g : 0; };
  const int all = first_row(k0 + 31), my_first = first_row(key);

  const size_t q_row0 = (sample * a.seq.tq + e.q_start) * sh.hq + head * sh.g;
  const T *qp = a.q + q_row0 * sh.d, *gp = a.gy + q_row0 * sh.d;
  const uint32_t ring = lds0 + (uint32_t)wave * (2 * S * kTile);
  const uint32_t values0 = lds0 + (uint32_t)W * (2 * S * kTile) + (uint32_t)wave * (S * 64 * 4);
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  constexpr int kStep = 32 * W;
  Loader lq_, lg_;
  lq_.init(sh.g, sh.hq * sh.d, sh.d, lane);
  lg_ = lq_;
  float value = 0.f;
  Range range;
  int rr = first_row(k0) / 32 * 32 + 32 * wave;
  RowWalk walk((uint32_t)rr, sh);
  // the rows from `from` on, where the walk stands, into stage s; lane 2 i + e brings value e of row i
  auto fetch = [&](int from, int s) {
    const size_t off = from < rows ? (size_t)walk.t0 * sh.hq * sh.d : 0;
    const int left = min(32, rows - from);
    const uint32_t stage = ring + (uint32_t)s * 2 * kTile;
    lq_.fetch(qp + off, left, walk.in0, sh.g, sh.inv_g, sh.hq * sh.d, sh.d, (int)sh.d, stage, lane);
    lg_.fetch(gp + off, left, walk.in0, sh.g, sh.inv_g, sh.hq * sh.d, sh.d, (int)sh.d, stage + kTile, lane);
    const bool in = (lane >> 1) < left;
    const float *p = reinterpret_cast<const float *>(a.values + q_row0 + (from < rows ? (size_t)walk.t0 * sh.hq : 0));
    const uint32_t r = walk.in0 + ((uint32_t)lane >> 1), t = (r * sh.inv_g) >> 22;
    const uint32_t at_value = 2 * (t * sh.hq + (r - t * sh.g)) + (lane & 1);
    if constexpr (DMA) lds_dma_b32(buffer_words(p, 0x7fffffffu), values0 + (uint32_t)(s * 64 * 4), in ? at_value * 4 : kOutOfRange);
    else value = in ? p[at_value] : 0.f;
    walk.advance(kStep);
  };
  Frag<T> kf[DP / 16], vf[DP / 16];
  load_row<T>(kf, a.k + row * sh.d, valid, sh, lane);
  load_row<T>(vf, a.v + row * sh.d, valid, sh, lane);
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(rr + s * kStep, s);

  arrived(kf);
  arrived(vf);
  f32x16 gk[DP / 32], gv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) gk[db] = gv[db] = f32x16{};

  for (int s = 0; rr < rows; rr += kStep, s = s + 1 == S ? 0 : s + 1) {
    const uint32_t stage = ring + (uint32_t)s * 2 * kTile, in = values0 + (uint32_t)(s * 64 * 4);
    if constexpr (DMA) {
      wait_loads<(S - 1) * (2 * Loader::kInstr + 1)>();
      if (!sh.whole) {
        Loader::clean(stage, (int)sh.d, lane);
        Loader::clean(stage + kTile, (int)sh.d, lane);
      }
    } else {
      lq_.put(stage, lane);
      lg_.put(stage + kTile, lane);
      *lds_ptr<float>(in + (uint32_t)lane * 4) = value;
      fetch(rr + kStep, 0);
    }
    keys_block<T, DP>(gk, gv, kf, vf, stage, kTile, in, rr < all, my_first - rr, valid, range, sh.scale_log2, row_at, col_at,
                      lane);
    if constexpr (DMA) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile's reads are done before its place is filled again
      fetch(rr + S * kStep, s);
    }
  }
  wait_loads<0>();
  if constexpr (kRanged<T>) {
    settle(gk, kLower<T> / range.scale);
    settle(gv, kLower<T>);
  }
  auto in_k = [&](int i) { return i < exist ? a.gk + (row_0 + (size_t)i * sh.hk) * sh.d : (T *)nullptr; };
  auto in_v = [&](int i) { return i < exist ? a.gv + (row_0 + (size_t)i * sh.hk) * sh.d : (T *)nullptr; };
  // the two gradients may be one tensor: one after the other, by the same thread
  emit_sum<T, DP, W>(gk, lds, sh.scale, a.acc_k, sh.d, a.vec != 0, in_k, lk - k0);
  emit_sum<T, DP, W>(gv, lds, 1.f, a.acc_v, sh.d, a.vec != 0, in_v, lk - k0);
}

template <auto *KERNEL, typename T>
int launch_kernel(phip_ctx *ctx, const char *name, const BwArgs<T> &a, uint64_t blocks, int threads, int lds) {
  const int rc = allow_lds<KERNEL>(ctx, lds);
  if (rc != PHIP_OK) return rc;
  hipLaunchKernelGGL(KERNEL, dim3((uint32_t)blocks), dim3((uint32_t)threads), lds, ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  note_kernel(ctx, name);
  return PHIP_OK;
}

// The workgroups of the two kernels.
struct Plan {
  struct Side {
    Way way;
    uint64_t wide, narrow;  // with tiles of 128, of 32
    bool launchable() const {
      return way == Way::Shared ? attention::launchable(wide, kThreads)
                                : attention::launchable(narrow, way == Way::One ? 64 : 256);
    }
  };
  Side q, k;
  uint64_t most_k;          // keys of the longest sequence
};

template <typename T>
Plan make_plan(phip_ctx *ctx, const BwArgs<T> &a, const phip_sequences *seqs) {
  const uint64_t most_q = (uint64_t)(seqs != nullptr ? seqs->max_q : a.seq.tq) * a.s.g;
  const uint64_t most_k = seqs != nullptr ? seqs->max_k : a.seq.tk;
  Plan p = {{Way::Shared, slots(a.seq, 128, a.s.g, false) * a.s.hk, slots(a.seq, 32, a.s.g, false) * a.s.hk},
            {Way::Shared, slots(a.seq, 128, 1, true) * a.s.hk, slots(a.seq, 32, 1, true) * a.s.hk},
            most_k};
  p.q.way = choose_way<T>(ctx, p.q.wide, p.q.narrow, most_q, most_k);
  p.k.way = choose_way<T>(ctx, p.k.wide, p.k.narrow, most_k, most_q);
  return p;
}

template <typename T, int DP, bool DMA>
int launch(phip_ctx *ctx, BwArgs<T> a, const Plan &plan) {
  constexpr int lds_q = 4 * kKeys<T> * Tile<T, DP>::kPitch;
  constexpr int lds_k = 4 * kRows<T> * Tile<T, DP>::kPitch + 4 * kRows<T> * 4;
  const Way way_q = plan.q.way, way_k = plan.k.way;
  const uint64_t rows = (uint64_t)a.seq.tq * a.s.g, keys = a.seq.tk;
  a.tiles = (uint32_t)(way_q == Way::Shared ? (rows + 127) / 128 : (rows + 31) / 32);
  auto queries = [&](auto fix) {
    constexpr bool FIX = decltype(fix)::value;
    if (way_q == Way::Four)
      return launch_kernel<few_queries_kernel<T, DP, DMA, 4, FIX>>(
          ctx, FIX ? "attention_few_queries_fix" : "attention_few_queries", a, plan.q.narrow, 256, kFewLds<T, DP, 4>);
    if constexpr (sizeof(T) == 4) {
      if (way_q == Way::One)
        return launch_kernel<few_queries_kernel<T, DP, DMA, 1, FIX>>(ctx, "attention_few1_queries", a, plan.q.narrow, 64,
                                                                     kFewLds<T, DP, 1>);
    }
    return launch_kernel<queries_kernel<T, DP, DMA, FIX>>(ctx, FIX ? "attention_queries_fix" : "attention_queries", a,
                                                          plan.q.wide, kThreads, lds_q);
  };
  int rc = PHIP_OK;
  if constexpr (sizeof(T) == 2) rc = plan.most_k <= kFixKeys ? queries(std::true_type()) : queries(std::false_type());
  else rc = queries(std::false_type());
  if (rc != PHIP_OK) return rc;
  a.tiles = (uint32_t)(way_k == Way::Shared ? (keys + 127) / 128 : (keys + 31) / 32);
  if (way_k == Way::Four)
    return launch_kernel<few_keys_kernel<T, DP, DMA, 4>>(ctx, "attention_few_keys", a, plan.k.narrow, 256, kFewLds<T, DP, 4>);
  if constexpr (sizeof(T) == 4) {
    if (way_k == Way::One)
      return launch_kernel<few_keys_kernel<T, DP, DMA, 1>>(ctx, "attention_few1_keys", a, plan.k.narrow, 64, kFewLds<T, DP, 1>);
  }
  return launch_kernel<keys_kernel<T, DP, DMA>>(ctx, "attention_keys", a, plan.k.wide, kThreads, lds_k);
}

template <typename T, bool DMA>
int dispatch(phip_ctx *ctx, const BwArgs<T> &a, const Plan &plan) {
  switch ((a.s.d + 31) / 32) {
    case 1: return launch<T, 32, DMA>(ctx, a, plan);
    case 2: return launch<T, 64, DMA>(ctx, a, plan);
    case 3: return launch<T, 96, DMA>(ctx, a, plan);
    default: return launch<T, 128, DMA>(ctx, a, plan);
  }
}

template <typename T>
int backward(phip_ctx *ctx, const T *q, const T *k, const T *v, const T *y, const float *stats, const T *gy, T *gq, T *gk,
             T *gv, uint32_t d, uint32_t hq, uint32_t hk, uint32_t tq, uint32_t tk, uint32_t bs,
             const phip_sequences *seqs, int causal, float scale) {
  PHIP_ENTER_KEEP_ZEROS(ctx);
  BwArgs<T> a = {};
  int rc = make_shape(d, hq, hk, tq, tk, bs, causal, scale, sizeof(T), &a.s);
  if (rc != PHIP_OK) return rc;
  rc = sequence_view(ctx, seqs, tq, tk, bs, true, &a.seq);
  if (rc != PHIP_OK) return rc;
  PHIP_REQUIRE(q && k && v && y && stats && gy && gq && gk && gv, "null pointer");
  PHIP_REQUIRE(elements_aligned(sizeof(T), {q, k, v, y, gy, gq, gk, gv}) && elements_aligned(4, {stats}),
               "an address is no multiple of the element size");
  const size_t nq = (size_t)d * hq * tq * bs * sizeof(T), nk = (size_t)d * hk * tk * bs * sizeof(T);
  const size_t ns = (size_t)hq * tq * bs * sizeof(float);
  auto is_read = [&](const void *g, size_t n) {
    return shares_memory(g, n, q, nq) || shares_memory(g, n, k, nk) || shares_memory(g, n, v, nk) ||
           shares_memory(g, n, y, nq) || shares_memory(g, n, gy, nq) || shares_memory(g, n, stats, ns);
  };
  PHIP_REQUIRE(!is_read(gq, nq) && !is_read(gk, nk) && !is_read(gv, nk), "a gradient shares memory with an operand");
  // the same tensor may be queries, keys and values, and then its one gradient is passed for each; anything in between
  // would have two lanes add to one element, or two layouts in one tensor
  const bool alike = hq == hk && tq == tk;
  PHIP_REQUIRE((gk == gv || !shares_memory(gk, nk, gv, nk)) && (gq == gk ? alike : !shares_memory(gq, nq, gk, nk)) &&
                   (gq == gv ? alike : !shares_memory(gq, nq, gv, nk)),
               "two gradients overlap without being the same tensor");
  const Plan plan = make_plan<T>(ctx, a, seqs);
  PHIP_REQUIRE(plan.q.launchable() && plan.k.launchable(), "too many rows");
  void *values = nullptr;
  rc = phip_pool_alloc(ctx, 2 * ns, &values, nullptr);
  if (rc != PHIP_OK) return rc;
  // Nothing is refused from here on: gradients noted as zero and not yet filled are written instead of added into.  gq is
  // written before gk and gk before gv, so of gradients that are one tensor the first takes the note.
  a.acc_q = !zeros_take(ctx, gq, nq);
  a.acc_k = !zeros_take(ctx, gk, nk);
  a.acc_v = !zeros_take(ctx, gv, nk);
  PHIP_FLUSH_ZEROS(ctx);
  a.q = q;
  a.k = k;
  a.v = v;
  a.y = y;
  a.gy = gy;
  a.stats = stats;
  a.values = static_cast<float2 *>(values);
  a.gq = gq;
  a.gk = gk;
  a.gv = gv;
  auto vec = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0; };
  a.vec = d % 4 == 0 && vec(gq) && vec(gk) && vec(gv);
  a.s.whole = rows_aligned(d, sizeof(T), 16, {q, k, v, y, gy});
  // fp32 rows are always whole dwords; 16-bit rows of an odd size are not
  bool dma = true;
  if constexpr (sizeof(T) == 2) {
    dma = rows_aligned(d, sizeof(T), 4, {q, k, v, gy});
    if (!dma) rc = dispatch<T, false>(ctx, a, plan);
  }
  if (dma) rc = dispatch<T, true>(ctx, a, plan);
  phip_pool_free(ctx, values);
  return rc;
}

}  // namespace
}  // namespace attention
}  // namespace phip

using namespace phip;

extern "C" {

int phip_attention_bw_f32(phip_ctx *ctx, const float *q, const float *k, const float *v, const float *y,
                          const float *stats, const float *gy, float *gq, float *gk, float *gv, uint32_t d, uint32_t hq,
                          uint32_t hk, uint32_t tq, uint32_t tk, uint32_t bs, const phip_sequences *seqs, int causal,
                          float scale) {
  return attention::backward<float>(ctx, q, k, v, y, stats, gy, gq, gk, gv, d, hq, hk, tq, tk, bs, seqs, causal, scale);
}

#define PHIP_EXPORT_ATTENTION_BW(SUF, T)                                                                                 \
  int phip_attention_bw_##SUF(phip_ctx *ctx, const void *q, const void *k, const void *v, const void *y,                 \
                              const float *stats, const void *gy, void *gq, void *gk, void *gv, uint32_t d, uint32_t hq, \
                              uint32_t hk, uint32_t tq, uint32_t tk, uint32_t bs, const phip_sequences *seqs,            \
                              int causal, float scale) {                                                                 \
    return attention::backward<T>(ctx, static_cast<const T *>(q), static_cast<const T *>(k), static_cast<const T *>(v),  \
                                  static_cast<const T *>(y), stats, static_cast<const T *>(gy), static_cast<T *>(gq),    \
                                  static_cast<T *>(gk), static_cast<T *>(gv), d, hq, hk, tq, tk, bs, seqs, causal,       \
                                  scale);                                                                                \
  }

PHIP_EXPORT_ATTENTION_BW(f16, f16_t)
PHIP_EXPORT_ATTENTION_BW(bf16, bf16_t)

#undef PHIP_EXPORT_ATTENTION_BW

}  // extern "C"
