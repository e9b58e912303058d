// Gradients of attention.  With P = exp(scale q k^T - stats) (stats: the log of the sum of exponentials that the forward
// call left), dP = gy v^T, delta = the sum of gy * y over a row and dS = P * (dP - delta):
//   gv += P^T gy,   gq += scale dS k,   gk += scale dS^T q.
//
// Two kernels, one that walks over the keys for 32 queries per wavefront (gq, and delta on the way) and one that walks
// over the queries for 32 keys per wavefront (gk, gv).  P and dP are computed in both, which is 7 products instead of 5,
// and in exchange every gradient is summed in registers in a fixed order and written once: no atomics, no fp32 copy of
// gq in memory, the same bits on every run.  The heads that share a key head are rows of one problem (as in the forward
// kernel), so their contributions to gk and gv meet in the same registers.
#include <algorithm>

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
  float *delta;                 // scratch: one value per row, written by the first kernel
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

// exp(score - stats) as a power of two; a row without keys has stats = -inf and must give 0.
__device__ inline float row_base(float stats) { return stats == -INFINITY ? INFINITY : stats * kLog2e; }

template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;

// gq and delta: the loop of the forward kernel with P recomputed instead of the running softmax.
template <typename T, int DP, bool DMA>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void queries_kernel(const BwArgs<T> a) {
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
  const int64_t r0 = (int64_t)at.t * BM;
  if (r0 >= (int64_t)tokens * sh.g) return;
  const int lq = behind ? 0 : (int)e.q_len, lk = (int)e.k_len;

  const int64_t r = r0 + 32 * wave + (lane & 31);
  const uint32_t tok = (uint32_t)(r / sh.g);
  const bool exists = tok < tokens, valid = exists && (int)tok < lq;
  const size_t row = ((sample * a.seq.tq + token0 + (exists ? tok : 0)) * sh.hq + head * sh.g + (uint32_t)(r % sh.g));
  const int lim = !valid ? 0 : sh.causal ? min(lk, max(0, (int)tok + lk - lq + 1)) : lk;

  const int64_t last = min((int64_t)lq * sh.g, r0 + BM) - 1;
  const int wg_keys = last < r0 ? 0 : sh.causal ? min(lk, max(0, (int)(last / sh.g) + lk - lq + 1)) : lk;
  const int64_t w_first = r0 + 32 * wave, w_last = min((int64_t)lq * sh.g - 1, w_first + 31);
  int w_keys = 0, w_all = 0;
  if (w_last >= w_first) {
    w_keys = sh.causal ? min(lk, max(0, (int)(w_last / sh.g) + lk - lq + 1)) : lk;
    w_all = sh.causal ? min(lk, max(0, (int)(w_first / sh.g) + lk - lq + 1)) : lk;
  }

  Frag<T> qf[DP / 16], gf[DP / 16];
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    const int d0 = 16 * c + 8 * (lane >> 5);
    qf[c] = load_frag(a.q + row * sh.d, valid, d0, (int)sh.d, (Frag<T> *)nullptr);
    gf[c] = load_frag(a.gy + row * sh.d, valid, d0, (int)sh.d, (Frag<T> *)nullptr);
    const Frag<T> yf = load_frag(a.y + row * sh.d, valid, d0, (int)sh.d, (Frag<T> *)nullptr);
#pragma unroll
    for (int j = 0; j < 8; ++j) delta = fmaf(element(gf[c], j), element(yf, j), delta);
  }
  delta = halves_sum(delta);
  const float base = valid ? row_base(a.stats[row]) : INFINITY;
  if (valid && lane < 32) a.delta[row] = delta;

  f32x16 acc[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
  const uint32_t stride = sh.hk * sh.d;
  const T *kp = a.k + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const T *vp = a.v + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  Loader lk_, lv_;
  auto fetch = [&](int t) {
    const uint32_t stage = lds0 + (uint32_t)(t & 1) * 2 * kTile;
    const size_t off = (size_t)t * KT * stride;
    lk_.fetch(kp + off, lk - t * KT, 0, 1, 0, stride, 0, (int)sh.d, stage, tid);
    lv_.fetch(vp + off, lk - t * KT, 0, 1, 0, stride, 0, (int)sh.d, stage + kTile, tid);
  };
  const int n = (wg_keys + KT - 1) / KT;
  if (n > 0) fetch(0);
  for (int t = 0; t < n; ++t) {
    const uint32_t stage = lds0 + (uint32_t)(t & 1) * 2 * kTile;
    if constexpr (DMA) {
      wait_loads<0>();
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
      f32x16 p = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) mma(p, L::row_frag(stage + row_at, kb, c), qf[c]);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) mma(dp, L::row_frag(stage + kTile + row_at, kb, c), gf[c]);
      const int first = t * KT + 32 * kb + 4 * (lane >> 5);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = exp2_fast(fmaf(p[i], sh.scale_log2, -base)) * (dp[i] - delta);
        p[i] = masked && first + block_row(i) >= lim ? 0.f : x;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> ds = as_operand(p, c, (Frag<T> *)nullptr);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) mma(acc[db], L::col_frag(stage + col_at, 2 * kb + c, db), ds);
      }
    }
  }
  if (exists) emit_row<T, DP>(a.gq + row * sh.d, acc, sh.scale, valid, a.acc_q, sh.d, a.vec != 0, lane);
}

// gk and gv: a workgroup takes 128 keys, 32 per wavefront, and walks over the rows (queries of the group) that see any of
// them in tiles of QT.
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
  const uint32_t values0 = lds0 + 4 * kTile;  // per stage: QT bases, QT deltas

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shape &sh = a.s;
  const uint32_t head = blockIdx.x % sh.hk, slot = blockIdx.x / sh.hk;
  const Place at = find_place(a.seq, slot, a.tiles, BN, 1, true, false);
  const SequenceEntry &e = at.e;
  const bool behind = e.sample == kNoSequence;
  const uint32_t token0 = behind ? a.seq.k_total : e.k_start;
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tk - a.seq.k_total : a.seq.packed ? e.k_len : a.seq.tk;
  const int64_t k0 = (int64_t)at.t * BN;
  if (k0 >= (int64_t)tokens) return;
  const int lq = (int)e.q_len, lk = behind ? 0 : (int)e.k_len;

  const int64_t key = k0 + 32 * wave + (lane & 31);
  const bool exists = key < (int64_t)tokens, valid = exists && key < lk;
  const size_t row = ((sample * a.seq.tk + token0 + (exists ? (uint32_t)key : 0)) * sh.hk + head);

  // rows that see any key of the workgroup / the lane's key / any key and all keys of the wavefront: from `*_first` on
  const int64_t rows = k0 < lk ? (int64_t)lq * sh.g : 0;
  auto first_row = [&](int64_t kk) { return sh.causal ? max((int64_t)0, kk - (lk - lq)) * (int64_t)sh.g : (int64_t)0; };
  const int64_t wg_first = first_row(k0) / QT * QT;
  const int64_t w_k0 = k0 + 32 * wave;
  const int64_t w_first = w_k0 < lk ? first_row(w_k0) : rows, w_all = first_row(w_k0 + 31);
  const int64_t my_first = first_row(key);

  Frag<T> kf[DP / 16], vf[DP / 16];
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    const int d0 = 16 * c + 8 * (lane >> 5);
    kf[c] = load_frag(a.k + row * sh.d, valid, d0, (int)sh.d, (Frag<T> *)nullptr);
    vf[c] = load_frag(a.v + row * sh.d, valid, d0, (int)sh.d, (Frag<T> *)nullptr);
  }
  f32x16 gk[DP / 32], gv[DP / 32];
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) gk[db] = gv[db] = f32x16{};

  const size_t q_row0 = (sample * a.seq.tq + e.q_start) * sh.hq + head * sh.g;
  const T *qp = a.q + q_row0 * sh.d, *gp = a.gy + q_row0 * sh.d;
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  Loader lq_, lg_;
  float value = 0.f;
  auto fetch = [&](int64_t r, int stage_no) {
    const uint32_t stage = lds0 + (uint32_t)stage_no * 2 * kTile;
    const uint32_t t0 = (uint32_t)(r / sh.g), in_group = (uint32_t)(r % sh.g);
    const size_t off = (size_t)t0 * sh.hq * sh.d;
    const int left = (int)min((int64_t)QT, rows - r);
    lq_.fetch(qp + off, left, in_group, sh.g, sh.inv_g, sh.hq * sh.d, sh.d, (int)sh.d, stage, tid);
    lg_.fetch(gp + off, left, in_group, sh.g, sh.inv_g, sh.hq * sh.d, sh.d, (int)sh.d, stage + kTile, tid);
    if (tid < 2 * QT) {
      const int i = tid & (QT - 1);
      const uint32_t rr = in_group + (uint32_t)i, t = (rr * sh.inv_g) >> 22;
      const size_t w = q_row0 + (size_t)(t0 + t) * sh.hq + (rr - t * sh.g);
      value = tid < QT ? INFINITY : 0.f;
      if (i < left) value = tid < QT ? row_base(a.stats[w]) : a.delta[w];
    }
  };
  if (wg_first < rows) fetch(wg_first, 0);
  int s = 0;
  for (int64_t r = wg_first; r < rows; r += QT, s ^= 1) {
    const uint32_t stage = lds0 + (uint32_t)s * 2 * kTile;
    const uint32_t values = values0 + (uint32_t)(s * 2 * QT * 4);
    if (tid < 2 * QT) *lds_ptr<float>(values + (uint32_t)tid * 4) = value;
    if constexpr (DMA) {
      wait_loads<0>();
    } else {
      lq_.put(stage, tid);
      lg_.put(stage + kTile, tid);
    }
    __syncthreads();
    if (r + QT < rows) fetch(r + QT, s ^ 1);
    if (r + QT <= w_first) continue;  // none of these rows sees a key of the wavefront
    const bool masked = r < w_all;
#pragma unroll 1
    for (int qb = 0; qb < QT / 32; ++qb) {
      const uint32_t q_at = stage + (uint32_t)(qb * 32 * L::kPitch), g_at = q_at + kTile;
      const uint32_t in = values + (uint32_t)((32 * qb + 4 * (lane >> 5)) * 4);
      const int hidden = (int)max((int64_t)0, min((int64_t)QT, my_first - r)) - 32 * qb - 4 * (lane >> 5);
      f32x16 p = f32x16{};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) mma(p, L::row_frag(q_at + row_at, 0, c), kf[c]);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 base = *lds_ptr<f32x4>(in + 32 * i4);
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int i = 4 * i4 + e4;
          p[i] = exp2_fast(fmaf(p[i], sh.scale_log2, -base[e4]));
          if (masked && block_row(i) < hidden) p[i] = 0.f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> pf = as_operand(p, c, (Frag<T> *)nullptr);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) mma(gv[db], L::col_frag(g_at + col_at, c, db), pf);
      }
      f32x16 dp = f32x16{};
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) mma(dp, L::row_frag(g_at + row_at, 0, c), vf[c]);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 delta = *lds_ptr<f32x4>(in + QT * 4 + 32 * i4);
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4) {
          const int i = 4 * i4 + e4;
          dp[i] = p[i] == 0.f ? 0.f : p[i] * (dp[i] - delta[e4]);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag<T> ds = as_operand(dp, c, (Frag<T> *)nullptr);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) mma(gk[db], L::col_frag(q_at + col_at, c, db), ds);
      }
    }
  }
  if (!exists) return;
  // the two gradients may be one tensor (the same tensor as keys and values): one after the other, by the same lane
  emit_row<T, DP>(a.gk + row * sh.d, gk, sh.scale, valid, a.acc_k, sh.d, a.vec != 0, lane);
  emit_row<T, DP>(a.gv + row * sh.d, gv, 1.f, valid, a.acc_v, sh.d, a.vec != 0, lane);
}

template <typename T, int DP, bool DMA>
int launch(phip_ctx *ctx, BwArgs<T> a) {
  constexpr int BM = 32 * kWaves;
  constexpr int lds_q = 4 * kKeys<T> * Tile<T, DP>::kPitch;
  constexpr int lds_k = 4 * kRows<T> * Tile<T, DP>::kPitch + 4 * kRows<T> * 4;
  int rc = allow_lds<queries_kernel<T, DP, DMA>>(ctx, lds_q);
  if (rc == PHIP_OK) rc = allow_lds<keys_kernel<T, DP, DMA>>(ctx, lds_k);
  if (rc != PHIP_OK) return rc;
  const uint64_t blocks_q = slots(a.seq, BM, a.s.g, false) * a.s.hk, blocks_k = slots(a.seq, BM, 1, true) * a.s.hk;
  PHIP_REQUIRE(blocks_q < 0x7fffffffu && blocks_k < 0x7fffffffu, "too many rows");
  a.tiles = (uint32_t)(((uint64_t)a.seq.tq * a.s.g + BM - 1) / BM);
  hipLaunchKernelGGL((queries_kernel<T, DP, DMA>), dim3((uint32_t)blocks_q), dim3(kThreads), lds_q, ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  a.tiles = (uint32_t)((a.seq.tk + BM - 1) / BM);
  hipLaunchKernelGGL((keys_kernel<T, DP, DMA>), dim3((uint32_t)blocks_k), dim3(kThreads), lds_k, ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  return PHIP_OK;
}

template <typename T>
int dispatch(phip_ctx *ctx, const BwArgs<T> &a, bool dma) {
  switch ((a.s.d + 31) / 32) {
    case 1: return dma ? launch<T, 32, true>(ctx, a) : launch<T, 32, false>(ctx, a);
    case 2: return dma ? launch<T, 64, true>(ctx, a) : launch<T, 64, false>(ctx, a);
    case 3: return dma ? launch<T, 96, true>(ctx, a) : launch<T, 96, false>(ctx, a);
    default: return dma ? launch<T, 128, true>(ctx, a) : launch<T, 128, false>(ctx, a);
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
  const size_t nq = (size_t)d * hq * tq * bs * sizeof(T), nk = (size_t)d * hk * tk * bs * sizeof(T);
  const size_t ns = (size_t)hq * tq * bs * sizeof(float);
  auto is_read = [&](const void *g, size_t n) {
    return shares_memory(g, n, q, nq) || shares_memory(g, n, k, nk) || shares_memory(g, n, v, nk) ||
           shares_memory(g, n, y, nq) || shares_memory(g, n, gy, nq) || shares_memory(g, n, stats, ns);
  };
  PHIP_REQUIRE(!is_read(gq, nq) && !is_read(gk, nk) && !is_read(gv, nk), "a gradient shares memory with an operand");
  // the same tensor may be queries, keys and values, and then its one gradient is passed for each; anything in between
  // would have two lanes add to one element
  PHIP_REQUIRE((gk == gv || !shares_memory(gk, nk, gv, nk)) &&
                   ((const void *)gq == gk || !shares_memory(gq, nq, gk, nk)) &&
                   ((const void *)gq == gv || !shares_memory(gq, nq, gv, nk)),
               "two gradients overlap without being the same tensor");
  // gradients noted as zero and not yet filled are written instead of added into; gq is written before gk and gk before
  // gv, so of gradients that are one tensor the first takes the note
  a.acc_q = !zeros_take(ctx, gq, nq);
  a.acc_k = !zeros_take(ctx, gk, nk);
  a.acc_v = !zeros_take(ctx, gv, nk);
  PHIP_FLUSH_ZEROS(ctx);
  void *delta = nullptr;
  rc = phip_pool_alloc(ctx, ns, &delta, nullptr);
  if (rc != PHIP_OK) return rc;
  a.q = q;
  a.k = k;
  a.v = v;
  a.y = y;
  a.gy = gy;
  a.stats = stats;
  a.delta = static_cast<float *>(delta);
  a.gq = gq;
  a.gk = gk;
  a.gv = gv;
  auto vec = [&](const void *p) { return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0; };
  a.vec = d % 4 == 0 && vec(gq) && vec(gk) && vec(gv);
  rc = dispatch<T>(ctx, a, rows_movable(d, sizeof(T), {q, k, v, gy}));
  phip_pool_free(ctx, delta);
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
