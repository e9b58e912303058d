// Attention forward: y = softmax(scale q k^T) v per sequence and head, with the running maximum and sum of the softmax
// (one pass over the keys; the scores are never in memory).
//
// The heads that share a key head are rows of the same problem: row r of a (sequence, key head) pair is query token
// r / g, head r % g of the group, so keys and values are read once for the group.
#include <algorithm>

#include "phip_attention.h"

namespace phip {
namespace attention {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;

template <typename T>
struct FwArgs {
  const T *q, *k, *v;
  T *y;
  float *stats;         // log of the sum of exponentials per row, may be null
  Shape s;
  SequenceView seq;
  uint32_t tiles;       // row tiles of a whole sample
  uint32_t vec_y;       // y's rows are aligned to four elements
  // key ranges (few rows): keys per range, ranges, partial results
  uint32_t chunk, splits;
  float *partial;       // per tile and range: rows x DP sums, then rows maxima, rows sums
  uint32_t *tickets;
};

// The state of 32 rows of a wavefront: the running maximum (raw scores) and sum, and the unnormalised result transposed
// (block db holds elements 32 db .. + 31 of the head, rows across).
template <int DP>
struct Rows {
  f32x16 o[DP / 32];
  float m, l;           // l: this half's keys only
};

// One step: 32 KB keys whose rows lie in LDS.  lim: keys below it are visible to the lane's row.
template <typename T, int DP, int KB>
__device__ inline void step(Rows<DP> &st, const Frag<T> (&qf)[DP / 16], uint32_t k_at, uint32_t v_at, int key0, int lim,
                            bool masked, float scale_log2, int lane) {
  typedef Tile<T, DP> L;
  f32x16 s[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    s[kb] = f32x16{};
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) mma(s[kb], L::row_frag(k_at, kb, c), qf[c]);
  }
  if (masked) {
    const int first = key0 + 4 * (lane >> 5);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[kb][i] = first + 32 * kb + block_row(i) < lim ? s[kb][i] : -INFINITY;
  }
  float mx = s[0][0];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
  mx = fmaxf(halves_max(mx), st.m);
  const float base = mx == -INFINITY ? 0.f : mx * scale_log2;  // a row that has seen no key yet stays empty
  if (__any(mx > st.m)) {
    const float alpha = exp2_fast(fmaf(st.m, scale_log2, -base));
    st.l *= alpha;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] *= alpha;
    st.m = mx;
  }
  float sum = 0.f;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[kb][i] = exp2_fast(fmaf(s[kb][i], scale_log2, -base));
      sum += s[kb][i];
    }
  st.l += sum;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Frag<T> p = as_operand(s[kb], c, (Frag<T> *)nullptr);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) mma(st.o[db], L::col_frag(v_at, 2 * kb + c, db), p);
    }
}

template <int DP>
__device__ inline void reset(Rows<DP> &st) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db) st.o[db] = f32x16{};
  st.m = -INFINITY;
  st.l = 0.f;
}

// Writes the lane's part of a row: x[db][i] * f, zeros for a row that saw no key.
template <typename T, int DP>
__device__ inline void store_row(T *row, const f32x16 (&x)[DP / 32], float f, bool some, uint32_t d, bool vec, int lane) {
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      const int d0 = 32 * db + 8 * i4 + 4 * (lane >> 5);
      float four[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) four[e] = some ? x[db][4 * i4 + e] * f : 0.f;
      if (d0 < (int)d) store4<T, false>(row + d0, four, (int)d - d0, vec);
    }
}

// Many rows: a workgroup of four wavefronts takes 128 rows, 32 per wavefront, and walks over the keys in tiles of KT.
// Tile t + 1 is on its way while tile t is worked on (two stages of K and V, one barrier per tile).
template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;

template <typename T, int DP, bool DMA>
__global__ __launch_bounds__(kThreads, 2) void rows_kernel(const FwArgs<T> a) {
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
  const uint32_t token0 = behind ? a.seq.q_total : e.q_start;  // of the sample
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tq - a.seq.q_total : a.seq.packed ? e.q_len : a.seq.tq;  // that this workgroup writes
  const int64_t r0 = (int64_t)at.t * BM;
  if (r0 >= (int64_t)tokens * sh.g) return;
  const int lq = behind ? 0 : (int)e.q_len, lk = (int)e.k_len;

  // the lane's row
  const int64_t r = r0 + 32 * wave + (lane & 31);
  const uint32_t tok = (uint32_t)(r / sh.g);
  const bool exists = tok < tokens, valid = exists && (int)tok < lq;
  const size_t row = ((sample * a.seq.tq + token0 + (exists ? tok : 0)) * sh.hq + head * sh.g + (uint32_t)(r % sh.g));
  const int lim = !valid ? 0 : sh.causal ? min(lk, max(0, (int)tok + lk - lq + 1)) : lk;

  // keys that any row of the workgroup, all rows of the wavefront, any row of the wavefront sees
  const int64_t last = min((int64_t)lq * sh.g, r0 + BM) - 1;
  const int wg_keys = last < r0 ? 0 : sh.causal ? min(lk, max(0, (int)(last / sh.g) + lk - lq + 1)) : lk;
  const int64_t w_first = r0 + 32 * wave, w_last = min((int64_t)lq * sh.g - 1, w_first + 31);
  int w_keys = 0, w_all = 0;
  if (w_last >= w_first) {
    w_keys = sh.causal ? min(lk, max(0, (int)(w_last / sh.g) + lk - lq + 1)) : lk;
    w_all = sh.causal ? min(lk, max(0, (int)(w_first / sh.g) + lk - lq + 1)) : lk;
  }

  Frag<T> qf[DP / 16];
#pragma unroll
  for (int c = 0; c < DP / 16; ++c)
    qf[c] = load_frag(a.q + row * sh.d, valid, 16 * c + 8 * (lane >> 5), (int)sh.d, (Frag<T> *)nullptr);

  Rows<DP> st;
  reset(st);
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
    __syncthreads();  // tile t is in LDS, and nobody reads the other stage any more
    if (t + 1 < n) fetch(t + 1);
    if (t * KT < w_keys)
      step<T, DP, KT / 32>(st, qf, stage + row_at, stage + kTile + col_at, t * KT, lim, (t + 1) * KT > w_all,
                           sh.scale_log2, lane);
  }

  const float l = halves_sum(st.l);
  if (!exists) return;
  store_row<T, DP>(a.y + row * sh.d, st.o, 1.f / l, valid && l != 0.f, sh.d, a.vec_y != 0, lane);
  if (a.stats != nullptr && lane < 32) a.stats[row] = !valid || l == 0.f ? -INFINITY : fmaf(st.m, sh.scale, logf(l));
}

template <typename T, int DP, bool DMA>
int launch_rows(phip_ctx *ctx, FwArgs<T> a) {
  constexpr int BM = 32 * kWaves;
  constexpr int lds = 4 * kKeys<T> * Tile<T, DP>::kPitch;
  a.tiles = (uint32_t)(((uint64_t)a.seq.tq * a.s.g + BM - 1) / BM);
  const uint64_t blocks = slots(a.seq, BM, a.s.g, false) * a.s.hk;
  PHIP_REQUIRE(blocks < 0x7fffffffu, "too many rows");
  const int rc = allow_lds<rows_kernel<T, DP, DMA>>(ctx, lds);
  if (rc != PHIP_OK) return rc;
  hipLaunchKernelGGL((rows_kernel<T, DP, DMA>), dim3((uint32_t)blocks), dim3(kThreads), lds, ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  return PHIP_OK;
}

template <typename T, int DP>
int launch(phip_ctx *ctx, const FwArgs<T> &a, bool dma) {
  return dma ? launch_rows<T, DP, true>(ctx, a) : launch_rows<T, DP, false>(ctx, a);
}

template <typename T>
int forward(phip_ctx *ctx, const T *q, const T *k, const T *v, T *y, float *stats, uint32_t d, uint32_t hq, uint32_t hk,
            uint32_t tq, uint32_t tk, uint32_t bs, const phip_sequences *seqs, int causal, float scale) {
  PHIP_ENTER(ctx);
  FwArgs<T> a = {};
  int rc = make_shape(d, hq, hk, tq, tk, bs, causal, scale, sizeof(T), &a.s);
  if (rc != PHIP_OK) return rc;
  rc = sequence_view(ctx, seqs, tq, tk, bs, true, &a.seq);
  if (rc != PHIP_OK) return rc;
  PHIP_REQUIRE(q != nullptr && k != nullptr && v != nullptr && y != nullptr, "null pointer");
  const size_t ny = (size_t)d * hq * tq * bs * sizeof(T), nk = (size_t)d * hk * tk * bs * sizeof(T);
  PHIP_REQUIRE(!shares_memory(y, ny, q, ny) && !shares_memory(y, ny, k, nk) && !shares_memory(y, ny, v, nk),
               "the result shares memory with an operand");
  a.q = q;
  a.k = k;
  a.v = v;
  a.y = y;
  a.stats = stats;
  a.vec_y = d % 4 == 0 && reinterpret_cast<uintptr_t>(y) % (4 * sizeof(T)) == 0;
  const bool dma = rows_movable(d, sizeof(T), {k, v});
  switch ((d + 31) / 32) {
    case 1: return launch<T, 32>(ctx, a, dma);
    case 2: return launch<T, 64>(ctx, a, dma);
    case 3: return launch<T, 96>(ctx, a, dma);
    default: return launch<T, 128>(ctx, a, dma);
  }
}

}  // namespace
}  // namespace attention
}  // namespace phip

using namespace phip;

extern "C" {

int phip_attention_fw_f32(phip_ctx *ctx, const float *q, const float *k, const float *v, float *y, float *stats,
                          uint32_t d, uint32_t hq, uint32_t hk, uint32_t tq, uint32_t tk, uint32_t bs,
                          const phip_sequences *seqs, int causal, float scale) {
  return attention::forward<float>(ctx, q, k, v, y, stats, d, hq, hk, tq, tk, bs, seqs, causal, scale);
}

#define PHIP_EXPORT_ATTENTION_FW(SUF, T)                                                                               \
  int phip_attention_fw_##SUF(phip_ctx *ctx, const void *q, const void *k, const void *v, void *y, float *stats,       \
                              uint32_t d, uint32_t hq, uint32_t hk, uint32_t tq, uint32_t tk, uint32_t bs,             \
                              const phip_sequences *seqs, int causal, float scale) {                                   \
    return attention::forward<T>(ctx, static_cast<const T *>(q), static_cast<const T *>(k), static_cast<const T *>(v), \
                                 static_cast<T *>(y), stats, d, hq, hk, tq, tk, bs, seqs, causal, scale);              \
  }

PHIP_EXPORT_ATTENTION_FW(f16, f16_t)
PHIP_EXPORT_ATTENTION_FW(bf16, bf16_t)

#undef PHIP_EXPORT_ATTENTION_FW

}  // extern "C"
