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
  // key ranges (few rows): keys per range, partial results
  uint32_t chunk;
  uint32_t splits;      // ranges of the longest sequence; a workgroup for each range of each tile, or,
  uint32_t listed;      // if not 0: workgroups for the ranges that the listed sequences have (see find_range): their slots
  uint32_t part_rows;   // rows of a tile that exist at most
  float *partial;       // per tile and range: part_rows x (DP sums, maximum, sum, 2 unused)
  uint32_t *tickets;
};

// The state of 32 rows of a wavefront: the running maximum (raw scores) and sum, and the unnormalised result transposed
// (block db holds elements 32 db .. + 31 of the head, rows across).
template <int DP>
struct Rows {
  f32x16 o[DP / 32];
  float m, l;           // l: this half's keys only, raised like the result
};

// One step over 32 KB keys whose rows lie in LDS, in three parts.  The scores:
template <int KB>
struct Scores {
  f32x16 s[KB];
};
template <typename T, int DP, int KB>
__device__ inline void scores(Scores<KB> &sc, const Frag<T> (&qf)[DP / 16], uint32_t k_at) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    sc.s[kb] = f32x16{};
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) mma(sc.s[kb], Tile<T, DP>::row_frag(k_at, kb, c), qf[c]);
  }
}

// The running softmax: the scores become exp(score - maximum), raised by kRaise.  lim: keys below it are visible to the
// lane's row.
template <typename T, int DP, int KB>
__device__ inline void softmax(Rows<DP> &st, Scores<KB> &sc, int key0, int lim, bool masked, float scale_log2, int lane) {
  f32x16 (&s)[KB] = sc.s;
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
  const float raised = base - kRaise<T>;
  float sum = 0.f;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[kb][i] = exp2_fast(fmaf(s[kb][i], scale_log2, -raised));
      sum += s[kb][i];
    }
  st.l += sum;
}

// A value of a masked key may be infinite or no number: 0 times it must not reach the rows that do not see the key.  Tells
// whether any of the fragment's elements is one.
template <typename T>
__device__ inline bool not_finite(const Frag16<T> &f) {
  constexpr uint32_t kOnes = __is_same(T, bf16_t) ? 0x7f80u : 0x7c00u;
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t w = f.v[e];
    bad = bad || (w & kOnes) == kOnes || ((w >> 16) & kOnes) == kOnes;
  }
  return bad;
}
__device__ inline bool not_finite(const f32x8 &f) {
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) bad = bad || !(fabsf(f[j]) <= 3.4028234e38f);
  return bad;
}
// The fragment with only element j of half h kept.
template <typename T>
__device__ inline Frag16<T> only(const Frag16<T> &f, int j, bool mine) {
  Frag16<T> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.v[e] = mine && e == (j >> 1) ? f.v[e] & ((j & 1) ? 0xffff0000u : 0xffffu) : 0u;
  return r;
}
__device__ inline f32x8 only(const f32x8 &f, int j, bool mine) {
  f32x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = mine && e == j ? f[e] : 0.f;
  return r;
}

// The product with the values of a tile that holds masked keys.  If all values are finite it is the plain product; if not,
// key after key is added to the rows that see it (slow, and rare: a value that is no number spoils the result anyway, only
// not of the rows before it).
template <typename T, int DP, int KB>
__device__ inline bool values_masked(Rows<DP> &st, const Scores<KB> &sc, uint32_t v_at, int key0, int lim, int lane) {
  bool bad = false;
#pragma unroll
  for (int rc = 0; rc < 2 * KB; ++rc)
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) bad = bad || not_finite(Tile<T, DP>::col_frag(v_at, rc, db));
  if (!__any(bad)) return false;
#pragma unroll
  for (int rc = 0; rc < 2 * KB; ++rc) {
    const Frag<T> p = as_operand(sc.s[rc / 2], rc % 2, (Frag<T> *)nullptr);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
      const Frag<T> v = Tile<T, DP>::col_frag(v_at, rc, db);
#pragma unroll 1
      for (int k = 0; k < 16; ++k) {
        const int h = k >> 3, j = k & 7, key = key0 + 16 * rc + (j & 3) + 8 * (j >> 2) + 4 * h;
        f32x16 one = f32x16{};
        mma(one, only(v, j, (lane >> 5) == h), only(p, j, (lane >> 5) == h));
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[db][i] += key < lim ? one[i] : 0.f;
      }
    }
  }
  return true;
}

// What the rounding of an operand left out, rounded in turn.
template <typename T>
__device__ inline Frag16<T> left_out(const f32x16 &p, int c, const Frag16<T> &f) {
  Frag16<T> r;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    r.v[e] = round_pair<T>(p[8 * c + 2 * e] - element(f, 2 * e), p[8 * c + 2 * e + 1] - element(f, 2 * e + 1));
  return r;
}

// The product with the values.  EXACT (16-bit storage): the probabilities in two parts, which together carry 16 bits (bf16) or
// 22 (fp16).  Taken where a sequence's rows are one tile, the single tokens of a serving loop: those calls wait for memory, so
// the second product costs 1 to 2 % (one token of 16 streams of 1 to 8192 keys, 32/8 heads of 128, bf16: 55.1 -> 56.2 us; 130001
// keys, fp16: 104.2 -> 105.1) and the result is as far from the exact one as its own rounding (root mean square error 1.27 and
// 1.33 -> 1.0 times that).  Prompts are bound by the products and the vector instructions and take one part.
template <typename T, int DP, int KB, bool EXACT>
__device__ inline void values(Rows<DP> &st, const Scores<KB> &sc, uint32_t v_at) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const Frag<T> p = as_operand(sc.s[kb], c, (Frag<T> *)nullptr);
      if constexpr (EXACT) {
        const Frag<T> rest = left_out<T>(sc.s[kb], c, p);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) {
          const Frag<T> v = Tile<T, DP>::col_frag(v_at, 2 * kb + c, db);
          mma(st.o[db], v, p);
          mma(st.o[db], v, rest);
        }
      } else {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) mma(st.o[db], Tile<T, DP>::col_frag(v_at, 2 * kb + c, db), p);
      }
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
// Tile t + 1 is on its way while tile t is worked on (two stages of K and V, one barrier per tile; 64 KiB of LDS and at most
// 256 registers, so that two workgroups share a CU and one's products run beside the other's exponentials).
// Bound by the two pipes: 16 Ki packed tokens, 32/8 heads of 128, bf16, causal: 889 us, 920 TFLOP/s, the matrix pipe busy 43 %
// and the vector pipe 51 % of the time (an exponential per score costs about what its 4 x 128 flops do); fp32, 8 x 2048
// tokens, 16 heads of 64: 556 us, 124 TFLOP/s of the 139 that a large product reaches.
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
  if ((uint64_t)at.t * BM >= (uint64_t)tokens * sh.g) return;
  const int lq = behind ? 0 : (int)e.q_len, lk = (int)e.k_len, g = (int)sh.g;
  const int r0 = (int)at.t * BM, rows = lq * g;

  // the lane's row
  const uint32_t r = (uint32_t)(r0 + 32 * wave + (lane & 31)), tok = r / sh.g;
  const bool exists = tok < tokens, valid = exists && (int)tok < lq;
  const size_t row = ((sample * a.seq.tq + token0 + (exists ? tok : 0)) * sh.hq + head * sh.g + (r - tok * sh.g));
  const int lim = !valid ? 0 : sh.causal ? min(lk, max(0, (int)tok + lk - lq + 1)) : lk;

  // keys that any row of the workgroup, all rows of the wavefront, any row of the wavefront sees
  auto seen_by = [&](int rr) { return sh.causal ? min(lk, max(0, rr / g + lk - lq + 1)) : lk; };
  const int last = min(rows, r0 + BM) - 1, wg_keys = last < r0 ? 0 : seen_by(last);
  const int w_first = r0 + 32 * wave, w_last = min(rows - 1, w_first + 31);
  const int w_keys = w_last < w_first ? 0 : seen_by(w_last), w_all = w_last < w_first ? 0 : seen_by(w_first);

  Frag<T> qf[DP / 16];
  load_row<T>(qf, a.q + row * sh.d, valid, sh, lane);

  Rows<DP> st;
  reset(st);
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
      if (!sh.whole) {  // the parts of the tile that this thread cleans may be another wavefront's
        __syncthreads();
        Loader::clean(stage, (int)sh.d, tid);
      }
    } else {
      lk_.put(stage, tid);
      lv_.put(stage + kTile, tid);
    }
    __syncthreads();  // tile t is in LDS, and nobody reads the other stage any more
    if (t + 1 < n) fetch(t + 1);
    if (t * KT < w_keys) {
      Scores<KT / 32> sc;
      scores<T, DP, KT / 32>(sc, qf, stage + row_at);
      softmax<T, DP, KT / 32>(st, sc, t * KT, lim, (t + 1) * KT > w_all, sh.scale_log2, lane);
      const bool masked = (t + 1) * KT > w_all;
      if (!masked || !values_masked<T, DP, KT / 32>(st, sc, stage + kTile + col_at, t * KT, lim, lane))
        values<T, DP, KT / 32, false>(st, sc, stage + kTile + col_at);
    }
  }

  const float l = halves_sum(st.l);
  if (!exists) return;
  store_row<T, DP>(a.y + row * sh.d, st.o, 1.f / l, valid && l != 0.f, sh.d, a.vec_y != 0, lane);
  if (a.stats != nullptr && lane < 32) a.stats[row] = !valid || l == 0.f ? -INFINITY : fmaf(st.m, sh.scale, logf(l * kLower<T>));
}

// Few rows (a new token per sequence against its cache, short prompts): what takes the time is reading the keys and values
// once, so a workgroup takes 32 rows and a range of the keys, its four wavefronts take blocks of 32 keys in turn, and the
// partial results (maximum, sum, unnormalised rows) meet in LDS, and between the ranges of a tile in memory: the workgroup
// that finishes last of a tile's ranges merges them in order.
//
// Every wavefront has a ring of LDS tiles of its own and waits for nobody else: K and V blocks alternate in it, and the
// block `kRing` positions ahead is ordered as soon as a block has been used, so that up to three quarters of 128 KiB are on
// their way to every CU.  Bound by memory: one token against 130001 keys, 8 key heads of 128, fp16: 105 us, 5.1 TB/s, the
// rate of a large copy; one token of 16 streams against 1 to 8192 keys: 56 us, 3.9 TB/s.
template <typename T, int DP, int W>
constexpr int kFewLds = W * std::max(2 * kStages<T, DP> * 32 * Tile<T, DP>::kPitch, (DP * 33 + 64) * 4);

// Device-scope accesses for what travels between workgroups, which may sit behind different L2 caches.
__device__ inline void store_shared(float *p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ inline float load_shared(const float *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// True in the workgroup that is the last of `count` to get here.  Each lane waits until memory has acknowledged its own
// stores, the barrier puts all of them before thread 0's ticket, and the ticket is a device-scope atomic on one address,
// so whoever draws the last one finds what the others stored.  The counter is left zeroed for the next launch.
__device__ inline bool last_of_tile(uint32_t *ticket, uint32_t count, uint32_t *flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t drawn = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const bool last = drawn == count - 1u;
    if (last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last ? 1u : 0u;
  }
  __syncthreads();
  return *flag != 0;
}

// Which tile and range of keys a workgroup of the kernel for few rows takes, and where the tile's partial results and its
// ticket lie.
struct RangePlace {
  Place at;
  uint32_t range;
  uint32_t part, step;  // partial result of the tile's first range, and how far the next is behind it
  uint32_t ticket;
};

// listed == 0: every tile has `splits` ranges, of which a short sequence leaves most without work.  Otherwise entry i of the
// list, with k_cum keys before it, owns the slots from floor(k_cum / chunk) + i on, which is room for its ranges (as in
// find_place for tiles), and a slot has `tiles` tiles; behind the slots come the tiles of tokens of no sequence.
template <typename T>
__device__ inline RangePlace find_range(const FwArgs<T> &a, uint32_t index, uint32_t head, int lane) {
  const Shape &sh = a.s;
  if (a.listed == 0) {
    const uint32_t slot = index / a.splits, tile = slot * sh.hk + head;
    return {find_place(a.seq, slot, a.tiles, 32, sh.g, false, sh.causal != 0), index - slot * a.splits, tile * a.splits, 1,
            tile};
  }
  const uint32_t slot = index / a.tiles, t = index - slot * a.tiles;
  if (slot >= a.listed)
    return {{{kNoSequence, 0, 0, 0, 0, 0, 0, 0}, uniform(index - a.listed * a.tiles)}, 0, 0, 0, 0};
  // the last entry whose first slot is not behind `slot`: 64 candidates at a time, one per lane
  uint32_t lo = 0, count = a.seq.n;
  while (count > 1) {
    const uint32_t stride = (count + 63) / 64, i = lo + (uint32_t)lane * stride;
    const bool mine = (uint32_t)lane * stride < count && a.seq.entries[i].k_cum / a.chunk + i <= slot;
    const uint32_t found = (uint32_t)__popcll(__ballot(mine)) - 1;  // lane 0's is true
    lo += found * stride;
    count = min(stride, count - found * stride);
  }
  lo = uniform(lo);
  const SequenceEntry e = uniform(a.seq.entries[lo]);
  const uint32_t first = e.k_cum / a.chunk + lo;
  const uint32_t own = a.seq.packed ? (uint32_t)(((uint64_t)e.q_len * sh.g + 31) / 32) : a.tiles;
  return {{e, uniform(sh.causal && t < own ? own - 1 - t : t)}, slot - first, (first * a.tiles + t) * sh.hk + head,
          a.tiles * sh.hk, (lo * a.tiles + t) * sh.hk + head};
}

template <typename T, int DP, bool DMA, int W, bool EXACT>
__global__ __launch_bounds__(64 * W, 1) void few_kernel(const FwArgs<T> a) {
  constexpr int BM = 32, S = kStages<T, DP>, kThreads = 64 * W;
  typedef Tile<T, DP> L;
  typedef TileLoader<T, DP, 32, 64, DMA> Loader;
  constexpr uint32_t kTile = (uint32_t)Loader::kBytes;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  __shared__ uint32_t flag;
  const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) unsigned char *)lds;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Shape &sh = a.s;
  const uint32_t head = blockIdx.x % sh.hk;
  const RangePlace place = find_range(a, blockIdx.x / sh.hk, head, lane);
  const Place &at = place.at;
  const uint32_t range = place.range;
  const SequenceEntry &e = at.e;
  const bool behind = e.sample == kNoSequence;
  const uint32_t token0 = behind ? a.seq.q_total : e.q_start;
  const size_t sample = behind ? 0 : e.sample;
  const uint32_t tokens = behind ? a.seq.tq - a.seq.q_total : a.seq.packed ? e.q_len : a.seq.tq;
  if ((uint64_t)at.t * BM >= (uint64_t)tokens * sh.g) return;
  const int lq = behind ? 0 : (int)e.q_len, lk = (int)e.k_len, g = (int)sh.g;
  const int r0 = (int)at.t * BM, rows = min((int)(tokens * sh.g) - r0, BM), filled = min(lq * g - r0, BM);

  // the lane's row; keys that it, any row and all rows of the tile see
  auto seen_by = [&](int rr) { return sh.causal ? min(lk, max(0, rr / g + lk - lq + 1)) : lk; };
  const bool exists = (lane & 31) < rows, valid = (lane & 31) < filled;
  const int lim = valid ? seen_by(r0 + (lane & 31)) : 0;
  const int keys = filled <= 0 ? 0 : seen_by(r0 + filled - 1), first_sees = filled <= 0 ? 0 : seen_by(r0);
  const int all = filled < BM ? 0 : first_sees;
  const uint32_t ranges = max(1u, ((uint32_t)keys + a.chunk - 1) / a.chunk);
  if (range >= ranges) return;
  const int from = (int)(range * a.chunk), to = min(keys, from + (int)a.chunk);

  const RowWalk walk((uint32_t)r0, sh);
  const size_t row_base = (sample * a.seq.tq + token0) * sh.hq + head * sh.g;
  Frag<T> qf[DP / 16];
  {
    const size_t row = row_base + walk.at(exists ? lane & 31 : 0, sh.hq);
    load_row<T>(qf, a.q + row * sh.d, valid, sh, lane);
  }
  Rows<DP> st;
  reset(st);
  const uint32_t stride = sh.hk * sh.d;
  const T *kp = a.k + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const T *vp = a.v + ((sample * a.seq.tk + e.k_start) * sh.hk + head) * (size_t)sh.d;
  const uint32_t ring = lds0 + (uint32_t)wave * (2 * S * kTile);
  const uint32_t row_at = L::row_lane(lane), col_at = L::col_lane(lane);
  Loader lk_, lv_;
  lk_.init(1, stride, 0, lane);
  lv_ = lk_;
  auto fetch_k = [&](int key, int s) {
    lk_.fetch(kp + (size_t)min(key, to) * stride, to - key, 0, 1, 1u << 22, stride, 0, (int)sh.d, ring + (uint32_t)s * 2 * kTile, lane);
  };
  auto fetch_v = [&](int key, int s) {
    lv_.fetch(vp + (size_t)min(key, to) * stride, to - key, 0, 1, 1u << 22, stride, 0, (int)sh.d, ring + (uint32_t)s * 2 * kTile + kTile, lane);
  };
  constexpr int kStep = 32 * W;
  int key = from + 32 * wave;
  if constexpr (DMA) {
    // blocks past the end are ordered too (they read nothing and write zeros), so that the waits count the same
    constexpr int kInFlight = (2 * S - 1) * Loader::kInstr;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      fetch_k(key + s * kStep, s);
      fetch_v(key + s * kStep, s);
    }
    arrived(qf);
    for (int s = 0; key < to; key += kStep, s = s + 1 == S ? 0 : s + 1) {
      const uint32_t stage = ring + (uint32_t)s * 2 * kTile;
      wait_loads<kInFlight>();
      if (!sh.whole) Loader::clean(stage, (int)sh.d, lane);
      Scores<1> sc;
      scores<T, DP, 1>(sc, qf, stage + row_at);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the block's reads are done before its place is filled again
      fetch_k(key + S * kStep, s);
      softmax<T, DP, 1>(st, sc, key, lim, key + 32 > all, sh.scale_log2, lane);
      wait_loads<kInFlight>();
      if (key + 32 <= first_sees || !values_masked<T, DP, 1>(st, sc, stage + kTile + col_at, key, lim, lane))
        values<T, DP, 1, EXACT>(st, sc, stage + kTile + col_at);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      fetch_v(key + S * kStep, s);
    }
    wait_loads<0>();  // nothing may land in the LDS that is used for something else below
  } else {
    if (key < to) {
      fetch_k(key, 0);
      fetch_v(key, 0);
    }
    for (; key < to; key += kStep) {
      lk_.put(ring, lane);
      lv_.put(ring + kTile, lane);
      if (key + kStep < to) {
        fetch_k(key + kStep, 0);
        fetch_v(key + kStep, 0);
      }
      Scores<1> sc;
      scores<T, DP, 1>(sc, qf, ring + row_at);
      softmax<T, DP, 1>(st, sc, key, lim, key + 32 > all, sh.scale_log2, lane);
      if (key + 32 <= first_sees || !values_masked<T, DP, 1>(st, sc, ring + kTile + col_at, key, lim, lane))
        values<T, DP, 1, EXACT>(st, sc, ring + kTile + col_at);
    }
  }

  if constexpr (W == 1) {  // nothing to merge (the keys are not divided either): as the kernel for many rows
    const float l = halves_sum(st.l);
    if (!exists) return;
    const size_t row = row_base + walk.at(lane & 31, sh.hq);
    store_row<T, DP>(a.y + row * sh.d, st.o, 1.f / l, valid && l != 0.f, sh.d, a.vec_y != 0, lane);
    if (a.stats != nullptr && lane < 32) a.stats[row] = !valid || l == 0.f ? -INFINITY : fmaf(st.m, sh.scale, logf(l * kLower<T>));
    return;
  }
  // the wavefronts' results: per wavefront DP columns of 33 floats (rows across), then 32 maxima and 32 sums
  __syncthreads();
  float *const area = reinterpret_cast<float *>(lds);
  constexpr int kPer = DP * 33 + 64;
  {
    float *mine = area + wave * kPer;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) mine[(32 * db + block_row(i) + 4 * (lane >> 5)) * 33 + (lane & 31)] = st.o[db][i];
    const float l = halves_sum(st.l);
    if (lane < 32) {
      mine[DP * 33 + lane] = valid ? st.m : -INFINITY;
      mine[DP * 33 + 32 + lane] = valid ? l : 0.f;
    }
  }
  __syncthreads();
  const bool whole = ranges == 1;
  const size_t part_size = (size_t)a.part_rows * (DP + 4);
  float *const all_parts = a.partial + place.part * part_size, *const part = all_parts + (size_t)range * place.step * part_size;
  // four elements of a row
  auto finish = [&](int row, uint32_t dd, const float (&o)[4], float m, float l) {
    const size_t at_row = row_base + walk.at((uint32_t)row, sh.hq);
    const float f = l == 0.f ? 0.f : 1.f / l;
    const float four[4] = {o[0] * f, o[1] * f, o[2] * f, o[3] * f};
    if (dd < sh.d) store4<T, false>(a.y + at_row * sh.d + dd, four, (int)(sh.d - dd), a.vec_y != 0);
    if (dd == 0 && a.stats != nullptr) a.stats[at_row] = l == 0.f ? -INFINITY : fmaf(m, sh.scale, logf(l * kLower<T>));
  };
  for (uint32_t i = tid; i < (uint32_t)rows * (DP / 4); i += kThreads) {
    const int row = (int)(i / (DP / 4));
    const uint32_t dd = i % (DP / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, area[w * kPer + DP * 33 + row]);
    const float base = m == -INFINITY ? 0.f : m * sh.scale_log2;
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float *his = area + w * kPer;
      const float lw = his[DP * 33 + 32 + row];
      // a wavefront that has seen no key of this row has a sum of 0 and its rows are 0
      const float f = lw == 0.f ? 0.f : exp2_fast(fmaf(his[DP * 33 + row], sh.scale_log2, -base));
      l = fmaf(lw, f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = lw == 0.f ? o[e] : fmaf(his[(dd + e) * 33 + row], f, o[e]);
    }
    if (whole) {
      finish(row, dd, o, m, l);
    } else {
      float *p = part + row * (DP + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) store_shared(p + dd + e, o[e]);
      if (dd == 0) {
        store_shared(p + DP, m);
        store_shared(p + DP + 1, l);
      }
    }
  }
  if (whole || !last_of_tile(a.tickets + place.ticket, ranges, &flag)) return;
  // The last of the tile: each thread has an element of a row at a time and takes the ranges 16 at a time, all their
  // loads in flight together.
  for (uint32_t i = tid; i < (uint32_t)rows * DP; i += kThreads) {
    const int row = (int)(i / DP);
    const uint32_t dd = i % DP;
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (uint32_t p0 = 0; p0 < ranges; p0 += 16) {
      float pm[16], pl[16], po[16];
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) {
        const float *p = all_parts + (size_t)min(p0 + u, ranges - 1) * place.step * part_size + row * (DP + 4);
        pm[u] = load_shared(p + DP);
        pl[u] = load_shared(p + DP + 1);
        po[u] = load_shared(p + dd);
      }
      float top = m;
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) top = fmaxf(top, pm[u]);
      const float base = top == -INFINITY ? 0.f : top * sh.scale_log2;
      const float f = l == 0.f ? 0.f : exp2_fast(fmaf(m, sh.scale_log2, -base));
      l *= f;
      o *= f;
      m = top;
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) {
        const bool none = p0 + u >= ranges || pl[u] == 0.f;
        const float fu = none ? 0.f : exp2_fast(fmaf(pm[u], sh.scale_log2, -base));
        l = none ? l : fmaf(pl[u], fu, l);
        o = none ? o : fmaf(po[u], fu, o);
      }
    }
    if (dd >= sh.d) continue;
    const size_t at_row = row_base + walk.at((uint32_t)row, sh.hq);
    a.y[at_row * sh.d + dd] = from_f32<T>(l == 0.f ? 0.f : o / l);
    if (dd == 0 && a.stats != nullptr) a.stats[at_row] = l == 0.f ? -INFINITY : fmaf(m, sh.scale, logf(l * kLower<T>));
  }
}

template <typename T, int DP, bool DMA>
int launch_rows(phip_ctx *ctx, FwArgs<T> a) {
  constexpr int BM = 32 * kWaves;
  constexpr int lds = 4 * kKeys<T> * Tile<T, DP>::kPitch;
  a.tiles = (uint32_t)(((uint64_t)a.seq.tq * a.s.g + BM - 1) / BM);
  const uint64_t blocks = slots(a.seq, BM, a.s.g, false) * a.s.hk;
  PHIP_REQUIRE(launchable(blocks, kThreads), "too many rows");
  const int rc = allow_lds<rows_kernel<T, DP, DMA>>(ctx, lds);
  if (rc != PHIP_OK) return rc;
  hipLaunchKernelGGL((rows_kernel<T, DP, DMA>), dim3((uint32_t)blocks), dim3(kThreads), lds, ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  note_kernel(ctx, "attention_rows");
  return PHIP_OK;
}

// Keys per range of the kernel for few rows.  One workgroup of four wavefronts fits on a CU (its ring of tiles), so the
// time is about the keys of a range times the rounds that the ranges take on the chip: a range is a CU's share of all keys,
// and where the longest sequence is less than two shares it is left whole, because its second range would wait for a CU.
// One token each, 32/8 heads of 128, bf16, us whole -> cut: 17 streams of 4096 keys (1.9 shares) 50 -> 64, 31 of them (1.03)
// 51 -> 102, 32 streams of 1 to 8192 (1.8) 92 -> 117; four of 8192 beside 60 of 1000 (2.8) 90 -> 58, one of 8192 beside 31 of
// 512 (11) 89 -> 25.
uint32_t few_chunk(phip_ctx *ctx, const SequenceView &view, const phip_sequences *seqs, uint64_t tiles) {
  const uint64_t cus = (uint64_t)ctx->prop.multiProcessorCount;
  const uint64_t most = seqs != nullptr ? seqs->max_k : view.tk;
  const uint64_t sum = seqs != nullptr ? seqs->k_sum : (uint64_t)view.n * view.tk;
  const uint64_t share = sum * tiles / view.n / cus;
  if (most < 2 * share || tiles > (uint64_t)kTicketSlots) return (uint32_t)most + 1;
  return (uint32_t)std::min<uint64_t>((std::max<uint64_t>(share, 256) + 127) / 128 * 128, 1u << 30);
}

template <typename T, int DP, bool DMA, int W, bool EXACT = false>
int launch_few(phip_ctx *ctx, FwArgs<T> a, const phip_sequences *seqs) {
  constexpr int lds = kFewLds<T, DP, W>;
  const int rc = allow_lds<few_kernel<T, DP, DMA, W, EXACT>>(ctx, lds);
  if (rc != PHIP_OK) return rc;
  a.tiles = (uint32_t)(((uint64_t)a.seq.tq * a.s.g + 31) / 32);
  const uint64_t tiles = slots(a.seq, 32, a.s.g, false) * a.s.hk;
  const uint32_t most = seqs != nullptr ? seqs->max_k : a.seq.tk;
  a.chunk = W == 1 ? most + 1 : few_chunk(ctx, a.seq, seqs, tiles);
  a.splits = most <= a.chunk ? 1 : (most + a.chunk - 1) / a.chunk;
  uint64_t blocks = tiles * a.splits, parts = blocks;
  const uint64_t most_rows = std::max<uint64_t>(1, (uint64_t)(a.seq.packed ? seqs->max_q : a.seq.tq) * a.s.g);
  a.part_rows = (uint32_t)std::min<uint64_t>(32, most_rows);
  if (a.splits > 1 && seqs != nullptr && seqs->k_sum <= 0xffffffffu) {
    // One long sequence among many short ones: its ranges times all tiles would be mostly empty workgroups, each with a place
    // in the scratch memory (131072 keys beside 127 times 64, one key head: 512 MB and 137 us; listed 4 MB and 62 us).  With
    // fewer than four places per range that exists the plain order is the faster one (31 streams of 1 to 8192 keys, 8 key
    // heads, 2.5 places: 67 us, listed 80).
    const uint64_t per = (most_rows + 31) / 32, listed = seqs->k_sum / a.chunk + a.seq.n, own = listed * per * a.s.hk;
    const uint64_t behind = a.seq.packed ? ((uint64_t)(a.seq.tq - a.seq.q_total) * a.s.g + 31) / 32 * a.s.hk : 0;
    if (4 * (own + behind) <= blocks && a.seq.n * per * a.s.hk <= (uint64_t)kTicketSlots) {
      a.listed = (uint32_t)listed;
      a.tiles = (uint32_t)per;
      blocks = own + behind;
      parts = own;
    }
  }
  PHIP_REQUIRE(launchable(blocks, 64 * W), "too many rows");
  void *partial = nullptr;
  if (a.splits > 1) {
    const int rc2 = phip_pool_alloc(ctx, (size_t)parts * a.part_rows * (DP + 4) * sizeof(float), &partial, nullptr);
    if (rc2 != PHIP_OK) return rc2;
    a.partial = static_cast<float *>(partial);
    a.tickets = tile_tickets(ctx);
  }
  hipLaunchKernelGGL((few_kernel<T, DP, DMA, W, EXACT>), dim3((uint32_t)blocks), dim3(64 * W), lds, ctx->stream, a);
  const hipError_t e = hipGetLastError();
  if (partial != nullptr) phip_pool_free(ctx, partial);
  if (e != hipSuccess) return fail(PHIP_ERR_RUNTIME, "launching the attention kernel failed: %s", hipGetErrorString(e));
  note_kernel(ctx, W == 1 ? "attention_few1" : a.listed ? "attention_few_listed" : a.splits > 1 ? "attention_few_split" : "attention_few");
  return PHIP_OK;
}

template <typename T, int DP, bool DMA>
int launch(phip_ctx *ctx, const FwArgs<T> &a, const phip_sequences *seqs) {
  const uint64_t wide = slots(a.seq, 128, a.s.g, false) * a.s.hk, narrow = slots(a.seq, 32, a.s.g, false) * a.s.hk;
  const uint64_t most = (uint64_t)(seqs != nullptr ? seqs->max_q : a.seq.tq) * a.s.g;
  Way way = choose_way<T>(ctx, wide, narrow, most, seqs != nullptr ? seqs->max_k : a.seq.tk);
  if (way == Way::Shared && most <= 32) way = Way::Four;
  if constexpr (sizeof(T) == 4) {
    if (way == Way::One) return launch_few<T, DP, DMA, 1>(ctx, a, seqs);
  }
  if (way == Way::Four) {
    if constexpr (sizeof(T) == 2) {  // a tile per sequence
      if ((a.seq.packed ? most : (uint64_t)a.seq.tq * a.s.g) <= 32) return launch_few<T, DP, DMA, 4, true>(ctx, a, seqs);
    }
    return launch_few<T, DP, DMA, 4>(ctx, a, seqs);
  }
  return launch_rows<T, DP, DMA>(ctx, a);
}

template <typename T, bool DMA>
int dispatch(phip_ctx *ctx, const FwArgs<T> &a, const phip_sequences *seqs) {
  switch ((a.s.d + 31) / 32) {
    case 1: return launch<T, 32, DMA>(ctx, a, seqs);
    case 2: return launch<T, 64, DMA>(ctx, a, seqs);
    case 3: return launch<T, 96, DMA>(ctx, a, seqs);
    default: return launch<T, 128, DMA>(ctx, a, seqs);
  }
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
  PHIP_REQUIRE(elements_aligned(sizeof(T), {q, k, v, y}) && elements_aligned(4, {stats}),
               "an address is no multiple of the element size");
  const size_t ny = (size_t)d * hq * tq * bs * sizeof(T), nk = (size_t)d * hk * tk * bs * sizeof(T);
  const size_t ns = (size_t)hq * tq * bs * sizeof(float);
  PHIP_REQUIRE(!shares_memory(y, ny, q, ny) && !shares_memory(y, ny, k, nk) && !shares_memory(y, ny, v, nk),
               "the result shares memory with an operand");
  PHIP_REQUIRE(stats == nullptr || (!shares_memory(stats, ns, q, ny) && !shares_memory(stats, ns, k, nk) &&
                                    !shares_memory(stats, ns, v, nk) && !shares_memory(stats, ns, y, ny)),
               "stats share memory with an operand or the result");
  a.q = q;
  a.k = k;
  a.v = v;
  a.y = y;
  a.stats = stats;
  a.vec_y = d % 4 == 0 && reinterpret_cast<uintptr_t>(y) % (4 * sizeof(T)) == 0;
  a.s.whole = rows_aligned(d, sizeof(T), 16, {q, k, v});
  // fp32 rows are always whole dwords; 16-bit rows of an odd size are not
  if constexpr (sizeof(T) == 2) {
    if (!rows_aligned(d, sizeof(T), 4, {q, k, v})) return dispatch<T, false>(ctx, a, seqs);
  }
  return dispatch<T, true>(ctx, a, seqs);
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
