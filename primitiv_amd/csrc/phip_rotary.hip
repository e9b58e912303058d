// Rotary positions of queries and keys, with or without a norm of each head in the same pass, forward and gradients.
//
//   n = x                                     or  x r w with r = 1 / sqrt(mean(x^2) + eps) over the head's d elements
//   (y0, y1) = A (n0 cos a - n1 sin a, n1 cos a + n0 sin a) for the pairs of the first 2 `pairs` elements, y = n behind them
//   a = position * f[pair]
// and back: g = the rotation by -a of gy (times A), gw += sum over rows of g x r, gx += r (g w - x r^2 mean(g w x)).
//
// A streaming kernel: x (or gy and x) is read once, y (or gx) written once, and that is what bounds it.  A workgroup
// takes a few tokens with all their heads of queries and keys: the cosines and sines are the same for all heads, so they
// are computed once per token into LDS.  A row is spread over the fewest lanes that hold it at two 16-byte chunks each, one
// for either side of its pairs, so a pair never leaves its lane and the norm is a few exchanges between neighbours.
#include <algorithm>
#include <initializer_list>

#include "phip_pointwise.h"
#include "phip_sequences.h"

namespace phip {
namespace rotary {
namespace {

using pointwise::kBlock;

constexpr uint32_t kMostSize = 128;
constexpr int kMostTokens = 8;   // per workgroup and step

// One of the two tensors of a call: queries or keys.
template <typename T>
struct Side {
  const T *x;             // forward: the operand; backward: the same (norm only)
  const T *w;             // weights of the norm
  const T *gy;            // backward
  T *o;                   // y, or gx
  uint32_t heads, inv;    // inv: ceil(2^32 / heads), 0 for one head
  uint32_t acc;           // backward: add into what is there
  uint32_t blocks;        // workgroups that have tokens (and, with weights, leave sums)
  uint32_t tt;            // tokens per step of a workgroup
};

template <typename T>
struct Args {
  Side<T> side[2];        // queries, keys; blockIdx.y tells which
  float *partial;         // backward with weights: per workgroup of either side, d sums
  SequenceView seq;
  uint32_t tokens;        // tq * batch
  uint32_t d;
  uint32_t pairs, items, lanes;  // items: lanes of a row that have work; lanes: the power of two that a row takes
  int32_t first;
  float amplitude, eps;
  float f[kMostSize / 2];
};

// sin and cos of p * f.  The product and its reduction to an eighth of a turn take 64 bits: at position 10^6 a product
// rounded to 32 bits would be off by 0.03 radian.  What is left, |r| <= pi / 4, goes through the Taylor series (first
// dropped terms r^11 / 11! < 2e-9 and r^12 / 12! < 2e-10).
__device__ inline float2 turn(int64_t p, float f) {
  const double turns = (double)p * (double)f * 0.15915494309189533577;  // / (2 pi)
  const double part = turns - rint(turns);
  const double quarter = rint(part * 4.0);
  const float r = (float)((part - quarter * 0.25) * 6.28318530717958647693);
  const float r2 = r * r;
  const float s = fmaf(r * r2, fmaf(r2, fmaf(r2, fmaf(r2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), r);
  const float c = fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, fmaf(r2, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int q = (int)quarter & 3;
  const float c2 = (q & 1) ? s : c, s2 = (q & 1) ? c : s;
  return {q == 1 || q == 2 ? -c2 : c2, q >= 2 ? -s2 : s2};
}

// The position of token n of the batch, or false when it belongs to no sequence.
__device__ inline bool position(const SequenceView &s, uint32_t n, int32_t first, int64_t *p) {
  const uint32_t b = n / s.tq, t = n - b * s.tq;
  if (s.places == nullptr) {
    *p = (int64_t)first + t;
    return true;
  }
  uint32_t i = b;
  if (s.packed) {
    uint32_t lo = 0, hi = s.n;  // the last sequence that starts at or before t
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (s.places[mid].q_start <= t) lo = mid;
      else hi = mid;
    }
    i = lo;
  }
  const SequencePlace e = s.places[i];
  *p = (int64_t)first + e.shift + (t - e.q_start);
  return t - e.q_start < e.q_len;
}

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T v[V];
};

// A lane's part of a row: z[0 .. V) and z[V .. 2 V).
template <int V, bool INTER>
struct Place {
  uint32_t a, b;     // where the two chunks lie in the row
  bool use, use_b;   // the lane has work; its second chunk exists
  bool turns;        // its elements are rotated (else they lie behind the pairs)
  uint32_t angle;    // first of the lane's V angles

  __device__ inline Place(uint32_t l, uint32_t pairs, uint32_t items, uint32_t d) {
    use = l < items;
    turns = l < pairs / V;
    angle = turns ? V * l : 0;
    if (turns) {
      a = INTER ? 2 * V * l : V * l;
      b = INTER ? a + V : pairs + V * l;
    } else {
      a = use ? 2 * pairs + 2 * V * (l - pairs / V) : 0;
      b = a + V;
    }
    use_b = use && b < d;
    if (!use_b) b = a;
  }
};

template <typename T, int V>
__device__ inline void load_row(const T *row, uint32_t a, uint32_t b, bool use, bool use_b, float (&z)[2 * V]) {
  const Vec<T, V> x = *reinterpret_cast<const Vec<T, V> *>(row + a), y = *reinterpret_cast<const Vec<T, V> *>(row + b);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    z[i] = use ? to_f32(x.v[i]) : 0.f;
    z[V + i] = use_b ? to_f32(y.v[i]) : 0.f;
  }
}

template <typename T, int V>
__device__ inline void store_row(T *row, uint32_t a, uint32_t b, bool use, bool use_b, bool acc, const float (&z)[2 * V]) {
  auto put = [&](uint32_t at, int o) {
    Vec<T, V> *p = reinterpret_cast<Vec<T, V> *>(row + at);
    Vec<T, V> x;
    if (acc) {
      const Vec<T, V> old = *p;
#pragma unroll
      for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(to_f32(old.v[i]) + z[o + i]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x.v[i] = from_f32<T>(z[o + i]);
    }
    *p = x;
  };
  if (use) put(a, 0);
  if (use_b) put(b, V);
}

// z rotated by the angles at `at` (cosine, sine); sign: +1 forward, -1 back.
template <int V, bool INTER>
__device__ inline void rotate(float (&z)[2 * V], const float2 *at, float sign) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 cs = at[i];
    float &x0 = z[INTER ? 2 * i : i], &x1 = z[INTER ? 2 * i + 1 : V + i];
    const float s = cs.y * sign, a = x0, b = x1;
    x0 = fmaf(a, cs.x, -b * s);
    x1 = fmaf(b, cs.x, a * s);
  }
}

__device__ inline float row_sum(float x, uint32_t lanes) {
  for (uint32_t o = lanes / 2; o > 0; o >>= 1) x += __shfl_xor(x, (int)o);
  return x;
}

// Angles of the step's tokens into LDS (zeros for tokens of no sequence), and which tokens belong to one.
template <typename T>
__device__ inline void make_table(const Args<T> &a, uint32_t n0, uint32_t count, float2 *table, uint32_t *valid) {
  for (uint32_t i = threadIdx.x; i < count * a.pairs; i += kBlock) {
    const uint32_t t = i / a.pairs, j = i - t * a.pairs;
    int64_t p;
    const bool in = position(a.seq, n0 + t, a.first, &p);
    const float2 cs = in ? turn(p, a.f[j]) : float2{0.f, 0.f};
    table[t * (kMostSize / 2) + j] = {cs.x * a.amplitude, cs.y * a.amplitude};
  }
  if (threadIdx.x < count) {
    int64_t p;
    valid[threadIdx.x] = position(a.seq, n0 + threadIdx.x, a.first, &p) ? 1u : 0u;
  }
}

// BACK: gradients.  NORM: with the norm of each head.
//
// Queries and keys take workgroups of their own (one launch), so that a workgroup needs one set of weights and sums; the
// second computation of a token's angles costs less than the registers of the other set (gradients with 16/4 heads of 64:
// 143 registers per lane and 53 us with both in one workgroup, 4 x 16 Ki tokens).
template <typename T, int V, bool INTER, bool NORM, bool BACK>
__global__ __launch_bounds__(kBlock) void rotary_kernel(const Args<T> a) {
  __shared__ float2 table[kMostTokens * (kMostSize / 2)];
  __shared__ uint32_t valid[kMostTokens];
  // rows at a time, their loads in flight together (single elements: four, or two with a second operand)
  constexpr uint32_t U = V > 1 ? (NORM && BACK ? 1 : 2) : NORM && BACK ? 2 : 4;
  const Side<T> &side = a.side[blockIdx.y];
  if (blockIdx.x >= side.blocks) return;
  const uint32_t l = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = kBlock / a.lanes;
  const Place<V, INTER> at(l, a.pairs, a.items, a.d);
  const float inv_d = 1.f / (float)a.d;

  float w[NORM ? 2 * V : 1], sums_of[NORM && BACK ? 2 * V : 1];
  if constexpr (NORM) {
    load_row<T, V>(side.w, at.a, at.b, at.use, at.use_b, w);
    if constexpr (BACK) {
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) sums_of[i] = 0.f;
    }
  }

  for (uint64_t n = (uint64_t)blockIdx.x * side.tt; n < a.tokens; n += (uint64_t)side.blocks * side.tt) {
    const uint32_t n0 = (uint32_t)n, count = min(side.tt, a.tokens - n0), rows = count * side.heads;
    const size_t base = (size_t)n0 * side.heads * a.d;
    make_table(a, n0, count, table, valid);
    __syncthreads();
    for (uint32_t r0 = 0; r0 < rows; r0 += groups * U) {
      float z[U][2 * V];
      [[maybe_unused]] float xs[NORM && BACK ? U : 1][2 * V];
      bool exists[U], in[U];
      size_t off[U];
      const float2 *cs[U];
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t ru = r0 + u * groups + group;
        exists[u] = ru < rows;
        const uint32_t r = exists[u] ? ru : rows - 1;  // lanes without a row go along for the exchanges
        const uint32_t t = side.inv == 0 ? r : __umulhi(r, side.inv);
        in[u] = valid[t] != 0;
        cs[u] = table + t * (kMostSize / 2) + at.angle;
        off[u] = base + (size_t)r * a.d;
        if constexpr (!BACK) load_row<T, V>(side.x + off[u], at.a, at.b, at.use, at.use_b, z[u]);
        else load_row<T, V>(side.gy + off[u], at.a, at.b, at.use && in[u], at.use_b && in[u], z[u]);
        if constexpr (NORM && BACK) load_row<T, V>(side.x + off[u], at.a, at.b, at.use && in[u], at.use_b && in[u], xs[u]);
      }
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) {
        T *out = side.o + off[u];
        if constexpr (!BACK) {
          if constexpr (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) ss = fmaf(z[u][i], z[u][i], ss);
            const float inv = 1.f / sqrtf(fmaf(row_sum(ss, a.lanes), inv_d, a.eps));
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) z[u][i] = z[u][i] * inv * w[i];
          }
          if (at.turns) rotate<V, INTER>(z[u], cs[u], 1.f);
          if (!in[u]) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) z[u][i] = 0.f;
          }
          if (exists[u]) store_row<T, V>(out, at.a, at.b, at.use, at.use_b, false, z[u]);
        } else {
          if (at.turns) rotate<V, INTER>(z[u], cs[u], -1.f);
          if constexpr (NORM) {
            float (&x)[2 * V] = xs[u];
            float ss = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
              ss = fmaf(x[i], x[i], ss);
              dot = fmaf(z[u][i] * w[i], x[i], dot);
            }
            // tokens of no sequence come as zeros, which with eps == 0 have no finite norm: they add nothing
            const float r = 1.f / sqrtf(fmaf(row_sum(ss, a.lanes), inv_d, a.eps)), inv = in[u] ? r : 0.f;
            const float mean = row_sum(dot, a.lanes) * inv_d * inv * inv;
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
              const float g = z[u][i];
              sums_of[i] += exists[u] ? g * x[i] * inv : 0.f;
              z[u][i] = inv * (g * w[i] - x[i] * mean);
            }
          }
          const bool acc = side.acc != 0;
          if (exists[u] && (in[u] || !acc)) store_row<T, V>(out, at.a, at.b, at.use, at.use_b, acc, z[u]);
        }
      }
    }
    __syncthreads();
  }

  if constexpr (NORM && BACK) {
    // the workgroup's sums: first between the rows of a wavefront, then wavefront after wavefront, in a fixed order
    __shared__ float sums[kMostSize];
    for (uint32_t i = threadIdx.x; i < kMostSize; i += kBlock) sums[i] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * V; ++i)
      for (uint32_t o = a.lanes; o < 64; o <<= 1) sums_of[i] += __shfl_xor(sums_of[i], (int)o);
    for (uint32_t v = 0; v < kBlock / 64; ++v) {
      __syncthreads();
      if (threadIdx.x / 64 == v && (threadIdx.x & 63) < a.lanes) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (at.use) sums[at.a + i] += sums_of[i];
          if (at.use_b) sums[at.b + i] += sums_of[V + i];
        }
      }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.d; i += kBlock)
      a.partial[((size_t)(blockIdx.y ? a.side[0].blocks : 0) + blockIdx.x) * a.d + i] = sums[i];
  }
}

// gw (+)= the sum over the workgroups of a side of one column of the partial sums: a workgroup takes 16 columns, 16 threads
// each.
template <typename T>
__global__ __launch_bounds__(kBlock) void weights_kernel(const float *partial, uint32_t blocks_q, uint32_t blocks_k, uint32_t d,
                                                         T *gwq, T *gwk, uint32_t acc_q, uint32_t acc_k) {
  __shared__ float part[kBlock];
  const bool is_q = blockIdx.y == 0;
  const uint32_t c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4, blocks = is_q ? blocks_q : blocks_k;
  const float *from = partial + (is_q ? 0 : (size_t)blocks_q * d);
  float s = 0.f;
  if (c < d)
    for (uint32_t b0 = k; b0 < blocks; b0 += 16 * 16) {  // 16 loads in flight
      float x[16];
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) x[u] = b0 + 16 * u < blocks ? from[(size_t)(b0 + 16 * u) * d + c] : 0.f;
#pragma unroll
      for (uint32_t u = 0; u < 16; ++u) s += x[u];
    }
  part[threadIdx.x] = s;
  __syncthreads();
  if (k != 0 || c >= d) return;
  for (uint32_t i = 1; i < 16; ++i) s += part[threadIdx.x + 16 * i];
  T *p = (is_q ? gwq : gwk) + c;
  *p = from_f32<T>((is_q ? acc_q : acc_k) ? to_f32(*p) + s : s);
}

// What the four entry points share.
template <typename T>
int make_args(phip_ctx *ctx, uint32_t d, uint32_t hq, uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs,
              int32_t first, const float *freqs, uint32_t pairs, float amplitude, float eps, bool has_k, Args<T> *out) {
  PHIP_REQUIRE(d >= 1 && d <= kMostSize, "head sizes of 1 to %u are supported, got %u", kMostSize, d);
  PHIP_REQUIRE(hq >= 1 && t >= 1 && bs >= 1, "empty tensors");
  PHIP_REQUIRE(has_k ? hk >= 1 : hk == 0, "%u heads of keys, and the keys are %s", hk, has_k ? "given" : "null");
  PHIP_REQUIRE(hq <= 16384 && hk <= 16384, "more than 16384 heads");  // rows of 8 tokens divided by a multiplication
  PHIP_REQUIRE(pairs <= d / 2, "%u pairs in a head of %u elements", pairs, d);
  PHIP_REQUIRE(pairs == 0 || freqs != nullptr, "null frequencies");
  PHIP_REQUIRE(eps >= 0.f && eps <= 3.4e38f, "eps must be finite and not negative");
  PHIP_REQUIRE((uint64_t)t * bs <= 0x7fffffffu, "more than 2^31 - 1 tokens");
  Args<T> a = {};
  const int rc = sequence_view(ctx, seqs, t, 0, bs, false, &a.seq);
  if (rc != PHIP_OK) return rc;
  a.tokens = t * bs;
  a.d = d;
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = i == 0 ? hq : hk;
    a.side[i].heads = h;
    a.side[i].inv = h <= 1 ? 0 : (uint32_t)(((1ull << 32) + h - 1) / h);
  }
  a.pairs = pairs;
  a.first = first;
  a.amplitude = amplitude;
  a.eps = eps;
  for (uint32_t i = 0; i < pairs; ++i) a.f[i] = freqs[i];
  *out = a;
  return PHIP_OK;
}

inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
inline bool all_aligned(size_t n, std::initializer_list<const void *> ptrs) {
  return std::all_of(ptrs.begin(), ptrs.end(), [n](const void *p) { return aligned(p, n); });
}

template <typename T, int V, bool INTER, bool NORM, bool BACK>
int launch_kernel(phip_ctx *ctx, Args<T> a) {
  a.items = a.pairs / V + (a.d - 2 * a.pairs + 2 * V - 1) / (2 * V);
  a.lanes = 1;
  while (a.lanes < a.items) a.lanes *= 2;
  const uint32_t blocks = std::max(a.side[0].blocks, a.side[1].blocks);
  hipLaunchKernelGGL((rotary_kernel<T, V, INTER, NORM, BACK>), dim3(blocks, a.side[1].heads != 0 ? 2 : 1), dim3(kBlock), 0,
                     ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  return PHIP_OK;
}

template <typename T, bool NORM, bool BACK>
int launch(phip_ctx *ctx, const Args<T> &a, bool interleaved) {
  constexpr uint32_t W = 16 / sizeof(T);
  auto fits = [&](uint32_t v) {
    bool ok = a.d % v == 0 && a.pairs % v == 0;
    for (const Side<T> &s : a.side)
      ok = ok && aligned(s.x, v * sizeof(T)) && aligned(s.w, v * sizeof(T)) && aligned(s.gy, v * sizeof(T)) && aligned(s.o, v * sizeof(T));
    return ok;
  };
  if (fits(W)) return interleaved ? launch_kernel<T, W, true, NORM, BACK>(ctx, a) : launch_kernel<T, W, false, NORM, BACK>(ctx, a);
  if constexpr (sizeof(T) == 2) {
    if (fits(2)) return interleaved ? launch_kernel<T, 2, true, NORM, BACK>(ctx, a) : launch_kernel<T, 2, false, NORM, BACK>(ctx, a);
  }
  return interleaved ? launch_kernel<T, 1, true, NORM, BACK>(ctx, a) : launch_kernel<T, 1, false, NORM, BACK>(ctx, a);
}

// Tokens per step of a side's workgroups: as many as leave a few workgroups for every CU.  looping: every workgroup leaves
// a row of partial sums, so their number is limited and they take several steps; without sums, a launch's 2^32 threads are
// the limit.
template <typename T>
void choose(phip_ctx *ctx, Args<T> *a, bool looping) {
  const uint64_t cus = (uint64_t)ctx->prop.multiProcessorCount;
  for (Side<T> &s : a->side) {
    if (s.heads == 0) continue;
    const uint64_t tt = a->tokens / (cus * 8), blocks_cap = looping ? cus * 4 : 1u << 23;
    s.tt = (uint32_t)(tt < 1 ? 1 : tt > kMostTokens ? kMostTokens : tt);
    s.blocks = (uint32_t)std::min<uint64_t>((a->tokens + s.tt - 1) / s.tt, blocks_cap);
  }
}

template <typename T, bool NORM>
int forward(phip_ctx *ctx, const T *xq, const T *xk, const T *wq, const T *wk, T *yq, T *yk, uint32_t d, uint32_t hq,
            uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs, int32_t first, const float *freqs,
            uint32_t pairs, int interleaved, float amplitude, float eps) {
  PHIP_ENTER(ctx);
  Args<T> a;
  const int rc = make_args<T>(ctx, d, hq, hk, t, bs, seqs, first, freqs, pairs, amplitude, eps, xk != nullptr, &a);
  if (rc != PHIP_OK) return rc;
  PHIP_REQUIRE(xq != nullptr && yq != nullptr && (xk == nullptr) == (yk == nullptr), "null pointer");
  PHIP_REQUIRE(!NORM || (wq != nullptr && (xk == nullptr) == (wk == nullptr)), "null weights");
  PHIP_REQUIRE(all_aligned(sizeof(T), {xq, xk, wq, wk, yq, yk}), "an address is no multiple of the element size");
  const size_t nq = (size_t)d * hq * a.tokens * sizeof(T), nk = (size_t)d * hk * a.tokens * sizeof(T);
  auto read = [&](const void *y, size_t n) {
    return shares_memory(y, n, wq, d * sizeof(T)) || shares_memory(y, n, wk, d * sizeof(T)) ||
           (y != xq && shares_memory(y, n, xq, nq)) || (y != xk && shares_memory(y, n, xk, nk));
  };
  // a result may take its own operand's place; nothing else may overlap
  PHIP_REQUIRE(!read(yq, nq) && yq != xk && (yk == nullptr || (!read(yk, nk) && yk != xq && !shares_memory(yq, nq, yk, nk))),
               "a result shares memory with an operand or with the other result");
  a.side[0].x = xq;
  a.side[1].x = xk;
  a.side[0].w = wq;
  a.side[1].w = wk;
  a.side[0].o = yq;
  a.side[1].o = yk;
  choose(ctx, &a, false);
  return launch<T, NORM, false>(ctx, a, interleaved != 0);
}

// partial: room for the sums of both sides' workgroups (norm only).
template <typename T, bool NORM>
int backward_one(phip_ctx *ctx, Args<T> a, bool interleaved, float *partial, T *gwq, T *gwk, bool acc_wq, bool acc_wk) {
  a.partial = partial;
  const int rc = launch<T, NORM, true>(ctx, a, interleaved);
  if (!NORM || rc != PHIP_OK) return rc;
  hipLaunchKernelGGL((weights_kernel<T>), dim3((a.d + 15) / 16, a.side[1].heads != 0 ? 2 : 1), dim3(kBlock), 0, ctx->stream,
                     a.partial, a.side[0].blocks, a.side[1].blocks, a.d, gwq, gwk, acc_wq ? 1u : 0u, acc_wk ? 1u : 0u);
  PHIP_LAUNCH_CHECK();
  return PHIP_OK;
}

template <typename T, bool NORM>
int backward(phip_ctx *ctx, const T *xq, const T *xk, const T *wq, const T *wk, const T *gyq, const T *gyk, T *gxq, T *gxk,
             T *gwq, T *gwk, uint32_t d, uint32_t hq, uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs,
             int32_t first, const float *freqs, uint32_t pairs, int interleaved, float amplitude, float eps) {
  PHIP_ENTER_KEEP_ZEROS(ctx);
  Args<T> a;
  int rc = make_args<T>(ctx, d, hq, hk, t, bs, seqs, first, freqs, pairs, amplitude, eps, gyk != nullptr, &a);
  if (rc != PHIP_OK) return rc;
  const bool has_k = gyk != nullptr;
  PHIP_REQUIRE(gyq != nullptr && gxq != nullptr && has_k == (gxk != nullptr), "null pointer");
  PHIP_REQUIRE(!NORM || (xq != nullptr && wq != nullptr && gwq != nullptr && has_k == (xk != nullptr) &&
                         has_k == (wk != nullptr) && has_k == (gwk != nullptr)),
               "null operand, weights or gradient of the weights");
  PHIP_REQUIRE(all_aligned(sizeof(T), {xq, xk, wq, wk, gyq, gyk, gxq, gxk, gwq, gwk}),
               "an address is no multiple of the element size");
  const size_t nq = (size_t)d * hq * a.tokens * sizeof(T), nk = (size_t)d * hk * a.tokens * sizeof(T), nw = d * sizeof(T);
  auto is_read = [&](const void *g, size_t n) {
    return shares_memory(g, n, xq, nq) || shares_memory(g, n, xk, nk) || shares_memory(g, n, wq, nw) ||
           shares_memory(g, n, wk, nw) || shares_memory(g, n, gyq, nq) || shares_memory(g, n, gyk, nk);
  };
  PHIP_REQUIRE(!is_read(gxq, nq) && !(has_k && is_read(gxk, nk)) && !(NORM && is_read(gwq, nw)) &&
                   !(NORM && has_k && is_read(gwk, nw)),
               "a gradient shares memory with an operand");
  PHIP_REQUIRE(!has_k || gxq == gxk ? !has_k || hq == hk : !shares_memory(gxq, nq, gxk, nk),
               "two gradients overlap without being the same tensor");
  PHIP_REQUIRE(!NORM || (!shares_memory(gwq, nw, gxq, nq) && !shares_memory(gwq, nw, gxk, nk) &&
                         !shares_memory(gwk, nw, gxq, nq) && !shares_memory(gwk, nw, gxk, nk) &&
                         (!has_k || gwq == gwk || !shares_memory(gwq, nw, gwk, nw))),
               "a gradient of the weights overlaps another gradient");
  choose(ctx, &a, NORM);
  void *partial = nullptr;
  if (NORM) {
    rc = phip_pool_alloc(ctx, (size_t)(a.side[0].blocks + a.side[1].blocks) * d * sizeof(float), &partial, nullptr);
    if (rc != PHIP_OK) return rc;
  }
  // nothing is refused from here on: gradients noted as zero and not yet filled are written instead of added into
  a.side[0].acc = !zeros_take(ctx, gxq, nq);
  a.side[1].acc = has_k && !zeros_take(ctx, gxk, nk);
  const bool acc_wq = NORM && !zeros_take(ctx, gwq, nw), acc_wk = NORM && has_k && !zeros_take(ctx, gwk, nw);
  PHIP_FLUSH_ZEROS(ctx);
  a.side[0].x = xq;
  a.side[1].x = xk;
  a.side[0].w = wq;
  a.side[1].w = wk;
  a.side[0].gy = gyq;
  a.side[1].gy = gyk;
  a.side[0].o = gxq;
  a.side[1].o = gxk;
  float *const sums = static_cast<float *>(partial);
  if (!has_k || (gxq != gxk && (!NORM || gwq != gwk))) {
    rc = backward_one<T, NORM>(ctx, a, interleaved != 0, sums, gwq, gwk, acc_wq, acc_wk);
  } else {
    // one tensor for both gradients (a tensor or a weight used as queries' and as keys'): one after the other
    Args<T> one = a;
    one.side[1] = Side<T>{};
    rc = backward_one<T, NORM>(ctx, one, interleaved != 0, sums, gwq, nullptr, acc_wq, false);
    one.side[0] = a.side[1];
    if (rc == PHIP_OK) rc = backward_one<T, NORM>(ctx, one, interleaved != 0, sums, gwk, nullptr, acc_wk, false);
  }
  if (partial != nullptr) phip_pool_free(ctx, partial);
  return rc;
}

}  // namespace
}  // namespace rotary
}  // namespace phip

using namespace phip;

extern "C" {

#define PHIP_EXPORT_ROTARY(SUF, T, PTR)                                                                                   \
  int phip_rotary_fw_##SUF(phip_ctx *ctx, const PTR *xq, const PTR *xk, PTR *yq, PTR *yk, uint32_t d, uint32_t hq,        \
                           uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs, int32_t first,               \
                           const float *freqs, uint32_t pairs, int interleaved, float amplitude) {                        \
    return rotary::forward<T, false>(ctx, static_cast<const T *>(xq), static_cast<const T *>(xk), nullptr, nullptr,       \
                                     static_cast<T *>(yq), static_cast<T *>(yk), d, hq, hk, t, bs, seqs, first, freqs,    \
                                     pairs, interleaved, amplitude, 0.f);                                                 \
  }                                                                                                                       \
  int phip_rotary_bw_##SUF(phip_ctx *ctx, const PTR *gyq, const PTR *gyk, PTR *gxq, PTR *gxk, uint32_t d, uint32_t hq,    \
                           uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs, int32_t first,               \
                           const float *freqs, uint32_t pairs, int interleaved, float amplitude) {                        \
    return rotary::backward<T, false>(ctx, nullptr, nullptr, nullptr, nullptr, static_cast<const T *>(gyq),               \
                                      static_cast<const T *>(gyk), static_cast<T *>(gxq), static_cast<T *>(gxk), nullptr, \
                                      nullptr, d, hq, hk, t, bs, seqs, first, freqs, pairs, interleaved, amplitude, 0.f); \
  }                                                                                                                       \
  int phip_norm_rotary_fw_##SUF(phip_ctx *ctx, const PTR *xq, const PTR *xk, const PTR *wq, const PTR *wk, PTR *yq,       \
                                PTR *yk, uint32_t d, uint32_t hq, uint32_t hk, uint32_t t, uint32_t bs,                   \
                                const phip_sequences *seqs, int32_t first, const float *freqs, uint32_t pairs,            \
                                int interleaved, float amplitude, float eps) {                                            \
    return rotary::forward<T, true>(ctx, static_cast<const T *>(xq), static_cast<const T *>(xk),                          \
                                    static_cast<const T *>(wq), static_cast<const T *>(wk), static_cast<T *>(yq),         \
                                    static_cast<T *>(yk), d, hq, hk, t, bs, seqs, first, freqs, pairs, interleaved,       \
                                    amplitude, eps);                                                                      \
  }                                                                                                                       \
  int phip_norm_rotary_bw_##SUF(phip_ctx *ctx, const PTR *xq, const PTR *xk, const PTR *wq, const PTR *wk,                \
                                const PTR *gyq, const PTR *gyk, PTR *gxq, PTR *gxk, PTR *gwq, PTR *gwk, uint32_t d,       \
                                uint32_t hq, uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs,            \
                                int32_t first, const float *freqs, uint32_t pairs, int interleaved, float amplitude,      \
                                float eps) {                                                                              \
    return rotary::backward<T, true>(ctx, static_cast<const T *>(xq), static_cast<const T *>(xk),                         \
                                     static_cast<const T *>(wq), static_cast<const T *>(wk), static_cast<const T *>(gyq), \
                                     static_cast<const T *>(gyk), static_cast<T *>(gxq), static_cast<T *>(gxk),           \
                                     static_cast<T *>(gwq), static_cast<T *>(gwk), d, hq, hk, t, bs, seqs, first, freqs,  \
                                     pairs, interleaved, amplitude, eps);                                                 \
  }

PHIP_EXPORT_ROTARY(f32, float, float)
PHIP_EXPORT_ROTARY(f16, f16_t, void)
PHIP_EXPORT_ROTARY(bf16, bf16_t, void)

#undef PHIP_EXPORT_ROTARY

}  // extern "C"
