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
#include <type_traits>

#include "phip_pointwise.h"
#include "phip_sequences.h"

namespace phip {
namespace rotary {
namespace {

using pointwise::kBlock;

constexpr uint32_t kMostSize = 128;
constexpr int kMostTokens = 8;   // per workgroup and step

template <typename T>
struct Args {
  const T *xq, *xk;       // forward: the operands; backward: the same (norm only)
  const T *wq, *wk;       // weights of the norm
  const T *gyq, *gyk;     // backward
  T *oq, *ok;             // y, or gx
  float *partial;         // backward with weights: per workgroup, d sums for wq, then d for wk
  SequenceView seq;
  uint32_t tokens;        // tq * batch
  uint32_t d, hq, h;      // h: heads of queries and keys together
  uint32_t tt;            // tokens per step of a workgroup
  uint32_t pairs, items, lanes;  // items: lanes of a row that have work; lanes: the power of two that a row takes
  int32_t first;
  float amplitude, eps;
  uint32_t acc_q, acc_k;  // backward: add into what is there
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
template <typename T, int V, bool INTER, bool NORM, bool BACK>
__global__ __launch_bounds__(kBlock) void rotary_kernel(const Args<T> a) {
  __shared__ float2 table[kMostTokens * (kMostSize / 2)];
  __shared__ uint32_t valid[kMostTokens];
  const uint32_t l = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = kBlock / a.lanes;
  const Place<V, INTER> at(l, a.pairs, a.items, a.d);
  const float inv_d = 1.f / (float)a.d;

  float wq[NORM ? 2 * V : 1], wk[NORM ? 2 * V : 1], sq[NORM && BACK ? 2 * V : 1], sk[NORM && BACK ? 2 * V : 1];
  if constexpr (NORM) {
    load_row<T, V>(a.wq, at.a, at.b, at.use, at.use_b, wq);
    if (a.h > a.hq) load_row<T, V>(a.wk, at.a, at.b, at.use, at.use_b, wk);
    if constexpr (BACK) {
#pragma unroll
      for (int i = 0; i < 2 * V; ++i) sq[i] = sk[i] = 0.f;
    }
  }

  for (uint64_t n = (uint64_t)blockIdx.x * a.tt; n < a.tokens; n += (uint64_t)gridDim.x * a.tt) {
    const uint32_t n0 = (uint32_t)n, count = min(a.tt, a.tokens - n0), rows = count * a.h;
    make_table(a, n0, count, table, valid);
    __syncthreads();
    for (uint32_t r0 = 0; r0 < rows; r0 += groups) {
      const bool exists = r0 + group < rows;
      const uint32_t r = exists ? r0 + group : rows - 1;  // lanes without a row go along for the exchanges
      const uint32_t t = r / a.h, head = r - t * a.h;
      const bool is_q = head < a.hq;
      const size_t off = is_q ? ((size_t)(n0 + t) * a.hq + head) * a.d : ((size_t)(n0 + t) * (a.h - a.hq) + (head - a.hq)) * a.d;
      const bool in = valid[t] != 0;
      const float2 *cs = table + t * (kMostSize / 2) + at.angle;
      float z[2 * V];
      T *out = (is_q ? a.oq : a.ok) + off;
      if constexpr (!BACK) {
        load_row<T, V>((is_q ? a.xq : a.xk) + off, at.a, at.b, at.use, at.use_b, z);
        if constexpr (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) ss = fmaf(z[i], z[i], ss);
          const float inv = 1.f / sqrtf(fmaf(row_sum(ss, a.lanes), inv_d, a.eps));
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) z[i] = z[i] * inv * (is_q ? wq[i] : wk[i]);
        }
        if (at.turns) rotate<V, INTER>(z, cs, 1.f);
        if (!in) {
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) z[i] = 0.f;
        }
        if (exists) store_row<T, V>(out, at.a, at.b, at.use, at.use_b, false, z);
      } else {
        load_row<T, V>((is_q ? a.gyq : a.gyk) + off, at.a, at.b, at.use && in, at.use_b && in, z);
        if (at.turns) rotate<V, INTER>(z, cs, -1.f);
        if constexpr (NORM) {
          float x[2 * V];
          load_row<T, V>((is_q ? a.xq : a.xk) + off, at.a, at.b, at.use && in, at.use_b && in, x);
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            ss = fmaf(x[i], x[i], ss);
            dot = fmaf(z[i] * (is_q ? wq[i] : wk[i]), x[i], dot);
          }
          const float inv = 1.f / sqrtf(fmaf(row_sum(ss, a.lanes), inv_d, a.eps));
          const float mean = row_sum(dot, a.lanes) * inv_d * inv * inv;
#pragma unroll
          for (int i = 0; i < 2 * V; ++i) {
            const float g = z[i], add = exists ? g * x[i] * inv : 0.f;
            sq[i] += is_q ? add : 0.f;
            sk[i] += is_q ? 0.f : add;
            z[i] = inv * (g * (is_q ? wq[i] : wk[i]) - x[i] * mean);
          }
        }
        const bool acc = (is_q ? a.acc_q : a.acc_k) != 0;
        if (exists && (in || !acc)) store_row<T, V>(out, at.a, at.b, at.use, at.use_b, acc, z);
      }
    }
    __syncthreads();
  }

  if constexpr (NORM && BACK) {
    // the workgroup's sums: row groups one after another, in a fixed order
    __shared__ float sums[2 * kMostSize];
    for (uint32_t i = threadIdx.x; i < 2 * kMostSize; i += kBlock) sums[i] = 0.f;
    // first between the rows of a wavefront
#pragma unroll
    for (int i = 0; i < 2 * V; ++i)
      for (uint32_t o = a.lanes; o < 64; o <<= 1) {
        sq[i] += __shfl_xor(sq[i], (int)o);
        sk[i] += __shfl_xor(sk[i], (int)o);
      }
    for (uint32_t w = 0; w < kBlock / 64; ++w) {
      __syncthreads();
      if (threadIdx.x / 64 == w && (threadIdx.x & 63) < a.lanes) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (at.use) {
            sums[at.a + i] += sq[i];
            sums[kMostSize + at.a + i] += sk[i];
          }
          if (at.use_b) {
            sums[at.b + i] += sq[V + i];
            sums[kMostSize + at.b + i] += sk[V + i];
          }
        }
      }
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * a.d; i += kBlock)
      a.partial[(size_t)blockIdx.x * 2 * a.d + i] = i < a.d ? sums[i] : sums[kMostSize + i - a.d];
  }
}

// gw (+)= the sum over the workgroups of one column of the partial sums: a workgroup takes 16 columns, 16 threads each.
template <typename T>
__global__ __launch_bounds__(kBlock) void weights_kernel(const float *partial, uint32_t blocks, uint32_t d, T *gwq, T *gwk,
                                                         uint32_t acc_q, uint32_t acc_k) {
  __shared__ float part[kBlock];
  const uint32_t c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4;
  float s = 0.f;
  if (c < 2 * d)
    for (uint32_t b = k; b < blocks; b += 16) s += partial[(size_t)b * 2 * d + c];
  part[threadIdx.x] = s;
  __syncthreads();
  if (k != 0 || c >= 2 * d) return;
  for (uint32_t i = 1; i < 16; ++i) s += part[threadIdx.x + 16 * i];
  T *p = c < d ? gwq + c : gwk != nullptr ? gwk + (c - d) : nullptr;
  if (p != nullptr) *p = from_f32<T>((c < d ? acc_q : acc_k) ? to_f32(*p) + s : s);
}

// What the four entry points share.
template <typename T>
int make_args(phip_ctx *ctx, uint32_t d, uint32_t hq, uint32_t hk, uint32_t t, uint32_t bs, const phip_sequences *seqs,
              int32_t first, const float *freqs, uint32_t pairs, float amplitude, float eps, bool has_k, Args<T> *out) {
  PHIP_REQUIRE(d >= 1 && d <= kMostSize, "head sizes of 1 to %u are supported, got %u", kMostSize, d);
  PHIP_REQUIRE(hq >= 1 && t >= 1 && bs >= 1, "empty tensors");
  PHIP_REQUIRE(has_k ? hk >= 1 : hk == 0, "%u heads of keys, and the keys are %s", hk, has_k ? "given" : "null");
  PHIP_REQUIRE((uint64_t)hq + hk <= (1u << 20), "too many heads");
  PHIP_REQUIRE(pairs <= d / 2, "%u pairs in a head of %u elements", pairs, d);
  PHIP_REQUIRE(pairs == 0 || freqs != nullptr, "null frequencies");
  PHIP_REQUIRE(eps >= 0.f && eps <= 3.4e38f, "eps must be finite and not negative");
  PHIP_REQUIRE((uint64_t)t * bs <= 0x7fffffffu, "more than 2^31 - 1 tokens");
  Args<T> a = {};
  const int rc = sequence_view(ctx, seqs, t, 0, bs, false, &a.seq);
  if (rc != PHIP_OK) return rc;
  a.tokens = t * bs;
  a.d = d;
  a.hq = hq;
  a.h = hq + hk;
  a.pairs = pairs;
  a.first = first;
  a.amplitude = amplitude;
  a.eps = eps;
  for (uint32_t i = 0; i < pairs; ++i) a.f[i] = freqs[i];
  *out = a;
  return PHIP_OK;
}

inline bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename T, int V, bool INTER, bool NORM, bool BACK>
int launch_kernel(phip_ctx *ctx, Args<T> a, uint32_t blocks) {
  a.items = a.pairs / V + (a.d - 2 * a.pairs + 2 * V - 1) / (2 * V);
  a.lanes = 1;
  while (a.lanes < a.items) a.lanes *= 2;
  hipLaunchKernelGGL((rotary_kernel<T, V, INTER, NORM, BACK>), dim3(blocks), dim3(kBlock), 0, ctx->stream, a);
  PHIP_LAUNCH_CHECK();
  return PHIP_OK;
}

template <typename T, bool NORM, bool BACK>
int launch(phip_ctx *ctx, const Args<T> &a, bool interleaved, uint32_t blocks) {
  constexpr uint32_t W = 16 / sizeof(T);
  auto fits = [&](uint32_t v) {
    bool ok = a.d % v == 0 && a.pairs % v == 0;
    for (const void *p : {(const void *)a.xq, (const void *)a.xk, (const void *)a.wq, (const void *)a.wk, (const void *)a.gyq,
                          (const void *)a.gyk, (const void *)a.oq, (const void *)a.ok})
      ok = ok && aligned(p, v * sizeof(T));
    return ok;
  };
  if (fits(W))
    return interleaved ? launch_kernel<T, W, true, NORM, BACK>(ctx, a, blocks) : launch_kernel<T, W, false, NORM, BACK>(ctx, a, blocks);
  if (sizeof(T) == 2 && fits(2))
    return interleaved ? launch_kernel<T, 2, true, NORM, BACK>(ctx, a, blocks) : launch_kernel<T, 2, false, NORM, BACK>(ctx, a, blocks);
  return interleaved ? launch_kernel<T, 1, true, NORM, BACK>(ctx, a, blocks) : launch_kernel<T, 1, false, NORM, BACK>(ctx, a, blocks);
}

// Tokens per step: as many as leave a few workgroups for every CU.
template <typename T>
uint32_t choose(phip_ctx *ctx, Args<T> *a, bool looping) {
  const uint64_t cus = (uint64_t)ctx->prop.multiProcessorCount;
  uint64_t tt = a->tokens / (cus * 8);
  a->tt = (uint32_t)(tt < 1 ? 1 : tt > kMostTokens ? kMostTokens : tt);
  uint64_t blocks = (a->tokens + a->tt - 1) / a->tt;
  const uint64_t cap = looping ? cus * 4 : ~0ull;  // looping: every workgroup leaves a row of partial sums
  return (uint32_t)(blocks > cap ? cap : blocks);
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
  const size_t nq = (size_t)d * hq * a.tokens * sizeof(T), nk = (size_t)d * hk * a.tokens * sizeof(T);
  auto read = [&](const void *y, size_t n) {
    return shares_memory(y, n, wq, d * sizeof(T)) || shares_memory(y, n, wk, d * sizeof(T)) ||
           (y != xq && shares_memory(y, n, xq, nq)) || (y != xk && shares_memory(y, n, xk, nk));
  };
  // a result may take its own operand's place; nothing else may overlap
  PHIP_REQUIRE(!read(yq, nq) && yq != xk && (yk == nullptr || (!read(yk, nk) && yk != xq && !shares_memory(yq, nq, yk, nk))),
               "a result shares memory with an operand or with the other result");
  a.xq = xq;
  a.xk = xk;
  a.wq = wq;
  a.wk = wk;
  a.oq = yq;
  a.ok = yk;
  const uint32_t blocks = choose(ctx, &a, false);
  return launch<T, NORM, false>(ctx, a, interleaved != 0, blocks);
}

template <typename T, bool NORM>
int backward_one(phip_ctx *ctx, Args<T> a, bool interleaved, T *gwq, T *gwk, bool acc_wq, bool acc_wk) {
  const uint32_t blocks = choose(ctx, &a, NORM);
  if constexpr (!NORM) return launch<T, false, true>(ctx, a, interleaved, blocks);
  void *partial = nullptr;
  int rc = phip_pool_alloc(ctx, (size_t)blocks * 2 * a.d * sizeof(float), &partial, nullptr);
  if (rc != PHIP_OK) return rc;
  a.partial = static_cast<float *>(partial);
  rc = launch<T, NORM, true>(ctx, a, interleaved, blocks);
  if (rc == PHIP_OK) {
    hipLaunchKernelGGL((weights_kernel<T>), dim3((2 * a.d + 15) / 16), dim3(kBlock), 0, ctx->stream, a.partial, blocks, a.d,
                       gwq, gwk, acc_wq ? 1u : 0u, acc_wk ? 1u : 0u);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) rc = fail(PHIP_ERR_RUNTIME, "launching the sum of the weights' gradients failed: %s", hipGetErrorString(e));
  }
  phip_pool_free(ctx, partial);
  return rc;
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
  // gradients noted as zero and not yet filled are written instead of added into
  a.acc_q = !zeros_take(ctx, gxq, nq);
  a.acc_k = has_k && !zeros_take(ctx, gxk, nk);
  const bool acc_wq = NORM && !zeros_take(ctx, gwq, nw), acc_wk = NORM && has_k && !zeros_take(ctx, gwk, nw);
  PHIP_FLUSH_ZEROS(ctx);
  a.xq = xq;
  a.xk = xk;
  a.wq = wq;
  a.wk = wk;
  a.gyq = gyq;
  a.gyk = gyk;
  a.oq = gxq;
  a.ok = gxk;
  if (!has_k || (gxq != gxk && (!NORM || gwq != gwk)))
    return backward_one<T, NORM>(ctx, a, interleaved != 0, gwq, gwk, acc_wq, acc_wk);
  // one tensor for both gradients (a tensor or a weight used as queries' and as keys'): one after the other
  Args<T> q = a, k = a;
  q.h = hq;
  q.xk = q.wk = q.gyk = nullptr;
  q.ok = nullptr;
  rc = backward_one<T, NORM>(ctx, q, interleaved != 0, gwq, nullptr, acc_wq, false);
  if (rc != PHIP_OK) return rc;
  k.h = k.hq = hk;
  k.xq = xk;
  k.wq = wk;
  k.gyq = gyk;
  k.oq = gxk;
  k.acc_q = a.acc_k;
  k.xk = k.wk = k.gyk = nullptr;
  k.ok = nullptr;
  return backward_one<T, NORM>(ctx, k, interleaved != 0, gwk, nullptr, acc_wk, false);
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
