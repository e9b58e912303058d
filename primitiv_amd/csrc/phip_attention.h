// Shared pieces of the attention kernels (forward and gradients).
//
// Everything is built from 32 x 32 blocks of the matrix instructions, and every product is arranged so that its result
// can be the right operand of the next one without leaving the registers.  A lane of a result block holds one column
// (lane % 32) and the rows (i & 3) + 8 (i >> 2) + 4 (lane / 32), i < 16; a right operand over 16 of those rows wants 8 of
// them from each half of the wavefront.  Which 8 does not matter as long as the left operand is read in the same order:
// chunk c of 16 rows gives half h the rows 16 c + 4 h + j (j < 4) and 16 c + 8 + 4 h + (j - 4), which are the registers
// 8 c + j.  So the scores are computed transposed (keys down, queries across): a lane then owns a query, the softmax
// needs one exchange between the halves per tile, and exp(scores) is the right operand of the product with the values.
//
// The three storage types share the code.  A fragment is 8 elements per lane for one 16-deep step: one
// v_mfma_f32_32x32x16 for 16-bit storage, eight v_mfma_f32_32x32x2_f32 for fp32.
#ifndef PHIP_ATTENTION_H_
#define PHIP_ATTENTION_H_

#include <atomic>
#include <initializer_list>

#include "phip_internal.h"
#include "phip_sequences.h"
#include "phip_types.h"

namespace phip {
namespace attention {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf8v __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kOutOfRange = 0x80000000u;  // past the end of any buffer described here

template <class T>
__device__ inline __attribute__((address_space(3))) T *lds_ptr(uint32_t addr) {
  return (__attribute__((address_space(3))) T *)(size_t)addr;
}

// ---- arguments ---------------------------------------------------------------------------------------------------

struct Shape {
  uint32_t d, hq, hk, g;      // head size, query heads, key heads, hq / hk
  uint32_t inv_g;
  uint32_t causal;
  float scale_log2;           // scale * log2(e): scores are exponents of 2
  float scale;
  uint32_t whole;             // rows are whole 16-byte chunks at addresses that are multiples of 16
};

// ---- fragments ------------------------------------------------------------------------------------------------------

template <typename T>
struct Frag16 {
  u32x4 v;  // elements 2 e, 2 e + 1 in v[e]
};
template <typename T>
struct FragOf {
  typedef Frag16<T> type;
};
template <>
struct FragOf<float> {
  typedef f32x8 type;
};
template <typename T>
using Frag = typename FragOf<T>::type;

__device__ inline void mma(f32x16 &c, const Frag16<bf16_t> &a, const Frag16<bf16_t> &b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8v, a.v), __builtin_bit_cast(bf8v, b.v), c, 0, 0, 0);
}
__device__ inline void mma(f32x16 &c, const Frag16<f16_t> &a, const Frag16<f16_t> &b) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8v, a.v), __builtin_bit_cast(half8v, b.v), c, 0, 0, 0);
}
__device__ inline void mma(f32x16 &c, const f32x8 &a, const f32x8 &b) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
}

// Two values rounded to nearest even and packed, x0 in the low half.  Left to the compiler, which knows the distance that
// a matrix instruction needs from the conversion that writes its operand.
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <typename T>
__device__ inline uint32_t round_pair(float x0, float x1) {
  const f32x2 x = {x0, x1};
  if constexpr (__is_same(T, bf16_t)) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, pair));
  } else {
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, pair));
  }
}

// Registers 8 c .. 8 c + 7 of a block as the right operand of the next product.  16-bit storage rounds here: the matrix
// instruction takes no wider operand, and the probabilities carry one rounding as a stored probability matrix would (the
// kernel for few rows adds what the rounding leaves out; dS is rounded once, too).
// fp16 rounds to a fixed step below 2^-14, and the thousands of probabilities that add up to a result may all lie there: they
// are kept kRaise powers of two higher (2^14 for a probability of 1, of the 2^16 that fp16 holds), so that only those below
// 2^-28 of the largest lose bits.  It costs nothing forward: the raise is part of the exponent, and the sum carries it too.
template <typename T>
constexpr float kRaise = __is_same(T, f16_t) ? 14.f : 0.f;
template <typename T>
constexpr float kLower = __is_same(T, f16_t) ? 0x1p-14f : 1.f;  // 2^-kRaise
template <typename T>
__device__ inline Frag16<T> as_operand(const f32x16 &p, int c, Frag16<T> *) {
  Frag16<T> f;
#pragma unroll
  for (int e = 0; e < 4; ++e) f.v[e] = round_pair<T>(p[8 * c + 2 * e], p[8 * c + 2 * e + 1]);
  return f;
}
__device__ inline f32x8 as_operand(const f32x16 &p, int c, f32x8 *) {
  f32x8 f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = p[8 * c + j];
  return f;
}

// ---- global memory --------------------------------------------------------------------------------------------------

template <typename T>
struct alignas(sizeof(T)) Chunk {  // 16 bytes at any address that suits the element
  T v[16 / sizeof(T)];
};

// 16 bytes of a row of d elements from element c0 on (a multiple of 16 bytes), zeros behind the row's end; all zeros unless
// `in`, which says that the row exists and c0 < d.
// WHOLE: d is a whole number of 16-byte chunks and the rows are aligned to them.  Otherwise the last chunk is read so that
// it ends with the row, and shifted into place by the same amount in all lanes: nothing waits for a load in either case, so
// that all of a lane's loads are in flight together.  Only rows shorter than one chunk (TINY: they may be) go element by
// element.  A lane
// without a part of the row then loads nothing: 16-byte loads at addresses that are no multiple of 16 cost their time per
// lane (fp32 heads of 65: 39 against 51 us with every lane loading).
template <bool WHOLE, bool TINY, typename T>
__device__ inline u32x4 load_part(const T *row, bool in, int c0, int d) {
  constexpr int N = 16 / (int)sizeof(T);
  u32x4 x = {0, 0, 0, 0};
  if constexpr (WHOLE) {
    x = *reinterpret_cast<const u32x4 *>(row + (in ? c0 : 0));
  } else if (!TINY || d >= N) {
    if (in) __builtin_memcpy(&x, reinterpret_cast<const Chunk<T> *>(row + min(c0, d - N)), 16);
    const int missing = d % N;
    if (missing != 0) {
      const uint32_t bytes = (uint32_t)(N - missing) * (uint32_t)sizeof(T);
      u32x4 y = x;
      if (bytes & 4) y = u32x4{y[1], y[2], y[3], 0};
      if (bytes & 8) y = u32x4{y[2], y[3], 0, 0};
      if (bytes & 2) y = u32x4{y[0] >> 16 | y[1] << 16, y[1] >> 16 | y[2] << 16, y[2] >> 16 | y[3] << 16, y[3] >> 16};
      x = c0 > d - N ? y : x;
    }
  } else if (in) {
    T e[N] = {};
#pragma unroll
    for (int i = 0; i < N - 1; ++i)
      if (c0 + i < d) e[i] = row[c0 + i];
    __builtin_memcpy(&x, e, 16);
  }
  return in ? x : u32x4{0, 0, 0, 0};
}

// A lane's 8 elements d0 .. d0 + 7 of a row, zeros behind the row's end or for a row that is not `valid` (the address of an
// existing row is needed all the same).
template <bool WHOLE, bool TINY, typename T>
__device__ inline Frag<T> load_frag(const T *row, bool valid, int d0, int d) {
  if constexpr (sizeof(T) == 2) {
    return {load_part<WHOLE, TINY>(row, valid && d0 < d, d0, d)};
  } else {
    const u32x4 lo = load_part<WHOLE, TINY>(row, valid && d0 < d, d0, d);
    const u32x4 hi = load_part<WHOLE, TINY>(row, valid && d0 + 4 < d, d0 + 4, d);
    f32x8 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t l = lo[e], h = hi[e];  // a bit cast of a vector's element itself takes the first one
      f[e] = __builtin_bit_cast(float, l);
      f[e + 4] = __builtin_bit_cast(float, h);
    }
    return f;
  }
}

// All of a lane's parts of a row: 16 c + 8 (lane / 32) + 0 .. 7.
template <typename T, int NC>
__device__ inline void load_row(Frag<T> (&f)[NC], const T *row, bool valid, const Shape &s, int lane) {
  if (s.whole) {
#pragma unroll
    for (int c = 0; c < NC; ++c) f[c] = load_frag<true, false>(row, valid, 16 * c + 8 * (lane >> 5), (int)s.d);
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) f[c] = load_frag<false, NC == 2>(row, valid, 16 * c + 8 * (lane >> 5), (int)s.d);
  }
}

// The compiler has waited for these loads when it gets here: a loop that counts its own loads behind this would otherwise
// wait for all of them in every round, because the first one may find these still on their way.
template <typename F, int N>
__device__ inline void arrived(const F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (sizeof(F) == 16) {
      asm volatile("" ::"v"(f[i].v) : "memory");
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = f[i][j];
        asm volatile("" ::"v"(x) : "memory");
      }
    }
  }
}

template <typename T>
__device__ inline float element(const Frag16<T> &f, int j) {
  const uint32_t bits = (j & 1) ? f.v[j >> 1] >> 16 : f.v[j >> 1] & 0xffffu;
  if constexpr (__is_same(T, bf16_t)) return __builtin_bit_cast(float, bits << 16);
  else return to_f32(__builtin_bit_cast(f16_t, (uint16_t)bits));
}
__device__ inline float element(const f32x8 &f, int j) { return f[j]; }

__device__ inline u32x4 buffer_words(const void *p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  // the address is the same in all lanes, which the compiler cannot always see
  u32x4 r = {(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
             (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)),
             (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
  return r;
}

// One 16-byte-per-lane buffer load whose destination is LDS: lane l's data lands at lds_addr + 16 l, zeros for lanes
// past the end of the buffer.  Inline assembly keeps the compiler from waiting for it in front of every later LDS read;
// the kernels wait themselves (wait_loads) before the barrier that publishes a tile.  m0 is scratch; the wait state
// between its write and the load is the one the instruction set asks for.
__device__ inline void lds_dma_b128(u32x4 rsrc, uint32_t lds_addr, uint32_t voffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds_addr)), "v"(voffset), "s"(rsrc)
               : "memory");
}
// The 4-byte form: lane l's data lands at lds_addr + 4 l.
__device__ inline void lds_dma_b32(u32x4 rsrc, uint32_t lds_addr, uint32_t voffset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)lds_addr)), "v"(voffset), "s"(rsrc)
               : "memory");
}
template <int N>
__device__ inline void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// ---- tiles in LDS ---------------------------------------------------------------------------------------------------
//
// A tile is ROWS rows of DP elements (the head size rounded up to a multiple of 32, zeros behind the row's end) at a
// pitch of a power of two.  The 16-byte chunk c of a row sits at position c ^ swizzle(row), so that both the reads along
// a row (16 consecutive rows, the same chunk) and the transposing reads (4 consecutive rows, 4 neighbouring chunks)
// spread over all 64 banks.
template <typename T, int DP>
struct Tile {
  static constexpr int kPitch = (DP <= 32 ? 32 : DP <= 64 ? 64 : 128) * (int)sizeof(T);  // bytes
  static constexpr int kChunks = kPitch / 16;
  static constexpr int kPerChunk = 16 / (int)sizeof(T);

  __device__ static inline int swizzle(int row) {
    if constexpr (kChunks >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (kChunks == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
  }

  // What a lane adds to a tile's address for the reads along rows: row lane % 32 of a 32-row block, half lane / 32.
  __device__ static inline uint32_t row_lane(int lane) {
    const int row = lane & 31, h = lane >> 5;
    const int c = sizeof(T) == 2 ? h : 2 * h;
    return (uint32_t)(row * kPitch + ((c ^ swizzle(row)) << 4));
  }
  // Elements 16 c + 8 h .. + 7 of the lane's row of block `blk`; `at` = tile address + row_lane.
  __device__ static inline Frag<T> row_frag(uint32_t at, int blk, int c) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t a = (at ^ (uint32_t)(c << 5)) + (uint32_t)(blk * 32 * kPitch);
      return {*lds_ptr<u32x4>(a)};
    } else {
      const uint32_t a = (at ^ (uint32_t)(c << 6));
      const f32x4 lo = *lds_ptr<f32x4>(a + (uint32_t)(blk * 32 * kPitch));
      const f32x4 hi = *lds_ptr<f32x4>((a ^ 16u) + (uint32_t)(blk * 32 * kPitch));
      return {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }

  // The same for the transposing reads: the fragment of column 32 db + lane % 32 over the 16 rows of chunk rc in the
  // order described at the top (rows 16 rc + 4 h + j, then 16 rc + 8 + 4 h + j).
  __device__ static inline uint32_t col_lane(int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      // ds_read_b64_tr_b16: of 16 lanes, lane 4 a + b receives element b of the 8 bytes that lanes a, 4 + a, 8 + a and
      // 12 + a point to; lane s points to row 4 h + s / 4, columns 4 (s % 4) .. + 3 of its 16
      const int s = lane & 15, row = 4 * h + (s >> 2), col = 16 * ((lane >> 4) & 1) + 4 * (s & 3);
      return (uint32_t)(row * kPitch + (((col >> 3) ^ swizzle(row)) << 4) + (col & 7) * 2);
    } else {
      const int row = 4 * h, col = lane & 31;
      return (uint32_t)(row * kPitch + (((col >> 2) ^ swizzle(row)) << 4) + (col & 3) * 4);
    }
  }
  __device__ static inline Frag<T> col_frag(uint32_t at, int rc, int db) {
    if constexpr (sizeof(T) == 2) {
      // rows 8 further on: the swizzle's low bits move by 2
      const uint32_t a = (at ^ (uint32_t)(db << 6)) + (uint32_t)(16 * rc * kPitch);
      const uint32_t b = (at ^ (uint32_t)(db << 6) ^ 32u) + (uint32_t)((16 * rc + 8) * kPitch);
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr<s16x4>(a)));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(lds_ptr<s16x4>(b)));
      return {{lo[0], lo[1], hi[0], hi[1]}};
    } else {
      f32x8 f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = 16 * rc + (j & 3) + 8 * (j >> 2);  // + 4 h, which is in `at`
        f[j] = *lds_ptr<float>((at ^ (uint32_t)(db << 7) ^ flip(j)) + (uint32_t)(row * kPitch));
      }
      return f;
    }
  }
  // (fp32) swizzle(4 h + row offset of element j) ^ swizzle(4 h), in bytes: the same for both halves
  __device__ static inline uint32_t flip(int j) {
    const int off = (j & 3) + 8 * (j >> 2);
    if constexpr (kChunks >= 16) return (uint32_t)((((off & 3) << 2) | (((off >> 3) & 1) << 1)) << 4);
    else return (uint32_t)(((((off >> 1) & 1) << 2) | (((off >> 3) & 1) << 1)) << 4);
  }
};

// Moves tiles of ROWS rows from global memory to LDS with NT threads.  Row r of a tile is at base + offset(r), where
// offset(r) = (r / g) * stride + (r % g) * inner (g rows lie `inner` apart, then `stride`): g = 1 for keys and values, the
// heads of a group for queries.  DMA: rows at 4-byte aligned addresses go straight to LDS, 16 bytes per lane (the chunk
// that holds a row's end brings the beginning of the next row along, see `clean`); otherwise they pass through registers
// (fetch before the computation on the tile before, put after it).
template <typename T, int DP, int ROWS, int NT, bool DMA>
struct TileLoader {
  typedef Tile<T, DP> L;
  static constexpr int kBytes = ROWS * L::kPitch;
  static constexpr int kInstr = kBytes / 16 / NT;
  static_assert(kBytes % (16 * NT) == 0, "a tile is a whole number of chunks per thread");
  static constexpr int kRowsPer = NT / L::kChunks;  // rows that one load per thread covers
  u32x4 held[DMA ? 1 : kInstr];
  // Load q of a thread takes row q kRowsPer + lane_row of the tile.  The swizzle is linear over the bits of the row, so the
  // thread's chunk is the one of its first row, exclusive-or a constant of q; and with g a divisor of kRowsPer the rows of q
  // lie `step` bytes behind each other.  So three registers describe a thread's part of every tile.
  uint32_t rowpart, c16, step;
  int lane_row;
  bool linear;

  __device__ inline void init(uint32_t g, uint32_t stride, uint32_t inner, int tid) {
    lane_row = tid / L::kChunks;
    c16 = (uint32_t)(((tid % L::kChunks) ^ L::swizzle(lane_row)) << 4);
    linear = kRowsPer % g == 0;
    rowpart = ((uint32_t)lane_row / g * stride + (uint32_t)lane_row % g * inner) * (uint32_t)sizeof(T);
    step = kRowsPer / g * stride * (uint32_t)sizeof(T);
  }

  // rows_left: rows of the tile that exist (may be <= 0 or more than ROWS).  first: where the tile's first row lies in
  // its group of g (0 when g == 1); base is the address of row -first (any address when no row exists).
  __device__ inline void fetch(const T *base, int rows_left, uint32_t first, uint32_t g, uint32_t inv_g, uint32_t stride,
                               uint32_t inner, int d, uint32_t lds_addr, int tid) {
    if constexpr (DMA) {
      uint32_t bytes = 0x7fffffffu;
      if (d % L::kPerChunk != 0) {  // the buffer ends with the last row that exists: nothing behind it is read
        const uint32_t last = first + (uint32_t)max(0, min(rows_left, ROWS) - 1), t = (last * inv_g) >> 22;
        bytes = rows_left > 0 ? (t * stride + (last - t * g) * inner + (uint32_t)d) * (uint32_t)sizeof(T) : 0;
      }
      const u32x4 rsrc = buffer_words(base, bytes);
      const uint32_t wave_at = (uint32_t)__builtin_amdgcn_readfirstlane((tid & ~63) * 16);
      const uint32_t row_bytes = (uint32_t)d * (uint32_t)sizeof(T);
      if (linear) {
#pragma unroll
        for (int q = 0; q < kInstr; ++q) {
          const uint32_t c = c16 ^ (uint32_t)(L::swizzle(q * kRowsPer) << 4), off = rowpart + c + (uint32_t)q * step;
          const bool in = lane_row < rows_left - q * kRowsPer && c < row_bytes;
          lds_dma_b128(rsrc, lds_addr + wave_at + (uint32_t)(q * NT * 16), in ? off : kOutOfRange);
        }
      } else {
#pragma unroll
        for (int q = 0; q < kInstr; ++q) {
          const uint32_t c = c16 ^ (uint32_t)(L::swizzle(q * kRowsPer) << 4);
          const uint32_t r = first + (uint32_t)(lane_row + q * kRowsPer), t = (r * inv_g) >> 22;
          const uint32_t off = (t * stride + (r - t * g) * inner) * (uint32_t)sizeof(T) + c;
          const bool in = lane_row < rows_left - q * kRowsPer && c < row_bytes;
          lds_dma_b128(rsrc, lds_addr + wave_at + (uint32_t)(q * NT * 16), in ? off : kOutOfRange);
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < kInstr; ++q) {
        const int c0 = (int)(c16 ^ (uint32_t)(L::swizzle(q * kRowsPer) << 4)) / (int)sizeof(T);
        const uint32_t r = first + (uint32_t)(lane_row + q * kRowsPer), t = (r * inv_g) >> 22;
        const bool in = lane_row + q * kRowsPer < rows_left && c0 < d;
        held[q] = load_part<false, DP == 32>(base + (in ? t * stride + (r - t * g) * inner : 0), in, c0, d);
      }
    }
  }
  __device__ inline void put(uint32_t lds_addr, int tid) {
    if constexpr (!DMA) {
#pragma unroll
      for (int q = 0; q < kInstr; ++q) *lds_ptr<u32x4>(lds_addr + (uint32_t)((q * NT + tid) * 16)) = held[q];
    }
  }
  // (DMA, d no whole number of chunks) After a tile has landed: zeros behind every row's end, so that the other operand's
  // zeros there meet zeros whatever the next row holds.  ROWS threads.
  __device__ static inline void clean(uint32_t lds_addr, int d, int tid) {
    if constexpr (DMA) {
      if (d % L::kPerChunk == 0 || tid >= ROWS) return;
      const uint32_t chunk = lds_addr + (uint32_t)(tid * L::kPitch) + (uint32_t)(((d / L::kPerChunk) ^ L::swizzle(tid)) << 4);
#pragma unroll
      for (int w = 0; w < 4; ++w)  // rows are whole dwords
        if (w * 4 >= d % L::kPerChunk * (int)sizeof(T)) *lds_ptr<uint32_t>(chunk + 4 * w) = 0;
    }
  }
};

// ceil(2^22 / g): (r * inverse(g)) >> 22 == r / g for r * g < 2^22.  Rows near a tile: r < 192 + g, g <= kMostGroup.
inline uint32_t inverse(uint32_t g) { return ((1u << 22) + g - 1) / g; }
constexpr uint32_t kMostGroup = 1024;

// Rows r0, r0 + 1, ... of a key head: row r is query token r / g, head r % g of the group.  `walk` finds the row r0 + i
// for i < 192 without a division.
struct RowWalk {
  uint32_t t0, in0, g, inv_g;
  // r0 is the same in all lanes, which the compiler cannot always see
  __device__ inline RowWalk(uint32_t r0, const Shape &s) : g(s.g), inv_g(s.inv_g) {
    t0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(r0 / s.g));
    in0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(r0 - t0 * s.g));
  }
  // where row r0 + i lies among rows of hq heads per token
  __device__ inline size_t at(uint32_t i, uint32_t hq) const {
    const uint32_t r = in0 + i, t = (r * inv_g) >> 22;
    return (size_t)(t0 + t) * hq + (r - t * g);
  }
  __device__ inline void advance(uint32_t n) {
    const uint32_t r = in0 + n, t = (r * inv_g) >> 22;
    t0 += t;
    in0 = r - t * g;
  }
};

// ---- small things ---------------------------------------------------------------------------------------------------

// Maximum and sum over the two halves of a wavefront (lanes l and l ^ 32), the same bits in both.
template <typename OP>
__device__ inline float over_halves(float x, OP op) {
  // the swap of a register's upper half with the lower half of its copy leaves the two halves in two registers
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return op(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ inline float halves_max(float x) {
  return over_halves(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline float halves_sum(float x) {
  return over_halves(x, [](float a, float b) { return a + b; });
}

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Row of register i of a result block, without the 4 (lane / 32).
__host__ __device__ constexpr int block_row(int i) { return (i & 3) + 8 * (i >> 2); }

// Four consecutive elements p[0..3], of which the first `n` exist; `vec`: p is aligned to four elements.
template <typename T, bool ACC>
__device__ inline void store4(T *p, const float (&x)[4], int n, bool vec) {
  if (vec && n >= 4) {
    struct alignas(4 * sizeof(T)) Quad {
      T v[4];
    } q;
    if constexpr (ACC) q = *reinterpret_cast<const Quad *>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) q.v[e] = from_f32<T>(ACC ? to_f32(q.v[e]) + x[e] : x[e]);
    *reinterpret_cast<Quad *>(p) = q;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = from_f32<T>(ACC ? to_f32(p[e]) + x[e] : x[e]);
  }
}

// Where a workgroup's tile lies: tile `t` of sequence `e`, or (e.sample == kNoSequence) tile `t` of the rows behind the
// last packed sequence.  `slot` counts the tiles of all sequences.
//  * whole and padded samples: n tiles per step, the last tile of every sample first when `last_first` (with a causal mask
//    the last rows see the most keys, so the long tiles start first);
//  * packed: sequence i starts at slot floor(rows before it / size) + i, which leaves room for its ceil(rows / size)
//    tiles; a slot that is left over has a tile past the end.
constexpr uint32_t kNoSequence = 0xffffffffu;
struct Place {
  SequenceEntry e;
  uint32_t t;
};
// The same value in all lanes, which the compiler cannot always see: kept in a scalar register.
__device__ inline uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
__device__ inline SequenceEntry uniform(const SequenceEntry &e) {
  return {uniform(e.sample), uniform(e.q_start), uniform(e.q_len), uniform(e.k_start), uniform(e.k_len), uniform(e.q_cum),
          uniform(e.k_cum), 0};
}
// rows_per: rows per token (g for queries, 1 for keys); tiles: tiles of a whole sample; by_keys: tiles of keys.
__device__ inline Place find_place(const SequenceView &s, uint32_t slot, uint32_t tiles, uint32_t size, uint32_t rows_per,
                                   bool by_keys, bool last_first) {
  if (!s.packed) {
    const uint32_t t = slot / s.n;
    return {uniform(s.at(uniform(slot - t * s.n))), uniform(last_first ? tiles - 1 - t : t)};
  }
  const uint32_t total = by_keys ? s.k_total : s.q_total;
  const uint32_t behind = (uint32_t)((uint64_t)total * rows_per / size) + s.n;
  if (slot >= behind) return {{kNoSequence, 0, 0, 0, 0, 0, 0, 0}, uniform(slot - behind)};
  uint32_t lo = 0, hi = s.n;  // the last entry whose first slot is not behind `slot`
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    const uint32_t cum = by_keys ? s.entries[mid].k_cum : s.entries[mid].q_cum;
    if ((uint32_t)((uint64_t)cum * rows_per / size) + mid <= slot) lo = mid;
    else hi = mid;
  }
  const SequenceEntry e = uniform(s.entries[lo]);
  const uint32_t t = slot - ((uint32_t)((uint64_t)(by_keys ? e.k_cum : e.q_cum) * rows_per / size) + lo);
  const uint32_t own = (uint32_t)(((uint64_t)(by_keys ? e.k_len : e.q_len) * rows_per + size - 1) / size);
  return {e, uniform(last_first && t < own ? own - 1 - t : t)};
}
// Slots that find_place can be asked for, per key head.
inline uint64_t slots(const SequenceView &s, uint32_t size, uint32_t rows_per, bool by_keys) {
  const uint64_t tokens = by_keys ? s.tk : s.tq, total = by_keys ? s.k_total : s.q_total;
  if (!s.packed) return (uint64_t)s.n * ((tokens * rows_per + size - 1) / size);
  return total * rows_per / size + s.n + ((tokens - total) * rows_per + size - 1) / size;
}

// ---- which kernel ---------------------------------------------------------------------------------------------------

// Stages of a wavefront's own ring of pairs of 32-row tiles: four wavefronts take 128 KiB of LDS at most.
template <typename T, int DP>
constexpr int kStages = 32 * Tile<T, DP>::kPitch <= 8192 ? 2 : 1;

// Which kernel walks over a call's tiles: the one whose workgroup shares every tile between 128 rows (or keys), or the one
// where each wavefront walks over tiles of its own, four or one of them with the same 32 rows (keys).
//
// Shared tiles cost the least per product, so they are taken wherever their workgroups fill the chip; with one for every
// second CU or fewer the finer division wins.  Both sides, us per training step, causal:
//   bf16, 16/4 heads of 128:   4 x 128 tokens 70 -> 41,   4 x 512 192 -> 94,   1 x 2048 672 -> 281
//   fp32, 16/4 heads of 128:   4 x 128       223 -> 83,   4 x 512 803 -> 360,  1 x 2048 3129 -> 1085
//   and the other way with a workgroup per CU: bf16, 16 heads of 65, 4 x 512: 149 shared, 301 with tiles of their own.
// fp32 products take four times as long per tile, which hides the loads of the finer division: there it also wins with a
// workgroup per CU when the walk is long (16 heads of 65, 1 x 2048: 1068 -> 740).
// One wavefront per workgroup: fp32 sequences so short that a 128-row tile is mostly empty and so many that every SIMD has
// one anyway (in 16-bit storage it does not pay: 16 heads of 65, 64 x 35 tokens: 125 against 157).  us per training step
// without -> with, by the number of 32-row tiles:
//                                512            1024           4096
//   8 tokens, 8 heads of 128     80 -> 44       154 -> 50      619 -> 185
//   32 tokens, 16 of 64          50 -> 32       98 -> 43       370 -> 164
//   35 tokens, 10 of 65          66 -> 71       116 -> 87      441 -> 295
//   64 tokens, 16 of 64          40 -> 43       69 -> 52       240 -> 196  (forward alone 43 -> 51)
//   96 tokens, 16 of 64          52 -> 54       92 -> 62       253 -> 221
//   128 tokens, 16 of 64         64 -> 65       70 -> 73       233 -> 250
// Walks of more than 256 keys (rows) want the 1024 tiles too: 4 queries, 500 keys, 8 heads of 128, forward: 58 -> 84 and
// 117 -> 96.
enum class Way { Shared, Four, One };
// wide, narrow: workgroups with tiles of 128 and of 32; most: rows (keys) of the longest sequence; walked: what its
// workgroups walk over.
template <typename T>
inline Way choose_way(phip_ctx *ctx, uint64_t wide, uint64_t narrow, uint64_t most, uint64_t walked) {
  const uint64_t cus = (uint64_t)ctx->prop.multiProcessorCount;
  if (sizeof(T) == 4 && most <= 64 && narrow >= (most <= 32 && walked <= 256 ? 2 : 4) * cus) return Way::One;
  if (wide * 2 <= cus || (sizeof(T) == 4 && wide <= cus && walked >= 1024)) return Way::Four;
  return Way::Shared;
}

constexpr uint32_t kMostSize = 128;  // largest head size
// A launch has fewer than 2^32 threads.
inline bool launchable(uint64_t blocks, uint64_t threads) { return blocks < (1ull << 32) / threads; }

// Checks what the forward and the gradient calls have in common.
inline int make_shape(uint32_t d, uint32_t hq, uint32_t hk, uint32_t tq, uint32_t tk, uint32_t bs, int causal, float scale,
                      size_t item, Shape *out) {
  PHIP_REQUIRE(d >= 1 && d <= kMostSize, "head sizes of 1 to %u are supported, got %u", kMostSize, d);
  PHIP_REQUIRE(hq >= 1 && hk >= 1 && hq % hk == 0, "%u query heads cannot share %u key heads", hq, hk);
  PHIP_REQUIRE(hq / hk <= kMostGroup, "more than %u query heads per key head", kMostGroup);
  PHIP_REQUIRE(tq >= 1 && tk >= 1 && bs >= 1, "empty tensors");
  // rows of a key head (queries times heads of the group) are counted in 32 bits, with room for a tile
  PHIP_REQUIRE((uint64_t)tq * (hq / hk) <= 0x7fffff00u && tk <= 0x7fffff00u, "more than 2^31 - 256 rows per key head");
  // offsets inside a tile of 64 rows are 32 bits wide
  PHIP_REQUIRE((uint64_t)d * hq * item * 72 < 0x7fffffffu, "heads of %u x %u elements are too large", hq, d);
  PHIP_REQUIRE(scale > 0.f && scale <= 1e30f, "the scale must be positive and at most 1e30");
  *out = {d, hq, hk, hq / hk, inverse(hq / hk), causal != 0 ? 1u : 0u, scale * kLog2e, scale, 0};
  return PHIP_OK;
}

// Lets KERNEL use `bytes` of dynamic LDS (more than the default 64 KiB) on the context's device; done once per device.
template <auto *KERNEL>
int allow_lds(phip_ctx *ctx, int bytes) {
  static std::atomic<uint64_t> done{0};
  if (bytes <= 64 * 1024 || (ctx->device < 64 && ((done.load() >> ctx->device) & 1))) return PHIP_OK;
  PHIP_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (ctx->device < 64) done.fetch_or(1ull << ctx->device);
  return PHIP_OK;
}

// True when rows of d elements at all the pointers are multiples of `unit` bytes: 4 to be moved to LDS without passing
// through registers, 16 for plain 16-byte loads.
inline bool rows_aligned(uint32_t d, size_t item, size_t unit, std::initializer_list<const void *> ptrs) {
  if (d * item % unit != 0) return false;
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % unit != 0) return false;
  return true;
}

inline bool elements_aligned(size_t item, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % item != 0) return false;
  return true;
}

}  // namespace attention
}  // namespace phip

#endif  // PHIP_ATTENTION_H_
