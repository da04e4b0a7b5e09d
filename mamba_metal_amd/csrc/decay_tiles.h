// Tiles of decaying linear attention: matrix-core operands read from shared memory, and a run's decays.
//
// All products are 16 x 16 tiles with fp32 accumulators.  Lane l = 16 g + i (g = l / 16) holds of an operand the row
// (or column) i and kE of the kStep elements of the sum, and of an accumulator column i, rows 4 g .. 4 g + 3.  Which
// elements of the sum a lane holds is free as long as both operands agree:
//   row order   k = kE g + j                            one 16-byte read of a row
//   acc order   k = 4 g + j, and 16 + 4 g + (j - 4)     the rows of two accumulator tiles, so that an accumulator is an
//                                                       operand of the next product without leaving its registers
// (fp32 operands: kE = 4, and the two orders are one).
#pragma once

#include "mm_common.h"

#include "decay_shape.h"

namespace mm {
namespace dattn {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
struct Op {
  using T = typename Ty<DT>::T;
  static constexpr bool kWide = DT == MM_F32;
  static constexpr int kE = kWide ? 4 : 8;      // elements of an operand in a lane
  static constexpr int kStep = 4 * kE;          // elements of the sum an operand covers
  static constexpr int kTiles = kWide ? 1 : 2;  // accumulator tiles an operand is made of
};

template <int DT>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MM_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == MM_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
}

// Two fp32 values as a pair of T in one word (round to nearest even).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == MM_BF16) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), bf2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2{static_cast<_Float16>(a), static_cast<_Float16>(b)}));
  }
}
template <int DT>
__device__ __forceinline__ void unpack2(uint32_t v, float& a, float& b) {
  if constexpr (DT == MM_BF16) {
    a = __uint_as_float(v << 16);
    b = __uint_as_float(v & 0xffff0000u);
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = __builtin_bit_cast(h2, v);
    a = static_cast<float>(h[0]);
    b = static_cast<float>(h[1]);
  }
}

// An operand in acc order of kTiles accumulator tiles.
template <int DT>
__device__ __forceinline__ u32x4 from_acc(const f32x4* t) {
  if constexpr (Op<DT>::kWide) return __builtin_bit_cast(u32x4, t[0]);
  else
    return u32x4{pack2<DT>(t[0][0], t[0][1]), pack2<DT>(t[0][2], t[0][3]), pack2<DT>(t[1][0], t[1][1]),
                 pack2<DT>(t[1][2], t[1][3])};
}

// 16-bit operands of a product whose result is a state in fp32: the value as a sum of TERMS of them.  bf16: three are
// fp32's own 24 bits.  fp16: two hold 22 bits, the second one 2^11 times too large (and summed by itself), since the rest of a
// value below 1/8 would be subnormal.  The matrix cores take subnormals as they are, but those hold fewer bits: a value below
// 2^-14 is off by up to 2^-36.
constexpr float kRestUp = 2048.0f;
template <int DT, int TERMS>
__device__ __forceinline__ void split_operand(const float (&x)[8], u32x4 (&out)[TERMS]) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    rest[j] = x[j];
    // (x, a product, as it is in fp32: its first term would else be one rounding of the exact product in the operand and the
    // rounding of an fp32 one where it is subtracted, next to a tie two numbers that are a step apart)
    if (DT == MM_F16) asm("" : "+v"(rest[j]));
  }
#pragma unroll
  for (int n = 0; n < TERMS; ++n)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float up = DT == MM_F16 && n == 1 ? kRestUp : 1.0f;
      const uint32_t w = pack2<DT>(rest[j] * up, rest[j + 1] * up);
      out[n][j / 2] = w;
      if (n + 1 < TERMS) {
        float a, b;
        unpack2<DT>(w, a, b);
        rest[j] -= a;
        rest[j + 1] -= b;
      }
    }
}

// Scores (accumulator tiles, in acc order) as operands, rounded once.  A score's rounding is the same in all channels of its
// token, so that few tokens may all be off by nearly half a step where many are by a third: `fine` ones, of calls of few
// tokens, take a second term, the rest.  (Forward pass of 32 heads of 128 by 64 in bf16 (fp16), 65536 tokens x heads: 41.1 us
// and 42.0 with it (42.7 and 43.7); 262144: 70 and 75 (78 and 87).)
template <int DT>
__device__ __forceinline__ void score_operand(const f32x4* t, bool fine, u32x4& whole, u32x4& rest) {
  whole = from_acc<DT>(t);
  if constexpr (!Op<DT>::kWide) {
    if (fine) {
      const float x[8] = {t[0][0], t[0][1], t[0][2], t[0][3], t[1][0], t[1][1], t[1][2], t[1][3]};
      u32x4 terms[2];
      split_operand<DT, 2>(x, terms);
      whole = terms[0];
      rest = terms[1];
    }
  }
}
// fp16 has 5 exponent bits: a token's scores go through a power of two that puts the largest of them, m, at 2^13, and what
// they are added to with them (2^40 at most, which leaves an output's other parts in fp32's range).  All of scores near 1e-5
// would be subnormal, and off by 2^-8 of them and more.
__device__ __forceinline__ void score_range(float m, float& up, float& down) {
  const int e = static_cast<int>(__float_as_uint(m) >> 23) - 127, k = e > 53 ? -40 : e < -27 ? 40 : 13 - e;
  const bool ok = m > 0.0f && e < 128;
  up = ok ? __uint_as_float((127 + k) << 23) : 1.0f;
  down = ok ? __uint_as_float((127 - k) << 23) : 1.0f;
}
template <int N>
__device__ __forceinline__ float largest(const f32x4 (&t)[N]) {  // of a column of accumulator tiles, in its four lanes
  float m = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(t[n][r]));
  m = fmaxf(m, lane_xor(m, 16));
  return fmaxf(m, lane_xor(m, 32));
}
// The product with the rest.
template <int DT>
__device__ __forceinline__ f32x4 mma_rest(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == MM_F16) return c + mma<DT>(a, b, f32x4{0.0f, 0.0f, 0.0f, 0.0f}) * (1.0f / kRestUp);
  else return mma<DT>(a, b, c);
}

// A tile of W columns in shared memory.  16-bit rows are cut into chunks of 16 bytes, and chunk c of row r is kept at
// place c ^ turn(r), without bank conflicts: a transposing read touches pairs of chunks of 8 rows, whose turns differ above
// the lowest bit; a 16-byte row read goes in four parts of 16 lanes, 0-3, 12-15 and 20-27 and so on, so that rows 4 to 11 of
// one chunk and the other rows of its neighbour meet, and those have both turns of each pair.  (fp32: rows 4 words longer.)
template <int DT, int W>
struct Tile {
  using T = typename Ty<DT>::T;
  static constexpr bool kWide = Op<DT>::kWide;
  static constexpr int kLd = kWide ? W + 4 : W;
  static __device__ __forceinline__ int turn(int r) {
    return W == 128 ? ((r & 7) ^ (r >> 1 & 4)) << 1 | (r >> 3 & 1) : ((r >> 1 & 3) ^ (r >> 2 & 2)) << 1 | (r >> 3 & 1);
  }
  static __device__ __forceinline__ int at(int r, int e) {
    return kWide ? r * kLd + e : r * kLd + (((e >> 3) ^ turn(r)) << 3) + (e & 7);
  }
  // at(r0 + r, e0 + e) for an r0 that 16 divides, which does not turn, and an e0 that has no bit of e's: it only flips bits of
  // what is the same for all of a lane's accesses, an instruction each where `at` would take four.
  static __device__ __forceinline__ int at(int r0, int e0, int r, int e) {
    return kWide ? (r0 + r) * kLd + e0 + e : r0 * kLd + ((r * kLd + (((e >> 3) ^ turn(r)) << 3) + (e & 7)) ^ e0);
  }
  // Row r0 + i, elements k0 on, in row order.
  static __device__ __forceinline__ u32x4 row(const T* tile, int r0, int k0, int lane) {
    return *reinterpret_cast<const u32x4*>(tile + at(r0, k0, lane & 15, Op<DT>::kE * (lane >> 4)));
  }
  // ... in acc order.
  static __device__ __forceinline__ u32x4 row_acc(const T* tile, int r0, int k0, int lane) {
    const int r = lane & 15, e = 4 * (lane >> 4);
    if constexpr (kWide) {
      return *reinterpret_cast<const u32x4*>(tile + at(r0, k0, r, e));
    } else {
      const u32x2 a = *reinterpret_cast<const u32x2*>(tile + at(r0, k0, r, e));
      const u32x2 b = *reinterpret_cast<const u32x2*>(tile + at(r0, k0 + 16, r, e));
      return u32x4{a[0], a[1], b[0], b[1]};
    }
  }
  // Four elements of column c0 + i of rows r0 + 4 g on, 16-bit types: the transposing read, in which each group of 16
  // lanes reads 4 rows of 16 elements, 8 bytes a lane, and gets a column each.
  static __device__ __forceinline__ u32x2 column4(const T* tile, int r0, int c0, int lane) {
    const T* const p = tile + at(r0, c0, 4 * (lane >> 4) + ((lane & 15) >> 2), 4 * (lane & 3));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)const_cast<T*>(p)));
  }
  // Column c0 + i, rows k0 on, in acc order: an operand whose sum runs over a tile's rows.
  static __device__ __forceinline__ u32x4 column(const T* tile, int k0, int c0, int lane) {
    if constexpr (kWide) {
      u32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = __float_as_uint(tile[at(k0 + 4 * (lane >> 4) + j, c0 + (lane & 15))]);
      return v;
    } else {
      const u32x2 a = column4(tile, k0, c0, lane), b = column4(tile, k0 + 16, c0, lane);
      return u32x4{a[0], a[1], b[0], b[1]};
    }
  }
};

// 64 rows of W elements of one head, as a workgroup of `Threads` stages them, 16 bytes a thread and step, held in
// registers between the load and the write to shared memory.
template <int DT, int W, int Threads>
struct Staged {
  using T = typename Ty<DT>::T;
  static constexpr int kE = Op<DT>::kE;
  static constexpr int kUnits = W / kE;                  // 16-byte units of a row
  static constexpr int kSteps = kRun * kUnits / Threads;
  static constexpr int kRows = Threads / kUnits;         // of a step
  static_assert(kSteps >= 1, "a unit for every thread");
  static_assert(Op<DT>::kWide || kRows % 16 == 0, "steps do not turn");
  u32x4 v[kSteps];
  static __device__ __forceinline__ int row() { return static_cast<int>(threadIdx.x) / kUnits; }
  static __device__ __forceinline__ int elem() { return static_cast<int>(threadIdx.x) % kUnits * kE; }
  // Rows r >= rows and elements >= width come as zeros.  16-byte aligned rows that 16 bytes divide, 64 of them within
  // 4 GB: `first` is the first row's (wave-uniform) address, `off` row() and elem() in bytes, `step` kRows rows in bytes.
  __device__ __forceinline__ void load(const char* first, uint32_t off, int64_t step, int rows, int width) {
    if (rows == kRun && width == W) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s, first += step) v[s] = *reinterpret_cast<const u32x4*>(first + off);
      return;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s, first += step) {
      v[s] = u32x4{0, 0, 0, 0};
      if (s * kRows + row() < rows && elem() < width) v[s] = *reinterpret_cast<const u32x4*>(first + off);
    }
  }
  // Any rows.
  __device__ __forceinline__ void load_any(const char* first, int64_t stride, int rows, int width) {
    const T* const base = reinterpret_cast<const T*>(first) + row() * stride + elem();
    for (int s = 0; s < kSteps; ++s) {
      T t[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j)
        t[j] = s * kRows + row() < rows && elem() + j < width ? base[s * kRows * stride + j] : static_cast<T>(0);
      u32x4 w;
      __builtin_memcpy(&w, t, 16);
#pragma unroll
      for (int q = 0; q < kSteps; ++q) v[q] = q == s ? w : v[q];
    }
  }
  __device__ __forceinline__ void store(T* tile, int tid) const {  // tid: threadIdx.x
#pragma unroll
    for (int s = 0; s < kSteps; ++s) *reinterpret_cast<u32x4*>(tile + Tile<DT, W>::at(s * kRows, 0, tid / kUnits, tid % kUnits * kE)) = v[s];
  }
};

// A run's decays: c_t, the running sum of the log decays to token t and with it, in log2 units.  Sums are 64-bit and
// kept as two floats, so that a difference is exact to fp32 however far both lie down.
struct alignas(16) Decays {
  float hi[kRun], lo[kRun];
  float into[kRun];    // exp(c_t): what the state before the run still counts at t
  float onward[kRun];  // exp(c_last - c_t): what token t still counts at the run's end
  float whole;         // exp(c_last)
};

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// Inclusive sum over the lanes up to each.
__device__ __forceinline__ double prefix_sum(double v) {
  v += dpp_or_zero<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8 within 16 lanes
  v += dpp_or_zero<0x112, 0xF>(v);
  v += dpp_or_zero<0x114, 0xF>(v);
  v += dpp_or_zero<0x118, 0xF>(v);
  v += dpp_or_zero<0x142, 0xA>(v);  // lane 15 of each row to the next, rows 1 and 3
  v += dpp_or_zero<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
  return v;
}

// g: lane t's log decay.  One that vanishes in fp32 anyway (exp(-1000) = 0, as for -inf) is cut off, so that sums stay
// finite and later differences exact.
__device__ __forceinline__ void run_decays(Decays& d, float g, int lane) {
  g = g < -1000.0f ? -1000.0f : g;
  const double c = prefix_sum(static_cast<double>(g)) * 1.4426950408889634;
  const float hi = static_cast<float>(c);
  const double last = __shfl(c, 63, 64);
  d.hi[lane] = hi;
  d.lo[lane] = static_cast<float>(c - hi);
  d.into[lane] = exp2_acc(hi) * (1.0f + static_cast<float>(c - hi) * kLn2);
  const double rest = last - c;
  const float rh = static_cast<float>(rest);
  d.onward[lane] = exp2_acc(rh) * (1.0f + static_cast<float>(rest - rh) * kLn2);
  if (lane == 63) d.whole = exp2_acc(hi) * (1.0f + static_cast<float>(c - hi) * kLn2);
}

// exp(c_t - c_s), or with `back` exp(c_s - c_t)
template <int DT>
__device__ __forceinline__ float between(float hi_t, float lo_t, float hi_s, float lo_s, bool back = false) {
  const float d = (hi_t - hi_s) + (lo_t - lo_s), x = back ? -d : d;
  const float e = exp2_decay<DT>(x);
  return DT == MM_F32 && x != x ? x : e;  // (exp2_acc's clamp would lose a NaN)
}

}  // namespace dattn
}  // namespace mm
