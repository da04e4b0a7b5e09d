// Products of large tiles on the matrix cores: C[m, n] = sum_k A(m, k) B(n, k), both operands streamed through shared
// memory by loads that go there directly, several stages deep.
//
// A stage is a slab of 64 bytes of k (32 16-bit elements, 16 fp32 ones) of the tile's rows, and four are under way.  What
// the 32 units of a die read at once is shared in its cache, so that all of them wait for the same misses: a stage's loads
// take 1.5 to 2 us, twice what its products take, and it is the bytes under way that keep the matrix cores fed.  bf16, 8192
// rows (7377 of them counted) of 2560 by 50280: 1890 us with two stages of 128 bytes behind flat loads, 1.67 to 1.72 ms now,
// 1.12 PFLOP/s; the cores' cycles are 58% busy at the 1.9 GHz that the card holds under it (a library product of the whole
// shape reaches 1.19).  fp32, 2048 by 16384 of 1024: 117 TFLOP/s (123 without the short sums below).
//
// An operand lies in memory either way:
//   kAlong   k is contiguous: a row of the slab is 64 bytes of a row of the matrix, four 16-byte chunks.  Chunk c of
//            row r is kept at place c ^ (r / 4 % 4), so that the rows whose reads meet fall into different banks.
//   kAcross  rows (m or n) are contiguous: the slab is 32 (16) rows of k by the tile's width, read with the transposing
//            read (fp32: element by element), which takes 64 bytes of each of 4 rows of k: those lie side by side.
// The direct load writes 16 bytes a lane at consecutive places, so the arrangement is of the addresses that the lanes
// read.  They are buffer loads: a lane whose element lies past the matrix's k (or past its width, kAcross) is given an
// offset past the buffer's end, which loads zeros, and reads of shared memory wait for themselves alone (behind flat ones
// the compiler waits for all reads under way).  Rows past a matrix's end are its last row again, whose results are not stored.
//
// The 32 x 32 tiles' operand layout: lane l holds row l % 32 and 16 bytes of k, chunk 2 s + l / 32 of the slab at step s
// of 2; an accumulator holds column l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4.
#pragma once

#include <type_traits>

#include "direct_load.h"
#include "mm_common.h"

namespace mm {
namespace slab {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kSlab = 64;  // bytes of k
constexpr int kSteps = 2;  // of 32 bytes
enum Lie { kAlong, kAcross };

template <int DT>
constexpr int kParts = DT == MM_F32 ? 4 : 1;  // products that 16 bytes of each operand make
template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, int part, f32x16 c) {
  if constexpr (DT == MM_F16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == MM_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[part]), __uint_as_float(b[part]), c, 0, 0, 0);
  }
}

struct Matrix {
  const char* base;
  int64_t ld;       // bytes from one row in memory to the next; a tile's rows lie within 2 GB
  int64_t rows;     // kAlong: rows of the operand; kAcross: its columns, in elements
  int64_t k;        // elements of a row
};

// One operand of a workgroup's tile: R rows, staged by NW waves.
template <int DT, Lie LIE, int R, int NW>
struct Side {
  using T = typename Ty<DT>::T;
  static constexpr int kEs = sizeof(T), kWidth = R;
  static constexpr int kDepth = kSlab / kEs;               // elements of k in a slab
  static constexpr int kLoads = R * kSlab / 1024 / NW;     // of a wave, 64 lanes of 16 bytes each
  static_assert(kLoads >= 1 && kLoads * 1024 * NW == R * kSlab, "whole loads");
  // kAcross: a load is kRows rows of k.  16-bit: 64 bytes of each of kSide rows side by side, then the next 64 bytes of
  // them; where a load has but 2 rows, the next one's are 128 bytes further on in the banks.
  static constexpr int kRows = 1024 / (R * kEs), kSide = kRows < 4 ? kRows : 4, kGroups = R * kEs / 64;
  static constexpr int kLoadBytes = LIE == kAcross && kEs == 2 && kRows == 2 ? 1024 + 128 : 1024;  // a load's place
  static constexpr int kBytes = kLoads * NW * kLoadBytes;
  const char* base;       // of the next slab: wave-uniform, and a lane's offset from it fits 32 bits
  uint32_t off[kLoads];
  int64_t step;
  int k_at[kLoads];       // a lane's first element of k in a slab

  // Lane's row of k (kAcross) or first element of k (kAlong), and column of the tile, in its load q.
  static __device__ __forceinline__ int k_of(int q, int wave, int lane) {
    if constexpr (LIE == kAlong) return (lane % 4 ^ (lane >> 4 & 3)) * 16 / kEs;
    else if constexpr (kEs == 2) return (q * NW + wave) * kRows + lane / 4 / kSide / kGroups * kSide + lane / 4 % kSide;
    else return (q * NW + wave) * kRows + lane * 16 / (R * kEs);
  }
  static __device__ __forceinline__ int col_of(int lane) {
    if constexpr (kEs == 2) return lane / 4 / kSide % kGroups * 32 + lane % 4 * 8;
    else return lane * 4 % R;
  }
  __device__ __forceinline__ void init(const Matrix& m, int64_t row0, int64_t k0, int wave, int lane) {
    step = LIE == kAlong ? kSlab : kDepth * m.ld;
    // (a tile may lie past the matrix's end: kAlong its rows are all the last one, kAcross its columns all zeros)
    const int64_t first = LIE == kAlong && row0 >= m.rows ? m.rows - 1 : row0;
    base = m.base + (LIE == kAlong ? first * m.ld + k0 * kEs : k0 * m.ld + first * kEs);
    const int64_t over = m.rows - 1 - first;                 // kAlong: not negative
    const int last = over < R ? static_cast<int>(over) : R;  // row of the tile
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int r = ((q * NW + wave) * 64 + lane) / 4;
      k_at[q] = k_of(q, wave, lane);
      if constexpr (LIE == kAlong) {
        off[q] = static_cast<uint32_t>((r < last ? r : last) * m.ld) + k_at[q] * kEs;
      } else {
        const int col = col_of(lane);
        off[q] = static_cast<uint32_t>(k_at[q] * m.ld) + col * kEs;
        if (row0 + col >= m.rows) k_at[q] = kDepth;  // (never within k)
      }
    }
  }
  // Issues the loads of one slab, of whose k `left` elements are in the matrix, and moves on.  (Without a branch: behind
  // one the compiler waits for all reads of shared memory instead of the oldest.)
  __device__ __forceinline__ void load(char* tile, int64_t left, int wave) {
    const int here = left < kDepth ? static_cast<int>(left < 0 ? 0 : left) : kDepth;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) load_direct(base, k_at[q] < here ? off[q] : kNowhere, tile + (q * NW + wave) * kLoadBytes);
    base += step;
  }
  // Rows r0 .. r0 + 31 at step s of a staged slab.
  static __device__ __forceinline__ u32x4 operand(const char* tile, int r0, int s, int lane) {
    if constexpr (LIE == kAlong) {
      const int r = r0 + (lane & 31), c = 2 * s + (lane >> 5);
      return *reinterpret_cast<const u32x4*>(tile + r * kSlab + ((c ^ (r >> 2 & 3)) << 4));
    } else {
      u32x4 v;
      const char* const p = tile + (8 * s + 4 * (lane >> 5)) * R * kEs + (r0 + (lane & 31)) * kEs;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(p + j * R * kEs);
      return v;
    }
  }
};

// 16-bit kAcross: where a lane's reads of columns r0 on begin, and what a column tile, a step and 4 rows of k are further.
// 16 lanes read 4 rows of k by 16 columns, 8 bytes each, and get a column each.
template <typename SIDE>
struct Across {
  static constexpr int kFour = SIDE::kRows == 2 ? 2 * SIDE::kLoadBytes : 4 * SIDE::kWidth * 2, kStep = 4 * kFour, kTile = SIDE::kSide * 64;
  static __device__ __forceinline__ uint32_t lane_at(int r0, int lane) {
    const int row = (lane & 15) >> 2, in = ((lane & 16) >> 3 | (lane & 3) >> 1) * 16 + (lane & 1) * 8;
    return (r0 >> 5) * kTile + 2 * (lane >> 5) * kFour + (SIDE::kRows == 2 ? (row >> 1) * SIDE::kLoadBytes + (row & 1) * 64 : row * 64) + in;
  }
};
// The operands of N column tiles, or of N and M of both sides, at step S: all reads and their wait in one piece.  (The
// compiler knows of no address in a transposing read, and would have each wait for all loads that fill other stages.)
#define MM_TR "ds_read_b64_tr_b16 "
template <typename C, int S>
__device__ __forceinline__ void across2(uint32_t at, u32x4 (&o)[2]) {
  u32x2 r[4];
  constexpr int s = S * C::kStep, f = C::kFour, t = C::kTile;
  asm volatile(MM_TR "%0, %4 offset:%5\n" MM_TR "%1, %4 offset:%6\n" MM_TR "%2, %4 offset:%7\n" MM_TR "%3, %4 offset:%8\n"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3])
               : "v"(at), "n"(s), "n"(s + f), "n"(s + t), "n"(s + t + f)
               : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) o[i] = u32x4{r[2 * i][0], r[2 * i][1], r[2 * i + 1][0], r[2 * i + 1][1]};
}
template <typename C, typename D, int S>
__device__ __forceinline__ void across22(uint32_t at, uint32_t bt, u32x4 (&o)[2], u32x4 (&p)[2]) {
  u32x2 r[8];
  constexpr int s = S * C::kStep, f = C::kFour, t = C::kTile, s2 = S * D::kStep, f2 = D::kFour, t2 = D::kTile;
  asm volatile(MM_TR "%0, %8 offset:%10\n" MM_TR "%1, %8 offset:%11\n" MM_TR "%2, %8 offset:%12\n" MM_TR "%3, %8 offset:%13\n"
               MM_TR "%4, %9 offset:%14\n" MM_TR "%5, %9 offset:%15\n" MM_TR "%6, %9 offset:%16\n" MM_TR "%7, %9 offset:%17\n"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
               : "v"(at), "v"(bt), "n"(s), "n"(s + f), "n"(s + t), "n"(s + t + f), "n"(s2), "n"(s2 + f2), "n"(s2 + t2), "n"(s2 + t2 + f2)
               : "memory");
#pragma unroll
  for (int i = 0; i < 2; ++i) o[i] = u32x4{r[2 * i][0], r[2 * i][1], r[2 * i + 1][0], r[2 * i + 1][1]};
#pragma unroll
  for (int i = 0; i < 2; ++i) p[i] = u32x4{r[4 + 2 * i][0], r[4 + 2 * i][1], r[5 + 2 * i][0], r[5 + 2 * i][1]};
}
template <typename C, typename D, int S>
__device__ __forceinline__ void across42(uint32_t at, uint32_t bt, u32x4 (&o)[4], u32x4 (&p)[2]) {
  u32x2 r[12];
  constexpr int s = S * C::kStep, f = C::kFour, t = C::kTile, s2 = S * D::kStep, f2 = D::kFour, t2 = D::kTile;
  asm volatile(MM_TR "%0, %12 offset:%14\n" MM_TR "%1, %12 offset:%15\n" MM_TR "%2, %12 offset:%16\n" MM_TR "%3, %12 offset:%17\n"
               MM_TR "%4, %12 offset:%18\n" MM_TR "%5, %12 offset:%19\n" MM_TR "%6, %12 offset:%20\n" MM_TR "%7, %12 offset:%21\n"
               MM_TR "%8, %13 offset:%22\n" MM_TR "%9, %13 offset:%23\n" MM_TR "%10, %13 offset:%24\n" MM_TR "%11, %13 offset:%25\n"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]), "=&v"(r[8]),
                 "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11])
               : "v"(at), "v"(bt), "n"(s), "n"(s + f), "n"(s + t), "n"(s + t + f), "n"(s + 2 * t), "n"(s + 2 * t + f), "n"(s + 3 * t),
                 "n"(s + 3 * t + f), "n"(s2), "n"(s2 + f2), "n"(s2 + t2), "n"(s2 + t2 + f2)
               : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = u32x4{r[2 * i][0], r[2 * i][1], r[2 * i + 1][0], r[2 * i + 1][1]};
#pragma unroll
  for (int i = 0; i < 2; ++i) p[i] = u32x4{r[8 + 2 * i][0], r[8 + 2 * i][1], r[9 + 2 * i][0], r[9 + 2 * i][1]};
}
#undef MM_TR

// A tile's shape: BM x BN by WM x WN waves, each TM x TN tiles of 32 x 32; ST stages.
template <int BM_, int BN_, int WM_, int WN_, int ST_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
  static constexpr int ST = ST_;                                   // stages, and the bytes of one
  static constexpr int kStage = (BM + BN) * kSlab / 8 * (BM == 256 || BN == 256 ? 9 : 8);
};

// A tile's stages: separate objects, so that the compiler sees that one's reads and another's loads do not meet.
#define MM_SLAB_STAGES(S, name)                                                                  \
  __shared__ __attribute__((aligned(16))) char name##0[S::kStage];                               \
  __shared__ __attribute__((aligned(16))) char name##1[S::kStage];                               \
  __shared__ __attribute__((aligned(16))) char name##2[S::kStage];                               \
  __shared__ __attribute__((aligned(16))) char name##3[S::kStage];

// Waits until all but the wave's last `Left` loads are done and its reads of shared memory too, then for the others.
template <int Left>
__device__ __forceinline__ void meet() {
  static_assert(Left < 64, "the counter's range");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((Left & 15) | (Left >> 4) << 14 | 7 << 4);  // vmcnt, expcnt free, lgkmcnt 0
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// acc += the sum over `k` elements from k0 on.  All threads of the workgroup; returns when nobody reads or loads the
// stages any more.
template <int DT, Lie LA, Lie LB, typename S>
__device__ __forceinline__ void product(const Matrix& A, const Matrix& B, int64_t m0, int64_t n0, int64_t k0, int64_t k,
                                        char* s0, char* s1, char* s2, char* s3,
                                         f32x16 (&acc)[S::TM][S::TN]) {
  static_assert(S::ST == 4, "as many objects");
  using SA = Side<DT, LA, S::BM, S::NW>;
  using SB = Side<DT, LB, S::BN, S::NW>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / S::WN * (32 * S::TM), wn = wave % S::WN * (32 * S::TN);
  SA a;
  SB b;
  a.init(A, m0, k0, wave, lane);
  b.init(B, n0, k0, wave, lane);
  const int64_t slabs = (k + SA::kDepth - 1) / SA::kDepth;
  auto load = [&](char* to, int64_t t) __attribute__((always_inline)) {
    const int64_t left = k - t * SA::kDepth;
    a.load(to, left, wave);
    b.load(to + SA::kBytes, left, wave);
  };
  // A step's operands, read while the step before is multiplied.
  struct Step {
    u32x4 a[S::TM], b[S::TN];
  };
  constexpr bool kTrA = LA == kAcross && SA::kEs == 2, kTrB = LB == kAcross && SB::kEs == 2;
  uint32_t tr_a = 0, tr_b = 0;
  if constexpr (kTrA) tr_a = Across<SA>::lane_at(wm, lane);
  if constexpr (kTrB) tr_b = Across<SB>::lane_at(wn, lane) + SA::kBytes;
  auto read = [&](const char* from, auto step) __attribute__((always_inline)) {
    constexpr int s = decltype(step)::value;
    const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)from));
    Step q;
    if constexpr (!kTrA) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i) q.a[i] = SA::operand(from, wm + 32 * i, s, lane);
    }
    if constexpr (!kTrB) {
#pragma unroll
      for (int j = 0; j < S::TN; ++j) q.b[j] = SB::operand(from + SA::kBytes, wn + 32 * j, s, lane);
    }
    if constexpr (kTrA && S::TM == 4) across42<Across<SA>, Across<SB>, s>(at + tr_a, at + tr_b, q.a, q.b);
    else if constexpr (kTrA) across22<Across<SA>, Across<SB>, s>(at + tr_a, at + tr_b, q.a, q.b);
    else if constexpr (kTrB) across2<Across<SB>, s>(at + tr_b, q.b);
    static_assert(!kTrA || kTrB, "both, or B alone");
    return q;
  };
  using First = std::integral_constant<int, 0>;
  using Second = std::integral_constant<int, 1>;
  // fp32: 256 elements at a time are summed by themselves and then added.  (A sum's own rounding grows with the root of the
  // addends behind one another: gradients of 700 rows of 4000 by 9000 tokens are off by 3e-7, in one chain by over 1e-6;
  // it costs 5%.  16-bit inputs bring more than that with them.)
  constexpr bool kShort = DT == MM_F32;
  f32x16 part_sum[kShort ? S::TM : 1][kShort ? S::TN : 1];
  auto& sum = [&]() -> auto& {
    if constexpr (kShort) return part_sum;
    else return acc;
  }();
  auto flush = [&](bool go_on) __attribute__((always_inline)) {
    if constexpr (kShort) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) {
          if (go_on) acc[i][j] += part_sum[i][j];
#pragma unroll
          for (int r = 0; r < 16; ++r) part_sum[i][j][r] = 0.0f;
        }
    }
  };
  flush(false);
  auto multiply = [&](const Step& q) __attribute__((always_inline)) {
#pragma unroll
    for (int part = 0; part < kParts<DT>; ++part)  // (neighbours in time add to different sums)
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) sum[i][j] = mma<DT>(q.a[i], q.b[j], part, sum[i][j]);
  };
  constexpr int kLoads = SA::kLoads + SB::kLoads;
  static_assert(kSteps == 2, "a slab's first step before the others are met, its second behind it");
  load(s0, 0);
  load(s1, 1);
  load(s2, 2);
  load(s3, 3);
  meet<(S::ST - 1) * kLoads>();
  Step q0 = read(s0, First{}), q1;
  // The slab's second step is multiplied when nobody reads the slab any more and the next one is there: that one's first
  // operands are read, and the loads that take the slab's place issued, under those products.  (Past the last slab zeros
  // are loaded, so that the count of loads under way stays the same.)
  auto slab = [&](char* here, const char* there, int64_t t) __attribute__((always_inline)) {
    if constexpr (kTrB) {
      // (these reads end with a wait: under it the other wave's products, and this one's that are under way)
      multiply(q0);
      __builtin_amdgcn_sched_barrier(0);
      q1 = read(here, Second{});
      meet<(S::ST - 2) * kLoads>();
      load(here, t + S::ST);
      __builtin_amdgcn_sched_barrier(0);
      multiply(q1);
      __builtin_amdgcn_sched_barrier(0);
      q0 = read(there, First{});
      __builtin_amdgcn_sched_barrier(0);
    } else {
      q1 = read(here, Second{});
      __builtin_amdgcn_sched_barrier(0);  // (the reads first: the compiler would put each next to its use)
      multiply(q0);
      __builtin_amdgcn_sched_barrier(0);
      meet<(S::ST - 2) * kLoads>();
      q0 = read(there, First{});
      load(here, t + S::ST);
      __builtin_amdgcn_sched_barrier(0);
      multiply(q1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int64_t t = 0;
  for (; t + S::ST <= slabs; t += S::ST) {
    slab(s0, s1, t);
    slab(s1, s2, t + 1);
    slab(s2, s3, t + 2);
    slab(s3, s0, t + 3);
    if (kShort && t % (256 / SA::kDepth) == 256 / SA::kDepth - S::ST) flush(true);
  }
  if (t < slabs) slab(s0, s1, t);
  if (t + 1 < slabs) slab(s1, s2, t + 1);
  if (t + 2 < slabs) slab(s2, s3, t + 2);
  flush(true);
  meet<0>();
}

template <typename S>
__device__ __forceinline__ void clear(f32x16 (&acc)[S::TM][S::TN]) {
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
}

// Workgroup `id` of `total` to a tile of mt x nt: each die (workgroup ids go round the 8) takes a contiguous share, in
// bands of 8 rows of tiles, so that what runs there at once shares its operands in the die's cache.
__device__ __forceinline__ void tile_of(uint32_t id, uint32_t mt, uint32_t nt, uint32_t& m, uint32_t& n) {
  const uint32_t total = mt * nt, share = total / 8, over = total % 8, die = id % 8;
  const uint32_t at = die * share + (die < over ? die : over) + id / 8;
  const uint32_t band = at / (8 * nt), in = at % (8 * nt);
  const uint32_t rows = mt - band * 8 < 8 ? mt - band * 8 : 8;
  m = band * 8 + in % rows;
  n = in / rows;
}

}  // namespace slab
}  // namespace mm
