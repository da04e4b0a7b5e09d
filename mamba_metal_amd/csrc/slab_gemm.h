// Products of large tiles on the matrix cores: C[m, n] = sum_k A(m, k) B(n, k), both operands streamed through shared
// memory by loads that go there directly, two stages deep.
//
// A stage is a slab of 128 bytes of k (64 16-bit elements, 32 fp32 ones) of the tile's rows.  An operand lies in memory
// either way:
//   kAlong   k is contiguous: a row of the slab is 128 bytes of a row of the matrix, eight 16-byte chunks.  Chunk c of
//            row r is kept at place c ^ (r / 2 % 8), so that 16 rows' reads of one chunk fall into different banks.
//   kAcross  rows (m or n) are contiguous: the slab is 64 (32) rows of k by the tile's width, read with the transposing
//            read (fp32: element by element).  Its chunks are kept at c ^ f(k), for the same reason.
// The direct load writes 16 bytes a lane at consecutive places, so the permutation is of the addresses that the lanes
// read.  Elements past the matrix's k (and columns past its width, kAcross) come from a block of zeros; rows past its end
// are its last row again, whose results are not stored.
//
// The 32 x 32 tiles' operand layout: lane l holds row l % 32 and 16 bytes of k, chunk 2 s + l / 32 of the slab at step s
// of 4; an accumulator holds column l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4.
#pragma once

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

constexpr int kSlab = 128;  // bytes of k
enum Lie { kAlong, kAcross };

template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (DT == MM_F16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == MM_BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
    return c;
  }
}

struct Matrix {
  const char* base;
  int64_t ld;       // bytes from one row in memory to the next
  int64_t rows;     // kAlong: rows of the operand; kAcross: its columns, in elements
  int64_t k;        // elements of the sum
  const char* zeros;  // 16 bytes of them
};

__device__ __forceinline__ void load_direct(const char* from, char* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// One operand of a workgroup's tile: R rows, staged by NW waves.
template <int DT, Lie LIE, int R, int NW>
struct Side {
  using T = typename Ty<DT>::T;
  static constexpr int kEs = sizeof(T);
  static constexpr int kDepth = kSlab / kEs;               // elements of k in a slab
  static constexpr int kBytes = R * kSlab;
  static constexpr int kLoads = kBytes / 1024 / NW;        // of a wave, 64 lanes of 16 bytes each
  static constexpr int kRowChunks = R * kEs / 16;          // kAcross: chunks of a row of k
  static_assert(kLoads >= 1 && kLoads * 1024 * NW == kBytes, "whole loads");
  const char* at[kLoads];
  int32_t k_at[kLoads];  // the lane's first element of k within the slab
  int64_t step;
  const char* zeros;

  static __device__ __forceinline__ int place(int k) {  // kAcross: what a row of k has its chunks permuted by
    return kEs != 2 ? 0 : kRowChunks >= 16 ? (k & 3) << 2 : kRowChunks == 8 ? (k >> 1 & 1) << 2 : 0;
  }
  __device__ __forceinline__ void init(const Matrix& m, int64_t row0, int64_t k0, int wave, int lane) {
    zeros = m.zeros;
    step = LIE == kAlong ? kSlab : kDepth * m.ld;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int s = (q * NW + wave) * 64 + lane;
      if constexpr (LIE == kAlong) {
        const int r = s / 8, c = s % 8 ^ (r >> 1 & 7);
        const int64_t row = row0 + r < m.rows ? row0 + r : m.rows - 1;
        k_at[q] = c * 16 / kEs;
        at[q] = m.base + row * m.ld + k0 * kEs + c * 16;
      } else {
        const int k = s / kRowChunks, c = s % kRowChunks ^ place(k);
        const int64_t col = row0 + c * (16 / kEs);
        k_at[q] = col < m.rows ? k : 1 << 30;  // (never within k)
        at[q] = m.base + (k0 + k) * m.ld + col * kEs;
      }
    }
  }
  // Issues the loads of one slab, of whose k `left` elements are in the matrix, and moves on.
  __device__ __forceinline__ void load(char* tile, int64_t left, int wave) {
    const bool all = LIE == kAlong && left >= kDepth;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const char* const from = all || k_at[q] < left ? at[q] : zeros;
      load_direct(from, tile + (q * NW + wave) * 1024);
      at[q] += step;
    }
  }
  // Rows r0 .. r0 + 31 at step s (of 4), of a staged slab.
  static __device__ __forceinline__ u32x4 operand(const char* tile, int r0, int s, int lane) {
    if constexpr (LIE == kAlong) {
      const int r = r0 + (lane & 31), c = 2 * s + (lane >> 5);
      return *reinterpret_cast<const u32x4*>(tile + r * kSlab + ((c ^ (r >> 1 & 7)) << 4));
    } else if constexpr (kEs == 2) {
      // 16 lanes read 4 rows of k by 16 columns, 8 bytes each, and get a column each
      const int col = r0 + (lane & 16) + 4 * (lane & 3), k = 16 * s + 8 * (lane >> 5) + ((lane & 15) >> 2);
      const char* const p = tile + k * R * kEs + (((col >> 3) ^ place(k)) << 4) + (col & 7) * 2;
      typedef __attribute__((address_space(3))) s16x4 Lds;
      const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p)));
      const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds*)(p + 4 * R * kEs)));
      return u32x4{a[0], a[1], b[0], b[1]};
    } else {
      u32x4 v;
      const char* const p = tile + (8 * s + 4 * (lane >> 5)) * R * kEs + (r0 + (lane & 31)) * kEs;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint32_t*>(p + j * R * kEs);
      return v;
    }
  }
};

// A tile's shape: BM x BN by WM x WN waves, each TM x TN tiles of 32 x 32.
template <int BM_, int BN_, int WM_, int WN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
};

// acc += the sum over `k` elements from k0 on.  All threads of the workgroup; s0 and s1 are (BM + BN) * 128 bytes each
// and must be two objects, so that the compiler sees that a stage's reads and the next one's loads do not meet.
template <int DT, Lie LA, Lie LB, typename S>
__device__ __forceinline__ void product(const Matrix& A, const Matrix& B, int64_t m0, int64_t n0, int64_t k0, int64_t k, char* s0,
                                        char* s1, f32x16 (&acc)[S::TM][S::TN]) {
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
  auto multiply = [&](const char* from) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4 ao[S::TM], bo[S::TN];
#pragma unroll
      for (int i = 0; i < S::TM; ++i) ao[i] = SA::operand(from, wm + 32 * i, s, lane);
#pragma unroll
      for (int j = 0; j < S::TN; ++j) bo[j] = SB::operand(from + SA::kBytes, wn + 32 * j, s, lane);
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc[i][j] = mma<DT>(ao[i], bo[j], acc[i][j]);
    }
  };
  if (slabs > 0) load(s0, 0);
  int64_t t = 0;
  for (; t + 1 < slabs; t += 2) {
    __syncthreads();  // s0 is loaded, and nobody reads s1
    load(s1, t + 1);
    multiply(s0);
    __syncthreads();
    if (t + 2 < slabs) load(s0, t + 2);
    multiply(s1);
  }
  if (t < slabs) {
    __syncthreads();
    multiply(s0);
  }
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
__device__ __forceinline__ int acc_row(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

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
