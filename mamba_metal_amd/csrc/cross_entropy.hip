// Softmax cross entropy of the rows before a language model's head, without keeping the logits.
//
//   l = W x      loss = log sum_v exp(l_v) - l_t      dl = (softmax(l) - onehot(t)) dloss      dx = W^T dl   dW = dl x^T
//
// Forward: the product W x by tiles, whose epilogue leaves of a tile the maximum and the sum of exponentials of every row
// (and the target's logit): 8 bytes for 256 logits.  Backward: piece by piece of the vocabulary the logits are computed
// again, and the epilogue turns them into dl in the inputs' type (its one rounding); the piece is then multiplied with W
// (adding to dx, in fp32) and with x (its rows of dW).  The four products are the time; everything else is 3%.
// A product's tile has the vocabulary along the accumulators' rows, so that the softmax's sums run within a lane.
// bf16, 8192 rows (7377 counted) of 2560 by 50280 tokens, in a kernel trace: 1.73 ms forward; backward in two pieces, each 0.92 ms
// for dl and 1.93 to 1.96 ms for dx and dW (0.98 PFLOP/s), and 0.11 for all else: 7.6 ms.  Untraced the pass takes 7.1 to 7.3,
// where three library products of whole matrices would take 5.3 and logits of 0.8 GB.  fp32, 999 (894) of 1001 by 10007, in a
// trace: 195 us, 209 and 381, and 20 a pass to lay the odd rows out; 716 us untraced.
//
// Rows that are ignored take no part: the others are gathered first (their sums over rows are then never touched by what
// an ignored row holds, and a batch that is mostly ignored costs its share), and workgroups past their count end at once.
#include "cross_entropy.h"
#include "row_io.h"

namespace mm {
namespace xent {

using slab::Matrix;
using slab::f32x16;
using slab::kAcross;
using slab::kAlong;
using slab::u32x2;
using slab::u32x4;

using Big = slab::Tile<256, 256, 2, 4, 4>;
using Mid = slab::Tile<128, 128, 2, 2, 4>;
using Thin = slab::Tile<128, 64, 4, 1, 4>;  // few rows of x

constexpr int kThreads = 1024;

__device__ __forceinline__ int64_t target_of(const Loss& p, int64_t i) {
  return p.targets64 ? static_cast<const int64_t*>(p.targets)[i] : static_cast<const int32_t*>(p.targets)[i];
}

// A sum (or maximum) over a workgroup of 1024.
template <typename V, typename F>
__device__ __forceinline__ V all_of(V v, V* s, F join) {
#pragma unroll
  for (int x = 1; x < 64; x *= 2) v = join(v, __shfl_xor(v, x, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < kThreads / 64; ++w) v = join(v, s[w]);
  return v;
}

// The rows that count, in order, and for the backward pass what their gradients are multiplied by.  One workgroup: 8192 rows
// a turn, their loads all under way at once (8192 rows: 7.4 us).
__global__ __launch_bounds__(kThreads) void rows_kernel(const Loss p, bool backward) {
  constexpr int kTurn = 8;
  __shared__ int32_t s_wave[kTurn * kThreads / 64];
  __shared__ float s_f[kThreads / 64];
  static_assert(kTurn * kThreads / 64 == 128, "two counts a lane");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int32_t base = 0;
  float top = 0.0f;
  // One number for all rows is left out of the pieces and multiplies the sums: what a target's dl is nearly is then a power
  // of two, which its rounding keeps.  fp16: the pieces hold dl times a power of two that puts the largest at 2^12, so that
  // small probabilities are not subnormal; the sums take it back.
  const float uniform = p.dtype == MM_F16 ? 4096.0f : 1.0f;
  for (int64_t r0 = 0; r0 < p.rows; r0 += kTurn * kThreads) {
    int64_t t[kTurn];
    float d[kTurn], lse[kTurn];
    uint64_t on[kTurn];
#pragma unroll
    for (int j = 0; j < kTurn; ++j) {
      const int64_t r = r0 + j * kThreads + threadIdx.x, in = r < p.rows ? r : p.rows - 1;
      t[j] = target_of(p, in);
      d[j] = backward && !p.reduction ? p.dloss[in * p.dloss_stride] : 0.0f;
      lse[j] = backward ? p.lse[in] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kTurn; ++j) {
      on[j] = __ballot(r0 + j * kThreads + threadIdx.x < p.rows && t[j] != p.ignore);
      if (lane == 0) s_wave[j * (kThreads / 64) + wave] = __popcll(on[j]);
    }
    __syncthreads();
    int32_t lo = s_wave[lane], hi = s_wave[64 + lane];
    const int32_t own_lo = lo, own_hi = hi;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const int32_t a = __shfl_up(lo, x, 64), c = __shfl_up(hi, x, 64);
      lo += lane >= x ? a : 0;
      hi += lane >= x ? c : 0;
    }
    const int32_t half = __shfl(lo, 63, 64), all = half + __shfl(hi, 63, 64);
    lo -= own_lo;
    hi += half - own_hi;
#pragma unroll
    for (int j = 0; j < kTurn; ++j) {
      const int64_t r = r0 + j * kThreads + threadIdx.x;
      const int32_t at = base + __shfl(j < kTurn / 2 ? lo : hi, j % (kTurn / 2) * (kThreads / 64) + wave, 64) +
                         __popcll(on[j] & ((1ull << lane) - 1));
      const bool mine = on[j] >> lane & 1;
      if (r < p.rows) p.at[r] = mine ? at : -1;
      if (mine) {
        p.row[at] = static_cast<int32_t>(r);
        p.target_at[at] = t[j];
        if (backward) {
          p.weights[at] = p.reduction ? uniform : d[j];
          p.lse_at[at] = t[j] < 0 || t[j] >= p.vocab ? __builtin_nanf("") : lse[j];
          top = fmaxf(top, fabsf(d[j]));
        }
      }
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.count[0] = base;
  if (!backward) return;
  if (p.reduction) {
    if (threadIdx.x == 0)
      p.scalars[0] = base == 0 ? 0.0f : *p.dloss * (p.reduction == 1 ? 1.0f / static_cast<float>(base) : 1.0f) / uniform;
    return;
  }
  top = all_of(top, s_f, [](float a, float b) { return fmaxf(a, b); });
  float up = 1.0f;
  if (p.dtype == MM_F16) {
    const int e = static_cast<int>(__float_as_uint(top) >> 23) - 127;
    if (top > 0.0f && e > -100 && e < 100) up = __builtin_ldexpf(1.0f, 12 - e);
    for (int64_t i = threadIdx.x; i < base; i += kThreads) p.weights[i] *= up;  // (a thread's own or behind all_of's barrier)
  }
  if (threadIdx.x == 0) p.scalars[0] = 1.0f / up;
}

// Rows of a matrix to 16-byte aligned ones with zeros behind their end; gather: those that count.  A copy: 8192 rows of 2560
// in bf16 take 16 us, 5.2 TB/s.
template <int DT>
__global__ __launch_bounds__(256) void lay_out_kernel(const void* from, int64_t from_ld, char* to, int64_t to_ld, int64_t rows,
                                                     int64_t dim, const int32_t* row, const int32_t* count, bool vec) {
  using T = typename Ty<DT>::T;
  constexpr int kE = 16 / sizeof(T);
  const int64_t units = to_ld / 16, n = (count ? *count : rows) * units;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < n; e += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t r = e / units, c = e % units * kE;
    const T* const p = static_cast<const T*>(from) + (row ? row[r] : r) * from_ld + c;
    u32x4 v;
    if (vec) {
      v = *reinterpret_cast<const u32x4*>(p);
    } else {
      T t[kE];
#pragma unroll
      for (int j = 0; j < kE; ++j) t[j] = c + j < dim ? p[j] : static_cast<T>(0);
      __builtin_memcpy(&v, t, 16);
    }
    *reinterpret_cast<u32x4*>(to + r * to_ld + c * sizeof(T)) = v;
  }
}

__device__ __forceinline__ Matrix vocabulary(const Loss& p, int64_t v0) {
  const int64_t es = p.dtype == MM_F32 ? 4 : 2;
  Matrix m;
  m.base = (p.wc ? p.wc : static_cast<const char*>(p.weight));
  m.ld = p.wc ? p.ld : p.w_ld * es;
  m.base += v0 * m.ld;
  m.rows = p.vocab - v0;
  m.k = p.ld / es;
  return m;
}
__device__ __forceinline__ Matrix counted(const Loss& p, int32_t count) {
  Matrix m;
  m.base = p.xc;
  m.ld = p.ld;
  m.rows = count;
  m.k = p.ld / (p.dtype == MM_F32 ? 4 : 2);
  return m;
}

// Logits of a tile of the vocabulary (rows) and of x (columns).  The product is the time (its epilogue, an fma and the
// hardware's exp2 for a logit in 16 bits, another 6%).  Forward: each column's maximum and sum of exponentials.
// Backward: dl of the piece.
template <int DT, typename S, bool GRAD>
__global__ __launch_bounds__(64 * S::NW) void logits_kernel(const Loss p) {
  using T = typename Ty<DT>::T;
  MM_SLAB_STAGES(S, stages)
  const int32_t count = *p.count;
  const int64_t vocab = GRAD ? p.piece_n : p.vocab;
  const uint32_t vt = static_cast<uint32_t>((GRAD ? p.piece_ld / static_cast<int64_t>(sizeof(T)) : vocab) + S::BM - 1) / S::BM;
  const uint32_t rt = static_cast<uint32_t>((p.rows + S::BN - 1) / S::BN);
  uint32_t m, n;
  slab::tile_of(blockIdx.x, vt, rt, m, n);
  const int64_t v0 = static_cast<int64_t>(m) * S::BM, r0 = static_cast<int64_t>(n) * S::BN;
  if (r0 >= count) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / S::WN, wn = wave % S::WN;
  // what the end needs of this lane's columns
  int64_t target[S::TN];  // relative to the matrix's first row
  float lse[S::TN], weight[S::TN];
#pragma unroll
  for (int j = 0; j < S::TN; ++j) {
    const int64_t r = r0 + wn * 32 * S::TN + 32 * j + (lane & 31), in = r < count ? r : 0;
    const int64_t t = p.target_at[in];
    target[j] = r < count ? t - (GRAD ? p.piece0 : 0) : -1;
    lse[j] = GRAD ? p.lse_at[in] : 0.0f;
    weight[j] = GRAD ? p.weights[in] : 0.0f;
  }
  f32x16 acc[S::TM][S::TN];
  slab::clear<S>(acc);
  const Matrix w = vocabulary(p, GRAD ? p.piece0 : 0), x = counted(p, count);
  slab::product<DT, kAlong, kAlong, S>(w, x, v0, r0, 0, w.k, stages0, stages1, stages2, stages3, acc);

  const int64_t vw = v0 + wm * 32 * S::TM + 4 * (lane >> 5);  // of the lane's first accumulator
  const int here = vocab - vw < 1 << 20 ? static_cast<int>(vocab - vw) : 1 << 20;  // tokens from there on
  const bool edge = v0 + S::BM > vocab;  // (most tiles have none)
  if constexpr (!GRAD) {
    float* const s_stat = reinterpret_cast<float*>(stages0);  // (WM, BN, 2)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      const int col = wn * 32 * S::TN + 32 * j + (lane & 31);
      const int64_t r = r0 + col;
      const int64_t t = target[j] - vw;
      if (edge) {
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * i + 8 * (e >> 2) + (e & 3) >= here) acc[i][j][e] = -INFINITY;
      }
      if (__any(t >= 0 && t < 32 * S::TM && t < here)) {
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * i + 8 * (e >> 2) + (e & 3) == t && r < count) p.hit[r] = acc[i][j][e];
      }
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) top = fmaxf(top, acc[i][j][e]);
      top = fmaxf(top, lane_xor(top, 32));
      float sum = 0.0f;
      const float from = top == -INFINITY ? 0.0f : top;  // (all logits -inf: a sum of 0, not a NaN)
      if constexpr (DT == MM_F32) {
        bool bad = top == INFINITY;
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float l = acc[i][j][e];
            bad |= l != l;  // (lost by fmaxf and exp2_acc's clamp)
            sum += exp2_acc((l - from) * kLog2e);
          }
        if (bad) sum = __builtin_nanf("");
      } else {
        // (a NaN, and an infinity less itself, goes through the hardware's exp2)
        const float base = from * kLog2e;
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e) sum += exp2_hw(__builtin_fmaf(acc[i][j][e], kLog2e, -base));
      }
      sum += lane_xor(sum, 32);
      if (lane < 32) {
        s_stat[(wm * S::BN + col) * 2] = top;
        s_stat[(wm * S::BN + col) * 2 + 1] = sum;
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < S::BN; c += 64 * S::NW) {
      if (r0 + c >= count) continue;
      float top = s_stat[c * 2], sum = s_stat[c * 2 + 1];
#pragma unroll
      for (int k = 1; k < S::WM; ++k) {
        const float t2 = s_stat[(k * S::BN + c) * 2], s2 = s_stat[(k * S::BN + c) * 2 + 1];
        const float m2 = fmaxf(top, t2), from = m2 == -INFINITY ? 0.0f : m2;
        sum = sum * exp2_acc((top - from) * kLog2e) + s2 * exp2_acc((t2 - from) * kLog2e);
        top = m2;
      }
      float* const out = p.stats + ((r0 + c) * p.tiles + m) * 2;
      out[0] = top;
      out[1] = sum;
    }
  } else {
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      const int64_t t = target[j] - vw;
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if constexpr (DT == MM_F32) {
            const float z = (acc[i][j][e] - lse[j]) * kLog2e, g = exp2_acc(z);
            acc[i][j][e] = (z != z ? z : g) * weight[j];
          } else {
            acc[i][j][e] = exp2_hw(__builtin_fmaf(acc[i][j][e], kLog2e, -lse[j] * kLog2e)) * weight[j];
          }
        }
      if (__any(t >= 0 && t < 32 * S::TM)) {
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * i + 8 * (e >> 2) + (e & 3) == t) acc[i][j][e] -= weight[j];
      }
      if (edge) {
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (32 * i + 8 * (e >> 2) + (e & 3) >= here) acc[i][j][e] = 0.0f;
      }
    }
    // Out by rows: through the stages, half a tile's rows at a time where it is large, a row's 16-byte chunks turned by its
    // number.  (A row of the piece is a whole number of tiles of 256; fp32 is stored from the accumulators.)
    const int wide = static_cast<int>(p.piece_ld / static_cast<int64_t>(sizeof(T)) - v0);  // of this tile's columns
    if constexpr (DT == MM_F32) {
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        const int64_t r = r0 + wn * 32 * S::TN + 32 * j + (lane & 31);
        if (r >= count) continue;
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int v = wm * 32 * S::TM + 4 * (lane >> 5) + 32 * i + 8 * q;
            if (v >= wide) continue;
            float* const to = reinterpret_cast<float*>(p.piece + r * p.piece_ld) + v0 + v;
            *reinterpret_cast<slab::f32x4*>(to) = slab::f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          }
      }
    } else {
      constexpr int kChunks = S::BM * 2 / 16, kPart = S::BN / 4;  // of a row; rows that a stage holds
      static_assert(kPart * S::BM * 2 <= S::kStage && kPart % 16 == 0, "a quarter of the tile's rows in a stage");
      auto stage_of = [&](int row) { return row / kPart == 0 ? stages0 : row / kPart == 1 ? stages1 : row / kPart == 2 ? stages2 : stages3; };
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        const int row = wn * 32 * S::TN + 32 * j + (lane & 31);
        char* const to = stage_of(row) + row % kPart * (S::BM * 2) + 8 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < S::TM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            T d[4];
            round2<DT>(acc[i][j][4 * q], acc[i][j][4 * q + 1], d[0], d[1]);
            round2<DT>(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3], d[2], d[3]);
            u32x2 w2;
            __builtin_memcpy(&w2, d, 8);
            const int chunk = wm * 4 * S::TM + 4 * i + q;
            *reinterpret_cast<u32x2*>(to + ((chunk ^ (row % kChunks)) << 4)) = w2;
          }
      }
      __syncthreads();
#pragma unroll 4
      for (int u = threadIdx.x; u < S::BN * kChunks; u += 64 * S::NW) {
        const int row = u / kChunks, chunk = u % kChunks;
        if (r0 + row >= count || chunk * 8 >= wide) continue;
        *reinterpret_cast<u32x4*>(p.piece + (r0 + row) * p.piece_ld + (v0 + chunk * 8) * 2) =
            *reinterpret_cast<const u32x4*>(stage_of(row) + row % kPart * (S::BM * 2) + ((chunk ^ (row % kChunks)) << 4));
      }
    }
  }
}

// fp32, where tiles of logits are so few that most of the card would wait for their long sums: a split of them, kept as it is.
template <int DT>
__global__ __launch_bounds__(64 * Thin::NW) void split_logits_kernel(const Loss p, bool grad) {
  MM_SLAB_STAGES(Thin, stages)
  const int32_t count = *p.count;
  const uint32_t vt = static_cast<uint32_t>(p.logit_ld / Thin::BM), rt = static_cast<uint32_t>((p.rows + Thin::BN - 1) / Thin::BN);
  uint32_t m, n;
  slab::tile_of(blockIdx.x % (vt * rt), vt, rt, m, n);
  const int64_t split = blockIdx.x / (vt * rt), v0 = static_cast<int64_t>(m) * Thin::BM, r0 = static_cast<int64_t>(n) * Thin::BN;
  if (r0 >= count) return;
  f32x16 acc[Thin::TM][Thin::TN];
  slab::clear<Thin>(acc);
  const Matrix w = vocabulary(p, grad ? p.piece0 : 0), x = counted(p, count);
  const int64_t k0 = split * p.logit_k, k = w.k - k0 < p.logit_k ? w.k - k0 : p.logit_k;
  slab::product<DT, kAlong, kAlong, Thin>(w, x, v0, r0, k0, k, stages0, stages1, stages2, stages3, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / Thin::WN, wn = wave % Thin::WN;
#pragma unroll
  for (int j = 0; j < Thin::TN; ++j) {
    const int64_t r = r0 + wn * 32 * Thin::TN + 32 * j + (lane & 31);
    if (r >= count) continue;
    float* const to = p.logit_part + (split * p.rows + r) * p.logit_ld + v0 + wm * 32 * Thin::TM + 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < Thin::TM; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<slab::f32x4*>(to + 32 * i + 8 * q) = slab::f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
  }
}
// Their sums, in order, and what logits_kernel makes of them: a wave takes 128 tokens of a row.
template <bool GRAD>
__global__ __launch_bounds__(256) void join_logits_kernel(const Loss p) {
  const int lane = threadIdx.x & 63;
  const int64_t tiles = p.logit_ld / 128, unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t r = unit / tiles, m = unit % tiles, v = m * 128 + 2 * lane;
  if (r >= *p.count) return;
  float l[2] = {0.0f, 0.0f};
#pragma unroll 4
  for (int64_t s = 0; s < p.logit_splits; ++s) {
    const float* const from = p.logit_part + (s * p.rows + r) * p.logit_ld + v;
    l[0] += from[0];
    l[1] += from[1];
  }
  const int64_t vocab = GRAD ? p.piece_n : p.vocab, target = p.target_at[r] - (GRAD ? p.piece0 : 0);
  if constexpr (!GRAD) {
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (v + e >= vocab) l[e] = -INFINITY;
      else if (v + e == target) p.hit[r] = l[e];
      top = fmaxf(top, l[e]);
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, lane_xor(top, x));
    const float from = top == -INFINITY ? 0.0f : top;
    bool bad = top == INFINITY;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      bad |= l[e] != l[e];
      sum += exp2_acc((l[e] - from) * kLog2e);
    }
    if (bad) sum = __builtin_nanf("");
#pragma unroll
    for (int x = 1; x < 64; x *= 2) sum += lane_xor(sum, x);
    if (lane == 0 && m < p.tiles) {
      p.stats[(r * p.tiles + m) * 2] = top;
      p.stats[(r * p.tiles + m) * 2 + 1] = sum;
    }
  } else {
    const float lse = p.lse_at[r], weight = p.weights[r];
    float* const to = reinterpret_cast<float*>(p.piece + r * p.piece_ld) + v;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float z = (l[e] - lse) * kLog2e, g = exp2_acc(z);
      const float d = (z != z ? z : g) * weight - (v + e == target ? weight : 0.0f);
      to[e] = v + e < vocab ? d : 0.0f;
    }
  }
}

// A row's loss from its tiles' maxima and sums: a wave a row.  (8192 rows, 197 tiles: 9 us.)
__global__ __launch_bounds__(256) void merge_kernel(const Loss p) {
  const int lane = threadIdx.x & 63;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= p.rows) return;
  const int32_t at = p.at[r];
  float loss = 0.0f, lse = 0.0f;
  if (at >= 0) {
    const float* const s = p.stats + at * p.tiles * 2;
    float top = -INFINITY;
    for (int64_t t = lane; t < p.tiles; t += 64) top = fmaxf(top, s[2 * t]);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, lane_xor(top, x));
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (int64_t t = lane; t < p.tiles; t += 64) sum += s[2 * t + 1] * exp2_acc((s[2 * t] - from) * kLog2e);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) sum += lane_xor(sum, x);
    const int64_t t = p.target_at[at];
    lse = top + logf(sum);
    loss = t < 0 || t >= p.vocab ? __builtin_nanf("") : (top - p.hit[at]) + logf(sum);
  }
  if (lane == 0) {
    if (p.lse) p.lse[r] = lse;
    (p.row_loss ? p.row_loss : p.loss)[r] = loss;
  }
}

// The rows' sum or mean, in 64 bits and a fixed order.  One workgroup.
__global__ __launch_bounds__(kThreads) void total_kernel(const Loss p) {
  __shared__ double s_d[kThreads / 64];
  double sum = 0.0;
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < p.rows; r += kThreads) sum += p.row_loss[r];
  sum = all_of(sum, s_d, [](double a, double b) { return a + b; });
  if (threadIdx.x == 0) p.loss[0] = static_cast<float>(p.reduction == 1 ? sum / static_cast<double>(*p.count) : sum);
}

// A tile of dx's part of this piece: rows that count by channels, a split of the piece's tokens; added in fp32.
template <int DT, typename S>
__device__ __forceinline__ void dx_tile(const Loss& p, uint32_t id, int32_t count, char* s0, char* s1, char* s2, char* s3) {
  using T = typename Ty<DT>::T;
  const uint32_t mt = static_cast<uint32_t>((p.rows + S::BM - 1) / S::BM), nt = static_cast<uint32_t>((p.dim + S::BN - 1) / S::BN);
  uint32_t m, n;
  slab::tile_of(id % (mt * nt), mt, nt, m, n);
  const int64_t split = id / (mt * nt);
  const int64_t r0 = static_cast<int64_t>(m) * S::BM, c0 = static_cast<int64_t>(n) * S::BN;
  if (r0 >= count) return;
  const int64_t k0 = split * p.split_k, k1 = k0 + p.split_k < p.piece_n ? k0 + p.split_k : p.piece_n;
  f32x16 acc[S::TM][S::TN];
  slab::clear<S>(acc);
  Matrix dl, w = vocabulary(p, p.piece0);
  dl.base = p.piece;
  dl.ld = p.piece_ld;
  dl.rows = count;
  w.rows = p.ld / static_cast<int64_t>(sizeof(T));
  if (k1 > k0) slab::product<DT, kAlong, kAcross, S>(dl, w, r0, c0, k0, k1 - k0, s0, s1, s2, s3, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float* const out = p.dx_part + split * p.rows * p.dim;
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      const int64_t c = c0 + wave % S::WN * 32 * S::TN + 32 * j + (lane & 31);
      const int64_t rt = r0 + wave / S::WN * 32 * S::TM + 32 * i + 4 * (lane >> 5);
      const int here = c < p.dim ? static_cast<int>(count - rt) : 0;
      float* at = out + rt * p.dim + c;
#pragma unroll
      for (int q = 0; q < 4; ++q, at += 8 * p.dim)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (8 * q + e < here) {
            const float v = acc[i][j][4 * q + e];
            at[e * p.dim] = p.first_piece ? v : at[e * p.dim] + v;
          }
    }
}

// A tile of the piece's rows of dW.
template <int DT, typename S>
__device__ __forceinline__ void dw_tile(const Loss& p, uint32_t id, int32_t count, char* s0, char* s1, char* s2, char* s3) {
  using T = typename Ty<DT>::T;
  const uint32_t mt = static_cast<uint32_t>((p.piece_n + S::BM - 1) / S::BM), nt = static_cast<uint32_t>((p.dim + S::BN - 1) / S::BN);
  uint32_t m, n;
  slab::tile_of(id, mt, nt, m, n);
  const int64_t v0 = static_cast<int64_t>(m) * S::BM, c0 = static_cast<int64_t>(n) * S::BN;
  f32x16 acc[S::TM][S::TN];
  slab::clear<S>(acc);
  Matrix dl, x;
  dl.base = p.piece;
  dl.ld = p.piece_ld;
  dl.rows = p.piece_ld / static_cast<int64_t>(sizeof(T));
  x.base = p.xc;
  x.ld = p.ld;
  x.rows = p.ld / static_cast<int64_t>(sizeof(T));
  slab::product<DT, kAcross, kAcross, S>(dl, x, v0, c0, 0, count, s0, s1, s2, s3, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float down = p.scalars[0];
#pragma unroll
  for (int i = 0; i < S::TM; ++i)
#pragma unroll
    for (int j = 0; j < S::TN; ++j) {
      const int64_t c = c0 + wave % S::WN * 32 * S::TN + 32 * j + (lane & 31);
      const int64_t vt = v0 + wave / S::WN * 32 * S::TM + 32 * i + 4 * (lane >> 5);
      const int here = c < p.dim && vt < p.piece_n ? static_cast<int>(p.piece_n - vt) : 0;
      T* at = static_cast<T*>(p.dweight) + (p.piece0 + vt) * p.dim + c;
#pragma unroll
      for (int q = 0; q < 4; ++q, at += 8 * p.dim)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (8 * q + e < here) at[e * p.dim] = Ty<DT>::from(acc[i][j][4 * q + e] * down);
    }
}

// Both gradients of a piece in one launch, dx's longer sums first: the card is full until the last of dW's tiles.  (320
// tiles of dx alone on 256 compute units leave it three quarters empty for half their time: 1.47 ms, and 0.92 for dW; 1.93
// together.)
template <int DT, typename S>
__global__ __launch_bounds__(64 * S::NW) void grads_kernel(const Loss p) {
  MM_SLAB_STAGES(S, stages)
  const int32_t count = *p.count;
  if (blockIdx.x < p.dx_tiles) dx_tile<DT, S>(p, blockIdx.x, count, stages0, stages1, stages2, stages3);
  else dw_tile<DT, S>(p, blockIdx.x - p.dx_tiles, count, stages0, stages1, stages2, stages3);
}

// dx: the splits' sums in order, rounded; zeros in the rows that are ignored.
template <int DT>
__global__ __launch_bounds__(256) void finish_dx_kernel(const Loss p) {
  const int64_t r = blockIdx.x;
  const int32_t at = p.at[r];
  const float down = p.scalars[0];
  for (int64_t c = threadIdx.x; c < p.dim; c += 256) {
    float sum = 0.0f;
    if (at >= 0) {
#pragma unroll 4
      for (int64_t s = 0; s < p.splits; ++s) sum += p.dx_part[(s * p.rows + at) * p.dim + c];
    }
    st<DT>(p.dx, r * p.dim + c, sum * down);
  }
}

// ------------------------------------------------------------------------------------------------------------- host
constexpr int64_t kMaxRows = int64_t{1} << 30, kMaxVocab = int64_t{1} << 30, kMaxDim = int64_t{1} << 20;
constexpr int64_t kPieceBytes = int64_t{512} << 20;  // of dl kept at a time

enum Size { kBig, kMid, kThin };
static int64_t high(Size s) { return s == kBig ? 256 : 128; }
static int64_t wide(Size s) { return s == kBig ? 256 : s == kMid ? 128 : 64; }
static int64_t tiles_of(Size s, int64_t m, int64_t n) { return ceil_div(m, high(s)) * ceil_div(n, wide(s)); }
// 256 x 256 where there are enough of them to fill the card's rounds, else 128 x 128.  (bf16, 1024 rows of 1024 by 8192
// tokens, 128 large tiles: 33 us, 27 in small ones; 2048 rows, 256 of them: 39 us, 47 in small ones.)  fp32: 128 x 128, whose
// sums leave room for a second set of them, or 128 x 64.  (2048 rows of 1024 by 16384 tokens, 512 large tiles: 559 us, 595
// in small ones; 999 of 1001 by 10007, 160 of them: 208 us, 192 in small ones.)
static Size size_of(int dtype, int64_t big_tiles) {
  if (dtype == MM_F32) return big_tiles >= 512 ? kMid : kThin;
  return big_tiles >= 192 ? kBig : kMid;
}
// 128 x 64 also for few rows, where the vocabulary's rows are the traffic.
static Size logits_size(int dtype, int64_t vocab, int64_t rows) { return rows <= 64 ? kThin : size_of(dtype, tiles_of(kBig, vocab, rows)); }

// The gradients of a piece of n tokens: tiles, and the splits of dx's few, long sums.
struct Grads {
  Size size;
  int64_t splits, split_k;
};
static Grads grads_of(int dtype, int64_t rows, int64_t dim, int64_t n, bool dx, bool dw) {
  // in products of a tile's row and column
  auto work = [&](Size s) { return (dx ? tiles_of(s, rows, dim) * n : 0) + (dw ? tiles_of(s, n, dim) * rows : 0); };
  const int64_t sum = dw && rows > 512 ? rows : 512;
  Grads g{size_of(dtype, work(kBig) / sum), 1, n};
  if (!dx) return g;
  const int64_t most = n / 512 < 1 ? 1 : n / 512 < 16 ? n / 512 : 16, tiles = tiles_of(g.size, rows, dim);
  if (dw) {
    // none longer than the share of one place on the card (bf16, 2048 rows of 1024 by 8192 tokens: 195 us whole, 110 in
    // two, 85 in three and in four; 8192 of 2560 by 25344: 2.06 ms whole and in four; fp32 as above: 384 us in four)
    const int64_t places = 256 * (g.size == kBig ? 1 : g.size == kMid ? 2 : 3);
    g.splits = ceil_div(n * places, work(g.size));
  } else {
    // alone: the rounds that end first, a tile's ends counted as 512 tokens
    int64_t least = INT64_MAX;
    for (int64_t s = 1; s <= most; ++s) {
      const int64_t t = ceil_div(tiles * s, 256) * (ceil_div(n, s) + 512);
      if (t < least) least = t, g.splits = s;
    }
  }
  if (g.splits > most) g.splits = most;
  g.split_k = round_up(ceil_div(n, g.splits), 64);
  g.splits = ceil_div(n, g.split_k);
  return g;
}

struct Plan {
  int64_t ld, tiles, piece_n, pieces;
  bool copy_w;
  Size logits;
  Grads grads;
  int64_t logit_splits, logit_k, logit_ld, logit_part;
  int64_t at, row, count, scalars, weights, lse_at, target_at, xc, wc, stats, hit, row_loss, piece, dx_part, total;
};

static Plan plan_of(const mm_linear_cross_entropy_params* q, bool backward) {
  Plan s{};
  const int64_t es = dtype_size(q->dtype);
  s.ld = round_up(q->dim * es, 16);
  s.copy_w = s.ld != q->dim * es || q->weight_stride * es % 16 != 0 || q->weight_stride * es >= (int64_t{1} << 23) || !aligned(q->weight, 16);
  s.logits = logits_size(q->dtype, q->vocab, q->rows);
  s.tiles = ceil_div(q->vocab, high(s.logits));
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += round_up(bytes, 256);
    return was;
  };
  s.at = take(q->rows * 4);
  s.row = take(q->rows * 4);
  s.count = take(4);
  s.scalars = take(4);
  s.target_at = take(q->rows * 8);
  s.xc = take(q->rows * s.ld);
  if (s.copy_w) s.wc = take(q->vocab * s.ld);
  if (!backward) {
    s.stats = take(q->rows * s.tiles * 8);
    s.hit = take(q->rows * 4);
    s.row_loss = take(q->reduction ? q->rows * 4 : 0);
  } else {
    s.weights = take(q->rows * 4);
    s.lse_at = take(q->rows * 4);
    // pieces of equal sizes, whole tiles of 256
    int64_t most = kPieceBytes / (q->rows * es) / 256 * 256;
    if (most < 256) most = 256;
    s.pieces = ceil_div(q->vocab, most);
    s.piece_n = round_up(ceil_div(q->vocab, s.pieces), 256);
    s.pieces = ceil_div(q->vocab, s.piece_n);
    s.piece = take(q->rows * s.piece_n * es);
    s.logits = logits_size(q->dtype, s.piece_n, q->rows);
    // (the workspace's size does not hang on which of the gradients are asked for)
    const Grads both = grads_of(q->dtype, q->rows, q->dim, s.piece_n, true, true), one = grads_of(q->dtype, q->rows, q->dim, s.piece_n, true, false);
    s.grads = !q->dx ? grads_of(q->dtype, q->rows, q->dim, s.piece_n, false, true) : q->dweight ? both : one;
    s.dx_part = take((both.splits > one.splits ? both.splits : one.splits) * q->rows * q->dim * 4);
  }
  // (the piece's columns are whole tiles of 256)
  s.logit_splits = 1;
  s.logit_ld = backward ? s.piece_n : round_up(q->vocab, 128);
  if (q->dtype == MM_F32 && s.logits == kThin) {
    // 512 workgroups of 256 elements of the sum at least (a pass over the loss, 30 rows of 4000 by 5000 tokens: 155 us whole,
    // 49 in 13; 64 of 7000 by 8000: 258, and 92 in 9.  300 of 2000 by 5000, 200 tiles: 86 us whole, 88 in three.)
    const int64_t tiles = tiles_of(kThin, s.logit_ld, q->rows), most = s.ld / 4 / 256;
    if (tiles < 192 && most > 1) {
      s.logit_splits = ceil_div(512, tiles) < most ? ceil_div(512, tiles) : most;
      s.logit_k = round_up(ceil_div(s.ld / 4, s.logit_splits), 64);
      s.logit_splits = ceil_div(s.ld / 4, s.logit_k);
      s.logit_part = take(s.logit_splits * q->rows * s.logit_ld * 4);
    }
  }
  s.total = at;
  return s;
}

static int check(const mm_linear_cross_entropy_params* q) {
  if (!q) return fail(MM_ERR_NULL_POINTER, "params is NULL");
  if (!valid_dtype(q->dtype)) return fail(MM_ERR_DTYPE, "dtype %d", q->dtype);
  if (q->targets_dtype != 0 && q->targets_dtype != 1) return fail(MM_ERR_DTYPE, "targets_dtype %d", q->targets_dtype);
  if (q->reduction < 0 || q->reduction > 2) return fail(MM_ERR_SHAPE, "reduction %d", q->reduction);
  if (q->rows < 0 || q->dim < 1 || q->vocab < 1 || q->rows > kMaxRows || q->dim > kMaxDim || q->vocab > kMaxVocab ||
      q->rows * q->dim >= (int64_t{1} << 40) || q->vocab * q->dim >= (int64_t{1} << 40) ||
      ceil_div(q->rows, 64) * ceil_div(q->vocab, 128) >= (int64_t{1} << 31))
    return fail(MM_ERR_SHAPE, "%lld rows, dim %lld, vocab %lld: empty, negative or too large", (long long)q->rows, (long long)q->dim,
                (long long)q->vocab);
  if (q->rows > 0 && (!q->x || !q->weight || !q->targets)) return fail(MM_ERR_NULL_POINTER, "x, weight and targets are required");
  if (q->x_stride < 0 || q->weight_stride < 0 || q->dloss_stride < 0) return fail(MM_ERR_LAYOUT, "negative stride");
  return MM_OK;
}
static int check_workspace(const mm_linear_cross_entropy_params* q, const Plan& s) {
  if (q->rows > 0 && (!q->workspace || !aligned(q->workspace, 256) || q->workspace_bytes < static_cast<size_t>(s.total)))
    return fail(MM_ERR_WORKSPACE, "needs %lld bytes of 256-byte aligned workspace", (long long)s.total);
  return MM_OK;
}
static Loss loss_of(const mm_linear_cross_entropy_params* q, const Plan& s, bool backward) {
  char* const ws = static_cast<char*>(q->workspace);
  Loss p{};
  p.x = q->x;
  p.weight = q->weight;
  p.targets = q->targets;
  p.rows = q->rows;
  p.dim = q->dim;
  p.vocab = q->vocab;
  p.x_ld = q->x_stride;
  p.w_ld = q->weight_stride;
  p.ignore = q->ignore_index;
  p.dloss_stride = q->reduction ? 0 : q->dloss_stride;
  p.targets64 = q->targets_dtype;
  p.dtype = q->dtype;
  p.reduction = q->reduction;
  p.loss = q->loss;
  p.lse = q->lse;
  p.dloss = q->dloss;
  p.dx = q->dx;
  p.dweight = q->dweight;
  p.at = reinterpret_cast<int32_t*>(ws + s.at);
  p.row = reinterpret_cast<int32_t*>(ws + s.row);
  p.count = reinterpret_cast<int32_t*>(ws + s.count);
  p.scalars = reinterpret_cast<float*>(ws + s.scalars);
  p.target_at = reinterpret_cast<int64_t*>(ws + s.target_at);
  p.xc = ws + s.xc;
  p.wc = s.copy_w ? ws + s.wc : nullptr;
  p.ld = s.ld;
  p.tiles = s.tiles;
  p.logit_splits = s.logit_splits;
  p.logit_k = s.logit_k;
  p.logit_ld = s.logit_ld;
  p.logit_part = reinterpret_cast<float*>(ws + s.logit_part);
  if (!backward) {
    p.stats = reinterpret_cast<float*>(ws + s.stats);
    p.hit = reinterpret_cast<float*>(ws + s.hit);
    p.row_loss = q->reduction ? reinterpret_cast<float*>(ws + s.row_loss) : nullptr;
  } else {
    p.weights = reinterpret_cast<float*>(ws + s.weights);
    p.lse_at = reinterpret_cast<float*>(ws + s.lse_at);
    p.piece = ws + s.piece;
    p.piece_ld = s.piece_n * dtype_size(q->dtype);
    p.dx_part = reinterpret_cast<float*>(ws + s.dx_part);
    p.splits = s.grads.splits;
    p.split_k = s.grads.split_k;
  }
  return p;
}

template <int DT>
static void launch_gather(const Loss& p, const Plan& s, bool backward, hipStream_t st) {
  hipLaunchKernelGGL(rows_kernel, dim3(1), dim3(kThreads), 0, st, p, backward);
  const int64_t es = dtype_size(DT);
  auto grid = [&](int64_t rows) {
    const int64_t n = ceil_div(rows * (s.ld / 16), 256);
    return dim3(static_cast<unsigned>(n < 4096 ? n : 4096));
  };
  const bool vec = s.ld == p.dim * es && p.x_ld * es % 16 == 0 && aligned(p.x, 16);
  hipLaunchKernelGGL((lay_out_kernel<DT>), grid(p.rows), dim3(256), 0, st, p.x, p.x_ld, p.xc, s.ld, p.rows, p.dim, p.row, p.count, vec);
  if (p.wc)
    hipLaunchKernelGGL((lay_out_kernel<DT>), grid(p.vocab), dim3(256), 0, st, p.weight, p.w_ld, p.wc, s.ld, p.vocab, p.dim, nullptr,
                       nullptr, false);
}
template <int DT, typename S, bool GRAD>
static void launch_logits_t(const Loss& p, int64_t vocab, hipStream_t st) {
  hipLaunchKernelGGL((logits_kernel<DT, S, GRAD>), dim3(static_cast<unsigned>(ceil_div(vocab, S::BM) * ceil_div(p.rows, S::BN))),
                     dim3(64 * S::NW), 0, st, p);
}
template <int DT, bool GRAD>
static void launch_logits(const Loss& p, Size size, int64_t vocab, hipStream_t st) {
  if constexpr (DT == MM_F32) {
    if (p.logit_splits > 1) {
      hipLaunchKernelGGL((split_logits_kernel<DT>), dim3(static_cast<unsigned>(tiles_of(kThin, p.logit_ld, p.rows) * p.logit_splits)),
                         dim3(64 * Thin::NW), 0, st, p, GRAD);
      hipLaunchKernelGGL((join_logits_kernel<GRAD>), dim3(static_cast<unsigned>(ceil_div(p.rows * (p.logit_ld / 128), 4))), dim3(256),
                         0, st, p);
      return;
    }
  }
  switch (size) {
    case kBig:
      if constexpr (DT != MM_F32) launch_logits_t<DT, Big, GRAD>(p, vocab, st);
      break;
    case kMid: launch_logits_t<DT, Mid, GRAD>(p, vocab, st); break;
    case kThin: launch_logits_t<DT, Thin, GRAD>(p, vocab, st); break;
  }
}
template <int DT, typename S>
static void launch_grads_t(Loss p, hipStream_t st) {
  p.dx_tiles = p.dx ? static_cast<uint32_t>(ceil_div(p.rows, S::BM) * ceil_div(p.dim, S::BN) * p.splits) : 0;
  const int64_t dw = p.dweight ? ceil_div(p.piece_n, S::BM) * ceil_div(p.dim, S::BN) : 0;
  hipLaunchKernelGGL((grads_kernel<DT, S>), dim3(static_cast<unsigned>(p.dx_tiles + dw)), dim3(64 * S::NW), 0, st, p);
}
template <int DT>
static void launch_grads(const Loss& p, Size size, hipStream_t st) {
  if (size == kMid) return launch_grads_t<DT, Mid>(p, st);
  if constexpr (DT == MM_F32) launch_grads_t<DT, Thin>(p, st); else launch_grads_t<DT, Big>(p, st);
}

template <int DT>
static void forward(const Loss& p, const Plan& s, hipStream_t st) {
  launch_gather<DT>(p, s, false, st);
  launch_logits<DT, false>(p, s.logits, p.vocab, st);
  hipLaunchKernelGGL(merge_kernel, dim3(static_cast<unsigned>(ceil_div(p.rows, 4))), dim3(256), 0, st, p);
  if (p.reduction) hipLaunchKernelGGL(total_kernel, dim3(1), dim3(kThreads), 0, st, p);
}
template <int DT>
static void backward(Loss p, const Plan& s, hipStream_t st) {
  launch_gather<DT>(p, s, true, st);
  for (int64_t k = 0; k < s.pieces; ++k) {
    p.piece0 = k * s.piece_n;
    p.piece_n = p.piece0 + s.piece_n < p.vocab ? s.piece_n : p.vocab - p.piece0;
    p.first_piece = k == 0;
    launch_logits<DT, true>(p, s.logits, s.piece_n, st);
    if (p.dx || p.dweight) launch_grads<DT>(p, s.grads.size, st);
  }
  if (p.dx) hipLaunchKernelGGL((finish_dx_kernel<DT>), dim3(static_cast<unsigned>(p.rows)), dim3(256), 0, st, p);
}

}  // namespace xent
}  // namespace mm

extern "C" {

size_t mm_linear_cross_entropy_workspace_size(const mm_linear_cross_entropy_params* p, int32_t backward) {
  using namespace mm;
  using namespace mm::xent;
  if (check(p) != MM_OK || p->rows == 0) return 0;
  return static_cast<size_t>(plan_of(p, backward != 0).total);
}

int mm_linear_cross_entropy_fwd(const mm_linear_cross_entropy_params* q, void* stream) {
  using namespace mm;
  using namespace mm::xent;
  clear_error();
  int e = check(q);
  if (e != MM_OK || q->rows == 0) return e;
  if (!q->loss) return fail(MM_ERR_NULL_POINTER, "loss is required");
  const Plan s = plan_of(q, false);
  if ((e = check_workspace(q, s)) != MM_OK) return e;
  const Loss p = loss_of(q, s, false);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (q->dtype) {
    case MM_F32: forward<MM_F32>(p, s, st); break;
    case MM_F16: forward<MM_F16>(p, s, st); break;
    default: forward<MM_BF16>(p, s, st); break;
  }
  return check_launch("linear_cross_entropy_fwd");
}

int mm_linear_cross_entropy_bwd(const mm_linear_cross_entropy_params* q, void* stream) {
  using namespace mm;
  using namespace mm::xent;
  clear_error();
  int e = check(q);
  if (e != MM_OK || q->rows == 0) return e;
  if (!q->lse || !q->dloss) return fail(MM_ERR_NULL_POINTER, "lse and dloss are required");
  const Plan s = plan_of(q, true);
  if ((e = check_workspace(q, s)) != MM_OK) return e;
  if (!q->dx && !q->dweight) return MM_OK;
  const Loss p = loss_of(q, s, true);
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (q->dtype) {
    case MM_F32: backward<MM_F32>(p, s, st); break;
    case MM_F16: backward<MM_F16>(p, s, st); break;
    default: backward<MM_BF16>(p, s, st); break;
  }
  return check_launch("linear_cross_entropy_bwd");
}

}  // extern "C"
