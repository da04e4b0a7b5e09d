// Column sums of a row-major (rows, cols) fp32 matrix of partial sums, in double and in a fixed order.
#pragma once

#include "mm_common.h"

namespace mm {
namespace rows {

constexpr int kGroups = 8;    // row groups of a workgroup, one wave each
constexpr int kMaxRows = 512; // rows one workgroup sums by itself; more go through a first pass

// 64 columns a workgroup, rows [blockIdx.y * span, + span): wave g takes every kGroups-th row, the groups'
// sums are added in order.  store(c, sum) for pass two, part2[blockIdx.y][c] for the first of two passes.
template <typename Store>
__device__ __forceinline__ void sum_columns(const float* part, int64_t rows, int64_t cols, int64_t span, Store store) {
  __shared__ double s_part[kGroups][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  const int64_t r0 = static_cast<int64_t>(blockIdx.y) * span, r1 = r0 + span < rows ? r0 + span : rows;
  double s = 0.0;
  if (c < cols) {
#pragma unroll 8
    for (int64_t r = r0 + g; r < r1; r += kGroups) s += part[r * cols + c];
  }
  s_part[g][lane] = s;
  __syncthreads();
  if (g != 0 || c >= cols) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) s += s_part[k][lane];
  store(c, s);
}

// First of two passes: sums of kMaxRows rows each (kept in fp32: one more rounding).
static __global__ __launch_bounds__(64 * kGroups) void first_pass_kernel(const float* part, float* part2, int64_t rows,
                                                                        int64_t cols) {
  float* const out = part2 + static_cast<int64_t>(blockIdx.y) * cols;
  sum_columns(part, rows, cols, kMaxRows, [&](int64_t c, double s) { out[c] = static_cast<float>(s); });
}

// Floats of workspace for `rows` rows of partial sums: the rows, and the first pass's results.
inline int64_t floats(int64_t rows, int64_t cols) {
  return rows * cols + (rows > kMaxRows ? ceil_div(rows, kMaxRows) * cols : 0);
}
// Runs the first pass where it is needed; returns the rows that the last pass has to sum, and their count.
inline const float* reduce_first(float* part, int64_t& rows, int64_t cols, hipStream_t s) {
  if (rows <= kMaxRows) return part;
  float* const part2 = part + rows * cols;
  const int64_t n = ceil_div(rows, kMaxRows);
  hipLaunchKernelGGL(first_pass_kernel, dim3(static_cast<unsigned>(ceil_div(cols, 64)), static_cast<unsigned>(n)),
                     dim3(64 * kGroups), 0, s, part, part2, rows, cols);
  rows = n;
  return part2;
}

}  // namespace rows
}  // namespace mm
