// Column sums of a row-major (rows, cols) fp32 matrix of partial sums, in double and in a fixed order.
#pragma once

#include "mm_common.h"

namespace mm {
namespace rows {

constexpr int kGroups = 8;    // row groups of a workgroup, one wave each
constexpr int kMaxRows = 512; // rows one workgroup sums by itself; more go through a first pass

// Columns [64 block, + 64), rows [group * span, + span): wave g takes every kGroups-th row, the waves' sums are
// added in order, and store(c, sum) gets them.
template <typename Store>
__device__ __forceinline__ void sum_columns(const float* part, int64_t rows, int64_t cols, int64_t block, int64_t group,
                                            int64_t span, Store store) {
  __shared__ double s_part[kGroups][64];
  const int lane = threadIdx.x & 63, g = threadIdx.x >> 6;
  const int64_t c = block * 64 + lane;
  const int64_t r0 = group * span, r1 = r0 + span < rows ? r0 + span : rows;
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
                                                                        int64_t cols, uint32_t blocks) {
  const uint32_t block = blockIdx.x % blocks, group = blockIdx.x / blocks;
  float* const out = part2 + static_cast<int64_t>(group) * cols;
  sum_columns(part, rows, cols, block, group, kMaxRows, [&](int64_t c, double s) { out[c] = static_cast<float>(s); });
}

// Floats of workspace for `rows` rows of partial sums: the rows, and the first pass's results.
inline int64_t floats(int64_t rows, int64_t cols) {
  return rows * cols + (rows > kMaxRows ? ceil_div(rows, kMaxRows) * cols : 0);
}
// Runs the first pass where it is needed; returns the rows that the last pass has to sum, and their count.
inline const float* reduce_first(float* part, int64_t& rows, int64_t cols, hipStream_t s) {
  if (rows <= kMaxRows) return part;
  float* const part2 = part + rows * cols;
  const int64_t n = ceil_div(rows, kMaxRows), blocks = ceil_div(cols, 64);  // (fewer workgroups than the rows had)
  hipLaunchKernelGGL(first_pass_kernel, dim3(static_cast<unsigned>(n * blocks)), dim3(64 * kGroups), 0, s, part, part2, rows,
                     cols, static_cast<uint32_t>(blocks));
  rows = n;
  return part2;
}

}  // namespace rows
}  // namespace mm
