// Activations kept in 8 bits: blocks of 16 tokens of one channel as int8 codes times one power of two.
//
// A block's scale is 2^(e - 127) for its exponent byte e, the smallest power of two that keeps the codes
// within 127: with m = max |x| over the block, m / scale lies in [63.75, 127.5), so a code is off by at most
// half a step, m / 127.5 at worst.  A power of two costs up to one bit against m / 127 and makes everything
// exact: x / scale and code * scale round nowhere, a code times its scale is a bf16 or fp16 number, and
// the scale takes one byte.  Blocks run along time because a layer's outlier channels then keep their
// scale to themselves, and because the kernels hold a channel's 16 tokens in one lane: no reduction
// crosses lanes.  A block's 16 codes are 16 contiguous bytes, blocks of neighbouring channels next to each
// other, so that a lane moves a block in one access and a wave 1 KB.  e = 255 marks a block that held an infinity or a NaN: it stands for NaNs.
#pragma once

#include "mm_common.h"

namespace mm {
namespace act8 {

constexpr int kBlk = MM_ACT8_BLOCK;

// Exponent byte of a block whose largest magnitude has these bits (largest as whole numbers, so that a
// NaN wins).  Adding half a code's step to the mantissa carries into the exponent exactly where a code
// would round to 128; the largest exponent that carries on past float's range keeps 248 and codes of 127.
__device__ __forceinline__ uint32_t exponent_of(uint32_t amax_bits) {
  const int e = static_cast<int>((amax_bits + 0x10000u) >> 23) - 6;
  const int c = e < 1 ? 1 : e > 248 ? 248 : e;
  return amax_bits >= 0x7f800000u ? 255u : static_cast<uint32_t>(c);
}
// 1 / scale (0 for a block of NaNs: its codes are zeros) and scale of an exponent byte.
__device__ __forceinline__ float inv_scale(uint32_t e) {
  return e == 255u ? 0.0f : __uint_as_float((254u - e) << 23);
}
__device__ __forceinline__ float scale_of(uint32_t e) {
  return e == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(e << 23);
}
__device__ __forceinline__ int code_of(float x, float inv) {
  float q = __builtin_rintf(x * inv);
  q = fminf(fmaxf(q, -127.0f), 127.0f);  // (a NaN, in a block of them, gives -127: any code will do)
  return static_cast<int>(q);
}
// Codes of four values, the first in the lowest byte.
__device__ __forceinline__ uint32_t code4(float a, float b, float c, float d, float inv) {
  return (static_cast<uint32_t>(code_of(a, inv)) & 0xffu) | (static_cast<uint32_t>(code_of(b, inv)) & 0xffu) << 8 |
         (static_cast<uint32_t>(code_of(c, inv)) & 0xffu) << 16 | static_cast<uint32_t>(code_of(d, inv)) << 24;
}
// Value k of a block's 16 codes.
__device__ __forceinline__ float value_of(const uint4& w, int k, float scale) {
  const uint32_t v = k < 4 ? w.x : k < 8 ? w.y : k < 12 ? w.z : w.w;
  return static_cast<float>(static_cast<int8_t>(v >> (8 * (k % 4)))) * scale;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace act8
}  // namespace mm
