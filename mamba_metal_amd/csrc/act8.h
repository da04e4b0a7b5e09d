// Activations kept in 8 bits: blocks of 16 tokens of one channel as int8 codes times one power of two.
//
// A block's scale is 2^(e - 127) for its exponent byte e, the smallest power of two that keeps the codes
// within 127: with m = max |x| over the block, m / scale lies in [63.75, 127.5), so a code is off by at most
// half a step, m / 127.5 at worst.  A power of two costs up to one bit against m / 127 and makes everything
// exact: x / scale and code * scale round nowhere, a code times its scale is a number of the activation's own type
// (but for fp16's largest, whose code stands for 65536), and the scale takes one byte.  Blocks run along time because a layer's outlier channels then keep their
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

// Codes of a lane's 16 values, the first in the lowest byte, and their exponent byte.  x / scale + 1.5 * 2^23 in
// one multiply-add is rounded to a whole number, ties to even, and has the code in its lowest byte.  (Only the
// largest exponent leaves room for a code of 128: there values are cut to 127 first.  A broken block's codes are
// zeros: a NaN would leave its own lowest byte.)
__device__ __forceinline__ uint4 pack16(const float (&v)[kBlk], uint32_t& e) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < kBlk; ++k) top = max(top, __float_as_uint(v[k]) & 0x7fffffffu);
  e = exponent_of(top);
  const float inv = inv_scale(e);
  uint32_t w[kBlk / 4];
  auto codes = [&](auto value) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kBlk; k += 4) {
      uint32_t c[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) c[q] = __float_as_uint(__builtin_fmaf(value(v[k + q]), inv, 12582912.0f));
      // bytes 0 of two words: select 0 is the second operand's lowest byte, 4 the first's, 0xc zero
      const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
      w[k / 4] = lo | hi << 16;
    }
  };
  if (__any(e >= 248u)) {
    const float most = 127.0f * __uint_as_float(248u << 23);
    codes([&](float x) __attribute__((always_inline)) {
      const float cut = e == 248u ? fminf(fmaxf(x, -most), most) : x;
      return e == 255u ? 0.0f : cut;
    });
  } else {
    codes([](float x) __attribute__((always_inline)) { return x; });
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A lane's block of 16 codes: loaded, prepared once, read value by value.
struct Block {
  uint4 w;
  uint32_t e;
  float scale;
  // codes and exps of a row of blocks (wave-uniform), the lane's channel
  __device__ __forceinline__ void load(const int8_t* codes, const uint8_t* exps, uint32_t d) {
    w = *reinterpret_cast<const uint4*>(codes + static_cast<uint64_t>(d) * kBlk);
    e = exps[d];
  }
  __device__ __forceinline__ void prepare() { scale = scale_of(e); }
  __device__ __forceinline__ float value(int k) const {
    const uint32_t v = k < 4 ? w.x : k < 8 ? w.y : k < 12 ? w.z : w.w;
    return static_cast<float>(static_cast<int8_t>(v >> (8 * (k % 4)))) * scale;
  }
};

}  // namespace act8
}  // namespace mm
