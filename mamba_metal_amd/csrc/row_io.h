// Row by row access of kernels whose lanes are neighbouring channels and whose waves walk along time.
#pragma once

#include "mm_common.h"

namespace mm {

// Rows of a tensor: a wave-uniform address that moves on by a row, and a lane's 32-bit offset into it (dim is at
// most 2^30, an element at most 4 bytes), so that an access takes no vector address arithmetic.
template <int DT>
struct Rows {
  using T = typename Ty<DT>::T;
  typedef __attribute__((address_space(1))) char Byte;  // (the asm below would lose that it is global memory)
  typedef __attribute__((address_space(1))) T Elem;
  Byte* p;
  int64_t step;  // bytes
  __device__ __forceinline__ Rows(const void* base, const int64_t* stride, int64_t b, int64_t t)
      : p((Byte*)const_cast<void*>(base) + (b * stride[0] + t * stride[1]) * static_cast<int64_t>(sizeof(T))),
        step(stride[1] * static_cast<int64_t>(sizeof(T))) {}
  __device__ __forceinline__ Rows(void* base, int64_t row, int64_t dim)  // contiguous
      : p((Byte*)base + row * dim * static_cast<int64_t>(sizeof(T))),
        step(dim * static_cast<int64_t>(sizeof(T))) {}
  __device__ __forceinline__ T load(uint32_t off) const { return *(const Elem*)(p + off); }
  __device__ __forceinline__ void store(uint32_t off, T v) const { *(Elem*)(p + off) = v; }
  __device__ __forceinline__ void next(bool more = true) {
    p += more ? step : 0;
    // a running address, not a product a row, and no more than one ahead of its access: SGPRs are few
    asm("" : "+s"(p));
    __builtin_amdgcn_sched_barrier(0);
  }
};

// Takes v as computed here: the compiler otherwise moves what only the outputs need past the wait, and holds its
// several operands in registers over it instead (backward pass: 240 registers, or 180 spilled ones).
__device__ __forceinline__ void keep(float& v) { asm volatile("" : "+v"(v)); }

// Two tokens' outputs, rounded to nearest even (bf16: one v_cvt_pk_bf16_f32 for both).
template <int DT>
__device__ __forceinline__ void round2(float x, float y, typename Ty<DT>::T& a, typename Ty<DT>::T& b) {
  if constexpr (DT == MM_BF16) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const uint32_t v = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), bf2));
    a = static_cast<unsigned short>(v);
    b = static_cast<unsigned short>(v >> 16);
  } else {
    a = Ty<DT>::from(x);
    b = Ty<DT>::from(y);
  }
}

}  // namespace mm
