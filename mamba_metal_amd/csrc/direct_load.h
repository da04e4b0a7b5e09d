// Loads from memory straight into shared memory, 16 bytes a lane.
#pragma once

#include "mm_common.h"

namespace mm {

constexpr uint32_t kNowhere = 0x80000000u;  // an offset past a buffer's end: zeros are loaded
__device__ __forceinline__ void load_direct(const char* base, uint32_t off, char* to) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x7fffffff, 0x00027000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)to, 16, off, 0, 0, 0);
}

}  // namespace mm
