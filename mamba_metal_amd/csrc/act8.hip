// Activations in 8 bits (act8.h): mm_act8_pack and mm_act8_unpack.
//
// One thread per block of 16 tokens of a channel, neighbouring channels on neighbouring lanes.
#include "act8.h"

namespace mm {
namespace act8 {

constexpr int kThreads = 256;

template <int DT>
__global__ __launch_bounds__(kThreads) void pack_kernel(const void* x, int8_t* codes, uint8_t* exps,
                                                        int64_t seqlen, int64_t dim, int64_t nblk,
                                                        int64_t total, int64_t xsb, int64_t xst) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= total) return;
  const int64_t d = id % dim, row = id / dim, b = row / nblk, t0 = row % nblk * kBlk;
  float v[kBlk];
#pragma unroll
  for (int k = 0; k < kBlk; ++k) {
    const int64_t t = t0 + k < seqlen ? t0 + k : seqlen - 1;
    v[k] = ld<DT>(x, b * xsb + t * xst + d);
    if (t0 + k >= seqlen) v[k] = 0.0f;
  }
  uint32_t e;
  *reinterpret_cast<uint4*>(codes + id * kBlk) = pack16(v, e);
  exps[id] = static_cast<uint8_t>(e);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void unpack_kernel(const int8_t* codes, const uint8_t* exps,
                                                          void* y, int64_t seqlen, int64_t dim,
                                                          int64_t nblk, int64_t total, int64_t ysb,
                                                          int64_t yst) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (id >= total) return;
  const int64_t d = id % dim, row = id / dim, b = row / nblk, t0 = row % nblk * kBlk;
  Block w;
  w.load(codes + (id - d) * kBlk, exps + (id - d), static_cast<uint32_t>(d));
  w.prepare();
#pragma unroll
  for (int k = 0; k < kBlk; ++k) {
    float v = w.value(k);
    // fp16's largest numbers round to a code that stands for 65536
    if (DT == MM_F16 && fabsf(v) == 65536.0f) v = v < 0.0f ? -65504.0f : 65504.0f;
    if (t0 + k < seqlen) st<DT>(y, b * ysb + (t0 + k) * yst + d, v);
  }
}

static int check(const void* x, const void* codes, const void* exps, int64_t batch, int64_t seqlen,
                 int64_t dim, const int64_t stride[2], int32_t dtype) {
  if (batch < 0 || seqlen < 0 || dim < 0) return fail(MM_ERR_SHAPE, "negative size");
  if (!valid_dtype(dtype)) return fail(MM_ERR_DTYPE, "dtype=%d", dtype);
  if (batch == 0 || seqlen == 0 || dim == 0) return MM_OK;
  if (!x || !codes || !exps || !stride)
    return fail(MM_ERR_NULL_POINTER, "the tensor, its strides, codes and exps are required");
  if (!aligned(codes, kBlk)) return fail(MM_ERR_LAYOUT, "codes are not 16-byte aligned");
  if (stride[0] < 0 || stride[1] < 0) return fail(MM_ERR_LAYOUT, "negative stride");
  if (ceil_div(seqlen, kBlk) > INT64_MAX / kBlk / 4 / batch / dim ||
      ceil_div(batch * ceil_div(seqlen, kBlk) * dim, kThreads) > 0x7fffffff)
    return fail(MM_ERR_SHAPE, "too many blocks");
  return MM_OK;
}

}  // namespace act8
}  // namespace mm

extern "C" {

int mm_act8_pack(const void* x, int8_t* codes, uint8_t* exps, int64_t batch, int64_t seqlen,
                 int64_t dim, const int64_t x_stride[2], int32_t dtype, void* stream) {
  using namespace mm;
  using namespace mm::act8;
  clear_error();
  const int e = check(x, codes, exps, batch, seqlen, dim, x_stride, dtype);
  if (e != MM_OK || batch == 0 || seqlen == 0 || dim == 0) return e;
  const int64_t nblk = ceil_div(seqlen, kBlk), total = batch * nblk * dim;
  const dim3 grid(static_cast<unsigned>(ceil_div(total, kThreads)));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_PACK(D)                                                                                  \
  hipLaunchKernelGGL((pack_kernel<D>), grid, dim3(kThreads), 0, s, x, codes, exps, seqlen, dim, nblk, \
                     total, x_stride[0], x_stride[1])
  switch (dtype) {
    case MM_F32: MM_PACK(MM_F32); break;
    case MM_F16: MM_PACK(MM_F16); break;
    default: MM_PACK(MM_BF16); break;
  }
#undef MM_PACK
  return check_launch("act8_pack");
}

int mm_act8_unpack(const int8_t* codes, const uint8_t* exps, void* y, int64_t batch, int64_t seqlen,
                   int64_t dim, const int64_t y_stride[2], int32_t dtype, void* stream) {
  using namespace mm;
  using namespace mm::act8;
  clear_error();
  const int e = check(y, codes, exps, batch, seqlen, dim, y_stride, dtype);
  if (e != MM_OK || batch == 0 || seqlen == 0 || dim == 0) return e;
  const int64_t nblk = ceil_div(seqlen, kBlk), total = batch * nblk * dim;
  const dim3 grid(static_cast<unsigned>(ceil_div(total, kThreads)));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_UNPACK(D)                                                                                   \
  hipLaunchKernelGGL((unpack_kernel<D>), grid, dim3(kThreads), 0, s, codes, exps, y, seqlen, dim, nblk, \
                     total, y_stride[0], y_stride[1])
  switch (dtype) {
    case MM_F32: MM_UNPACK(MM_F32); break;
    case MM_F16: MM_UNPACK(MM_F16); break;
    default: MM_UNPACK(MM_BF16); break;
  }
#undef MM_UNPACK
  return check_launch("act8_unpack");
}

}  // extern "C"
