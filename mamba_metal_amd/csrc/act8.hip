// Activations in 8 bits (act8.h): mm_act8_pack and mm_act8_unpack.
//
// One thread per block of 16 tokens of a channel, neighbouring channels on neighbouring lanes.  Bound by memory: bf16
// 8 x 2048 x 2560 19 us packed and 20 us unpacked (6.6 TB/s, with the last-level cache's help; with a 64-bit index a
// thread, whose divisions were half of the instructions, 25 and 28).
#include "act8.h"
#include "row_io.h"

namespace mm {
namespace act8 {

constexpr int kMaxThreads = 256;

// The workgroup's row of blocks (of all sequences) and the thread's channel; lanes past the last channel do what the
// last one's does.
struct Place {
  uint32_t d;
  int64_t row, b, t0;
  __device__ __forceinline__ Place(int64_t dim, uint32_t nblk, uint32_t ncb) {
    d = min(blockIdx.x % ncb * blockDim.x + threadIdx.x, static_cast<uint32_t>(dim - 1));
    const uint32_t r = blockIdx.x / ncb;
    row = r;
    b = r / nblk;
    t0 = static_cast<int64_t>(r % nblk) * kBlk;
  }
};

template <int DT>
__global__ __launch_bounds__(kMaxThreads) void pack_kernel(const void* x, int8_t* codes, uint8_t* exps, int64_t seqlen,
                                                           int64_t dim, uint32_t nblk, uint32_t ncb, int64_t xsb, int64_t xst) {
  using T = typename Ty<DT>::T;
  const Place at(dim, nblk, ncb);
  const uint32_t off = at.d * static_cast<uint32_t>(sizeof(T));
  const int64_t stride[2] = {xsb, xst};
  Rows<DT> in(x, stride, at.b, at.t0);
  T raw[kBlk];
  float v[kBlk];
  if (at.t0 + kBlk <= seqlen) {
#pragma unroll
    for (int k = 0; k < kBlk; ++k) {
      raw[k] = in.load(off);
      in.next();
    }
#pragma unroll
    for (int k = 0; k < kBlk; ++k) v[k] = Ty<DT>::f(raw[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kBlk; ++k) {
      raw[k] = in.load(off);
      in.next(at.t0 + k + 1 < seqlen);
    }
#pragma unroll
    for (int k = 0; k < kBlk; ++k) v[k] = at.t0 + k < seqlen ? Ty<DT>::f(raw[k]) : 0.0f;
  }
  uint32_t e;
  const uint4 w = pack16(v, e);
  *reinterpret_cast<uint4*>(codes + at.row * dim * kBlk + static_cast<uint64_t>(at.d) * kBlk) = w;
  (exps + at.row * dim)[at.d] = static_cast<uint8_t>(e);
}

template <int DT>
__global__ __launch_bounds__(kMaxThreads) void unpack_kernel(const int8_t* codes, const uint8_t* exps, void* y, int64_t seqlen,
                                                             int64_t dim, uint32_t nblk, uint32_t ncb, int64_t ysb,
                                                             int64_t yst) {
  using T = typename Ty<DT>::T;
  const Place at(dim, nblk, ncb);
  const uint32_t off = at.d * static_cast<uint32_t>(sizeof(T));
  Block w;
  w.load(codes + at.row * dim * kBlk, exps + at.row * dim, at.d);
  w.prepare();
  const int64_t stride[2] = {ysb, yst};
  Rows<DT> out(y, stride, at.b, at.t0);
  const int n = at.t0 + kBlk <= seqlen ? kBlk : static_cast<int>(seqlen - at.t0);
#pragma unroll
  for (int k = 0; k < kBlk; k += 2) {
    float v[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      v[c] = w.value(k + c);
      // fp16's largest numbers round to a code that stands for 65536
      if (DT == MM_F16 && fabsf(v[c]) == 65536.0f) v[c] = v[c] < 0.0f ? -65504.0f : 65504.0f;
    }
    T r[2];
    round2<DT>(v[0], v[1], r[0], r[1]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (k + c < n) out.store(off, r[c]);
      out.next();
    }
  }
}

// Threads of a workgroup (whole waves, no more than the channels need) and workgroups of a row.
static int threads_of(int64_t dim) { return dim >= kMaxThreads ? kMaxThreads : static_cast<int>(round_up(dim, 64)); }

static int check(const void* x, const void* codes, const void* exps, int64_t batch, int64_t seqlen,
                 int64_t dim, const int64_t stride[2], int32_t dtype) {
  if (batch < 0 || seqlen < 0 || dim < 0) return fail(MM_ERR_SHAPE, "negative size");
  if (!valid_dtype(dtype)) return fail(MM_ERR_DTYPE, "dtype=%d", dtype);
  if (batch == 0 || seqlen == 0 || dim == 0) return MM_OK;
  if (!x || !codes || !exps || !stride)
    return fail(MM_ERR_NULL_POINTER, "the tensor, its strides, codes and exps are required");
  if (!aligned(codes, kBlk)) return fail(MM_ERR_LAYOUT, "codes are not 16-byte aligned");
  if (stride[0] < 0 || stride[1] < 0) return fail(MM_ERR_LAYOUT, "negative stride");
  if (dim > (int64_t{1} << 30) || ceil_div(seqlen, kBlk) > 0x7fffffff / batch ||
      batch * ceil_div(seqlen, kBlk) > 0x7fffffff / ceil_div(dim, threads_of(dim)))
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
  const uint32_t nblk = static_cast<uint32_t>(ceil_div(seqlen, kBlk));
  const int threads = threads_of(dim);
  const uint32_t ncb = static_cast<uint32_t>(ceil_div(dim, threads));
  const dim3 grid(static_cast<unsigned>(batch * nblk * ncb));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_PACK(D)                                                                                            \
  hipLaunchKernelGGL((pack_kernel<D>), grid, dim3(threads), 0, s, x, codes, exps, seqlen, dim, nblk, ncb, x_stride[0], \
                     x_stride[1])
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
  if (rows_overlap(batch, seqlen, dim, y_stride)) return fail(MM_ERR_LAYOUT, "rows of y overlap");
  const uint32_t nblk = static_cast<uint32_t>(ceil_div(seqlen, kBlk));
  const int threads = threads_of(dim);
  const uint32_t ncb = static_cast<uint32_t>(ceil_div(dim, threads));
  const dim3 grid(static_cast<unsigned>(batch * nblk * ncb));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_UNPACK(D)                                                                                            \
  hipLaunchKernelGGL((unpack_kernel<D>), grid, dim3(threads), 0, s, codes, exps, y, seqlen, dim, nblk, ncb, y_stride[0], \
                     y_stride[1])
  switch (dtype) {
    case MM_F32: MM_UNPACK(MM_F32); break;
    case MM_F16: MM_UNPACK(MM_F16); break;
    default: MM_UNPACK(MM_BF16); break;
  }
#undef MM_UNPACK
  return check_launch("act8_unpack");
}

}  // extern "C"
