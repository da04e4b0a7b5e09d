// Backward pass of the causal depthwise conv1d (+ SiLU): mm_causal_conv1d_bwd.
//
//   p_t = bias + sum_k w_k x_{t-(K-1)+k}     dp = dout * silu'(p)
//   dx_t = sum_k w_k dp_{t+(K-1)-k}          dw_k = sum_t dp_t x_{t-(K-1)+k}     dbias = sum_t dp_t
//
// One thread per channel and run of kRun tokens: it walks from the run's first token to K - 1 past its
// end, the last K values of x and of dp in registers, and recomputes p.  A run's sums for dw and dbias go
// to the workspace; a second kernel adds the runs up in a fixed order, in double.
#include <type_traits>

#include "act8.h"
#include "reduce_rows.h"

namespace mm {
namespace convb {

constexpr int kThreads = 64;
constexpr int kRun = 64;   // tokens per thread, a multiple of the 8-bit block
constexpr int kMaxW = 8;

struct Params {
  const void* x;
  const int8_t* codes;
  const uint8_t* exps;
  const void* w;
  const void* bias;
  const void* dout;
  void* dx;
  float* part;  // [runs of all sequences][K + 1][dim], or NULL
  int64_t seqlen, dim, nruns;
  int64_t xs0, xs1, ds0, ds1, ws0, ws1;
  uint32_t ncb;  // blocks of channels
  int32_t w_dtype, silu;
};

__device__ __forceinline__ int64_t round_up_dev(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
__device__ __forceinline__ float ld_any(const void* p, int64_t i, int32_t dt) {
  return dt == MM_F32 ? ld<MM_F32>(p, i) : dt == MM_F16 ? ld<MM_F16>(p, i) : ld<MM_BF16>(p, i);
}
__device__ __forceinline__ void st_any(void* p, int64_t i, float v, int32_t dt) {
  if (dt == MM_F32) st<MM_F32>(p, i, v);
  else if (dt == MM_F16) st<MM_F16>(p, i, v);
  else st<MM_BF16>(p, i, v);
}

template <int DT, int K, bool C8>
__global__ __launch_bounds__(kThreads) void conv1d_bwd_kernel(const Params p) {
  using T = typename Ty<DT>::T;
  constexpr int kB = act8::kBlk, H = K - 1;  // tokens loaded at once; history
  const uint32_t d = (blockIdx.x % p.ncb) * 64 + (threadIdx.x & 63);
  if (d >= p.dim) return;
  const int64_t row = blockIdx.x / p.ncb;  // of all sequences' runs
  const int64_t b = row / p.nruns, t0 = row % p.nruns * kRun;
  const int64_t t1 = t0 + kRun < p.seqlen ? t0 + kRun : p.seqlen;
  const int64_t nblk = (p.seqlen + kB - 1) / kB;
  const T* const xb = static_cast<const T*>(p.x) + b * p.xs0;
  const T* const yb = static_cast<const T*>(p.dout) + b * p.ds0;
  T* const dxb = static_cast<T*>(p.dx) + b * p.seqlen * p.dim;
  float w[K], dw[K];
  const float bias = p.bias ? ld_any(p.bias, d, p.w_dtype) : 0.0f;
  float db = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    w[k] = ld_any(p.w, d * p.ws0 + k * p.ws1, p.w_dtype);
    dw[k] = 0.0f;
  }
  // x[t0 + k], k < n, of the 16 tokens from t0 on (a block's); tokens past the sequence read its last one
  auto load_x = [&](float* x, int64_t t0, int k0, int n) __attribute__((always_inline)) {
    if constexpr (C8) {
      const int64_t o = (b * nblk + t0 / kB) * p.dim;
      act8::Block q;
      q.load(p.codes + o * kB, p.exps + o, d);
      q.prepare();
#pragma unroll
      for (int k = 0; k < n; ++k) x[k] = q.value(k0 + k);
    } else {
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const int64_t t = t0 + k0 + k;
        x[k] = Ty<DT>::f(xb[(t < p.seqlen ? t : p.seqlen - 1) * p.xs1 + d]);
      }
    }
  };
  auto slope = [&](float v) __attribute__((always_inline)) {  // silu'
    const float s = rcp_hw(1.0f + exp2_hw(-v * kLog2e));
    return s * __builtin_fmaf(v, 1.0f - s, 1.0f);
  };
  float x[H + kB], dp[H + kB];  // tokens t - H .. t + 15
#pragma unroll
  for (int k = 0; k < H; ++k) x[k] = dp[k] = 0.0f;
  if (H > 0 && t0 > 0) load_x(x, t0 - kB, kB - H, H);
  // tokens t + k0, k0 < n: p, dp, the sums (`own` tokens only) and dx of H tokens earlier
  auto tokens = [&](int64_t t, auto n_c, auto own_c) __attribute__((always_inline)) {
    constexpr int n = decltype(n_c)::value;
    constexpr bool own = decltype(own_c)::value;
    float dy[n];
#pragma unroll
    for (int k = 0; k < n; ++k) dy[k] = Ty<DT>::f(yb[(t + k < p.seqlen ? t + k : p.seqlen - 1) * p.ds1 + d]);
    load_x(x + H, t, 0, n);
#pragma unroll
    for (int k = 0; k < n; ++k) {
      float v = bias;
#pragma unroll
      for (int q = 0; q < K; ++q) v = __builtin_fmaf(w[q], x[k + q], v);
      const float s = p.silu ? slope(v) : 1.0f;
      dp[H + k] = t + k < p.seqlen ? dy[k] * s : 0.0f;
      if constexpr (own) {
        db += dp[H + k];
#pragma unroll
        for (int q = 0; q < K; ++q) dw[q] = __builtin_fmaf(dp[H + k], t + k < p.seqlen ? x[k + q] : 0.0f, dw[q]);
      }
      const int64_t o = t + k - H;
      if (p.dx != nullptr && o >= t0 && o < t1) {
        float u = 0.0f;
#pragma unroll
        for (int q = 0; q < K; ++q) u = __builtin_fmaf(w[q], dp[H + k - q], u);
        dxb[o * p.dim + d] = Ty<DT>::from(u);
      }
    }
#pragma unroll
    for (int k = 0; k < H; ++k) x[k] = x[n + k], dp[k] = dp[n + k];
  };
  for (int64_t t = t0; t < t1; t += kB) tokens(t, std::integral_constant<int, kB>{}, std::true_type{});
  // the last H tokens' dx: up to H tokens of the next run, or zeros
  if constexpr (H > 0) {
    const int64_t end = round_up_dev(t1, kB);
    if (end < p.seqlen) {
      tokens(end, std::integral_constant<int, H>{}, std::false_type{});
    } else if (p.dx != nullptr) {
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const int64_t o = end + k - H;
        float u = 0.0f;
#pragma unroll
        for (int q = k + 1; q < K; ++q) u = __builtin_fmaf(w[q], dp[H + k - q], u);
        if (o >= t0 && o < t1) dxb[o * p.dim + d] = Ty<DT>::from(u);
      }
    }
  }
  if (p.part != nullptr) {
    float* q = p.part + row * (K + 1) * p.dim + d;
#pragma unroll
    for (int k = 0; k < K; ++k) q[k * p.dim] = dw[k];
    q[K * p.dim] = db;
  }
}

// dw[c, k] and dbias[c] from the runs' sums, rows of [K + 1][dim].
__global__ __launch_bounds__(64 * rows::kGroups) void reduce_kernel(const float* part, void* dw, void* dbias, int64_t nrows,
                                                                  int64_t dim, int width, int32_t w_dtype) {
  rows::sum_columns(part, nrows, (width + 1) * dim, nrows, [&](int64_t c, double s) {
    const int64_t k = c / dim, d = c % dim;
    if (k < width) st_any(dw, d * width + k, static_cast<float>(s), w_dtype);
    else if (dbias != nullptr) st_any(dbias, d, static_cast<float>(s), w_dtype);
  });
}

static bool sizes_ok(int64_t batch, int64_t seqlen, int64_t dim) {
  return batch >= 0 && seqlen >= 0 && dim >= 0 && dim <= (int64_t{1} << 30) && seqlen <= (int64_t{1} << 40) &&
         (dim == 0 || seqlen == 0 || batch <= INT64_MAX / 64 / dim / (seqlen + kRun));
}

}  // namespace convb
}  // namespace mm

extern "C" {

size_t mm_causal_conv1d_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int64_t width) {
  using namespace mm;
  using namespace mm::convb;
  if (!sizes_ok(batch, seqlen, dim) || width < 1 || width > kMaxW) return 0;
  return static_cast<size_t>(rows::floats(batch * ceil_div(seqlen, kRun), (width + 1) * dim) * 4);
}

int mm_causal_conv1d_bwd(const void* x, const int8_t* x_codes, const uint8_t* x_exps,
                         const void* weight, const void* bias, const void* dout, void* dx, void* dw,
                         void* dbias, int64_t batch, int64_t seqlen, int64_t dim, int64_t width,
                         const int64_t x_stride[2], const int64_t dout_stride[2],
                         const int64_t w_stride[2], int32_t x_dtype, int32_t w_dtype,
                         int32_t apply_silu, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mm;
  using namespace mm::convb;
  clear_error();
  if (batch < 0 || seqlen < 0 || dim < 0) return fail(MM_ERR_SHAPE, "negative size");
  if (width < 1 || width > kMaxW) return fail(MM_ERR_SHAPE, "width=%lld not in 1..%d", (long long)width, kMaxW);
  if (!sizes_ok(batch, seqlen, dim)) return fail(MM_ERR_SHAPE, "too many elements");
  if (!valid_dtype(x_dtype) || !valid_dtype(w_dtype)) return fail(MM_ERR_DTYPE, "bad dtype");
  const bool c8 = x == nullptr;
  const int64_t nruns = ceil_div(seqlen, kRun), nrun_rows = batch * nruns;
  if (batch > 0 && seqlen > 0 && dim > 0) {
    if (c8 ? !x_codes || !x_exps : !x_stride)
      return fail(MM_ERR_NULL_POINTER, "x and its strides, or x_codes and x_exps, are required");
    if (!weight || !w_stride || !dout || !dout_stride)
      return fail(MM_ERR_NULL_POINTER, "weight, dout and their strides are required");
    if ((!c8 && (x_stride[0] < 0 || x_stride[1] < 0)) || dout_stride[0] < 0 || dout_stride[1] < 0 ||
        w_stride[0] < 0 || w_stride[1] < 0)
      return fail(MM_ERR_LAYOUT, "negative stride");
  }
  if (nrun_rows > 0x7fffffff / ceil_div(dim > 0 ? dim : 1, kThreads)) return fail(MM_ERR_SHAPE, "too many elements");
  if (dbias && !dw) return fail(MM_ERR_NULL_POINTER, "dbias needs dw");
  if (dim == 0 || (!dx && !dw)) return MM_OK;
  const size_t need = dw ? mm_causal_conv1d_bwd_workspace_size(batch, seqlen, dim, width) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(MM_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  if (c8 && !aligned(x_codes, act8::kBlk)) return fail(MM_ERR_LAYOUT, "x_codes are not 16-byte aligned");
  if (need > 0 && !aligned(workspace, 256)) return fail(MM_ERR_WORKSPACE, "workspace is not 256-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (nrun_rows > 0) {
    Params p{};
    p.x = x;
    p.codes = x_codes;
    p.exps = x_exps;
    p.w = weight;
    p.bias = bias;
    p.dout = dout;
    p.dx = dx;
    p.part = dw ? static_cast<float*>(workspace) : nullptr;
    p.seqlen = seqlen;
    p.dim = dim;
    p.nruns = nruns;
    if (!c8) p.xs0 = x_stride[0], p.xs1 = x_stride[1];
    p.ds0 = dout_stride[0], p.ds1 = dout_stride[1];
    p.ws0 = w_stride[0], p.ws1 = w_stride[1];
    p.w_dtype = w_dtype;
    p.silu = apply_silu != 0;
    p.ncb = static_cast<uint32_t>(ceil_div(dim, kThreads));
    const dim3 grid(static_cast<unsigned>(p.ncb * nrun_rows));
#define MM_CB1(D, K, C) hipLaunchKernelGGL((conv1d_bwd_kernel<D, K, C>), grid, dim3(kThreads), 0, s, p)
#define MM_CB2(D, K) \
  if (c8) MM_CB1(D, K, true); else MM_CB1(D, K, false); break
#define MM_CB(D)                 \
  switch (width) {               \
    case 1: MM_CB2(D, 1);        \
    case 2: MM_CB2(D, 2);        \
    case 3: MM_CB2(D, 3);        \
    case 4: MM_CB2(D, 4);        \
    case 5: MM_CB2(D, 5);        \
    case 6: MM_CB2(D, 6);        \
    case 7: MM_CB2(D, 7);        \
    default: MM_CB2(D, 8);       \
  }
    switch (x_dtype) {
      case MM_F32: MM_CB(MM_F32); break;
      case MM_F16: MM_CB(MM_F16); break;
      default: MM_CB(MM_BF16); break;
    }
#undef MM_CB
#undef MM_CB2
#undef MM_CB1
    const int e = check_launch("causal_conv1d_bwd");
    if (e != MM_OK) return e;
  }
  if (!dw) return MM_OK;
  const int64_t cols = (width + 1) * dim;
  int64_t nrows = nrun_rows;
  const float* part = rows::reduce_first(static_cast<float*>(workspace), nrows, cols, s);
  hipLaunchKernelGGL(reduce_kernel, dim3(static_cast<unsigned>(ceil_div(cols, 64))), dim3(64 * rows::kGroups), 0, s, part, dw,
                     dbias, nrows, dim, static_cast<int>(width), w_dtype);
  return check_launch("causal_conv1d_bwd_reduce");
}

}  // extern "C"
