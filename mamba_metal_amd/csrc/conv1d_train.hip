// Training form of the causal depthwise conv1d (+ SiLU): mm_causal_conv1d_bwd, and mm_causal_conv1d_fwd_act8, the
// forward pass that keeps its input in 8 bits.
//
//   p_t = bias + sum_k w_k x_{t-(K-1)+k}     dp = dout * silu'(p)
//   dx_t = sum_k w_k dp_{t+(K-1)-k}          dw_k = sum_t dp_t x_{t-(K-1)+k}     dbias = sum_t dp_t
//
// One thread per channel and run of tokens, four waves of neighbouring channels a workgroup: it walks the run in
// blocks of 16 tokens, all of a block loaded at once, with the last K - 1 values of x and dp in registers, and
// recomputes p.  A run's last dx need dp of the K - 1 tokens after it, which are computed again.  A run's sums
// for dw and dbias go to the workspace; another kernel adds the runs up in a fixed order, in double.
//
// bf16 8 x 2048 x 5120, width 4, 8-bit checkpoint: forward with the codes 81 us (5.3 TB/s, memory), backward 107 + 4 us
// (4.0 TB/s; 32 vector instructions an element keep the units 84% busy).  The next block's loads ahead of this one's
// arithmetic change nothing.
#include <type_traits>

#include "act8.h"
#include "reduce_rows.h"
#include "row_io.h"

namespace mm {
namespace convb {

constexpr int kThreads = 256;
constexpr int kB = act8::kBlk;  // tokens loaded at once
constexpr int kS = 8;             // tokens in registers at once, backward
constexpr int kMaxW = 8;

struct Params {
  const void* x;
  int8_t* codes;
  uint8_t* exps;
  const void* w;
  const void* bias;
  const void* dout;  // or, forward, out
  void* dx;
  float* part;  // [runs of all sequences][K + 1][dim], or NULL
  int64_t seqlen, dim, nruns, run;
  int64_t xs[2], ds[2], ws0, ws1;
  uint32_t ncb;  // workgroups of channels
  int32_t w_dtype, silu;
};

// Tokens of a run: 64 forward, 128 backward, where tokens done twice and partial sums are one in so many (8 x 2048 x
// 5120: 64 114 + 7 us with the sum, 128 107 + 4, 256 107 + 4), and fewer where that leaves the chip with less
// than 8 waves a CU.
static int64_t run_of(int64_t batch, int64_t seqlen, int64_t dim, bool backward) {
  int64_t run = backward ? 128 : 64;
  while (run > kB && batch * ceil_div(seqlen, run) * ceil_div(dim, 64) < 2048) run /= 2;
  return run;
}

__device__ __forceinline__ float ld_any(const void* p, int64_t i, int32_t dt) {
  return dt == MM_F32 ? ld<MM_F32>(p, i) : dt == MM_F16 ? ld<MM_F16>(p, i) : ld<MM_BF16>(p, i);
}
__device__ __forceinline__ void st_any(void* p, int64_t i, float v, int32_t dt) {
  if (dt == MM_F32) st<MM_F32>(p, i, v);
  else if (dt == MM_F16) st<MM_F16>(p, i, v);
  else st<MM_BF16>(p, i, v);
}

// The thread's channel and run.  Lanes past the last channel do what the last one's does.
struct Place {
  uint32_t d;
  int64_t row, b, t0, t1, nblk;
  __device__ __forceinline__ Place(const Params& p) {
    d = min((blockIdx.x % p.ncb) * kThreads + threadIdx.x, static_cast<uint32_t>(p.dim - 1));
    row = blockIdx.x / p.ncb;  // of all sequences' runs
    const uint32_t r = static_cast<uint32_t>(row), n = static_cast<uint32_t>(p.nruns);
    b = r / n;
    t0 = r % n * p.run;
    t1 = t0 + p.run < p.seqlen ? t0 + p.run : p.seqlen;
    nblk = (p.seqlen + kB - 1) / kB;
  }
};

// n tokens from t on; those past the sequence read its last one.
template <int DT, int n>
__device__ __forceinline__ void load_rows(float* v, const void* base, const int64_t* stride, int64_t b, int64_t t,
                                          int64_t seqlen, uint32_t off) {
  typename Ty<DT>::T raw[n > 0 ? n : 1];
  Rows<DT> in(base, stride, b, t);
  if (t + n <= seqlen) {
#pragma unroll
    for (int k = 0; k < n; ++k) {
      raw[k] = in.load(off);
      in.next();
    }
  } else {
#pragma unroll
    for (int k = 0; k < n; ++k) {
      raw[k] = in.load(off);
      in.next(t + k + 1 < seqlen);
    }
  }
#pragma unroll
  for (int k = 0; k < n; ++k) v[k] = Ty<DT>::f(raw[k]);
}

template <int DT, int K, bool C8>
__global__ __launch_bounds__(kThreads) void conv1d_bwd_kernel(const Params p) {
  using T = typename Ty<DT>::T;
  constexpr int H = K - 1;  // history
  const Place at(p);
  const uint32_t d = at.d, off = d * static_cast<uint32_t>(sizeof(T));
  const int64_t b = at.b;
  float w[K], dw[K];
  const float bias = p.bias ? ld_any(p.bias, d, p.w_dtype) : 0.0f;
  float db = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    w[k] = ld_any(p.w, d * p.ws0 + k * p.ws1, p.w_dtype);
    dw[k] = 0.0f;
  }
  using std::integral_constant;
  // Tokens t - H .. t + kS - 1: half a block at a time, for the registers (6 waves a SIMD at width 4, 4 at width 8).
  float x[H + kS], dp[H + kS];
#pragma unroll
  for (int k = 0; k < H; ++k) x[k] = dp[k] = 0.0f;
  act8::Block xc;  // the block of 16 tokens
  auto fetch = [&](int64_t t) __attribute__((always_inline)) {
    const int64_t o = (b * at.nblk + t / kB) * p.dim;
    xc.load(p.codes + o * kB, p.exps + o, d);
    xc.prepare();
  };
  if (H > 0 && at.t0 > 0) {
    if constexpr (C8) {
      fetch(at.t0 - kB);
#pragma unroll
      for (int k = 0; k < H; ++k) x[k] = xc.value(kB - H + k);
    } else {
      load_rows<DT, H>(x, p.x, p.xs, b, at.t0 - H, p.seqlen, off);
    }
  }
  // tokens t + k, k < n, from the block's token k0 on: p, dp, the sums (`own` tokens only) and dx of H tokens earlier
  auto tokens = [&](int64_t t, auto k0_c, auto n_c, auto own_c) __attribute__((always_inline)) {
    constexpr int k0 = decltype(k0_c)::value, n = decltype(n_c)::value;
    constexpr bool own = decltype(own_c)::value;
    float dy[n];
    load_rows<DT, n>(dy, p.dout, p.ds, b, t, p.seqlen, off);
    if constexpr (C8) {
#pragma unroll
      for (int k = 0; k < n; ++k) x[H + k] = xc.value(k0 + k);
    } else {
      load_rows<DT, n>(x + H, p.x, p.xs, b, t, p.seqlen, off);
    }
    Rows<DT> out(p.dx, b * p.seqlen + t - H, p.dim);
    auto walk = [&](auto whole_c) __attribute__((always_inline)) {
      constexpr bool whole = decltype(whole_c)::value;  // all tokens and their dx are the run's
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const bool in = whole || t + k < p.seqlen;
        float v = bias;
#pragma unroll
        for (int q = 0; q < K; ++q) v = __builtin_fmaf(w[q], x[k + q], v);
        float s = rcp_hw(1.0f + exp2_hw(-v * kLog2e));
        s *= __builtin_fmaf(v, 1.0f - s, 1.0f);  // silu'
        s = p.silu ? s : 1.0f;
        dp[H + k] = in ? dy[k] * s : 0.0f;
        if constexpr (own) {
          db += dp[H + k];
#pragma unroll
          for (int q = 0; q < K; ++q) dw[q] = __builtin_fmaf(dp[H + k], in ? x[k + q] : 0.0f, dw[q]);
        }
        const int64_t o = t + k - H;
        if (p.dx != nullptr && (whole || (o >= at.t0 && o < at.t1))) {
          float u = 0.0f;
#pragma unroll
          for (int q = 0; q < K; ++q) u = __builtin_fmaf(w[q], dp[H + k - q], u);
          T r, unused;
          round2<DT>(u, 0.0f, r, unused);
          out.store(off, r);
        }
        out.next();
      }
    };
    const bool whole = t - H >= at.t0 && t + n <= p.seqlen && t + n - H <= at.t1;
    if (whole) walk(std::true_type{});
    else walk(std::false_type{});
#pragma unroll
    for (int k = 0; k < H; ++k) x[k] = x[n + k], dp[k] = dp[n + k];
  };
  for (int64_t t = at.t0; t < at.t1; t += kB) {
    if constexpr (C8) fetch(t);
    tokens(t, integral_constant<int, 0>{}, integral_constant<int, kS>{}, std::true_type{});
    if (t + kS < at.t1) tokens(t + kS, integral_constant<int, kS>{}, integral_constant<int, kS>{}, std::true_type{});
  }
  // the last H tokens' dx: up to H tokens of the next run, or zeros
  if constexpr (H > 0) {
    const int64_t end = (at.t1 + kS - 1) / kS * kS;  // of the tokens walked
    if (p.dx != nullptr) {
      if (end < p.seqlen) {
        if constexpr (C8) fetch(end);
        tokens(end, integral_constant<int, 0>{}, integral_constant<int, H>{}, std::false_type{});
      } else {
        Rows<DT> out(p.dx, b * p.seqlen + end - H, p.dim);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const int64_t o = end + k - H;
          float u = 0.0f;
#pragma unroll
          for (int q = k + 1; q < K; ++q) u = __builtin_fmaf(w[q], dp[H + k - q], u);
          if (o >= at.t0 && o < at.t1) out.store(off, Ty<DT>::from(u));
          out.next();
        }
      }
    }
  }
  if (p.part != nullptr) {
    float* q = p.part + at.row * (K + 1) * p.dim;
#pragma unroll
    for (int k = 0; k < K; ++k) (q + k * p.dim)[d] = dw[k];
    (q + K * p.dim)[d] = db;
  }
}

// The forward pass with its input kept in 8 bits: x is read once for the outputs and the codes.  The outputs are
// mm_causal_conv1d_fwd's, bit for bit: the same multiply-adds in the same order.
template <int DT, int K>
__global__ __launch_bounds__(kThreads) void conv1d_fwd_act8_kernel(const Params p) {
  using T = typename Ty<DT>::T;
  constexpr int H = K - 1;
  const Place at(p);
  const uint32_t d = at.d, off = d * static_cast<uint32_t>(sizeof(T));
  float w[K];
  const float bias = p.bias ? ld_any(p.bias, d, p.w_dtype) : 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) w[k] = ld_any(p.w, d * p.ws0 + k * p.ws1, p.w_dtype);
  float x[H + kB];
#pragma unroll
  for (int k = 0; k < H; ++k) x[k] = 0.0f;
  if (H > 0 && at.t0 > 0) load_rows<DT, H>(x, p.x, p.xs, at.b, at.t0 - H, p.seqlen, off);
  for (int64_t t = at.t0; t < at.t1; t += kB) {
    load_rows<DT, kB>(x + H, p.x, p.xs, at.b, t, p.seqlen, off);
    float v[kB];
#pragma unroll
    for (int k = 0; k < kB; ++k) v[k] = t + k < p.seqlen ? x[H + k] : 0.0f;
    uint32_t e;
    const uint4 c = act8::pack16(v, e);
    const int64_t o = (at.b * at.nblk + t / kB) * p.dim;
    *reinterpret_cast<uint4*>(p.codes + o * kB + static_cast<uint64_t>(d) * kB) = c;
    (p.exps + o)[d] = static_cast<uint8_t>(e);
    Rows<DT> out(const_cast<void*>(p.dout), at.b * p.seqlen + t, p.dim);
#pragma unroll
    for (int k = 0; k < kB; k += 2) {
      float y[2];
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        float acc = bias;
#pragma unroll
        for (int q = 0; q < K; ++q) acc = __builtin_fmaf(w[q], x[k + c2 + q], acc);
        y[c2] = p.silu ? silu_f(acc) : acc;
      }
      T r[2];
      round2<DT>(y[0], y[1], r[0], r[1]);
#pragma unroll
      for (int c2 = 0; c2 < 2; ++c2) {
        if (t + k + c2 < p.seqlen) out.store(off, r[c2]);
        out.next();
      }
    }
#pragma unroll
    for (int k = 0; k < H; ++k) x[k] = x[kB + k];
  }
}

// dw[c, k] and dbias[c] from the runs' sums, rows of [K + 1][dim].
__global__ __launch_bounds__(64 * rows::kGroups) void reduce_kernel(const float* part, void* dw, void* dbias, int64_t nrows,
                                                                  int64_t dim, int width, int32_t w_dtype) {
  rows::sum_columns(part, nrows, (width + 1) * dim, blockIdx.x, 0, nrows, [&](int64_t c, double s) {
    const int64_t k = c / dim, d = c % dim;
    if (k < width) st_any(dw, d * width + k, static_cast<float>(s), w_dtype);
    else if (dbias != nullptr) st_any(dbias, d, static_cast<float>(s), w_dtype);
  });
}

static bool sizes_ok(int64_t batch, int64_t seqlen, int64_t dim) {
  return batch >= 0 && seqlen >= 0 && dim >= 0 && dim <= (int64_t{1} << 30) && seqlen <= (int64_t{1} << 40) &&
         (batch == 0 || dim == 0 || seqlen + 64 <= INT64_MAX / 256 / batch / (dim + kThreads));
}

// The checks and parameters that both entry points share.  x may be missing where there are codes.
static int prepare(Params& p, const void* x, const int8_t* codes, const uint8_t* exps, const void* weight, const void* bias,
                   const void* dout, int64_t batch, int64_t seqlen, int64_t dim, int64_t width, const int64_t x_stride[2],
                   const int64_t dout_stride[2], const int64_t w_stride[2], int32_t x_dtype, int32_t w_dtype,
                   int32_t apply_silu, bool backward) {
  if (batch < 0 || seqlen < 0 || dim < 0) return fail(MM_ERR_SHAPE, "negative size");
  if (width < 1 || width > kMaxW) return fail(MM_ERR_SHAPE, "width=%lld not in 1..%d", (long long)width, kMaxW);
  if (!sizes_ok(batch, seqlen, dim)) return fail(MM_ERR_SHAPE, "too many elements");
  if (!valid_dtype(x_dtype) || !valid_dtype(w_dtype)) return fail(MM_ERR_DTYPE, "bad dtype");
  if (batch == 0 || seqlen == 0 || dim == 0) return MM_OK;
  if (!x && (!codes || !exps)) return fail(MM_ERR_NULL_POINTER, "x, or x_codes and x_exps, are required");
  if (!codes != !exps) return fail(MM_ERR_NULL_POINTER, "codes and exps are given together");
  if ((x && !x_stride) || !weight || !w_stride || !dout || !dout_stride)
    return fail(MM_ERR_NULL_POINTER, "weight, the output's tensor and the strides are required");
  if ((x && (x_stride[0] < 0 || x_stride[1] < 0)) || dout_stride[0] < 0 || dout_stride[1] < 0 || w_stride[0] < 0 ||
      w_stride[1] < 0)
    return fail(MM_ERR_LAYOUT, "negative stride");
  if (!aligned(codes, kB)) return fail(MM_ERR_LAYOUT, "codes are not 16-byte aligned");
  p.x = x;
  p.codes = const_cast<int8_t*>(codes);
  p.exps = const_cast<uint8_t*>(exps);
  p.w = weight;
  p.bias = bias;
  p.dout = dout;
  p.seqlen = seqlen;
  p.dim = dim;
  p.run = run_of(batch, seqlen, dim, backward);
  p.nruns = ceil_div(seqlen, p.run);
  for (int k = 0; k < 2; ++k) p.xs[k] = x ? x_stride[k] : 0, p.ds[k] = dout_stride[k];
  p.ws0 = w_stride[0], p.ws1 = w_stride[1];
  p.ncb = static_cast<uint32_t>(ceil_div(dim, kThreads));
  p.w_dtype = w_dtype;
  p.silu = apply_silu != 0;
  if (batch * p.nruns > 0x7fffffff / static_cast<int64_t>(p.ncb)) return fail(MM_ERR_SHAPE, "too many elements");
  return MM_OK;
}

}  // namespace convb
}  // namespace mm

// One launch for each width of a kernel template F<DT, K, ...>.
#define MM_CONV_WIDTHS(LAUNCH, D) \
  switch (width) {                \
    case 1: LAUNCH(D, 1); break;  \
    case 2: LAUNCH(D, 2); break;  \
    case 3: LAUNCH(D, 3); break;  \
    case 4: LAUNCH(D, 4); break;  \
    case 5: LAUNCH(D, 5); break;  \
    case 6: LAUNCH(D, 6); break;  \
    case 7: LAUNCH(D, 7); break;  \
    default: LAUNCH(D, 8); break; \
  }
#define MM_CONV_DTYPES(LAUNCH)                        \
  switch (x_dtype) {                                  \
    case MM_F32: MM_CONV_WIDTHS(LAUNCH, MM_F32) break; \
    case MM_F16: MM_CONV_WIDTHS(LAUNCH, MM_F16) break; \
    default: MM_CONV_WIDTHS(LAUNCH, MM_BF16) break;    \
  }

extern "C" {

size_t mm_causal_conv1d_bwd_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int64_t width) {
  using namespace mm;
  using namespace mm::convb;
  if (!sizes_ok(batch, seqlen, dim) || width < 1 || width > kMaxW) return 0;
  return static_cast<size_t>(rows::floats(batch * ceil_div(seqlen, run_of(batch, seqlen, dim, true)), (width + 1) * dim) * 4);
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
  Params p{};
  int e = prepare(p, x, x ? nullptr : x_codes, x ? nullptr : x_exps, weight, bias, dout, batch, seqlen, dim, width, x_stride,
                  dout_stride, w_stride, x_dtype, w_dtype, apply_silu, true);
  if (e != MM_OK) return e;
  if (dbias && !dw) return fail(MM_ERR_NULL_POINTER, "dbias needs dw");
  if (dim == 0 || (!dx && !dw)) return MM_OK;
  const size_t need = dw ? mm_causal_conv1d_bwd_workspace_size(batch, seqlen, dim, width) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(MM_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
  if (need > 0 && !aligned(workspace, 256)) return fail(MM_ERR_WORKSPACE, "workspace is not 256-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  int64_t nrows = batch * p.nruns;
  if (nrows > 0) {
    p.dx = dx;
    p.part = dw ? static_cast<float*>(workspace) : nullptr;
    const dim3 grid(static_cast<unsigned>(p.ncb * nrows));
#define MM_CB(D, K)                                                                                  \
  if (x) hipLaunchKernelGGL((conv1d_bwd_kernel<D, K, false>), grid, dim3(kThreads), 0, s, p);         \
  else hipLaunchKernelGGL((conv1d_bwd_kernel<D, K, true>), grid, dim3(kThreads), 0, s, p)
    MM_CONV_DTYPES(MM_CB)
#undef MM_CB
    e = check_launch("causal_conv1d_bwd");
    if (e != MM_OK) return e;
  }
  if (!dw) return MM_OK;
  const int64_t cols = (width + 1) * dim;
  const float* part = rows::reduce_first(static_cast<float*>(workspace), nrows, cols, s);
  hipLaunchKernelGGL(reduce_kernel, dim3(static_cast<unsigned>(ceil_div(cols, 64))), dim3(64 * rows::kGroups), 0, s, part, dw,
                     dbias, nrows, dim, static_cast<int>(width), w_dtype);
  return check_launch("causal_conv1d_bwd_reduce");
}

int mm_causal_conv1d_fwd_act8(const void* x, const void* weight, const void* bias, void* out, int8_t* x_codes,
                              uint8_t* x_exps, int64_t batch, int64_t seqlen, int64_t dim, int64_t width,
                              const int64_t x_stride[2], const int64_t w_stride[2], int32_t x_dtype,
                              int32_t w_dtype, int32_t apply_silu, void* stream) {
  using namespace mm;
  using namespace mm::convb;
  clear_error();
  Params p{};
  const int64_t out_stride[2] = {0, 0};  // contiguous
  const int e = prepare(p, x, x_codes, x_exps, weight, bias, out, batch, seqlen, dim, width, x_stride, out_stride, w_stride,
                        x_dtype, w_dtype, apply_silu, false);
  if (e != MM_OK || batch == 0 || seqlen == 0 || dim == 0) return e;
  if (!x || !x_codes) return fail(MM_ERR_NULL_POINTER, "x, x_codes and x_exps are required");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(p.ncb * batch * p.nruns));
#define MM_CF(D, K) hipLaunchKernelGGL((conv1d_fwd_act8_kernel<D, K>), grid, dim3(kThreads), 0, s, p)
  MM_CONV_DTYPES(MM_CF)
#undef MM_CF
  return check_launch("causal_conv1d_fwd_act8");
}

}  // extern "C"
