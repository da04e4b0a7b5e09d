// Gated linear recurrence with one state a channel: mm_gated_scan_fwd, _bwd and _step.
//
//   r = sigmoid(a_gate)  i = sigmoid(x_gate)  a = exp(A r)  h_t = a h_{t-1} + sqrt(1 - a^2) i x
//
// Simple form: one thread per (batch, channel) walks the sequence.
#include "act8.h"

namespace mm {
namespace gscan {

constexpr int kThreads = 64;
constexpr int kBlk = MM_ACT8_BLOCK;

__device__ __forceinline__ float sigmoid_f(float x) { return rcp_hw(1.0f + exp2_hw(-x * kLog2e)); }

// a = exp(l) and beta^2 = 1 - a^2 for l = A r <= 0.  Next to a = 1 both come from q = 1 - a, taken from its
// series -l (1 + l/2 + l^2/6 + ... + l^5/720) (the first dropped term is 5e-8 of q at l = -1/4): 1 - a^2 keeps
// its precision, and a's rounding leans to no side, where the hardware exponential's would add up over the
// thousands of tokens that such a channel remembers.  Below, q >= 0.22 is 1 - a to a few 1e-7.
__device__ __forceinline__ void decay(float l, float& a, float& beta2) {
  float s = 1.0f / 720.0f;
  s = __builtin_fmaf(s, l, 1.0f / 120.0f);
  s = __builtin_fmaf(s, l, 1.0f / 24.0f);
  s = __builtin_fmaf(s, l, 1.0f / 6.0f);
  s = __builtin_fmaf(s, l, 0.5f);
  s = __builtin_fmaf(s, l, 1.0f);
  const float e = exp2_hw(l * kLog2e);
  const bool near = l > -0.25f;
  const float q = near ? -l * s : 1.0f - e;
  a = near ? 1.0f - q : e;
  beta2 = q * (1.0f + a);
}
// A as the kernels use it: A r stays finite at A = -inf (a = 0 all the same, and 0 * l = 0), a NaN stays.
__device__ __forceinline__ float rate_of(float A) { return A < -3.4028235e38f ? -3.4028235e38f : A; }

__device__ __forceinline__ int64_t length_of(const mm_gated_scan_params& p, int64_t b) {
  if (p.lengths == nullptr) return p.seqlen;
  const int64_t n = p.lengths_dtype ? static_cast<const int64_t*>(p.lengths)[b]
                                    : static_cast<const int32_t*>(p.lengths)[b];
  return n < 0 ? 0 : n > p.seqlen ? p.seqlen : n;
}

template <int DT, bool Z>
__global__ __launch_bounds__(kThreads) void fwd_kernel(const mm_gated_scan_params p) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, b = blockIdx.y;
  if (d >= p.dim) return;
  const int64_t len = length_of(p, b), nblk = (p.seqlen + kBlk - 1) / kBlk;
  const float A = rate_of(p.A[d]);
  float h = p.h0 ? p.h0[b * p.dim + d] : 0.0f;
  for (int64_t t0 = 0; t0 < p.seqlen; t0 += kBlk) {
    if (p.block_states) p.block_states[(b * nblk + t0 / kBlk) * p.dim + d] = h;
    float raw[4][kBlk];
#pragma unroll
    for (int k = 0; k < kBlk; ++k) {
      const int64_t t = t0 + k < p.seqlen ? t0 + k : p.seqlen - 1;
      const bool in = t0 + k < len;
      raw[0][k] = ld<DT>(p.x, b * p.x_stride[0] + t * p.x_stride[1] + d);
      raw[1][k] = ld<DT>(p.a_gate, b * p.a_gate_stride[0] + t * p.a_gate_stride[1] + d);
      raw[2][k] = ld<DT>(p.x_gate, b * p.x_gate_stride[0] + t * p.x_gate_stride[1] + d);
      raw[3][k] = Z ? ld<DT>(p.z, b * p.z_stride[0] + t * p.z_stride[1] + d) : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j][k] = in ? raw[j][k] : 0.0f;
    }
    if (p.codes[0]) {
#pragma unroll
      for (int j = 0; j < (Z ? 4 : 3); ++j) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kBlk; ++k) top = max(top, act8::abs_bits(raw[j][k]));
        const uint32_t e = act8::exponent_of(top);
        p.exps[j][(b * nblk + t0 / kBlk) * p.dim + d] = static_cast<uint8_t>(e);
#pragma unroll
        for (int k = 0; k < kBlk; ++k)
          if (t0 + k < p.seqlen)
            p.codes[j][(b * p.seqlen + t0 + k) * p.dim + d] = act8::code_of(raw[j][k], act8::inv_scale(e));
      }
    }
#pragma unroll
    for (int k = 0; k < kBlk; ++k) {
      const bool in = t0 + k < len;
      float a, beta2;
      decay(A * sigmoid_f(raw[1][k]), a, beta2);
      const float bu = __builtin_sqrtf(beta2) * sigmoid_f(raw[2][k]) * raw[0][k];
      h = in ? __builtin_fmaf(a, h, bu) : h;
      const float y = Z ? h * silu_f(raw[3][k]) : h;
      if (t0 + k < p.seqlen) st<DT>(p.y, b * p.y_stride[0] + (t0 + k) * p.y_stride[1] + d, in ? y : 0.0f);
    }
  }
  if (p.state_out) p.state_out[b * p.dim + d] = h;
}

template <int DT, bool Z, bool C8>
__global__ __launch_bounds__(kThreads) void bwd_kernel(const mm_gated_scan_params p, float* dA_part) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, b = blockIdx.y;
  if (d >= p.dim) return;
  const int64_t len = length_of(p, b), nblk = (p.seqlen + kBlk - 1) / kBlk;
  const float A = rate_of(p.A[d]);
  float carry = p.dstate ? p.dstate[b * p.dim + d] : 0.0f, dA = 0.0f;
  for (int64_t t0 = (nblk - 1) * kBlk; t0 >= 0; t0 -= kBlk) {
    float raw[4][kBlk], dy[kBlk], hp[kBlk];
    float scale[4] = {};
    if constexpr (C8) {
#pragma unroll
      for (int j = 0; j < (Z ? 4 : 3); ++j)
        scale[j] = act8::scale_of(p.exps[j][(b * nblk + t0 / kBlk) * p.dim + d]);
    }
#pragma unroll
    for (int k = 0; k < kBlk; ++k) {
      const int64_t t = t0 + k < p.seqlen ? t0 + k : p.seqlen - 1;
      const bool in = t0 + k < len;
      if constexpr (C8) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          raw[j][k] = j < (Z ? 4 : 3) ? scale[j] * p.codes[j][(b * p.seqlen + t) * p.dim + d] : 0.0f;
      } else {
        raw[0][k] = ld<DT>(p.x, b * p.x_stride[0] + t * p.x_stride[1] + d);
        raw[1][k] = ld<DT>(p.a_gate, b * p.a_gate_stride[0] + t * p.a_gate_stride[1] + d);
        raw[2][k] = ld<DT>(p.x_gate, b * p.x_gate_stride[0] + t * p.x_gate_stride[1] + d);
        raw[3][k] = Z ? ld<DT>(p.z, b * p.z_stride[0] + t * p.z_stride[1] + d) : 0.0f;
      }
      dy[k] = ld<DT>(p.dy, b * p.dy_stride[0] + t * p.dy_stride[1] + d);
      dy[k] = in ? dy[k] : 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[j][k] = in ? raw[j][k] : 0.0f;
    }
    float h = p.block_states[(b * nblk + t0 / kBlk) * p.dim + d];
#pragma unroll
    for (int k = 0; k < kBlk; ++k) {
      hp[k] = h;
      float a, beta2;
      decay(A * sigmoid_f(raw[1][k]), a, beta2);
      h = __builtin_fmaf(a, h, __builtin_sqrtf(beta2) * sigmoid_f(raw[2][k]) * raw[0][k]);
    }
#pragma unroll
    for (int k = kBlk - 1; k >= 0; --k) {
      const bool in = t0 + k < len;
      const float r = sigmoid_f(raw[1][k]), i = sigmoid_f(raw[2][k]), l = A * r;
      float a, beta2;
      decay(l, a, beta2);
      const float beta = __builtin_sqrtf(beta2), u = i * raw[0][k];
      float g = dy[k], dz = 0.0f;
      if constexpr (Z) {
        const float s = sigmoid_f(raw[3][k]), zs = raw[3][k] * s;
        dz = g * __builtin_fmaf(a, hp[k], beta * u) * (s + zs * (1.0f - s));
        g *= zs;
      }
      const float dh = g + carry;
      const float ratio = beta2 == 0.0f ? 0.0f : a * a / beta;
      const float dl = dh * (hp[k] * a - u * ratio), du = dh * beta;
      if (t0 + k < p.seqlen) {
        const int64_t o = (b * p.seqlen + t0 + k) * p.dim + d;
        st<DT>(p.dx, o, in ? du * i : 0.0f);
        st<DT>(p.da_gate, o, in ? dl * l * (1.0f - r) : 0.0f);
        st<DT>(p.dx_gate, o, in ? du * u * (1.0f - i) : 0.0f);
        if constexpr (Z) st<DT>(p.dz, o, in ? dz : 0.0f);
      }
      dA += in ? dl * r : 0.0f;
      carry = in ? a * dh : carry;
    }
  }
  if (p.dh0) p.dh0[b * p.dim + d] = carry;
  dA_part[b * p.dim + d] = dA;
}

__global__ __launch_bounds__(kThreads) void dA_kernel(const float* part, float* dA, int64_t rows, int64_t dim) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (d >= dim) return;
  double s = 0.0;
  for (int64_t k = 0; k < rows; ++k) s += part[k * dim + d];
  dA[d] = static_cast<float>(s);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void step_kernel(const float* state, float* state_out, const void* x,
                                                        const void* a_gate, const void* x_gate, const float* A,
                                                        const void* z, void* y, int64_t dim, int64_t xs,
                                                        int64_t as, int64_t gs, int64_t zs, int64_t ys) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, b = blockIdx.y;
  if (d >= dim) return;
  float a, beta2;
  decay(rate_of(A[d]) * sigmoid_f(ld<DT>(a_gate, b * as + d)), a, beta2);
  const float u = sigmoid_f(ld<DT>(x_gate, b * gs + d)) * ld<DT>(x, b * xs + d);
  const float h = __builtin_fmaf(a, state[b * dim + d], __builtin_sqrtf(beta2) * u);
  state_out[b * dim + d] = h;
  st<DT>(y, b * ys + d, z ? h * silu_f(ld<DT>(z, b * zs + d)) : h);
}

constexpr int kMaxBatch = 65535;  // grid y

static int check_sizes(int64_t batch, int64_t seqlen, int64_t dim) {
  if (batch < 0 || seqlen < 0 || dim < 0) return fail(MM_ERR_SHAPE, "negative size");
  if (batch > kMaxBatch) return fail(MM_ERR_SHAPE, "batch=%lld exceeds %d", (long long)batch, kMaxBatch);
  if (dim > (int64_t{1} << 30) || seqlen > (int64_t{1} << 40) ||
      (dim > 0 && seqlen > 0 && batch > INT64_MAX / 64 / dim / seqlen))
    return fail(MM_ERR_SHAPE, "too many elements");
  return MM_OK;
}

static int check_strides(const int64_t* s, const char* name) {
  if (s[0] < 0 || s[1] < 0) return fail(MM_ERR_LAYOUT, "%s has a negative stride", name);
  return MM_OK;
}

static int check_common(const mm_gated_scan_params* p) {
  if (!p) return fail(MM_ERR_NULL_POINTER, "params is NULL");
  int e = check_sizes(p->batch, p->seqlen, p->dim);
  if (e != MM_OK) return e;
  if (!valid_dtype(p->dtype)) return fail(MM_ERR_DTYPE, "dtype=%d", p->dtype);
  if (p->lengths && p->lengths_dtype != 0 && p->lengths_dtype != 1)
    return fail(MM_ERR_DTYPE, "lengths_dtype=%d", p->lengths_dtype);
  if (p->handoff_timeout_us < 0)
    return fail(MM_ERR_SHAPE, "handoff_timeout_us=%d is negative", p->handoff_timeout_us);
  return MM_OK;
}

// The four inputs (the last may be missing), as tensors or as codes.
static int check_inputs(const mm_gated_scan_params* p, bool tensors, bool z) {
  const void* in[4] = {p->x, p->a_gate, p->x_gate, p->z};
  const int64_t* st[4] = {p->x_stride, p->a_gate_stride, p->x_gate_stride, p->z_stride};
  static const char* const name[4] = {"x", "a_gate", "x_gate", "z"};
  if (!p->A) return fail(MM_ERR_NULL_POINTER, "A is required");
  for (int k = 0; k < (z ? 4 : 3); ++k) {
    if (tensors && !in[k]) return fail(MM_ERR_NULL_POINTER, "%s is required", name[k]);
    if (tensors) {
      const int e = check_strides(st[k], name[k]);
      if (e != MM_OK) return e;
    }
    if (!p->codes[k] != !p->exps[k] || !p->codes[k] != !p->codes[0])
      return fail(MM_ERR_NULL_POINTER, "codes and exps are given for every input or for none");
  }
  return MM_OK;
}

static int check_workspace(const mm_gated_scan_params* p, size_t need) {
  if (need == 0) return MM_OK;
  if (!p->workspace || p->workspace_bytes < need)
    return fail(MM_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need,
                p->workspace ? p->workspace_bytes : size_t{0});
  if (!aligned(p->workspace, 256)) return fail(MM_ERR_WORKSPACE, "workspace is not 256-byte aligned");
  return MM_OK;
}

}  // namespace gscan
}  // namespace mm

extern "C" {

size_t mm_gated_scan_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int32_t backward) {
  using namespace mm::gscan;
  if (batch <= 0 || seqlen < 0 || dim <= 0 || batch > kMaxBatch || !backward) return 0;
  return static_cast<size_t>(batch * dim * 4);
}

int mm_gated_scan_fwd(const mm_gated_scan_params* p, void* stream) {
  using namespace mm;
  using namespace mm::gscan;
  clear_error();
  int e = check_common(p);
  if (e != MM_OK || p->batch == 0 || p->dim == 0) return e;
  if (p->seqlen > 0) {
    if ((e = check_inputs(p, true, p->z != nullptr)) != MM_OK) return e;
    if (!p->y) return fail(MM_ERR_NULL_POINTER, "y is required");
    if ((e = check_strides(p->y_stride, "y")) != MM_OK) return e;
  } else if (!p->A) {
    return fail(MM_ERR_NULL_POINTER, "A is required");
  }
  if ((e = check_workspace(p, mm_gated_scan_workspace_size(p->batch, p->seqlen, p->dim, 0))) != MM_OK) return e;
  const dim3 grid(static_cast<unsigned>(ceil_div(p->dim, kThreads)), static_cast<unsigned>(p->batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_GS(D)                                                                            \
  if (p->z) hipLaunchKernelGGL((fwd_kernel<D, true>), grid, dim3(kThreads), 0, s, *p);      \
  else hipLaunchKernelGGL((fwd_kernel<D, false>), grid, dim3(kThreads), 0, s, *p)
  switch (p->dtype) {
    case MM_F32: MM_GS(MM_F32); break;
    case MM_F16: MM_GS(MM_F16); break;
    default: MM_GS(MM_BF16); break;
  }
#undef MM_GS
  return check_launch("gated_scan_fwd");
}

int mm_gated_scan_bwd(const mm_gated_scan_params* p, void* stream) {
  using namespace mm;
  using namespace mm::gscan;
  clear_error();
  int e = check_common(p);
  if (e != MM_OK || p->batch == 0 || p->dim == 0) return e;
  const bool c8 = p->codes[0] != nullptr, z = c8 ? p->z_present != 0 : p->z != nullptr;
  if (!p->dA) return fail(MM_ERR_NULL_POINTER, "dA is required");
  if (p->seqlen > 0) {
    if ((e = check_inputs(p, !c8, z)) != MM_OK) return e;
    if (!p->dy || !p->block_states) return fail(MM_ERR_NULL_POINTER, "dy and block_states are required");
    if (!p->dx || !p->da_gate || !p->dx_gate || (z && !p->dz))
      return fail(MM_ERR_NULL_POINTER, "dx, da_gate, dx_gate (and dz with z) are required");
    if ((e = check_strides(p->dy_stride, "dy")) != MM_OK) return e;
  } else if (!p->A) {
    return fail(MM_ERR_NULL_POINTER, "A is required");
  }
  if ((e = check_workspace(p, mm_gated_scan_workspace_size(p->batch, p->seqlen, p->dim, 1))) != MM_OK) return e;
  const dim3 grid(static_cast<unsigned>(ceil_div(p->dim, kThreads)), static_cast<unsigned>(p->batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(p->workspace);
#define MM_GS1(D, Z, C) hipLaunchKernelGGL((bwd_kernel<D, Z, C>), grid, dim3(kThreads), 0, s, *p, part)
#define MM_GS(D)                                            \
  if (c8) {                                                 \
    if (z) MM_GS1(D, true, true); else MM_GS1(D, false, true);   \
  } else {                                                  \
    if (z) MM_GS1(D, true, false); else MM_GS1(D, false, false); \
  }
  switch (p->dtype) {
    case MM_F32: MM_GS(MM_F32); break;
    case MM_F16: MM_GS(MM_F16); break;
    default: MM_GS(MM_BF16); break;
  }
#undef MM_GS
#undef MM_GS1
  e = check_launch("gated_scan_bwd");
  if (e != MM_OK) return e;
  hipLaunchKernelGGL(dA_kernel, dim3(grid.x), dim3(kThreads), 0, s, part, p->dA, p->batch, p->dim);
  return check_launch("gated_scan_dA");
}

int mm_gated_scan_step(const float* state, float* state_out, const void* x, const void* a_gate,
                       const void* x_gate, const float* A, const void* z, void* y, int64_t batch,
                       int64_t dim, int64_t x_stride_b, int64_t a_gate_stride_b,
                       int64_t x_gate_stride_b, int64_t z_stride_b, int64_t y_stride_b,
                       int32_t dtype, void* stream) {
  using namespace mm;
  using namespace mm::gscan;
  clear_error();
  int e = check_sizes(batch, 1, dim);
  if (e != MM_OK) return e;
  if (!valid_dtype(dtype)) return fail(MM_ERR_DTYPE, "dtype=%d", dtype);
  if (batch == 0 || dim == 0) return MM_OK;
  if (!state || !state_out || !x || !a_gate || !x_gate || !A || !y)
    return fail(MM_ERR_NULL_POINTER, "state, state_out, x, a_gate, x_gate, A and y are required");
  if (x_stride_b < 0 || a_gate_stride_b < 0 || x_gate_stride_b < 0 || (z && z_stride_b < 0) || y_stride_b < 0)
    return fail(MM_ERR_LAYOUT, "negative stride");
  const dim3 grid(static_cast<unsigned>(ceil_div(dim, kThreads)), static_cast<unsigned>(batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_GS(D)                                                                                       \
  hipLaunchKernelGGL((step_kernel<D>), grid, dim3(kThreads), 0, s, state, state_out, x, a_gate, x_gate, A, \
                     z, y, dim, x_stride_b, a_gate_stride_b, x_gate_stride_b, z_stride_b, y_stride_b)
  switch (dtype) {
    case MM_F32: MM_GS(MM_F32); break;
    case MM_F16: MM_GS(MM_F16); break;
    default: MM_GS(MM_BF16); break;
  }
#undef MM_GS
  return check_launch("gated_scan_step");
}

}  // extern "C"
