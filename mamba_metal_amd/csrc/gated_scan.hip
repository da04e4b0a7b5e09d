// Gated linear recurrence with one state a channel: mm_gated_scan_fwd, _bwd and _step.
//
//   r = sigmoid(a_gate)  i = sigmoid(x_gate)  a = exp(A r)  h_t = a h_{t-1} + sqrt(1 - a^2) i x
//
// One pass over the data, whatever the shape.  A workgroup takes a tile of W x 16 tokens by 64 C channels
// (lane = C channels, wave = 16 tokens): it loads all of the tile at once, turns it into the pairs (a, b)
// of h = a h + b in registers, composes them to one pair a wave and, through LDS, one pair (P, Q) a tile and
// channel, gets the state h before its first token, and runs the recurrence again from there to the outputs:
// two multiply-adds a token and channel for time in parallel.  The state comes from the tiles before it in
// the same channels: a tile publishes (P, Q) as soon as it has them and its last state as soon as it
// knows it; a tile waits for the nearest kWindow - 1 tiles' pairs or states and the next one's state and
// folds them, first tile first.  The state after tile k is P_k h + Q_k by the same operation for whoever
// folds it, so results do not depend on who was there first.  Tiles are claimed from a counter, in order of
// time, so that what a tile waits for is always running or done.
//
// The backward pass is the same in reverse: dh_t = g_t + c, c <- a_t dh_t, with each wave's 16 states
// recomputed from the stored state before its first token.
#include <type_traits>

#include "act8.h"
#include "reduce_rows.h"

namespace mm {
namespace gscan {

constexpr int kBlk = MM_ACT8_BLOCK;  // tokens of a wave
constexpr int kMaxWaves = 16;        // of a forward tile
constexpr int kMaxWavesBwd = 8;      // of a backward tile
constexpr int kWindow = 16;          // tiles that a tile looks back at
constexpr int kStepThreads = 64;

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


// ------------------------------------------------------------------------------ C neighbouring channels
template <int DT, int C>
struct Ch {
  using T = typename Ty<DT>::T;
  typedef T V __attribute__((ext_vector_type(C)));
  __device__ static __forceinline__ V load(const T* p) { return *reinterpret_cast<const V*>(p); }
  __device__ static __forceinline__ void store(T* p, const float (&v)[C]) {
    V o;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = cvt<DT>(v[c]);
    *reinterpret_cast<V*>(p) = o;
  }
  template <int D>
  __device__ static __forceinline__ T cvt(float x) {
    if constexpr (D == MM_BF16) return __builtin_bit_cast(unsigned short, static_cast<__bf16>(x));  // v_cvt_pk_bf16_f32
    else return Ty<DT>::from(x);
  }
};

// ------------------------------------------------------------------------------ the tiles' hand-off
// Workspace: [control: ticket, error][a pair of words for each tile and channel].  A word is a float and a tag
// in one 64-bit access, so a reader that sees the tag has the value: no fence, no cache write-back.
constexpr int kControlBytes = 256;
constexpr uint32_t kPair = 1, kState = 2;  // tags: (P, Q) so far, the state after the tile

struct Handoff {
  uint32_t* control;       // [0] tickets, [1] an expired wait
  unsigned long long* word; // [tile][2: Q or state, P][64 C]
  uint64_t spin_ticks;
  int32_t* status;
};

__device__ __forceinline__ void publish(unsigned long long* w, float v, uint32_t tag) {
  __hip_atomic_store(w, static_cast<unsigned long long>(tag) << 32 | __float_as_uint(v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* w) {
  return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ bool peek_error(const Handoff& hd) {
  return __hip_atomic_load(&hd.control[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
}

// The tile's claim: tickets count tiles in order of their turn, all channels of a turn first.
struct Claim {
  uint32_t strip, turn;
};
__device__ __forceinline__ Claim claim(const Handoff& hd, uint32_t nstrips, uint32_t nturns) {
  __shared__ uint32_t s_ticket;
  uint32_t ticket = blockIdx.x;
  if (nturns > 1) {
    if (threadIdx.x == 0) s_ticket = atomicAdd(&hd.control[0], 1u);
    __syncthreads();
    ticket = __builtin_amdgcn_readfirstlane(s_ticket);
  }
  return {ticket % nstrips, ticket / nstrips};
}

// What wave w of `waves` does between its tile's composition and the state before the tile: wave 0 publishes
// the tile's pair, and the waves fetch the kWindow tiles before it into s_back[distance - 1], a pair, or a
// state with P = -1 (a product of decays is never negative).  The wait is bounded by wall-clock time and
// sets the status word if it expires, which is not expected: the tiles waited for are running or done.
template <int C>
__device__ __forceinline__ void look_back(const Handoff& hd, uint32_t turn, uint32_t strip, uint32_t nstrips, int wave,
                                          int waves, float2 (&s_back)[kWindow][64 * C]) {
  const int lane = threadIdx.x & 63;
  for (int j = wave; j < kWindow && static_cast<uint32_t>(j) < turn; j += waves) {
    const unsigned long long* w =
        hd.word + (static_cast<uint64_t>(turn - 1 - j) * nstrips + strip) * (2 * 64 * C) + lane * C;
    const bool last = j == kWindow - 1;  // this one's state is needed
    const uint64_t t_start = wall_clock64();
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float2 v = make_float2(-1.0f, 0.0f);
      for (;;) {
        const unsigned long long q = peek(w + c), pw = peek(w + 64 * C + c);
        const uint32_t tag = static_cast<uint32_t>(q >> 32);
        v.y = __uint_as_float(static_cast<uint32_t>(q));
        if (tag == kState) {
          v.x = -1.0f;
          break;
        }
        if (tag == kPair && !last && static_cast<uint32_t>(pw >> 32) == kPair) {
          v.x = __uint_as_float(static_cast<uint32_t>(pw));
          break;
        }
        // one expired wait of the call makes the others return at once
        if (wall_clock64() - t_start > hd.spin_ticks || peek_error(hd)) {
          __hip_atomic_store(&hd.control[1], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          if (hd.status != nullptr)
            __hip_atomic_fetch_or(hd.status, MM_SCAN_STATUS_HANDOFF_TIMEOUT, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          v = make_float2(-1.0f, 0.0f);
          break;
        }
        __builtin_amdgcn_s_sleep(1);
      }
      s_back[j][lane * C + c] = v;
    }
  }
}

__global__ __launch_bounds__(256) void clear_kernel(uint4* p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = make_uint4(0, 0, 0, 0);
}

struct Launch {
  mm_gated_scan_params p;
  Handoff hd;
  float* dA_part;
  uint32_t nstrips, nturns, ncb;  // strips of 64 C channels of a sequence, tiles of a strip, strips a sequence
  int32_t waves;
};

// ------------------------------------------------------------------------------ forward
template <int DT, int C, bool Z, bool P8>
__global__ __launch_bounds__(64 * kMaxWaves) void fwd_kernel(const Launch k) {
  using V = typename Ch<DT, C>::V;
  using T = typename Ty<DT>::T;
  constexpr int N = Z ? 4 : 3;
  __shared__ float2 s_pair[kMaxWaves][64 * C];
  __shared__ float2 s_back[kWindow][64 * C];
  const mm_gated_scan_params& p = k.p;
  const Claim cl = claim(k.hd, k.nstrips, k.nturns);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = cl.strip / k.ncb;
  const uint32_t d = (cl.strip % k.ncb) * (64 * C) + lane * C;
  const bool live = d < p.dim;           // with C = 2 dim is even
  const uint32_t dd = live ? d : 0;      // loads of the other lanes stay in bounds
  const int64_t len = length_of(p, b), nblk = (p.seqlen + kBlk - 1) / kBlk;
  const int64_t blk = static_cast<int64_t>(cl.turn) * k.waves + wave, t0 = blk * kBlk;
  const bool here = t0 < p.seqlen;       // the wave has tokens

  // pairs (a, b), and the gate's inputs for later
  float a[kBlk][C], bu[kBlk][C];
  V zr[Z ? kBlk : 1];
  float P[C], Q[C];
#pragma unroll
  for (int c = 0; c < C; ++c) P[c] = 1.0f, Q[c] = 0.0f;
  auto load_all = [&](auto full_c) __attribute__((always_inline)) {
    constexpr bool full = decltype(full_c)::value;
    const T* src[4] = {static_cast<const T*>(p.x) + b * p.x_stride[0], static_cast<const T*>(p.a_gate) + b * p.a_gate_stride[0],
                       static_cast<const T*>(p.x_gate) + b * p.x_gate_stride[0],
                       Z ? static_cast<const T*>(p.z) + b * p.z_stride[0] : nullptr};
    const int64_t st[4] = {p.x_stride[1], p.a_gate_stride[1], p.x_gate_stride[1], Z ? p.z_stride[1] : 0};
    V raw[N][kBlk];
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const int64_t tt = full || t0 + t < p.seqlen ? t0 + t : p.seqlen - 1;
#pragma unroll
      for (int j = 0; j < N; ++j) raw[j][t] = Ch<DT, C>::load(src[j] + tt * st[j] + dd);
    }
    if constexpr (!full) {
#pragma unroll
      for (int t = 0; t < kBlk; ++t)
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
          for (int c = 0; c < C; ++c) raw[j][t][c] = t0 + t < len ? raw[j][t][c] : static_cast<T>(0);
    }
    if constexpr (P8) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          uint32_t top = 0;
#pragma unroll
          for (int t = 0; t < kBlk; ++t) top = max(top, act8::abs_bits(Ty<DT>::f(raw[j][t][c])));
          const uint32_t e = act8::exponent_of(top);
          const float inv = act8::inv_scale(e);
          uint32_t w[kBlk / 4];
#pragma unroll
          for (int t = 0; t < kBlk; t += 4) w[t / 4] = act8::code4(Ty<DT>::f(raw[j][t][c]), Ty<DT>::f(raw[j][t + 1][c]),
                                                                    Ty<DT>::f(raw[j][t + 2][c]), Ty<DT>::f(raw[j][t + 3][c]), inv);
          if (live) {
            const int64_t o = (b * nblk + blk) * p.dim + d + c;
            *reinterpret_cast<uint4*>(p.codes[j] + o * kBlk) = make_uint4(w[0], w[1], w[2], w[3]);
            p.exps[j][o] = static_cast<uint8_t>(e);
          }
        }
      }
    }
    float A[C];
#pragma unroll
    for (int c = 0; c < C; ++c) A[c] = rate_of(p.A[dd + c]);
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float beta2;
        decay(A[c] * sigmoid_f(Ty<DT>::f(raw[1][t][c])), a[t][c], beta2);
        bu[t][c] = __builtin_amdgcn_sqrtf(beta2) * (sigmoid_f(Ty<DT>::f(raw[2][t][c])) * Ty<DT>::f(raw[0][t][c]));
        if constexpr (!full) {
          a[t][c] = t0 + t < len ? a[t][c] : 1.0f;
          bu[t][c] = t0 + t < len ? bu[t][c] : 0.0f;
        }
        P[c] *= a[t][c];
        Q[c] = __builtin_fmaf(a[t][c], Q[c], bu[t][c]);
      }
      if constexpr (Z) zr[t] = raw[3][t];
    }
  };
  const bool full = t0 + kBlk <= len;
  if (full) load_all(std::true_type{});
  else if (here && (P8 || t0 < len)) load_all(std::false_type{});

  // the state before the tile
  float h[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    s_pair[wave][lane * C + c] = make_float2(P[c], Q[c]);
    h[c] = 0.0f;
  }
  __syncthreads();
  float tp[C], tq[C];
#pragma unroll
  for (int c = 0; c < C; ++c) tp[c] = 1.0f, tq[c] = 0.0f;
  unsigned long long* const mine = k.hd.word + (static_cast<uint64_t>(cl.turn) * k.nstrips + cl.strip) * (2 * 64 * C) + lane * C;
  if (k.nturns > 1 && wave == 0) {
    for (int w = 0; w < k.waves; ++w) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float2 v = s_pair[w][lane * C + c];
        tp[c] *= v.x;
        tq[c] = __builtin_fmaf(v.x, tq[c], v.y);
      }
    }
    if (cl.turn > 0 && cl.turn + 1 < k.nturns) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        publish(mine + 64 * C + c, tp[c], kPair);
        publish(mine + c, tq[c], kPair);
      }
    }
  }
  if (cl.turn == 0) {
    if (p.h0 != nullptr) {
#pragma unroll
      for (int c = 0; c < C; ++c) h[c] = p.h0[b * p.dim + dd + c];
    }
  } else {
    look_back<C>(k.hd, cl.turn, cl.strip, k.nstrips, wave, k.waves, s_back);
    __syncthreads();
    const int far = cl.turn < kWindow ? static_cast<int>(cl.turn) : kWindow;
    for (int j = far - 1; j >= 0; --j) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float2 v = s_back[j][lane * C + c];
        h[c] = v.x < 0.0f ? v.y : __builtin_fmaf(v.x, h[c], v.y);
      }
    }
  }
  if (k.nturns > 1 && wave == 0 && cl.turn + 1 < k.nturns) {
#pragma unroll
    for (int c = 0; c < C; ++c) publish(mine + c, __builtin_fmaf(tp[c], h[c], tq[c]), kState);
  }
  // the state before the wave
  for (int w = 0; w < wave; ++w) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float2 v = s_pair[w][lane * C + c];
      h[c] = __builtin_fmaf(v.x, h[c], v.y);
    }
  }
  if (here && live && p.block_states != nullptr) {
    float* const o = p.block_states + (b * nblk + blk) * p.dim + d;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = h[c];
  }

  // the recurrence and the outputs
  T* const yb = static_cast<T*>(p.y) + b * p.y_stride[0];
  if (full) {
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      float y[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        h[c] = __builtin_fmaf(a[t][c], h[c], bu[t][c]);
        y[c] = Z ? h[c] * silu_f(Ty<DT>::f(zr[Z ? t : 0][c])) : h[c];
      }
      if (live) Ch<DT, C>::store(yb + (t0 + t) * p.y_stride[1] + d, y);
    }
  } else if (here) {
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const bool in = t0 + t < len;
      float y[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (in) h[c] = __builtin_fmaf(a[t][c], h[c], bu[t][c]);
        y[c] = Z ? h[c] * silu_f(Ty<DT>::f(zr[Z ? t : 0][c])) : h[c];
        y[c] = in ? y[c] : 0.0f;
      }
      if (live && t0 + t < p.seqlen) Ch<DT, C>::store(yb + (t0 + t) * p.y_stride[1] + d, y);
    }
  }
  // (by the wave of the last block: the state is y's last one, bit for bit)
  if (p.state_out != nullptr && live && blk == (nblk > 0 ? nblk - 1 : 0)) {
#pragma unroll
    for (int c = 0; c < C; ++c) p.state_out[b * p.dim + d + c] = h[c];
  }
}

// ------------------------------------------------------------------------------ backward
// Turn 0 is the last tile of a sequence.  Of a token, what needs dh is dh times a number that does not:
//   dx = dh c1, c1 = i beta            dx_gate = dh c2, c2 = beta u (1 - i)
//   da_gate = dh c3, c3 = f l (1 - r)  dA += dh c4, c4 = f r      with f = h_{t-1} a - u a^2 / beta
// so these four, a and g are all that is kept in registers over the wait.
template <int DT, bool Z, bool C8>
__global__ __launch_bounds__(64 * kMaxWavesBwd, 2) void bwd_kernel(const Launch k) {
  using T = typename Ty<DT>::T;
  constexpr int N = Z ? 4 : 3;
  __shared__ float2 s_pair[kMaxWavesBwd][64];
  __shared__ float2 s_back[kWindow][64];
  __shared__ float s_dA[kMaxWavesBwd][64];
  const mm_gated_scan_params& p = k.p;
  const Claim cl = claim(k.hd, k.nstrips, k.nturns);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = cl.strip / k.ncb;
  const uint32_t d = (cl.strip % k.ncb) * 64 + lane;
  const bool live = d < p.dim;
  const uint32_t dd = live ? d : 0;
  const int64_t len = length_of(p, b), nblk = (p.seqlen + kBlk - 1) / kBlk;
  const int64_t blk = static_cast<int64_t>(k.nturns - 1 - cl.turn) * k.waves + wave, t0 = blk * kBlk;
  const bool here = t0 < p.seqlen;
  const int64_t row = (b * p.seqlen + t0) * p.dim;  // of the gradients

  float a[kBlk], g[kBlk], c1[kBlk], c2[kBlk], c3[kBlk], c4[kBlk];
  float P = 1.0f, Q = 0.0f;
  auto load_all = [&](auto full_c) __attribute__((always_inline)) {
    constexpr bool full = decltype(full_c)::value;
    const T* src[5] = {};
    int64_t st[5] = {};
    src[4] = static_cast<const T*>(p.dy) + b * p.dy_stride[0];
    st[4] = p.dy_stride[1];
    uint4 code[C8 ? N : 1];
    float scale[C8 ? N : 1];
    T raw[C8 ? 1 : N][kBlk], dyr[kBlk];
    if constexpr (C8) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int64_t o = (b * nblk + blk) * p.dim + dd;
        code[j] = *reinterpret_cast<const uint4*>(p.codes[j] + o * kBlk);
        scale[j] = act8::scale_of(p.exps[j][o]);
      }
    } else {
      src[0] = static_cast<const T*>(p.x) + b * p.x_stride[0], st[0] = p.x_stride[1];
      src[1] = static_cast<const T*>(p.a_gate) + b * p.a_gate_stride[0], st[1] = p.a_gate_stride[1];
      src[2] = static_cast<const T*>(p.x_gate) + b * p.x_gate_stride[0], st[2] = p.x_gate_stride[1];
      if constexpr (Z) src[3] = static_cast<const T*>(p.z) + b * p.z_stride[0], st[3] = p.z_stride[1];
    }
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const int64_t tt = full || t0 + t < p.seqlen ? t0 + t : p.seqlen - 1;
      if constexpr (!C8) {
#pragma unroll
        for (int j = 0; j < N; ++j) raw[j][t] = src[j][tt * st[j] + dd];
      }
      dyr[t] = src[4][tt * st[4] + dd];
    }
    const float A = rate_of(p.A[dd]);
    float h = p.block_states[(b * nblk + blk) * p.dim + dd];
    auto value = [&](int j, int t) __attribute__((always_inline)) {
      float v;
      if constexpr (C8) v = act8::value_of(code[j], t, scale[j]);
      else v = Ty<DT>::f(raw[j][t]);
      return full || t0 + t < len ? v : 0.0f;
    };
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      const bool in = full || t0 + t < len;
      const float x = value(0, t), r = sigmoid_f(value(1, t)), i = sigmoid_f(value(2, t)), l = A * r;
      float beta2;
      decay(l, a[t], beta2);
      // 1 / beta, or 0 at a = 1, where the root has no slope (and where beta^2 is below the smallest normal
      // number, whose reciprocal root the instruction takes as infinite; a NaN stays one)
      const float ib = fabsf(beta2) < 1.17549435e-38f ? 0.0f : __builtin_amdgcn_rsqf(beta2);
      const float beta = beta2 * ib, u = i * x, hp = h;
      const float f = __builtin_fmaf(hp, a[t], -u * (a[t] * a[t] * ib));
      c1[t] = i * beta;
      c2[t] = beta * u * (1.0f - i);
      c3[t] = f * l * (1.0f - r);
      c4[t] = f * r;
      h = __builtin_fmaf(a[t], h, beta * u);
      g[t] = Ty<DT>::f(dyr[t]);
      if constexpr (Z) {
        const float z = value(3, t), s = sigmoid_f(z), zs = z * s;
        const float dz = g[t] * h * __builtin_fmaf(zs, 1.0f - s, s);
        if (live && (full || t0 + t < p.seqlen))
          static_cast<T*>(p.dz)[row + t * p.dim + d] = Ch<DT, 1>::template cvt<DT>(in ? dz : 0.0f);
        g[t] *= zs;
      }
      if constexpr (!full) {
        a[t] = in ? a[t] : 1.0f;
        h = in ? h : hp;
        g[t] = in ? g[t] : 0.0f;
        c1[t] = in ? c1[t] : 0.0f;
        c2[t] = in ? c2[t] : 0.0f;
        c3[t] = in ? c3[t] : 0.0f;
        c4[t] = in ? c4[t] : 0.0f;
      }
    }
#pragma unroll
    for (int t = kBlk - 1; t >= 0; --t) {
      P *= a[t];
      Q = a[t] * (Q + g[t]);
    }
  };
  const bool full = t0 + kBlk <= len, some = here && t0 < len;
  if (full) load_all(std::true_type{});
  else if (some) load_all(std::false_type{});

  s_pair[wave][lane] = make_float2(P, Q);
  __syncthreads();
  float tp = 1.0f, tq = 0.0f, carry = 0.0f;
  unsigned long long* const mine = k.hd.word + (static_cast<uint64_t>(cl.turn) * k.nstrips + cl.strip) * 128 + lane;
  if (k.nturns > 1 && wave == 0) {
    for (int w = k.waves - 1; w >= 0; --w) {
      const float2 v = s_pair[w][lane];
      tp *= v.x;
      tq = __builtin_fmaf(v.x, tq, v.y);
    }
    if (cl.turn > 0 && cl.turn + 1 < k.nturns) {
      publish(mine + 64, tp, kPair);
      publish(mine, tq, kPair);
    }
  }
  if (cl.turn == 0) {
    if (p.dstate != nullptr) carry = p.dstate[b * p.dim + dd];
  } else {
    look_back<1>(k.hd, cl.turn, cl.strip, k.nstrips, wave, k.waves, s_back);
    __syncthreads();
    const int far = cl.turn < kWindow ? static_cast<int>(cl.turn) : kWindow;
    for (int j = far - 1; j >= 0; --j) {
      const float2 v = s_back[j][lane];
      carry = v.x < 0.0f ? v.y : __builtin_fmaf(v.x, carry, v.y);
    }
  }
  if (k.nturns > 1 && wave == 0 && cl.turn + 1 < k.nturns) publish(mine, __builtin_fmaf(tp, carry, tq), kState);
  for (int w = k.waves - 1; w > wave; --w) {
    const float2 v = s_pair[w][lane];
    carry = __builtin_fmaf(v.x, carry, v.y);
  }

  float dA = 0.0f;
  T* const dx = static_cast<T*>(p.dx) + row;
  T* const da = static_cast<T*>(p.da_gate) + row;
  T* const dg = static_cast<T*>(p.dx_gate) + row;
  auto out = [&](int t, float v1, float v2, float v3) __attribute__((always_inline)) {
    dx[t * p.dim + d] = Ch<DT, 1>::template cvt<DT>(v1);
    dg[t * p.dim + d] = Ch<DT, 1>::template cvt<DT>(v2);
    da[t * p.dim + d] = Ch<DT, 1>::template cvt<DT>(v3);
  };
  if (some) {
#pragma unroll
    for (int t = kBlk - 1; t >= 0; --t) {
      const float dh = g[t] + carry;
      carry = full || t0 + t < len ? a[t] * dh : carry;
      dA = __builtin_fmaf(dh, c4[t], dA);
      if (live && (full || t0 + t < p.seqlen)) {
        const bool in = full || t0 + t < len;  // (0 times an infinite dh is not 0)
        out(t, in ? dh * c1[t] : 0.0f, in ? dh * c2[t] : 0.0f, in ? dh * c3[t] : 0.0f);
      }
    }
  } else if (here && live) {
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      if (t0 + t >= p.seqlen) break;
      out(t, 0.0f, 0.0f, 0.0f);
      if constexpr (Z) static_cast<T*>(p.dz)[row + t * p.dim + d] = Ch<DT, 1>::template cvt<DT>(0.0f);
    }
  }
  if (p.dh0 != nullptr && live && cl.turn + 1 == k.nturns && wave == 0) p.dh0[b * p.dim + d] = carry;
  s_dA[wave][lane] = dA;
  __syncthreads();
  if (wave == 0 && live) {
    for (int w = 1; w < k.waves; ++w) dA += s_dA[w][lane];
    k.dA_part[(b * k.nturns + cl.turn) * p.dim + d] = dA;
  }
}

__global__ __launch_bounds__(64 * rows::kGroups) void dA_kernel(const float* part, float* dA, int64_t nrows, int64_t dim) {
  rows::sum_columns(part, nrows, dim, nrows, [&](int64_t c, double s) { dA[c] = static_cast<float>(s); });
}

template <int DT>
__global__ __launch_bounds__(kStepThreads) void step_kernel(const float* state, float* state_out, const void* x,
                                                        const void* a_gate, const void* x_gate, const float* A,
                                                        const void* z, void* y, int64_t dim, int64_t xs,
                                                        int64_t as, int64_t gs, int64_t zs, int64_t ys) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kStepThreads + threadIdx.x, b = blockIdx.y;
  if (d >= dim) return;
  float a, beta2;
  decay(rate_of(A[d]) * sigmoid_f(ld<DT>(a_gate, b * as + d)), a, beta2);
  const float u = sigmoid_f(ld<DT>(x_gate, b * gs + d)) * ld<DT>(x, b * xs + d);
  const float h = __builtin_fmaf(a, state[b * dim + d], __builtin_sqrtf(beta2) * u);
  state_out[b * dim + d] = h;
  st<DT>(y, b * ys + d, z ? h * silu_f(ld<DT>(z, b * zs + d)) : h);
}

#ifndef TW
#define TW 8
#define TWB 8
#define MM_C2 0
#endif
constexpr int kTileWaves = TW, kTileWavesBwd = TWB;         // of the tiles of longer sequences
constexpr int kMaxBatch = 65535;  // grid y

// Sizes whose products below stay within 64 bits: the element count, times what a workspace takes of each.
static bool sizes_ok(int64_t batch, int64_t seqlen, int64_t dim) {
  return batch <= kMaxBatch && dim <= (int64_t{1} << 30) && seqlen <= (int64_t{1} << 40) &&
         (batch == 0 || dim == 0 || seqlen + 1024 <= INT64_MAX / 4096 / batch / (dim + 128));
}
static int check_sizes(int64_t batch, int64_t seqlen, int64_t dim) {
  if (batch < 0 || seqlen < 0 || dim < 0) return fail(MM_ERR_SHAPE, "negative size");
  if (batch > kMaxBatch) return fail(MM_ERR_SHAPE, "batch=%lld exceeds %d", (long long)batch, kMaxBatch);
  if (!sizes_ok(batch, seqlen, dim)) return fail(MM_ERR_SHAPE, "too many elements");
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
    if (!aligned(p->codes[k], kBlk)) return fail(MM_ERR_LAYOUT, "codes are not 16-byte aligned");
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


// ------------------------------------------------------------------------------ shapes of a call
struct Shape {
  int waves;
  int64_t ncb, nstrips, nturns, handoff_bytes;
};
// C channels a lane.  Sequences of up to `most` blocks of 16 tokens are one tile: no hand-off, one launch.
static Shape shape_of(int64_t batch, int64_t seqlen, int64_t dim, int C, bool backward) {
  const int most = backward ? kMaxWavesBwd : kMaxWaves;
  const int64_t nblk = ceil_div(seqlen > 0 ? seqlen : 1, kBlk);
  Shape s;
  s.waves = nblk <= most ? static_cast<int>(nblk) : backward ? kTileWavesBwd : kTileWaves;
  s.ncb = ceil_div(dim, 64 * C);
  s.nstrips = batch * s.ncb;
  s.nturns = ceil_div(nblk, s.waves);
  s.handoff_bytes = s.nturns > 1 ? kControlBytes + s.nturns * s.nstrips * (2 * 64 * C * 8) : 0;
  return s;
}
static int64_t dA_bytes(const Shape& s, int64_t batch, int64_t dim) { return round_up(rows::floats(batch * s.nturns, dim) * 4, 256); }

static int prepare(Launch& k, const mm_gated_scan_params* p, const Shape& s, char* handoff, hipStream_t stream) {
  if (s.nstrips * s.nturns > 0x7fffffff) return fail(MM_ERR_SHAPE, "too many elements");
  k.p = *p;
  k.hd.control = reinterpret_cast<uint32_t*>(handoff);
  k.hd.word = reinterpret_cast<unsigned long long*>(handoff + kControlBytes);
  k.hd.status = p->status;
  if (s.nturns > 1) {
    static DeviceCache cache;
    const int khz = device_cached(
        cache,
        [] {
          int dev = 0, v = 0;
          return hipGetDevice(&dev) == hipSuccess &&
                         hipDeviceGetAttribute(&v, hipDeviceAttributeWallClockRate, dev) == hipSuccess
                     ? v
                     : 0;
        },
        100000);
    const int64_t us = p->handoff_timeout_us > 0 ? p->handoff_timeout_us : 2000000;
    k.hd.spin_ticks = static_cast<uint64_t>(us) * khz / 1000;
    const int64_t n = s.handoff_bytes / 16;
    hipLaunchKernelGGL(clear_kernel, dim3(static_cast<unsigned>(ceil_div(n, 256))), dim3(256), 0, stream,
                       reinterpret_cast<uint4*>(handoff), n);
  }
  k.nstrips = static_cast<uint32_t>(s.nstrips);
  k.nturns = static_cast<uint32_t>(s.nturns);
  k.ncb = static_cast<uint32_t>(s.ncb);
  k.waves = s.waves;
  return MM_OK;
}

// Whether lanes may take two neighbouring channels: pairs of them are aligned in every tensor.
static bool pairs_ok(const mm_gated_scan_params* p) {
  const int64_t vb = 2 * dtype_size(p->dtype);
  const void* ptr[5] = {p->x, p->a_gate, p->x_gate, p->z, p->y};
  const int64_t* st[5] = {p->x_stride, p->a_gate_stride, p->x_gate_stride, p->z_stride, p->y_stride};
  if (p->dim % 2 != 0) return false;
  for (int k = 0; k < 5; ++k)
    if (ptr[k] && (!aligned(ptr[k], vb) || st[k][0] % 2 != 0 || st[k][1] % 2 != 0)) return false;
  return true;
}

}  // namespace gscan
}  // namespace mm

extern "C" {

size_t mm_gated_scan_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int32_t backward) {
  using namespace mm::gscan;
  if (batch <= 0 || seqlen < 0 || dim <= 0 || !sizes_ok(batch, seqlen, dim)) return 0;
  const Shape s = shape_of(batch, seqlen, dim, 1, backward != 0);
  if (backward) return static_cast<size_t>(dA_bytes(s, batch, dim) + s.handoff_bytes);
  const Shape s2 = shape_of(batch, seqlen, dim, 2, false);
  return static_cast<size_t>(s2.handoff_bytes > s.handoff_bytes ? s2.handoff_bytes : s.handoff_bytes);
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int C = pairs_ok(p) && MM_C2 ? 2 : 1;
  const Shape s = shape_of(p->batch, p->seqlen, p->dim, C, false);
  Launch k{};
  if ((e = prepare(k, p, s, static_cast<char*>(p->workspace), st)) != MM_OK) return e;
  const dim3 grid(static_cast<unsigned>(s.nstrips * s.nturns)), block(64 * s.waves);
  const bool p8 = p->codes[0] != nullptr && p->seqlen > 0;
#define MM_GS1(D, C, Z, P8) hipLaunchKernelGGL((fwd_kernel<D, C, Z, P8>), grid, block, 0, st, k)
#define MM_GS2(D, C, Z) \
  if (p8) MM_GS1(D, C, Z, true); else MM_GS1(D, C, Z, false)
#define MM_GS3(D, C) \
  if (p->z) { MM_GS2(D, C, true); } else { MM_GS2(D, C, false); }
#define MM_GS(D) \
  if (C == 2) { MM_GS3(D, 2) } else { MM_GS3(D, 1) }
  switch (p->dtype) {
    case MM_F32: MM_GS(MM_F32); break;
    case MM_F16: MM_GS(MM_F16); break;
    default: MM_GS(MM_BF16); break;
  }
#undef MM_GS
#undef MM_GS3
#undef MM_GS2
#undef MM_GS1
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
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Shape s = shape_of(p->batch, p->seqlen, p->dim, 1, true);
  Launch k{};
  k.dA_part = static_cast<float*>(p->workspace);
  if ((e = prepare(k, p, s, static_cast<char*>(p->workspace) + dA_bytes(s, p->batch, p->dim), st)) != MM_OK) return e;
  const dim3 grid(static_cast<unsigned>(s.nstrips * s.nturns)), block(64 * s.waves);
#define MM_GS1(D, Z, C) hipLaunchKernelGGL((bwd_kernel<D, Z, C>), grid, block, 0, st, k)
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
  int64_t nrows = p->batch * s.nturns;
  const float* part = rows::reduce_first(k.dA_part, nrows, p->dim, st);
  hipLaunchKernelGGL(dA_kernel, dim3(static_cast<unsigned>(ceil_div(p->dim, 64))), dim3(64 * rows::kGroups), 0, st, part, p->dA,
                     nrows, p->dim);
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
  const dim3 grid(static_cast<unsigned>(ceil_div(dim, kStepThreads)), static_cast<unsigned>(batch));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define MM_GS(D)                                                                                       \
  hipLaunchKernelGGL((step_kernel<D>), grid, dim3(kStepThreads), 0, s, state, state_out, x, a_gate, x_gate, A, \
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
