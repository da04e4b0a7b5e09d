// Gated linear recurrence with one state a channel: mm_gated_scan_fwd, _bwd and _step.
//
//   r = sigmoid(a_gate)  i = sigmoid(x_gate)  a = exp(A r)  h_t = a h_{t-1} + sqrt(1 - a^2) i x
//
// One pass over the data, whatever the shape.  A workgroup takes a tile of W x 16 tokens by 64 channels
// (lane = channel, wave = 16 tokens): it loads all of the tile at once, turns it into the pairs (a, b)
// of h = a h + b in registers, composes them to one pair a wave and, through LDS, one pair (P, Q) a tile and
// channel, gets the state h before its first token, and has every token's state as a product and a sum of its own: two
// multiply-adds a token and channel for time in parallel.  The state comes from the tiles before it in
// the same channels: a tile publishes (P, Q) as soon as it has them and its last state as soon as it
// knows it; a tile waits for the nearest kWindow - 1 tiles' pairs or states and the next one's state and
// folds them, first tile first.  The state after tile k is P_k h + Q_k by the same operation for whoever
// folds it, so results do not depend on who was there first.  Workgroups claim the tiles of their strip of
// channels from its counter, in order of time, so that what a tile waits for is always running or done.
//
// The backward pass is the same in reverse: dh_t = g_t + c, c <- a_t dh_t, with each wave's 16 states
// recomputed from the stored state before its first token.
//
// Bound by memory, then by vector instructions (51 an element forward with the output gate, 78 backward).  bf16 with
// the output gate, us in passes one after another: forward 1 x 8192 x 5120 110 (3.8 TB/s; 4.99 is what a large copy
// reaches; without the wait for the states before a tile 98), 8 x 2048 x 5120 forward 240 and backward 343 (3.6 and 4.5
// TB/s), 4 x 8192 x 5120 with 8-bit checkpoints 548 and 562 (4.4 and 4.3 TB/s).
#include <type_traits>

#include "act8.h"
#include "gated_tiles.h"
#include "reduce_rows.h"
#include "row_io.h"

namespace mm {
namespace gscan {

constexpr int kWindow = 16;          // tiles that a tile looks back at
constexpr int kStepThreads = 64;

__device__ __forceinline__ float sigmoid_f(float x) { return rcp_hw(1.0f + exp2_hw(-x * kLog2e)); }

// a = exp(l) and beta^2 = 1 - a^2 for l = A r <= 0.  Next to a = 1 both come from q = 1 - a, taken from its
// series -l (1 + l/2 + l^2/6 + ...): 1 - a^2 keeps its precision, and a's rounding leans to no side, where the
// hardware exponential's would add up over the thousands of tokens that such a channel remembers.  fp32: from
// l = -1/4 on, to l^5/720 (the first dropped term is 5e-8 of q there; below, 1 - a is good to a few 1e-7).
// 16-bit types: from l = -1/16 on, to l^3/24 (1e-7; below, 1 - a is good to 2e-6, a 2000th of bf16's half step, a
// 250th of fp16's), two multiply-adds less.
template <int DT>
__device__ __forceinline__ void decay(float l, float& a, float& beta2) {
  constexpr bool wide = DT == MM_F32;
  float s = wide ? 1.0f / 720.0f : 1.0f / 24.0f;
  if constexpr (wide) {
    s = __builtin_fmaf(s, l, 1.0f / 120.0f);
    s = __builtin_fmaf(s, l, 1.0f / 24.0f);
  }
  s = __builtin_fmaf(s, l, 1.0f / 6.0f);
  s = __builtin_fmaf(s, l, 0.5f);
  s = __builtin_fmaf(s, l, 1.0f);
  const float e = exp2_hw(l * kLog2e);
  const bool near = l > (wide ? -0.25f : -0.0625f);
  const float q_near = -l * s, q_far = 1.0f - e;  // (both by name: as operands of ?: they became branches)
  const float q = near ? q_near : q_far;
  const float a_near = 1.0f - q;
  a = near ? a_near : e;
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

// ------------------------------------------------------------------------------ the tiles' hand-off
// Workspace: [control: an expired wait, then each strip's next turn, a line each][a word for each tile and channel].
// One counter for all tiles bounded the forward pass at about 25 ns a tile.  A word is the pair (P, Q), or (-1, the
// state after the tile): a product of decays is never negative.  It is one 64-bit access, so a reader has both or
// neither: no fence, no cache write-back.  All zeros is a word that is not there yet, and a P of 0 is written as -0.
struct Handoff {
  uint32_t* control;
  unsigned long long* word; // [tile][64]
  uint64_t spin_ticks;
  int32_t* status;
};

__device__ __forceinline__ void publish(unsigned long long* w, float p, float q) {
  __hip_atomic_store(w, static_cast<unsigned long long>(__float_as_uint(p)) << 32 | __float_as_uint(q), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long peek(const unsigned long long* w) {
  return __hip_atomic_load(w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool peek_error(const Handoff& hd) {
  return __hip_atomic_load(&hd.control[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
}

// The tile's claim: the workgroup's strip, its turn in time the next of its strip.
struct Claim {
  uint32_t strip, turn;
};
__device__ __forceinline__ bool claim(const Handoff& hd, const Spread& sp, Claim& cl) {
  __shared__ uint32_t s_turn;
  cl.turn = 0;
  cl.strip = blockIdx.x % sp.nstrips;
  if (sp.per_die) {
    const uint32_t j = blockIdx.x / kDies, s = place_of(blockIdx.x % kDies, j, sp);
    if (s >= sp.span) return false;
    cl.strip = span_of(j, sp) + s;
  }
  if (sp.nturns > 1) {
    if (threadIdx.x == 0) s_turn = atomicAdd(&hd.control[(1 + cl.strip) * (kControlBytes / 4)], 1u);
    __syncthreads();
    cl.turn = __builtin_amdgcn_readfirstlane(s_turn);
  }
  return true;
}

// f of the lane's pairs v[lo] .. v[hi - 1], or in reverse, eight LDS reads in flight at a time.
__device__ __forceinline__ float2 lane_pair(const float2 (*v)[64], int j) { return v[j][threadIdx.x & 63]; }
template <bool BACK, typename F>
__device__ __forceinline__ void each_pair(const float2 (*v)[64], int lo, int hi, F f) {  // lo .. hi - 1, or hi - 1 .. lo
  for (int j0 = 0; j0 < hi - lo; j0 += 8) {
    float2 q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int j = j0 + k < hi - lo ? j0 + k : 0;
      q[k] = lane_pair(v, BACK ? hi - 1 - j : lo + j);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (j0 + k < hi - lo) f(q[k]);
  }
}

// What a wave does between its tile's composition and the state before the tile: the waves fetch the kWindow tiles
// before it into s_back[distance - 1], a pair or a state (P = -1).  A wave's tiles are polled together, so that it
// takes one round trip where all are there.  The wait is bounded by wall-clock time and sets the status word if it
// expires, which is not expected: the tiles waited for are running or done.  At least kMinWaves waves.
constexpr int kMinWaves = 4, kPolls = kWindow / kMinWaves;
constexpr uint64_t kLongWait = 10000;  // ticks, 100 us
__device__ __forceinline__ void look_back(const Handoff& hd, uint32_t turn, uint32_t strip, uint32_t nstrips, int wave,
                                          int waves, float2 (&s_back)[kWindow][64]) {
  const int lane = threadIdx.x & 63;
  const unsigned long long* w[kPolls];
  unsigned long long q[kPolls];
  bool need[kPolls];
#pragma unroll
  for (int k = 0; k < kPolls; ++k) {
    const int j = wave + k * waves;
    need[k] = j < kWindow && static_cast<uint32_t>(j) < turn;
    w[k] = hd.word + (static_cast<uint64_t>(need[k] ? turn - 1 - j : turn) * nstrips + strip) * 64 + lane;
  }
  const uint64_t t_start = wall_clock64();
  for (;;) {
#pragma unroll
    for (int k = 0; k < kPolls; ++k)
      if (need[k]) q[k] = peek(w[k]);
    bool again = false;
#pragma unroll
    for (int k = 0; k < kPolls; ++k) {
      if (!need[k]) continue;
      const int j = wave + k * waves;
      const float pk = __uint_as_float(static_cast<uint32_t>(q[k] >> 32));
      // the farthest tile's state is needed, of the others the pair will do
      if (__all(j == kWindow - 1 ? pk < 0.0f : q[k] >> 32 != 0)) {
        s_back[j][lane] = make_float2(pk, __uint_as_float(static_cast<uint32_t>(q[k])));
        need[k] = false;
      } else {
        again = true;
      }
    }
    if (!again) break;
    // one expired wait of the call makes the others return soon (a look at its word is another round trip, so only
    // a wait that is already long takes it)
    const uint64_t waited = wall_clock64() - t_start;
    if (waited > hd.spin_ticks || (waited > kLongWait && peek_error(hd))) {
      __hip_atomic_store(&hd.control[0], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (hd.status != nullptr)
        __hip_atomic_fetch_or(hd.status, MM_SCAN_STATUS_HANDOFF_TIMEOUT, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int k = 0; k < kPolls; ++k)
        if (need[k]) s_back[wave + k * waves][lane] = make_float2(-1.0f, 0.0f);
      break;
    }
    __builtin_amdgcn_s_sleep(1);
  }
}
// The state before the tile from what look_back fetched, first tile first.
__device__ __forceinline__ float fold_back(uint32_t turn, const float2 (&s_back)[kWindow][64]) {
  float h = 0.0f;
  each_pair<true>(s_back, 0, turn < kWindow ? static_cast<int>(turn) : kWindow, [&](const float2& v) __attribute__((always_inline)) {
    const float joined = __builtin_fmaf(v.x, h, v.y);
    h = v.x < 0.0f ? v.y : joined;
  });
  return h;
}

__global__ __launch_bounds__(256) void clear_kernel(uint4* p, int64_t n) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) p[i] = make_uint4(0, 0, 0, 0);
}

struct Launch {
  mm_gated_scan_params p;
  Handoff hd;
  float* dA_part;
  Spread spread;
  uint32_t nstrips, nturns, ncb;  // strips of 64 channels of a sequence, tiles of a strip, strips a sequence
  int32_t waves;
};

// ------------------------------------------------------------------------------ forward
// A token's state is h_t = E_t h + H_t for the state h before the wave, E and H the products and sums so far: E, H
// and the gate's input are what is kept in registers over the wait.
template <int DT, bool Z, bool P8>
__global__ __launch_bounds__(64 * kMaxWaves) void fwd_kernel(const Launch k) {
  using T = typename Ty<DT>::T;
  constexpr int N = Z ? 4 : 3;
  __shared__ float2 s_pair[kMaxWaves][64];
  __shared__ float2 s_back[kWindow][64];
  const mm_gated_scan_params& p = k.p;
  Claim cl;
  if (!claim(k.hd, k.spread, cl)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = cl.strip / k.ncb;
  // lanes past the last channel do what the last one's does, stores and all
  const uint32_t d = min((cl.strip % k.ncb) * 64 + lane, static_cast<uint32_t>(p.dim - 1));
  const uint32_t off = d * static_cast<uint32_t>(sizeof(T));
  const int64_t len = length_of(p, b), nblk = (p.seqlen + kBlk - 1) / kBlk;
  const int64_t blk = static_cast<int64_t>(cl.turn) * k.waves + wave, t0 = blk * kBlk;
  const bool here = t0 < p.seqlen;  // the wave has tokens

  float E[kBlk], H[kBlk];
  T zr[Z ? kBlk : 1];
  float P = 1.0f, Q = 0.0f;
  auto load_all = [&](auto full_c) __attribute__((always_inline)) {
    constexpr bool full = decltype(full_c)::value;
    Rows<DT> in[4] = {{p.x, p.x_stride, b, t0}, {p.a_gate, p.a_gate_stride, b, t0}, {p.x_gate, p.x_gate_stride, b, t0},
                      {Z ? p.z : p.x, Z ? p.z_stride : p.x_stride, b, t0}};
    T raw[N][kBlk];
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        raw[j][t] = in[j].load(off);
        in[j].next(full || t0 + t + 1 < p.seqlen);
      }
    }
    const float A = rate_of(p.A[d]);
    if constexpr (!full) {
#pragma unroll
      for (int t = 0; t < kBlk; ++t)
#pragma unroll
        for (int j = 0; j < N; ++j) raw[j][t] = t0 + t < len ? raw[j][t] : static_cast<T>(0);
    }
    if constexpr (P8) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float v[kBlk];
#pragma unroll
        for (int t = 0; t < kBlk; ++t) v[t] = Ty<DT>::f(raw[j][t]);
        uint32_t e;
        const uint4 w = act8::pack16(v, e);
        const int64_t o = (b * nblk + blk) * p.dim;
        *reinterpret_cast<uint4*>(p.codes[j] + o * kBlk + static_cast<uint64_t>(d) * kBlk) = w;
        (p.exps[j] + o)[d] = static_cast<uint8_t>(e);
      }
    }
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      float a, beta2;
      decay<DT>(A * sigmoid_f(Ty<DT>::f(raw[1][t])), a, beta2);
      float bu = __builtin_amdgcn_sqrtf(beta2) * (sigmoid_f(Ty<DT>::f(raw[2][t])) * Ty<DT>::f(raw[0][t]));
      if constexpr (!full) {
        a = t0 + t < len ? a : 1.0f;
        bu = t0 + t < len ? bu : 0.0f;
      }
      P *= a;
      Q = __builtin_fmaf(a, Q, bu);
      keep(P);
      keep(Q);
      E[t] = P;
      H[t] = Q;
      if constexpr (Z) zr[t] = raw[3][t];
    }
  };
  const bool full = t0 + kBlk <= len, some = here && (P8 || t0 < len);
  if (full) load_all(std::true_type{});
  else if (some) load_all(std::false_type{});

  // The state before the tile, and before the wave.  A tile past the sequence's end has none to pass on: the tiles
  // after it are past it too, and the final state is written where the last token is.
  float h = 0.0f;
  const bool past = cl.turn > 0 && static_cast<int64_t>(cl.turn) * k.waves * kBlk >= len;
  if (!past) {
    if (k.waves > 1) {
      s_pair[wave][lane] = make_float2(P, Q);
      __syncthreads();
    }
    float tp = 1.0f, tq = 0.0f;
    unsigned long long* const mine = k.hd.word + (static_cast<uint64_t>(cl.turn) * k.nstrips + cl.strip) * 64 + lane;
    const bool more = cl.turn + 1 < k.nturns;
    if (more && wave == 0) {
      each_pair<false>(s_pair, 0, k.waves, [&](const float2& v) __attribute__((always_inline)) {
        tp *= v.x;
        tq = __builtin_fmaf(v.x, tq, v.y);
      });
      tp = tp == 0.0f ? -0.0f : tp;
      if (cl.turn > 0) publish(mine, tp, tq);
    }
    if (cl.turn == 0) {
      if (p.h0 != nullptr) h = p.h0[b * p.dim + d];
    } else {
      look_back(k.hd, cl.turn, cl.strip, k.nstrips, wave, k.waves, s_back);
      __syncthreads();
      h = fold_back(cl.turn, s_back);
    }
    if (more && wave == 0) publish(mine, -1.0f, __builtin_fmaf(tp, h, tq));
    each_pair<false>(s_pair, 0, wave, [&](const float2& v) __attribute__((always_inline)) { h = __builtin_fmaf(v.x, h, v.y); });
  }
  if (here && p.block_states != nullptr) (p.block_states + (b * nblk + blk) * p.dim)[d] = h;

  float last = h;
  auto finish = [&](auto full_c) __attribute__((always_inline)) {
    constexpr bool full = decltype(full_c)::value;
    Rows<DT> out(p.y, p.y_stride, b, t0);
#pragma unroll
    for (int t = 0; t < kBlk; t += 2) {
      float y[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = full || t0 + t + c < len;
        last = in ? __builtin_fmaf(E[t + c], h, H[t + c]) : last;
        y[c] = last;
        if constexpr (Z) {
          const float z = Ty<DT>::f(zr[t + c]);
          y[c] *= z * sigmoid_f(z);
        }
        y[c] = in ? y[c] : 0.0f;
      }
      T v[2];
      round2<DT>(y[0], y[1], v[0], v[1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (full || t0 + t + c < p.seqlen) out.store(off, v[c]);
        out.next();
      }
    }
  };
  if (full) {
    finish(std::true_type{});
  } else if (here) {
    if (!some) {
#pragma unroll
      for (int t = 0; t < kBlk; ++t) {
        E[t] = H[t] = 0.0f;
        if constexpr (Z) zr[t] = static_cast<T>(0);
      }
    }
    finish(std::false_type{});
  }
  // (by the wave of the last token: the state is that token's, bit for bit)
  if (p.state_out != nullptr && blk == (len > 0 ? (len - 1) / kBlk : 0)) p.state_out[b * p.dim + d] = last;
}

// ------------------------------------------------------------------------------ backward
// Turn 0 is the last tile of a sequence.  With c what comes from the tokens after the wave, dh_t = E_t c + G_t, E
// and G the products and sums of the recurrence in reverse.  What needs dh is dh times a number that does not:
//   dx = dh c1, c1 = i beta    dx_gate = dh c2, c2 = beta u (1 - i)    da_gate = dh c3, c3 = f l (1 - r)
// with f = h_{t-1} a - u a^2 / beta, and dA is c (sum of E f r) + (sum of G f r): five numbers a token and two more
// are all that is kept in registers over the wait.
template <int DT, bool Z, bool C8>
__global__ __launch_bounds__(64 * kMaxWavesBwd, 4) void bwd_kernel(const Launch k) {
  using T = typename Ty<DT>::T;
  constexpr int N = Z ? 4 : 3;
  __shared__ float2 s_pair[kMaxWavesBwd][64];
  __shared__ float2 s_back[kWindow][64];
  // A lane's own f r, and c3 of the first 12 tokens: 28 registers less, which 4 waves a SIMD do not have
  __shared__ float4 s_c4[kMaxWavesBwd][kBlk / 4][64], s_c3[kMaxWavesBwd][3][64];
  __shared__ float s_dA[kMaxWavesBwd][64];
  const mm_gated_scan_params& p = k.p;
  Claim cl;
  if (!claim(k.hd, k.spread, cl)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t b = cl.strip / k.ncb;
  const uint32_t d = min((cl.strip % k.ncb) * 64 + lane, static_cast<uint32_t>(p.dim - 1));
  const uint32_t off = d * static_cast<uint32_t>(sizeof(T));
  const int64_t len = length_of(p, b), nblk = (p.seqlen + kBlk - 1) / kBlk;
  const int64_t blk = static_cast<int64_t>(k.nturns - 1 - cl.turn) * k.waves + wave, t0 = blk * kBlk;
  const bool here = t0 < p.seqlen;
  const int64_t row = b * p.seqlen + t0;  // of the gradients

  float E[kBlk], G[kBlk], c1[kBlk], c2[kBlk], c3[kBlk];
  float P = 1.0f, Q = 0.0f, dA_c = 0.0f, dA_0 = 0.0f;
  auto load_all = [&](auto full_c) __attribute__((always_inline)) {
    constexpr bool full = decltype(full_c)::value;
    act8::Block code[C8 ? N : 1];
    T raw[C8 ? 1 : N][kBlk], dyr[kBlk];
    Rows<DT> dyp(p.dy, p.dy_stride, b, t0);
    if constexpr (C8) {
      const int64_t o = (b * nblk + blk) * p.dim;
#pragma unroll
      for (int j = 0; j < N; ++j) code[j].load(p.codes[j] + o * kBlk, p.exps[j] + o, d);
    } else {
      Rows<DT> in[4] = {{p.x, p.x_stride, b, t0}, {p.a_gate, p.a_gate_stride, b, t0}, {p.x_gate, p.x_gate_stride, b, t0},
                        {Z ? p.z : p.x, Z ? p.z_stride : p.x_stride, b, t0}};
#pragma unroll
      for (int t = 0; t < kBlk; ++t)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          raw[j][t] = in[j].load(off);
          in[j].next(full || t0 + t + 1 < p.seqlen);
        }
    }
#pragma unroll
    for (int t = 0; t < kBlk; ++t) {
      dyr[t] = dyp.load(off);
      dyp.next(full || t0 + t + 1 < p.seqlen);
    }
    const float A = rate_of(p.A[d]);
    float h = (p.block_states + (b * nblk + blk) * p.dim)[d];
    if constexpr (C8) {
#pragma unroll
      for (int j = 0; j < N; ++j) code[j].prepare();
    }
    auto value = [&](int j, int t) __attribute__((always_inline)) {
      float v;
      if constexpr (C8) v = code[j].value(t);
      else v = Ty<DT>::f(raw[j][t]);
      return full || t0 + t < len ? v : 0.0f;
    };
    float a[kBlk], c4[4];
    Rows<DT> dzp(p.dz, row, p.dim);
#pragma unroll
    for (int t = 0; t < kBlk; t += 2) {
      float dz[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int tt = t + c;
        const bool in = full || t0 + tt < len;
        const float x = value(0, tt), r = sigmoid_f(value(1, tt)), i = sigmoid_f(value(2, tt)), l = A * r;
        float beta2;
        decay<DT>(l, a[tt], beta2);
        // 1 / beta, or 0 at a = 1, where the root has no slope (and where beta^2 is below the smallest normal
        // number, whose reciprocal root the instruction takes as infinite; a NaN stays one)
        const float root = __builtin_amdgcn_rsqf(beta2);
        const float ib = fabsf(beta2) < 1.17549435e-38f ? 0.0f : root;
        const float beta = beta2 * ib, u = i * x, bu = beta * u;
        const float f = __builtin_fmaf(h, a[tt], -u * (a[tt] * a[tt] * ib));
        c1[tt] = i * beta;
        c2[tt] = __builtin_fmaf(-bu, i, bu);
        c4[tt % 4] = f * r;
        c3[tt] = f * __builtin_fmaf(-l, r, l);
        const float hn = __builtin_fmaf(a[tt], h, bu);
        h = in ? hn : h;
        G[tt] = Ty<DT>::f(dyr[tt]);
        if constexpr (Z) {
          const float z = value(3, tt), s = sigmoid_f(z), zs = z * s;
          dz[c] = in ? G[tt] * h * __builtin_fmaf(zs, 1.0f - s, s) : 0.0f;
          G[tt] *= zs;
        }
        if constexpr (!full) {
          a[tt] = in ? a[tt] : 1.0f;
          G[tt] = in ? G[tt] : 0.0f;
          c1[tt] = in ? c1[tt] : 0.0f;
          c2[tt] = in ? c2[tt] : 0.0f;
          c3[tt] = in ? c3[tt] : 0.0f;
          c4[tt % 4] = in ? c4[tt % 4] : 0.0f;
        }
      }
      if constexpr (Z) {
        T v[2];
        round2<DT>(dz[0], dz[1], v[0], v[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (full || t0 + t + c < p.seqlen) dzp.store(off, v[c]);
          dzp.next();
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        keep(c1[t + c]);
        keep(c2[t + c]);
        if (t >= 12) keep(c3[t + c]);
      }
      if (t % 4 == 2) {
        s_c4[wave][t / 4][lane] = make_float4(c4[0], c4[1], c4[2], c4[3]);
        if (t < 12) s_c3[wave][t / 4][lane] = make_float4(c3[t - 2], c3[t - 1], c3[t], c3[t + 1]);
      }
    }
    float4 q4[kBlk / 4];
#pragma unroll
    for (int t = 0; t < kBlk / 4; ++t) q4[t] = s_c4[wave][t][lane];
#pragma unroll
    for (int t = kBlk - 1; t >= 0; --t) {
      E[t] = P;
      G[t] += Q;
      const float4 q = q4[t / 4];
      const float c = t % 4 == 0 ? q.x : t % 4 == 1 ? q.y : t % 4 == 2 ? q.z : q.w;
      dA_c = __builtin_fmaf(P, c, dA_c);
      dA_0 = __builtin_fmaf(G[t], c, dA_0);
      P *= a[t];
      Q = a[t] * G[t];
    }
  };
  const bool full = t0 + kBlk <= len, some = here && t0 < len;
  if (full) load_all(std::true_type{});
  else if (some) load_all(std::false_type{});

  // what comes from the tokens after the tile, and after the wave: past the sequence's end just dstate
  float carry = 0.0f;
  const bool past = static_cast<int64_t>(k.nturns - 1 - cl.turn) * k.waves * kBlk >= len;
  if ((past || cl.turn == 0) && p.dstate != nullptr) carry = p.dstate[b * p.dim + d];
  if (!past && k.waves > 1) {
    s_pair[wave][lane] = make_float2(P, Q);
    __syncthreads();
  }
  float tp = 1.0f, tq = 0.0f;
  unsigned long long* const mine = k.hd.word + (static_cast<uint64_t>(cl.turn) * k.nstrips + cl.strip) * 64 + lane;
  const bool more = cl.turn + 1 < k.nturns;
  if (past) {
    if (more && wave == 0) publish(mine, -1.0f, carry);
  } else {
    if (more && wave == 0) {
      each_pair<true>(s_pair, 0, k.waves, [&](const float2& v) __attribute__((always_inline)) {
        tp *= v.x;
        tq = __builtin_fmaf(v.x, tq, v.y);
      });
      tp = tp == 0.0f ? -0.0f : tp;
      if (cl.turn > 0) publish(mine, tp, tq);
    }
    if (cl.turn > 0) {
      look_back(k.hd, cl.turn, cl.strip, k.nstrips, wave, k.waves, s_back);
      __syncthreads();
      carry = fold_back(cl.turn, s_back);
    }
    if (more && wave == 0) publish(mine, -1.0f, __builtin_fmaf(tp, carry, tq));
    each_pair<true>(s_pair, wave + 1, k.waves, [&](const float2& v) __attribute__((always_inline)) { carry = __builtin_fmaf(v.x, carry, v.y); });
  }

  auto finish = [&](auto full_c) __attribute__((always_inline)) {
    constexpr bool full = decltype(full_c)::value;
    Rows<DT> o[3] = {{p.dx, row, p.dim}, {p.dx_gate, row, p.dim}, {p.da_gate, row, p.dim}};
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      const float4 q = s_c3[wave][t][lane];
      c3[4 * t] = q.x, c3[4 * t + 1] = q.y, c3[4 * t + 2] = q.z, c3[4 * t + 3] = q.w;
    }
#pragma unroll
    for (int t = 0; t < kBlk; t += 2) {
      float v[3][2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool in = full || t0 + t + c < len;  // (0 times an infinite dh is not 0)
        const float dh = __builtin_fmaf(E[t + c], carry, G[t + c]);
        v[0][c] = in ? dh * c1[t + c] : 0.0f;
        v[1][c] = in ? dh * c2[t + c] : 0.0f;
        v[2][c] = in ? dh * c3[t + c] : 0.0f;
      }
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        T w[2];
        round2<DT>(v[j][0], v[j][1], w[0], w[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (full || t0 + t + c < p.seqlen) o[j].store(off, w[c]);
          o[j].next();
        }
      }
    }
  };
  if (full) {
    finish(std::true_type{});
  } else if (some) {
    finish(std::false_type{});
  } else if (here) {
    Rows<DT> o[4] = {{p.dx, row, p.dim}, {p.dx_gate, row, p.dim}, {p.da_gate, row, p.dim}, {Z ? p.dz : p.dx, row, p.dim}};
    for (int64_t t = t0; t < t0 + kBlk && t < p.seqlen; ++t) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        o[j].store(off, static_cast<T>(0));
        o[j].next();
      }
    }
  }
  const float dA = some ? __builtin_fmaf(dA_c, carry, dA_0) : 0.0f;
  if (p.dh0 != nullptr && cl.turn + 1 == k.nturns && wave == 0) p.dh0[b * p.dim + d] = __builtin_fmaf(P, carry, Q);
  s_dA[wave][lane] = dA;
  __syncthreads();
  if (wave == 0) {
    float sum = dA;
    for (int w = 1; w < k.waves; ++w) sum += s_dA[w][lane];
    k.dA_part[(b * k.nturns + cl.turn) * p.dim + d] = sum;
  }
}

__global__ __launch_bounds__(64 * rows::kGroups) void dA_kernel(const float* part, float* dA, int64_t nrows, int64_t dim) {
  rows::sum_columns(part, nrows, dim, blockIdx.x, 0, nrows, [&](int64_t c, double s) { dA[c] = static_cast<float>(s); });
}

template <int DT>
__global__ __launch_bounds__(kStepThreads) void step_kernel(const float* state, float* state_out, const void* x,
                                                        const void* a_gate, const void* x_gate, const float* A,
                                                        const void* z, void* y, int64_t dim, int64_t xs,
                                                        int64_t as, int64_t gs, int64_t zs, int64_t ys) {
  const int64_t d = static_cast<int64_t>(blockIdx.x) * kStepThreads + threadIdx.x, b = blockIdx.y;
  if (d >= dim) return;
  float a, beta2;
  decay<DT>(rate_of(A[d]) * sigmoid_f(ld<DT>(a_gate, b * as + d)), a, beta2);
  const float u = sigmoid_f(ld<DT>(x_gate, b * gs + d)) * ld<DT>(x, b * xs + d);
  const float h = __builtin_fmaf(a, state[b * dim + d], __builtin_sqrtf(beta2) * u);
  state_out[b * dim + d] = h;
  st<DT>(y, b * ys + d, z ? h * silu_f(ld<DT>(z, b * zs + d)) : h);
}

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

static int64_t dA_bytes(const Shape& s, int64_t batch, int64_t dim) { return round_up(rows::floats(batch * s.nturns, dim) * 4, 256); }

static int prepare(Launch& k, const mm_gated_scan_params* p, const Shape& s, char* handoff, hipStream_t stream) {
  if (s.tiles > 0x7fffffff) return fail(MM_ERR_SHAPE, "too many elements");
  k.p = *p;
  k.hd.control = reinterpret_cast<uint32_t*>(handoff);
  k.hd.word = reinterpret_cast<unsigned long long*>(handoff + s.control_bytes);
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
  k.spread = {k.nstrips, k.nturns, static_cast<uint32_t>(s.per_die), static_cast<uint32_t>(s.span)};
  k.waves = s.waves;
  return MM_OK;
}

}  // namespace gscan
}  // namespace mm

extern "C" {

size_t mm_gated_scan_workspace_size(int64_t batch, int64_t seqlen, int64_t dim, int32_t backward) {
  using namespace mm::gscan;
  if (batch <= 0 || seqlen < 0 || dim <= 0 || !sizes_ok(batch, seqlen, dim)) return 0;
  const Shape s = shape_of(batch, seqlen, dim, backward != 0);
  return static_cast<size_t>((backward ? dA_bytes(s, batch, dim) : 0) + s.handoff_bytes);
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
    if (rows_overlap(p->batch, p->seqlen, p->dim, p->y_stride)) return fail(MM_ERR_LAYOUT, "rows of y overlap");
  } else if (!p->A) {
    return fail(MM_ERR_NULL_POINTER, "A is required");
  }
  if ((e = check_workspace(p, mm_gated_scan_workspace_size(p->batch, p->seqlen, p->dim, 0))) != MM_OK) return e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Shape s = shape_of(p->batch, p->seqlen, p->dim, false, p->lengths != nullptr);
  Launch k{};
  if ((e = prepare(k, p, s, static_cast<char*>(p->workspace), st)) != MM_OK) return e;
  const dim3 grid(static_cast<unsigned>(s.tiles)), block(64 * s.waves);
  const bool p8 = p->codes[0] != nullptr && p->seqlen > 0;
#define MM_GS1(D, Z, P8) hipLaunchKernelGGL((fwd_kernel<D, Z, P8>), grid, block, 0, st, k)
#define MM_GS(D)                                                 \
  if (p8) {                                                      \
    if (p->z) MM_GS1(D, true, true); else MM_GS1(D, false, true);   \
  } else {                                                       \
    if (p->z) MM_GS1(D, true, false); else MM_GS1(D, false, false); \
  }
  switch (p->dtype) {
    case MM_F32: MM_GS(MM_F32); break;
    case MM_F16: MM_GS(MM_F16); break;
    default: MM_GS(MM_BF16); break;
  }
#undef MM_GS
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
  const Shape s = shape_of(p->batch, p->seqlen, p->dim, true, p->lengths != nullptr);
  Launch k{};
  k.dA_part = static_cast<float*>(p->workspace);
  if ((e = prepare(k, p, s, static_cast<char*>(p->workspace) + dA_bytes(s, p->batch, p->dim), st)) != MM_OK) return e;
  const dim3 grid(static_cast<unsigned>(s.tiles)), block(64 * s.waves);
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
  if (batch > 1 && y_stride_b < dim) return fail(MM_ERR_LAYOUT, "rows of y overlap");
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
