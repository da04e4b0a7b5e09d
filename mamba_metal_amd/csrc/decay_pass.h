// Linear attention with a decay for each head: the pass over the tokens, forward and mirrored.
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T      y_t = scale S_t^T q_t
//
// In runs of 64 tokens, with c_t the sum of g from the run's start to t and S the state before the run:
//   y_t = sum_{s <= t} scale (q_t . k_s) exp(c_t - c_s) v_s + scale exp(c_t) S^T q_t
//   S  <- exp(c_63) S + sum_s exp(c_63 - c_s) k_s v_s^T
// so that everything is matrix products.  The backward pass's dv and the gradient of the state are the same sums with
// time turned round and q and k exchanged:
//   dv_s = sum_{t >= s} scale (k_s . q_t) exp(c_t - c_s) dy_t + exp(c_63 - c_s) dS^T k_s
//   dS  <- exp(c_63) dS + sum_t scale exp(c_t) q_t dy_t^T
// A workgroup walks over the runs of one head and 64 value channels; wave w keeps columns 16 w .. 16 w + 15 of the
// state in registers, fp32, and leaves them in shared memory as operands of S^T q; token block w is its share of the
// outputs.  Where the heads alone do not fill the card the tokens are cut into segments: a first pass finds what each segment
// adds to the state, a small kernel joins them, and the second pass starts each segment from its state.
//
// A run is a chain (shared memory, scores, outputs, state) of which a workgroup's own instructions take less than half: it
// is hidden by other workgroups, so that registers and shared memory are held to what lets three share a compute unit in 16
// bits (q goes straight from memory to operands, addresses are made anew in every run).  bf16, 80 heads of 128 by 64 and one
// q and k, in a kernel trace: 8192 tokens of one sequence take 52 us for what the segments add, 8 to join them and 98 to 103 for
// the outputs; 8 sequences of 2048 tokens 280 to 290 us (0.7 GB with the states that are kept, 2.4 TB/s), mirrored 375 to 384 us
// (1.0 GB, 2.7 TB/s).  (Traced, kernels stand alone: with the gradients' 308 these are 970, and the pass takes 900.)  Two
// workgroups a unit: 339 and 498 us.
#pragma once

#include <type_traits>

#include "decay_attention.h"
#include "decay_tiles.h"

namespace mm {
namespace dattn {

template <int DT, int DKP, bool REV, bool OUT, bool VEC>
__global__ __launch_bounds__(256, DT == MM_F32 ? (DKP == 128 && OUT ? 1 : 2) : VEC ? 3 : 2) void pass_kernel(const Pass p) {
  using T = typename Ty<DT>::T;
  using O = Op<DT>;
  using TK = Tile<DT, DKP>;
  using TV = Tile<DT, kVBlock>;
  constexpr int ND = DKP / 16;  // state tiles of a wave
  constexpr int NU = DKP / O::kStep, NR = kRun / O::kStep;
  constexpr int TERMS = DT == MM_F32 ? 1 : DT == MM_F16 ? 2 : 3;
  constexpr int kDecayWave = REV ? 3 : 0;                                   // the one with the fewest scores
  __shared__ __attribute__((aligned(16))) T s_k[kRun * TK::kLd];               // what adds to the state: k, or q
  __shared__ __attribute__((aligned(16))) T s_v[kRun * TV::kLd];               // its values: v, or dy
  __shared__ __attribute__((aligned(16))) T s_s[OUT ? kVBlock * TK::kLd : 8];  // the state as an operand, a value channel a row
  __shared__ Decays s_d[2];
  __shared__ float s_max[4], s_x[4];
  int lane = threadIdx.x & 63, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;

  uint32_t id = blockIdx.x;
  const int vb = static_cast<int>(id % p.vblocks);
  id /= p.vblocks;
  // (what the last segment walked adds is asked for by nobody: the states-only pass leaves it out)
  const uint32_t segs = p.segments - (OUT ? 0 : 1);
  const int seg = static_cast<int>(id % segs) + (REV && !OUT ? 1 : 0);
  id /= segs;
  const int64_t head = id % static_cast<uint32_t>(p.heads), b = id / static_cast<uint32_t>(p.heads);
  const int64_t group = static_cast<uint32_t>(head) / static_cast<uint32_t>(p.per);
  const int64_t bh = b * p.heads + head;
  const int64_t len = length_of(p, b);
  const int64_t run0 = static_cast<int64_t>(seg) * p.seg_runs;
  const int64_t run_end = run0 + p.seg_runs < p.runs ? run0 + p.seg_runs : p.runs;
  const int vw = static_cast<int>(p.dv - vb * kVBlock < kVBlock ? p.dv - vb * kVBlock : kVBlock);
  const int dk = static_cast<int>(p.dk);

  // The state before the first run walked: zeros, the caller's, or what the segments before this one left.
  f32x4 S[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) S[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const bool first = REV ? seg == p.segments - 1 : seg == 0;
  const int vcol = vb * kVBlock + 16 * wave + i;
  if (OUT && !first) {
    const f32x4* const from = seg_state(p, bh, REV ? seg + 1 : seg - 1, vb) + (wave * ND) * 64 + lane;
#pragma unroll
    for (int t = 0; t < ND; ++t) S[t] = from[t * 64];
  } else if (OUT && p.init) {
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * t + 4 * g + r;
        if (d < dk && vcol < p.dv) S[t][r] = p.init[(bh * p.dk + d) * p.dv + vcol];
      }
  }

  Staged<DT, DKP, 256> rk;
  Staged<DT, kVBlock, 256> rv;
  // The run to fetch next: its rows' addresses (running ones: few scalar registers), which a step moves on by a run.
  constexpr int64_t kEs = sizeof(T);
  const int64_t live_runs = (len + kRun - 1) / kRun;
  const int64_t walk_end = run_end < live_runs ? run_end : live_runs;  // runs with tokens: [run0, walk_end)
  const int64_t walk = walk_end - run0;
  int64_t at_run = REV ? walk_end - 1 : run0;
  const char* qp = static_cast<const char*>(p.q) + (b * p.q_stride[0] + group * p.q_stride[2] + at_run * kRun * p.q_stride[1]) * kEs;
  const char* kp = static_cast<const char*>(p.k) + (b * p.k_stride[0] + group * p.k_stride[2] + at_run * kRun * p.k_stride[1]) * kEs;
  const char* vp = static_cast<const char*>(p.v) + (b * p.v_stride[0] + head * p.v_stride[2] + vb * kVBlock + at_run * kRun * p.v_stride[1]) * kEs;
  T* yp = static_cast<T*>(p.y) + ((b * p.seqlen + at_run * kRun) * p.heads + head) * p.dv + vb * kVBlock;  // (of the run at hand)
  int64_t g_at = b * p.g_stride[0] + head * p.g_stride[2] + at_run * kRun * p.g_stride[1];
  using Offset = std::conditional_t<VEC, uint32_t, int64_t>;  // (any rows: they may lie further apart)
  const Offset q_off = static_cast<Offset>(((16 * wave + i) * p.q_stride[1] + O::kE * g) * kEs);
  const uint32_t k_off = static_cast<uint32_t>((rk.row() * p.k_stride[1] + rk.elem()) * kEs);
  const uint32_t v_off = static_cast<uint32_t>((rv.row() * p.v_stride[1] + rv.elem()) * kEs);
  constexpr int kWay = REV ? -1 : 1;
  auto rows_of = [&](int64_t run) { return static_cast<int>(len - run * kRun < kRun ? len - run * kRun : kRun); };
  // Three parts, spread over a run's computation: issued at once they would wait for each other's way into the cache
  // (2400 of a run's 12000 cycles).
  auto fetch_k = [&](int rows) __attribute__((always_inline)) {
    if constexpr (VEC) rk.load(kp, k_off, rk.kRows * p.k_stride[1] * kEs, rows, dk);
    else rk.load_any(kp, p.k_stride[1], rows, dk);
    kp += kWay * kRun * p.k_stride[1] * kEs;
  };
  auto fetch_v = [&](int rows) __attribute__((always_inline)) {
    if constexpr (VEC) rv.load(vp, v_off, rv.kRows * p.v_stride[1] * kEs, rows, vw);
    else rv.load_any(vp, p.v_stride[1], rows, vw);
    vp += kWay * kRun * p.v_stride[1] * kEs;
  };
  // What asks (q, or k mirrored): token 16 wave + i as operands, which no other wave needs.
  u32x4 own[OUT ? NU : 1];
  auto fetch_q = [&](int rows) __attribute__((always_inline)) {
    const bool in = 16 * wave + i < rows;
#pragma unroll
    for (int u = 0; u < (OUT ? NU : 0); ++u) {
      const int e = u * O::kStep + O::kE * g;
      const T* const from = reinterpret_cast<const T*>(qp + q_off) + u * O::kStep;
      if constexpr (VEC) {
        own[u] = u32x4{0, 0, 0, 0};
        if (in && e < dk) own[u] = *reinterpret_cast<const u32x4*>(from);
      } else {
        T t[O::kE];
#pragma unroll
        for (int j = 0; j < O::kE; ++j) t[j] = in && e + j < dk ? from[j] : static_cast<T>(0);
        __builtin_memcpy(&own[u], t, 16);
      }
    }
    qp += kWay * kRun * p.q_stride[1] * kEs;
  };
  auto gate = [&](int rows) __attribute__((always_inline)) {
    const uint32_t raw = lane < rows ? load_gate(p, g_at + lane * p.g_stride[1]) : 0u;
    g_at += kWay * kRun * p.g_stride[1];
    return raw;
  };
  // fp16: the largest magnitude of the wave's columns
  auto note_max = [&]() __attribute__((always_inline)) {
    float m = 0.0f;
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(S[t][r]));
#pragma unroll
    for (int x = 1; x < 64; x *= 2) m = fmaxf(m, lane_xor(m, x));
    if (lane == 0) s_max[wave] = m;
  };
  // mirrored: the product of both states of a run, once all waves have left their parts
  const bool dot_wanted = OUT && REV && p.dot;
  auto note_dot = [&](int64_t run, const Decays& d) {
    const int64_t block = (bh * p.runs + run) * p.vblocks + vb;
    if (threadIdx.x == 0) p.dot[block] = (s_x[0] + s_x[1] + s_x[2] + s_x[3]) * d.whole * (DT == MM_F16 ? p.factors_with[block] : 1.0f);
  };
  double total = 0.0;   // the segment's log decay
  float factor = 1.0f;  // fp16: the state's power of two
  if (walk > 0) {
    fetch_k(rows_of(at_run));
    fetch_v(rows_of(at_run));
    if (OUT) fetch_q(rows_of(at_run));
    if (DT == MM_F16 && OUT) note_max();
    if (wave == kDecayWave) run_decays(s_d[0], gate_value(p, gate(rows_of(at_run))), lane);
  }
  for (int64_t n = 0; n < walk; ++n) {
    // addresses in shared memory are made anew in every run: held over it they would be dozens of registers
    asm volatile("" : "+v"(lane), "+v"(tid));
    const int g = lane >> 4, i = lane & 15;
    const int64_t run = at_run, next = n + 1 < walk ? run + kWay : run;
    at_run = next;
    __syncthreads();  // nobody reads the tiles of the run before
    if constexpr (OUT && REV) {
      if (dot_wanted && n > 0) note_dot(run - kWay, s_d[(n - 1) & 1]);
    }
    rk.store(s_k, tid);
    rv.store(s_v, tid);
    if constexpr (OUT) {
      if constexpr (DT == MM_F16) {
        // fp16 has 5 exponent bits: the state goes through a power of two that puts its largest element at 2^13
        const float m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        const int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
        factor = m > 0.0f && e < 128 ? __builtin_ldexpf(1.0f, e - 13 < -120 ? -120 : e - 13) : 1.0f;
      }
      // (rounded to 16 bits: products of 16-bit operands, off by half a step each at random)
      const float shrink = DT == MM_F16 ? 1.0f / factor : 1.0f;
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        const f32x4 x = DT == MM_F16 ? S[t] * shrink : S[t];
        T* const to = s_s + TK::at(16 * wave, 16 * t, i, 4 * g);
        if constexpr (O::kWide) *reinterpret_cast<f32x4*>(to) = x;
        else *reinterpret_cast<u32x2*>(to) = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
        if constexpr (!O::kWide) {
          // (a run's tokens share the roundings of its states: few of them get the rests, too)
          if (p.state_rests) {
            float a[4];
            unpack2<DT>(pack2<DT>(x[0], x[1]), a[0], a[1]);
            unpack2<DT>(pack2<DT>(x[2], x[3]), a[2], a[3]);
#pragma unroll
            for (int r = 0; r < 4; ++r) a[r] = (x[r] - a[r]) * kRestUp;
            *reinterpret_cast<u32x2*>(static_cast<T*>(p.state_rests) + ((bh * p.runs + run) * p.vblocks + vb) * kVBlock * DKP +
                                      (16 * wave + i) * DKP + 16 * t + 4 * g) = u32x2{pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3])};
          }
        }
      }
    }
    __syncthreads();
    const Decays& D = s_d[n & 1];
    const int64_t block = (bh * p.runs + run) * p.vblocks + vb;  // of the saved states
    // what the state's product with the saved ones of the forward pass needs, before the next run's loads
    constexpr int kSaved = OUT && REV ? ND : 1;
    u32x2 saved2[kSaved];
    f32x4 saved4[kSaved];
    if constexpr (OUT && REV) {
      if (dot_wanted) {
        const T* const before = static_cast<const T*>(p.dot_with) + block * kVBlock * DKP;
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          if constexpr (O::kWide) saved4[t] = *reinterpret_cast<const f32x4*>(before + ((wave * ND + t) * 64 + lane) * 4);
          else saved2[t] = *reinterpret_cast<const u32x2*>(before + (16 * wave + i) * DKP + 16 * t + 4 * g);
        }
      }
    }
    uint32_t g_next = 0;
    if (wave == kDecayWave && n + 1 < walk) g_next = gate(rows_of(next));
    if (n + 1 < walk) fetch_v(rows_of(next));
    if (!OUT && n + 1 < walk) fetch_k(rows_of(next));
    // The state kept for the backward pass, a quarter at a time, for the same reason as the loads.  16 bits: a value
    // channel a row; fp32: as operands over the value channels, a lane's four together.
    float dot = 0.0f;
    auto keep_state = [&](int quarter) __attribute__((always_inline)) {
      if (!OUT || !p.states) return;
      T* const to = static_cast<T*>(p.states) + block * kVBlock * DKP;
      if constexpr (O::kWide) {
#pragma unroll
        for (int c = 0; c < ND / 4; ++c) {
          const int t = quarter * (ND / 4) + c;
          const f32x4 v = __builtin_bit_cast(f32x4, TK::column(s_s, 16 * wave, 16 * t, lane));
          *reinterpret_cast<f32x4*>(to + ((wave * ND + t) * 64 + lane) * 4) = v;
          if (REV && dot_wanted) {
#pragma unroll
            for (int r = 0; r < 4; ++r) dot += v[r] * saved4[REV ? t : 0][r];
          }
        }
        return;
      }
      constexpr int kUnits = DKP / O::kE, kEach = kVBlock * kUnits / 256 / 4 > 0 ? kVBlock * kUnits / 256 / 4 : 1;
      if (quarter >= kVBlock * kUnits / 256) return;
#pragma unroll
      for (int s = 0; s < kEach; ++s) {
        const int u = (quarter * kEach + s) * 256 + tid, r = u / kUnits, e = u % kUnits * O::kE;
        *reinterpret_cast<u32x4*>(to + r * DKP + e) = *reinterpret_cast<const u32x4*>(s_s + TK::at(r, e));
      }
      if (DT == MM_F16 && quarter == 0 && threadIdx.x == 0) p.factors[block] = factor;
    };
    if constexpr (OUT) {
      if constexpr (REV && !O::kWide) {
        if (dot_wanted) {
#pragma unroll
          for (int t = 0; t < ND; ++t) {
            float x[4];
            unpack2<DT>(saved2[t][0], x[0], x[1]);
            unpack2<DT>(saved2[t][1], x[2], x[3]);
#pragma unroll
            for (int r = 0; r < 4; ++r) dot += x[r] * S[t][r];
          }
          if (p.rests_with) {
            const T* const rest = static_cast<const T*>(p.rests_with) + block * kVBlock * DKP + (16 * wave + i) * DKP + 4 * g;
            float more = 0.0f;
#pragma unroll
            for (int t = 0; t < ND; ++t) {
              const u32x2 w = *reinterpret_cast<const u32x2*>(rest + 16 * t);
              float x[4];
              unpack2<DT>(w[0], x[0], x[1]);
              unpack2<DT>(w[1], x[2], x[3]);
#pragma unroll
              for (int r = 0; r < 4; ++r) more += x[r] * S[t][r];
            }
            dot += more * (1.0f / kRestUp);
          }
        }
      }
      // Token block `wave` of the run: its scores, as accumulators (what adds) x (what asks) that are at once operands of
      // their product with the values.
      f32x4 acc[4];
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        acc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (REV ? st < wave : st > wave) continue;
#pragma unroll
        for (int u = 0; u < NU; ++u) acc[st] = mma<DT>(TK::row(s_k, 16 * st, u * O::kStep, lane), own[u], acc[st]);
      }
      if (n + 1 < walk) fetch_k(rows_of(next));
      keep_state(0);
      const float hi_r = D.hi[16 * wave + i], lo_r = D.lo[16 * wave + i];
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (REV ? st < wave : st > wave) continue;
        const f32x4 hi = *reinterpret_cast<const f32x4*>(D.hi + 16 * st + 4 * g);
        const f32x4 lo = *reinterpret_cast<const f32x4*>(D.lo + 16 * st + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float decay = REV ? between<DT>(hi[r], lo[r], hi_r, lo_r) : between<DT>(hi_r, lo_r, hi[r], lo[r]);
          const float x = acc[st][r] * p.scale * decay;
          acc[st][r] = st != wave || (REV ? 4 * g + r >= i : 4 * g + r <= i) ? x : 0.0f;
        }
      }
      float up = 1.0f, down = 1.0f;  // fp16: what the token's outputs stand in until the end
      if constexpr (DT == MM_F16) {
        score_range(largest(acc), up, down);
#pragma unroll
        for (int st = 0; st < 4; ++st) acc[st] *= up;
      }
      const bool fine = !O::kWide && p.fine;
      u32x4 po[NR], rest[NR];
#pragma unroll
      for (int u = 0; u < NR; ++u) score_operand<DT>(acc + u * O::kTiles, fine, po[u], rest[u]);
      keep_state(1);
      // outputs, turned over: 4 value channels of a token in a lane
      f32x4 y[4];
#pragma unroll
      for (int vt = 0; vt < 4; ++vt) y[vt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int vt = 0; vt < 4; ++vt) y[vt] = mma<DT>(TK::row(s_s, 16 * vt, u * O::kStep, lane), own[u], y[vt]);
      if (n + 1 < walk) fetch_q(rows_of(next));
      keep_state(2);
      float ws = (REV ? D.onward : D.into)[16 * wave + i] * ((REV ? 1.0f : p.scale) * factor);
      if constexpr (DT == MM_F16) ws *= up;
#pragma unroll
      for (int vt = 0; vt < 4; ++vt) y[vt] *= ws;
#pragma unroll
      for (int u = 0; u < NR; ++u) {
        if (REV ? (u + 1) * O::kStep <= 16 * wave : u * O::kStep > 16 * wave + 15) continue;
#pragma unroll
        for (int vt = 0; vt < 4; ++vt) y[vt] = mma<DT>(TV::column(s_v, u * O::kStep, 16 * vt, lane), po[u], y[vt]);
        if (fine) {
#pragma unroll
          for (int vt = 0; vt < 4; ++vt) y[vt] = mma_rest<DT>(TV::column(s_v, u * O::kStep, 16 * vt, lane), rest[u], y[vt]);
        }
      }
      if constexpr (DT == MM_F16) {
#pragma unroll
        for (int vt = 0; vt < 4; ++vt) y[vt] *= down;
      }
      const int left = static_cast<int>(p.seqlen - run * kRun < kRun ? p.seqlen - run * kRun : kRun), t = 16 * wave + i;
      if (t < left) {
        T* const to = yp + t * p.heads * p.dv + 4 * g;
        const bool in = t < rows_of(run);
#pragma unroll
        for (int vt = 0; vt < 4; ++vt) {
          if (!in) y[vt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (VEC) {
            if (16 * vt + 4 * g < vw) {
              if constexpr (O::kWide) *reinterpret_cast<f32x4*>(to + 16 * vt) = y[vt];
              else *reinterpret_cast<u32x2*>(to + 16 * vt) = u32x2{pack2<DT>(y[vt][0], y[vt][1]), pack2<DT>(y[vt][2], y[vt][3])};
            }
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (16 * vt + 4 * g + r < vw) to[16 * vt + r] = Ty<DT>::from(y[vt][r]);
          }
        }
      }
      yp += kWay * kRun * p.heads * p.dv;
    }
    if (wave == kDecayWave && n + 1 < walk) run_decays(s_d[(n + 1) & 1], gate_value(p, g_next), lane);
    // the state's step: this wave's value columns, weighted, as operands over the run's tokens
    const float whole = D.whole;
#pragma unroll
    for (int t = 0; t < ND; ++t) S[t] *= whole;
    const float* const weight = REV ? D.into : D.onward;
    const float ws = REV ? p.scale : 1.0f;
#pragma unroll
    for (int u = 0; u < NR; ++u) {
      if (u == NR - 1) keep_state(3);
      const u32x4 vo = TV::column(s_v, u * O::kStep, 16 * wave, lane);
      u32x4 terms[TERMS];
      if constexpr (O::kWide) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(weight + 16 * u + 4 * g) * ws;
        terms[0] = __builtin_bit_cast(u32x4, __builtin_bit_cast(f32x4, vo) * w);
      } else {
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(weight + 32 * u + 4 * g) * ws;
        const f32x4 w1 = *reinterpret_cast<const f32x4*>(weight + 32 * u + 16 + 4 * g) * ws;
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack2<DT>(vo[j], x[2 * j], x[2 * j + 1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] *= w0[j];
          x[4 + j] *= w1[j];
        }
        split_operand<DT, TERMS>(x, terms);
      }
      // four state tiles at a time: products that follow each other are independent
#pragma unroll
      for (int t0 = 0; t0 < ND; t0 += 4) {
        u32x4 ko[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) ko[t] = TK::column(s_k, u * O::kStep, 16 * (t0 + t), lane);
        if constexpr (DT == MM_F16) {
#pragma unroll
          for (int t = 0; t < 4; ++t) S[t0 + t] = mma<DT>(ko[t], terms[0], S[t0 + t]);
#pragma unroll
          for (int t = 0; t < 4; ++t) S[t0 + t] += mma<DT>(ko[t], terms[1], f32x4{0.0f, 0.0f, 0.0f, 0.0f}) * (1.0f / kRestUp);
        } else {
#pragma unroll
          for (int m = TERMS - 1; m >= 0; --m)
#pragma unroll
            for (int t = 0; t < 4; ++t) S[t0 + t] = mma<DT>(ko[t], terms[m], S[t0 + t]);
        }
      }
    }
    if (OUT && REV && dot_wanted) {
#pragma unroll
      for (int x = 1; x < 64; x *= 2) dot += lane_xor(dot, x);
      if (lane == 0) s_x[wave] = dot;
    }
    if (DT == MM_F16 && OUT) note_max();
    if (!OUT) total += static_cast<double>(D.hi[63]) + D.lo[63];
  }
  if constexpr (OUT && REV) {
    if (walk > 0 && dot_wanted) {
      __syncthreads();
      note_dot(run0, s_d[(walk - 1) & 1]);
    }
  }

  if constexpr (OUT) {
    // tokens of runs that hold none of the sequence
    const int64_t z0 = (walk_end > run0 ? walk_end : run0) * kRun;
    const int64_t z1 = run_end * kRun < p.seqlen ? run_end * kRun : p.seqlen;
    for (int64_t t = z0 + (threadIdx.x >> 6); t < z1; t += 4)
      if (lane < vw)
        static_cast<T*>(p.y)[((b * p.seqlen + t) * p.heads + head) * p.dv + vb * kVBlock + lane] = Ty<DT>::from(0.0f);
    const bool last = REV ? seg == 0 : seg == p.segments - 1;
    if (last && p.final_state) {
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = 16 * t + 4 * g + r;
          if (d < dk && vcol < p.dv) p.final_state[(bh * p.dk + d) * p.dv + vcol] = S[t][r];
        }
    }
  } else {
    f32x4* const to = seg_state(p, bh, seg, vb) + (wave * ND) * 64 + lane;
#pragma unroll
    for (int t = 0; t < ND; ++t) to[t * 64] = S[t];
    if (vb == 0 && threadIdx.x == 0) p.seg_decay[bh * p.segments + seg] = total;
  }
}

// What the segments add, joined: slot `seg` gets the state after it (mirrored: before it).  Memory traffic: 9 segments of 80
// heads, 45 MB in 8 us.
template <int DKP, bool REV>
__global__ __launch_bounds__(256) void join_kernel(const Pass p) {
  constexpr int ND = DKP / 16;
  const int64_t per_head = static_cast<int64_t>(p.vblocks) * kVBlock * DKP / 4;  // in fours
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= p.batch * p.heads * per_head) return;
  const int64_t bh = e / per_head, at = e % per_head;
  const int vb = static_cast<int>(at / (4 * ND * 64)), in = static_cast<int>(at % (4 * ND * 64));
  const int lane = in & 63, tile = in / 64 % ND, wave = in / 64 / ND;
  f32x4 S = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (p.init) {
    const int vcol = vb * kVBlock + 16 * wave + (lane & 15);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * tile + 4 * (lane >> 4) + r;
      if (d < p.dk && vcol < p.dv) S[r] = p.init[(bh * p.dk + d) * p.dv + vcol];
    }
  }
  f32x4* const slots = seg_state(p, bh, 0, vb) + in;
  const int64_t step = seg_state(p, bh, 1, vb) - seg_state(p, bh, 0, vb);
  const double* const decays = p.seg_decay + bh * p.segments;
  for (int n0 = 0; n0 + 1 < p.segments; n0 += 8) {
    f32x4 adds[8];
    double c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // (eight at a time under way)
      const int n = n0 + j + 1 < p.segments ? n0 + j : n0, seg = REV ? p.segments - 1 - n : n;
      adds[j] = slots[seg * step];
      c[j] = decays[seg];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = n0 + j, seg = REV ? p.segments - 1 - n : n;
      if (n + 1 >= p.segments) break;
      const float hi = static_cast<float>(c[j]);
      S = S * (exp2_acc(hi) * (1.0f + static_cast<float>(c[j] - hi) * kLn2)) + adds[j];
      slots[seg * step] = S;
    }
  }
}

template <int DT, int DKP, bool REV, bool VEC>
static void launch_pass_t(const Pass& p, hipStream_t s) {
  const unsigned per_seg = static_cast<unsigned>(p.batch * p.heads * p.vblocks);
  if (p.segments > 1) {
    hipLaunchKernelGGL((pass_kernel<DT, DKP, REV, false, VEC>), dim3(per_seg * (p.segments - 1)), dim3(256), 0, s, p);
    const int64_t n = p.batch * p.heads * p.vblocks * static_cast<int64_t>(kVBlock) * DKP / 4;
    hipLaunchKernelGGL((join_kernel<DKP, REV>), dim3(static_cast<unsigned>(ceil_div(n, 256))), dim3(256), 0, s, p);
  }
  hipLaunchKernelGGL((pass_kernel<DT, DKP, REV, true, VEC>), dim3(per_seg * p.segments), dim3(256), 0, s, p);
}
// vec: 16 bytes at a time where all rows allow it; any other layout element by element.
template <int DT, bool REV>
static void launch_pass_d(const Pass& p, hipStream_t s) {
  if (padded_dk(p.dk) == 64) {
    if (p.vec) launch_pass_t<DT, 64, REV, true>(p, s); else launch_pass_t<DT, 64, REV, false>(p, s);
  } else {
    if (p.vec) launch_pass_t<DT, 128, REV, true>(p, s); else launch_pass_t<DT, 128, REV, false>(p, s);
  }
}
template <bool REV>
static void launch_pass(const Pass& p, hipStream_t s) {
  switch (p.dtype) {
    case MM_F32: launch_pass_d<MM_F32, REV>(p, s); break;
    case MM_F16: launch_pass_d<MM_F16, REV>(p, s); break;
    default: launch_pass_d<MM_BF16, REV>(p, s); break;
  }
}

}  // namespace dattn
}  // namespace mm
