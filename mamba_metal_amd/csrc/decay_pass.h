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
// state in registers, fp32, as accumulators whose layout is at once the operand of S^T q.  Where the heads alone do not
// fill the card the tokens are cut into segments: a first pass finds what each segment adds to the state, a small kernel
// joins them, and the second pass starts each segment from its state.
#pragma once

#include "decay_attention.h"
#include "decay_tiles.h"

namespace mm {
namespace dattn {

// 16-bit operands of a product whose result is a state in fp32: the value as a sum of TERMS of them.  bf16: three are
// fp32's own 24 bits.  fp16: two hold 22 bits, the second one 2^11 times too large (and summed by itself), since the rest of a
// value below 1/8 would be subnormal, which the matrix cores take as 0; so would be values below 2^-14, which therefore
// are all rest.
constexpr float kRestUp = 2048.0f;
template <int DT, int TERMS>
__device__ __forceinline__ void split_operand(const float (&x)[8], u32x4 (&out)[TERMS]) {
  float rest[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = x[j];
#pragma unroll
  for (int n = 0; n < TERMS; ++n)
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float c[2] = {rest[j], rest[j + 1]};
      if (DT == MM_F16) {
#pragma unroll
        for (int e = 0; e < 2; ++e) c[e] = n == 0 ? (fabsf(c[e]) < 6.103515625e-05f ? 0.0f : c[e]) : c[e] * kRestUp;
      }
      const uint32_t w = pack2<DT>(c[0], c[1]);
      out[n][j / 2] = w;
      if (n + 1 < TERMS) {
        float a, b;
        unpack2<DT>(w, a, b);
        rest[j] -= a;
        rest[j + 1] -= b;
      }
    }
}

template <int DT, int DKP, bool REV, bool OUT>
__global__ __launch_bounds__(256) void pass_kernel(const Pass p) {
  using T = typename Ty<DT>::T;
  using O = Op<DT>;
  constexpr int LDK = DKP + O::kPad, LDV = kVBlock + O::kPad, LDP = kRun + O::kPad;
  constexpr int ND = DKP / 16;  // state tiles of a wave
  constexpr int TERMS = DT == MM_F32 ? 1 : DT == MM_F16 ? 2 : 3;
  __shared__ __attribute__((aligned(16))) T s_q[OUT ? kRun * LDK : 8];  // what asks: q, or k mirrored
  __shared__ __attribute__((aligned(16))) T s_k[kRun * LDK];            // what adds to the state: k, or q
  __shared__ __attribute__((aligned(16))) T s_v[kRun * LDV];            // its values: v, or dy
  __shared__ __attribute__((aligned(16))) T s_p[OUT ? kRun * LDP : 8];
  __shared__ __attribute__((aligned(16))) T s_s[OUT ? 4 * 16 * LDK : 8];  // a wave's state columns, to turn them over
  __shared__ Decays s_d;
  __shared__ float s_max[4];
  __shared__ double s_x[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;

  uint32_t id = blockIdx.x;
  const int vb = static_cast<int>(id % p.vblocks);
  id /= p.vblocks;
  const int seg = static_cast<int>(id % p.segments);
  id /= p.segments;
  const int64_t head = id % p.heads, b = id / p.heads;
  const int64_t group = head / p.per;
  const int64_t bh = b * p.heads + head;
  const int64_t len = length_of(p, b);
  const int64_t run0 = static_cast<int64_t>(seg) * p.seg_runs;
  const int64_t run_end = run0 + p.seg_runs < p.runs ? run0 + p.seg_runs : p.runs;
  const int vw = static_cast<int>(p.dv - vb * kVBlock < kVBlock ? p.dv - vb * kVBlock : kVBlock);
  const int dk = static_cast<int>(p.dk);

  const T* const qh = static_cast<const T*>(p.q) + b * p.q_stride[0] + group * p.q_stride[2];
  const T* const kh = static_cast<const T*>(p.k) + b * p.k_stride[0] + group * p.k_stride[2];
  const T* const vh = static_cast<const T*>(p.v) + b * p.v_stride[0] + head * p.v_stride[2] + vb * kVBlock;
  const int64_t gh = b * p.g_stride[0] + head * p.g_stride[2];

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

  Staged<DT, DKP> rq, rk;
  Staged<DT, kVBlock> rv;
  float rg = 0.0f;
  auto fetch = [&](int64_t run) __attribute__((always_inline)) {
    const int64_t t0 = run * kRun;
    const int rows = static_cast<int>(len - t0 < kRun ? len - t0 : kRun);
    if (OUT) rq.load(qh + t0 * p.q_stride[1], p.q_stride[1], rows, dk, p.vec & 1);
    rk.load(kh + t0 * p.k_stride[1], p.k_stride[1], rows, dk, p.vec & 2);
    rv.load(vh + t0 * p.v_stride[1], p.v_stride[1], rows, vw, p.vec & 4);
    rg = lane < rows ? load_gate(p, gh + (t0 + lane) * p.g_stride[1]) : 0.0f;
  };
  const int64_t live_runs = (len + kRun - 1) / kRun;
  const int64_t walk_end = run_end < live_runs ? run_end : live_runs;  // runs with tokens: [run0, walk_end)
  double total = 0.0;  // the segment's log decay
  float factor = 1.0f; // fp16: the state's power of two
  if (walk_end > run0) {
    if (DT == MM_F16 && OUT) {
      float m = 0.0f;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(S[t][r]));
#pragma unroll
      for (int x = 1; x < 64; x *= 2) m = fmaxf(m, lane_xor(m, x));
      if (lane == 0) s_max[wave] = m;
    }
    fetch(REV ? walk_end - 1 : run0);
  }
  for (int64_t n = 0; n < walk_end - run0; ++n) {
    const int64_t run = REV ? walk_end - 1 - n : run0 + n;
    if (OUT) rq.store(s_q);
    rk.store(s_k);
    rv.store(s_v);
    if (wave == (REV ? 3 : 0)) run_decays(s_d, rg, lane);
    __syncthreads();
    if (n + 1 < walk_end - run0) fetch(REV ? run - 1 : run + 1);

    u32x4 vo[kRun / O::kStep];  // this wave's value columns, as operands over the run's tokens
#pragma unroll
    for (int u = 0; u < kRun / O::kStep; ++u) vo[u] = column_operand<DT>(s_v, LDV, u * O::kStep, 16 * wave, lane);

    if constexpr (OUT) {
      if constexpr (DT == MM_F16) {
        // fp16 has 5 exponent bits: the state goes through a power of two that puts its largest element at 2^13
        const float m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
        const int e = static_cast<int>(__float_as_uint(m) >> 23) - 127;
        factor = m > 0.0f && e < 128 ? __builtin_ldexpf(1.0f, e - 13 < -120 ? -120 : e - 13) : 1.0f;
      }
      const float shrink = DT == MM_F16 ? 1.0f / factor : 1.0f;
      // the state as an operand (rounded to 16 bits: products of 16-bit operands, off by half a step each at random)
      u32x4 so[DKP / O::kStep];
#pragma unroll
      for (int u = 0; u < DKP / O::kStep; ++u) {
        f32x4 part[O::kTiles];
#pragma unroll
        for (int n2 = 0; n2 < O::kTiles; ++n2) part[n2] = S[u * O::kTiles + n2] * shrink;
        so[u] = from_acc<DT>(part);
      }
      if (p.states) {
        // for the backward pass: 16 columns turned over, so that its operands over them are whole reads
        T* const mine = s_s + wave * 16 * LDK;
#pragma unroll
        for (int u = 0; u < DKP / O::kStep; ++u) {
          if constexpr (O::kWide) {
            *reinterpret_cast<u32x4*>(mine + i * LDK + 16 * u + 4 * g) = so[u];
          } else {
            *reinterpret_cast<u32x2*>(mine + i * LDK + 32 * u + 4 * g) = u32x2{so[u][0], so[u][1]};
            *reinterpret_cast<u32x2*>(mine + i * LDK + 32 * u + 16 + 4 * g) = u32x2{so[u][2], so[u][3]};
          }
        }
        T* const out = run_state<T>(p.states, p, bh, run, vb, DKP);
        const T* const before = p.dot ? run_state<T>(const_cast<void*>(p.dot_with), p, bh, run, vb, DKP) : nullptr;
        float dot = 0.0f;
        wave_lds_fence();
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          const int64_t at = state_at<DT>(wave, t, ND, lane);
          if constexpr (O::kWide) {
            f32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = mine[(4 * g + j) * LDK + 16 * t + i];
            *reinterpret_cast<f32x4*>(out + at) = v;
            if (REV && before) {
              const f32x4 w = *reinterpret_cast<const f32x4*>(before + at);
#pragma unroll
              for (int j = 0; j < 4; ++j) dot += v[j] * w[j];
            }
          } else {
            const u32x2 v = column4<DT>(mine, LDK, 0, 16 * t, lane);
            *reinterpret_cast<u32x2*>(out + at) = v;
            if (REV && before) {
              const u32x2 w = *reinterpret_cast<const u32x2*>(before + at);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float a, b2, x, y;
                unpack2<DT>(v[j], a, b2);
                unpack2<DT>(w[j], x, y);
                dot += a * x + b2 * y;
              }
            }
          }
        }
        if (REV && before) {
          if constexpr (!O::kWide) {
            // what rounding the gradient's state left out, so that the sum has one rounded factor and not two
            wave_lds_fence();
#pragma unroll
            for (int u = 0; u < DKP / O::kStep; ++u) {
              f32x4 part[2];
#pragma unroll
              for (int n2 = 0; n2 < 2; ++n2)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  float a, b2;
                  unpack2<DT>(so[u][2 * n2 + r], a, b2);
                  part[n2][2 * r] = S[2 * u + n2][2 * r] * shrink - a;
                  part[n2][2 * r + 1] = S[2 * u + n2][2 * r + 1] * shrink - b2;
                }
              const u32x4 rest = from_acc<DT>(part);
              *reinterpret_cast<u32x2*>(mine + i * LDK + 32 * u + 4 * g) = u32x2{rest[0], rest[1]};
              *reinterpret_cast<u32x2*>(mine + i * LDK + 32 * u + 16 + 4 * g) = u32x2{rest[2], rest[3]};
            }
            wave_lds_fence();
#pragma unroll
            for (int t = 0; t < ND; ++t) {
              const u32x2 v = column4<DT>(mine, LDK, 0, 16 * t, lane);
              const u32x2 w = *reinterpret_cast<const u32x2*>(before + state_at<DT>(wave, t, ND, lane));
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float a, b2, x, y;
                unpack2<DT>(v[j], a, b2);
                unpack2<DT>(w[j], x, y);
                dot += a * x + b2 * y;
              }
            }
          }
#pragma unroll
          for (int x = 1; x < 64; x *= 2) dot += lane_xor(dot, x);
          if (lane == 0) s_x[wave] = dot;
        }
        if (DT == MM_F16 && threadIdx.x == 0) p.factors[(bh * p.runs + run) * p.vblocks + vb] = factor;
      }
      // scores of row block `wave`: tiles of (what adds) x (what asks), whose accumulators are rows of p
      const float hi_r = s_d.hi[16 * wave + i], lo_r = s_d.lo[16 * wave + i];
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        if (REV ? st < wave : st > wave) continue;
        f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < DKP / O::kStep; ++u)
          acc = mma<DT>(row_operand<DT>(s_k, LDK, 16 * st, u * O::kStep, lane),
                        row_operand<DT>(s_q, LDK, 16 * wave, u * O::kStep, lane), acc);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(s_d.hi + 16 * st + 4 * g);
        const f32x4 lo = *reinterpret_cast<const f32x4*>(s_d.lo + 16 * st + 4 * g);
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int other = 16 * st + 4 * g + r, row = 16 * wave + i;
          const bool in = REV ? other >= row : other <= row;
          const float decay = REV ? between<DT>(hi[r], lo[r], hi_r, lo_r) : between<DT>(hi_r, lo_r, hi[r], lo[r]);
          v[r] = in ? acc[r] * p.scale * decay : 0.0f;
        }
        T* const at = s_p + (16 * wave + i) * LDP + 16 * st + 4 * g;
        if constexpr (O::kWide) *reinterpret_cast<f32x4*>(at) = f32x4{v[0], v[1], v[2], v[3]};
        else *reinterpret_cast<u32x2*>(at) = u32x2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
      }
      // the tiles beside the diagonal that an operand's step takes in with it
      if constexpr (!O::kWide) {
        if (REV ? (wave & 1) : !(wave & 1))
          *reinterpret_cast<u32x2*>(s_p + (16 * wave + i) * LDP + 16 * (REV ? wave - 1 : wave + 1) + 4 * g) = u32x2{0, 0};
      }
      __syncthreads();
      if (REV && p.dot && threadIdx.x == 0)
        p.dot[(bh * p.runs + run) * p.vblocks + vb] =
            (s_x[0] + s_x[1] + s_x[2] + s_x[3]) * s_d.whole * factor *
            (DT == MM_F16 ? p.factors_with[(bh * p.runs + run) * p.vblocks + vb] : 1.0f);
      // outputs: row block by row block, this wave's 16 columns
      const float qs = (REV ? 1.0f : p.scale) * factor;
#pragma unroll
      for (int rt = 0; rt < 4; ++rt) {
        f32x4 acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < DKP / O::kStep; ++u)
          acc = mma<DT>(row_operand_acc<DT>(s_q, LDK, 16 * rt, u * O::kStep, lane), so[u], acc);
        acc *= *reinterpret_cast<const f32x4*>((REV ? s_d.onward : s_d.into) + 16 * rt + 4 * g) * qs;
#pragma unroll
        for (int u = 0; u < kRun / O::kStep; ++u) {
          if (REV ? (u + 1) * O::kStep <= 16 * rt : u * O::kStep > 16 * rt + 15) continue;
          acc = mma<DT>(row_operand_acc<DT>(s_p, LDP, 16 * rt, u * O::kStep, lane), vo[u], acc);
        }
        const int64_t t0 = run * kRun + 16 * rt + 4 * g;
        T* const y = static_cast<T*>(p.y) + ((b * p.seqlen + t0) * p.heads + head) * p.dv + vcol;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t0 + r < p.seqlen && vcol < p.dv) y[r * p.heads * p.dv] = Ty<DT>::from(t0 + r < len ? acc[r] : 0.0f);
      }
    }
    // the state's step
    const float whole = s_d.whole;
#pragma unroll
    for (int t = 0; t < ND; ++t) S[t] *= whole;
    const float* const weight = REV ? s_d.into : s_d.onward;
    const float ws = REV ? p.scale : 1.0f;
#pragma unroll
    for (int u = 0; u < kRun / O::kStep; ++u) {
      u32x4 terms[TERMS];
      if constexpr (O::kWide) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(weight + 16 * u + 4 * g) * ws;
        terms[0] = __builtin_bit_cast(u32x4, __builtin_bit_cast(f32x4, vo[u]) * w);
      } else {
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(weight + 32 * u + 4 * g) * ws;
        const f32x4 w1 = *reinterpret_cast<const f32x4*>(weight + 32 * u + 16 + 4 * g) * ws;
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack2<DT>(vo[u][j], x[2 * j], x[2 * j + 1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] *= w0[j];
          x[4 + j] *= w1[j];
        }
        split_operand<DT, TERMS>(x, terms);
      }
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        const u32x4 ko = column_operand<DT>(s_k, LDK, u * O::kStep, 16 * t, lane);
        if constexpr (DT == MM_F16) {
          S[t] = mma<DT>(ko, terms[0], S[t]);
          S[t] += mma<DT>(ko, terms[1], f32x4{0.0f, 0.0f, 0.0f, 0.0f}) * (1.0f / kRestUp);
        } else {
#pragma unroll
          for (int m = TERMS - 1; m >= 0; --m) S[t] = mma<DT>(ko, terms[m], S[t]);
        }
      }
    }
    if (DT == MM_F16 && OUT) {
      float m = 0.0f;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(S[t][r]));
#pragma unroll
      for (int x = 1; x < 64; x *= 2) m = fmaxf(m, lane_xor(m, x));
      if (lane == 0) s_max[wave] = m;
    }
    if (!OUT) total += static_cast<double>(s_d.hi[63]) + s_d.lo[63];
    __syncthreads();
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

// What the segments add, joined: slot `seg` gets the state after it (mirrored: before it).
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
  for (int n = 0; n + 1 < p.segments; ++n) {
    const int seg = REV ? p.segments - 1 - n : n;
    const double c = p.seg_decay[bh * p.segments + seg];
    f32x4* const slot = seg_state(p, bh, seg, vb) + in;
    const float hi = static_cast<float>(c);
    S = S * (exp2_acc(hi) * (1.0f + static_cast<float>(c - hi) * kLn2)) + *slot;
    *slot = S;
  }
}

template <int DT, int DKP, bool REV>
static void launch_pass_t(const Pass& p, hipStream_t s) {
  const unsigned per_seg = static_cast<unsigned>(p.batch * p.heads * p.vblocks);
  if (p.segments > 1) {
    hipLaunchKernelGGL((pass_kernel<DT, DKP, REV, false>), dim3(per_seg * p.segments), dim3(256), 0, s, p);
    const int64_t n = p.batch * p.heads * p.vblocks * static_cast<int64_t>(kVBlock) * DKP / 4;
    hipLaunchKernelGGL((join_kernel<DKP, REV>), dim3(static_cast<unsigned>(ceil_div(n, 256))), dim3(256), 0, s, p);
  }
  hipLaunchKernelGGL((pass_kernel<DT, DKP, REV, true>), dim3(per_seg * p.segments), dim3(256), 0, s, p);
}
template <int DT, bool REV>
static void launch_pass_d(const Pass& p, hipStream_t s) {
  if (padded_dk(p.dk) == 64) launch_pass_t<DT, 64, REV>(p, s);
  else launch_pass_t<DT, 128, REV>(p, s);
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
