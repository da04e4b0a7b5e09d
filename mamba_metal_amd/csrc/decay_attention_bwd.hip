// Linear attention with a decay for each head: gradients of q, k and the log decays.
//
// With the states before each run (S, from the forward pass) and the gradients of the states after it (dS, from the
// mirrored pass) every run stands alone.  D[t, s] = scale exp(c_t - c_s) for s <= t, else 0; dP = (dy v^T) D:
//   dq_t = sum_s dP[t, s] k_s + scale exp(c_t) S dy_t        dk_s = sum_t dP[t, s] q_t + exp(c_63 - c_s) dS v_s
// The log decay of token t scales what tokens t' >= t take from tokens s < t.  With M = dP (q k^T), elementwise:
//   dg_t = sum_{t' >= t} (row sum - column sum of M)(t') + sum_{t' >= t} scale exp(c_t') q_t' . S dy_t'
//        + sum_{s < t} exp(c_63 - c_s) k_s . dS v_s + exp(c_63) <S, dS>
// so that no sum reaches past the run, and what cancels in it cancels among 64 tokens.
//
// A workgroup takes one run and some heads that share q and k, which it stages once and whose gradients it sums over
// the heads in registers.  Waves 0 to 3 make dq, waves 4 to 7 dk, 16 tokens each: the two are one computation with the
// roles exchanged (own rows dy, others v, state S, sum over k; or own rows v, others dy, state dS, sum over q).
#include "decay_attention.h"
#include "decay_tiles.h"

namespace mm {
namespace dattn {

template <int DT, int DKP>
__global__ __launch_bounds__(512) void grad_kernel(const Grad p) {
  using T = typename Ty<DT>::T;
  using O = Op<DT>;
  using TK = Tile<DT, DKP>;
  using TV = Tile<DT, kVBlock>;
  constexpr int ND = DKP / 16, NU = kVBlock / O::kStep;
  __shared__ __attribute__((aligned(16))) T s_qk[2][kRun * TK::kLd];  // q, k
  __shared__ __attribute__((aligned(16))) T s_dv[2][kRun * TV::kLd];  // dy, v
  __shared__ Decays s_d;
  __shared__ float s_sum[2][kRun], s_inter[2][kRun];  // M's row and column sums; the states' parts
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, i = lane & 15;
  const int role = wave >> 2, blk = wave & 3;  // 0: dq, 1: dk

  uint32_t id = blockIdx.x;
  const int set = static_cast<int>(id % p.sets);
  id /= p.sets;
  const int64_t group = id % p.groups;
  id /= static_cast<uint32_t>(p.groups);
  const int64_t run = id % p.runs, b = id / p.runs;
  const int64_t len = length_of(p, b), t0 = run * kRun;
  const int rows = static_cast<int>(len - t0 < 0 ? 0 : len - t0 < kRun ? len - t0 : kRun);
  const int h0 = set * p.set_heads, h1 = h0 + p.set_heads < p.per ? h0 + p.set_heads : static_cast<int>(p.per);
  const int dk = static_cast<int>(p.dk);

  f32x4 out[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) out[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (rows > 0) {
    {
      Staged<DT, DKP, 512> r;
      r.load(static_cast<const T*>(p.q) + b * p.q_stride[0] + t0 * p.q_stride[1] + group * p.q_stride[2], p.q_stride[1],
             rows, dk, p.vec & 1);
      r.store(s_qk[0]);
      r.load(static_cast<const T*>(p.k) + b * p.k_stride[0] + t0 * p.k_stride[1] + group * p.k_stride[2], p.k_stride[1],
             rows, dk, p.vec & 2);
      r.store(s_qk[1]);
    }
    __syncthreads();
    const T* const s_own = s_qk[role];
    const T* const s_other = s_qk[1 - role];
    // scores of the own rows (columns of the tiles) with the others: the same for all heads
    f32x4 A[4];
#pragma unroll
    for (int ot = 0; ot < 4; ++ot) {
      A[ot] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < DKP / O::kStep; ++u)
        A[ot] = mma<DT>(TK::row(s_other, 16 * ot, u * O::kStep, lane),
                        TK::row(s_own, 16 * blk, u * O::kStep, lane), A[ot]);
    }

    Staged<DT, kVBlock, 512> ry, rv;
    float rg = 0.0f;
    auto fetch = [&](int h, int vb) __attribute__((always_inline)) {
      const int64_t head = group * p.per + h;
      const int vw = static_cast<int>(p.dv - vb * kVBlock < kVBlock ? p.dv - vb * kVBlock : kVBlock);
      ry.load(static_cast<const T*>(p.dy) + b * p.dy_stride[0] + t0 * p.dy_stride[1] + head * p.dy_stride[2] + vb * kVBlock,
              p.dy_stride[1], rows, vw, p.vec & 8);
      rv.load(static_cast<const T*>(p.v) + b * p.v_stride[0] + t0 * p.v_stride[1] + head * p.v_stride[2] + vb * kVBlock,
              p.v_stride[1], rows, vw, p.vec & 4);
      if (vb == 0) rg = lane < rows ? load_gate(p, b * p.g_stride[0] + (t0 + lane) * p.g_stride[1] + head * p.g_stride[2]) : 0.0f;
    };
    fetch(h0, 0);
    for (int h = h0; h < h1; ++h) {
      const int64_t head = group * p.per + h, bh = b * p.heads + head;
      f32x4 acc[4], tmp[ND];
#pragma unroll
      for (int ot = 0; ot < 4; ++ot) acc[ot] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < ND; ++t) tmp[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      float factor = 1.0f;
      for (int vb = 0; vb < p.vblocks; ++vb) {
        __syncthreads();
        ry.store(s_dv[0]);
        rv.store(s_dv[1]);
        if (vb == 0 && wave == 0) run_decays(s_d, rg, lane);
        __syncthreads();
        const T* const from = run_state<T>(const_cast<void*>(role ? p.dstates : p.states), p, bh, run, vb, DKP);
        if (vb + 1 < p.vblocks) fetch(h, vb + 1);
        else if (h + 1 < h1) fetch(h + 1, 0);
        const T* const own_t = s_dv[role];
        const T* const other_t = s_dv[1 - role];
        u32x4 own[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) own[u] = TV::row_acc(own_t, 16 * blk, u * O::kStep, lane);
        if constexpr (DT == MM_F16) {
          const float f = (role ? p.dfactors : p.factors)[(bh * p.runs + run) * p.vblocks + vb];
#pragma unroll
          for (int t = 0; t < ND; ++t) tmp[t] *= factor / f;
          factor = f;
        }
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int t = 0; t < ND; ++t)
            tmp[t] = mma<DT>(own[u], *reinterpret_cast<const u32x4*>(from + static_cast<int64_t>((u * ND + t) * 64 + lane) * O::kE),
                             tmp[t]);
#pragma unroll
        for (int ot = 0; ot < 4; ++ot) {
          if (role ? ot < blk : ot > blk) continue;
#pragma unroll
          for (int u = 0; u < NU; ++u) acc[ot] = mma<DT>(TV::row_acc(other_t, 16 * ot, u * O::kStep, lane), own[u], acc[ot]);
        }
      }
      // dP and M
      const float hi_r = s_d.hi[16 * blk + i], lo_r = s_d.lo[16 * blk + i];
      float sum = 0.0f;
#pragma unroll
      for (int ot = 0; ot < 4; ++ot) {
        if (role ? ot < blk : ot > blk) continue;
        const f32x4 hi = *reinterpret_cast<const f32x4*>(s_d.hi + 16 * ot + 4 * g);
        const f32x4 lo = *reinterpret_cast<const f32x4*>(s_d.lo + 16 * ot + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int other = 16 * ot + 4 * g + r, row = 16 * blk + i;
          const bool in = role ? other >= row : other <= row;
          const float decay = role ? between<DT>(hi[r], lo[r], hi_r, lo_r) : between<DT>(hi_r, lo_r, hi[r], lo[r]);
          acc[ot][r] = in ? acc[ot][r] * p.scale * decay : 0.0f;
          sum += in ? acc[ot][r] * A[ot][r] : 0.0f;
        }
      }
      u32x4 dp[kRun / O::kStep];
#pragma unroll
      for (int u = 0; u < kRun / O::kStep; ++u) dp[u] = from_acc<DT>(acc + u * O::kTiles);
      // the states' part, scaled row by row
      const f32x4 w = *reinterpret_cast<const f32x4*>((role ? s_d.onward : s_d.into) + 16 * blk + 4 * g) *
                      ((role ? 1.0f : p.scale) * factor);
      f32x4 inter = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        tmp[t] *= w;
        out[t] += tmp[t];
        if (p.dg) {
#pragma unroll
          for (int r = 0; r < 4; ++r) inter[r] += tmp[t][r] * Ty<DT>::f(s_own[TK::at(16 * blk + 4 * g + r, 16 * t + i)]);
        }
      }
#pragma unroll
      for (int u = 0; u < kRun / O::kStep; ++u) {
        if (role ? (u + 1) * O::kStep <= 16 * blk : u * O::kStep > 16 * blk + 15) continue;
#pragma unroll
        for (int t = 0; t < ND; ++t) out[t] = mma<DT>(dp[u], TK::column(s_other, u * O::kStep, 16 * t, lane), out[t]);
      }
      if (p.dg) {
        sum += lane_xor(sum, 16);
        sum += lane_xor(sum, 32);
        if (g == 0) s_sum[role][16 * blk + i] = sum;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int x = 1; x < 16; x *= 2) inter[r] += lane_xor(inter[r], x);
          if (i == 0) s_inter[role][16 * blk + 4 * g + r] = inter[r];
        }
        __syncthreads();
        if (wave == 0) {
          const double u = static_cast<double>(s_sum[0][lane]) - s_sum[1][lane] + s_inter[0][lane];
          const double kv = s_inter[1][lane];
          const double up = prefix_sum(u), all = __shfl(up, 63, 64);
          double dg = all - up + u + prefix_sum(kv) - kv;
          for (int vb = 0; vb < p.vblocks; ++vb) dg += p.dot[(bh * p.runs + run) * p.vblocks + vb];
          if (lane < rows) p.dg[(b * p.seqlen + t0 + lane) * p.heads + head] = static_cast<float>(dg);
        }
      }
    }
  }
  if (p.dg && wave == 0 && lane >= rows && t0 + lane < p.seqlen)
    for (int h = h0; h < h1; ++h) p.dg[(b * p.seqlen + t0 + lane) * p.heads + group * p.per + h] = 0.0f;
  const int64_t t = t0 + 16 * blk + 4 * g;
  const int64_t at = (((p.sets > 1 ? set * p.batch : 0) + b) * p.seqlen + t) * p.groups + group;
  void* const dst = role ? p.dk_out : p.dq;
#pragma unroll
  for (int c = 0; c < ND; ++c) {
    const int d = 16 * c + i;
    if (d >= dk) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (t + r >= p.seqlen) continue;
      const float v = 16 * blk + 4 * g + r < rows ? out[c][r] : 0.0f;
      const int64_t e = (at + r * p.groups) * p.dk + d;
      if (p.sets > 1) static_cast<float*>(dst)[e] = v;
      else static_cast<T*>(dst)[e] = Ty<DT>::from(v);
    }
  }
}

template <int DT>
static void launch_grad_t(const Grad& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.batch * p.runs * p.groups * p.sets));
  if (padded_dk(p.dk) == 64) hipLaunchKernelGGL((grad_kernel<DT, 64>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((grad_kernel<DT, 128>), grid, dim3(512), 0, s, p);
}
void launch_grad(const Grad& p, hipStream_t s) {
  switch (p.dtype) {
    case MM_F32: launch_grad_t<MM_F32>(p, s); break;
    case MM_F16: launch_grad_t<MM_F16>(p, s); break;
    default: launch_grad_t<MM_BF16>(p, s); break;
  }
}

}  // namespace dattn
}  // namespace mm
