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
// What a head needs, 48 KB with key_dim 128 in 16 bits, is loaded straight into shared memory while the head before is
// computed (two buffers, one barrier a head); fp32, whose buffers would not fit twice, and rows off 16 bytes go through
// registers instead.  8 sequences of 2048 tokens of 80 heads in bf16: 1.0 GB in 308 us, 3.3 TB/s; a head takes 4 us of a
// compute unit, of which its loads are 2.4 (reads that waited for the loads under way: 420 us).
#include <type_traits>

#include "decay_attention.h"
#include "decay_tiles.h"
#include "direct_load.h"

namespace mm {
namespace dattn {

// 16-bit types: operands of columns 16 t + i, over 32 rows of a tile, for N of t (Tile's column).  at[t]: where a lane's reads
// begin; ROWS: the first row.  The reads and their wait are one piece: of a transposing read in the compiler's hands it is not
// known where it reads, and each would wait for all direct loads under way.
#define MM_TR "ds_read_b64_tr_b16 "
template <typename TILE, int ROWS>
__device__ __forceinline__ void columns(const uint32_t (&at)[4], u32x4 (&o)[4]) {
  u32x2 r[8];
  constexpr int kA = ROWS * TILE::kLd * 2, kB = kA + 16 * TILE::kLd * 2;
  asm volatile(MM_TR "%0, %8 offset:%12\n" MM_TR "%1, %8 offset:%13\n" MM_TR "%2, %9 offset:%12\n" MM_TR "%3, %9 offset:%13\n"
               MM_TR "%4, %10 offset:%12\n" MM_TR "%5, %10 offset:%13\n" MM_TR "%6, %11 offset:%12\n" MM_TR "%7, %11 offset:%13\n"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
               : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(kA), "n"(kB)
               : "memory");
#pragma unroll
  for (int t = 0; t < 4; ++t) o[t] = u32x4{r[2 * t][0], r[2 * t][1], r[2 * t + 1][0], r[2 * t + 1][1]};
}
template <typename TILE, int ROWS>
__device__ __forceinline__ void columns(const uint32_t (&at)[8], u32x4 (&o)[8]) {
  u32x2 r[16];
  constexpr int kA = ROWS * TILE::kLd * 2, kB = kA + 16 * TILE::kLd * 2;
  asm volatile(MM_TR "%0, %16 offset:%24\n" MM_TR "%1, %16 offset:%25\n" MM_TR "%2, %17 offset:%24\n" MM_TR "%3, %17 offset:%25\n"
               MM_TR "%4, %18 offset:%24\n" MM_TR "%5, %18 offset:%25\n" MM_TR "%6, %19 offset:%24\n" MM_TR "%7, %19 offset:%25\n"
               MM_TR "%8, %20 offset:%24\n" MM_TR "%9, %20 offset:%25\n" MM_TR "%10, %21 offset:%24\n" MM_TR "%11, %21 offset:%25\n"
               MM_TR "%12, %22 offset:%24\n" MM_TR "%13, %22 offset:%25\n" MM_TR "%14, %23 offset:%24\n" MM_TR "%15, %23 offset:%25\n"
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]), "=&v"(r[8]),
                 "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
               : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]), "v"(at[7]), "n"(kA), "n"(kB)
               : "memory");
#pragma unroll
  for (int t = 0; t < 8; ++t) o[t] = u32x4{r[2 * t][0], r[2 * t][1], r[2 * t + 1][0], r[2 * t + 1][1]};
}
#undef MM_TR
// Where column4 of row 0 and column 16 t begins in a tile.  The rows' turn is the same 16 rows further on.
template <typename TILE, typename T, int N>
__device__ __forceinline__ void columns_at(const T* tile, int lane, uint32_t (&at)[N]) {
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const T*)tile));
#pragma unroll
  for (int t = 0; t < N; ++t) at[t] = base + TILE::at(0, 16 * t, 4 * (lane >> 4) + ((lane & 15) >> 2), 4 * (lane & 3)) * 2;
}

// FINE: of few tokens (decay_tiles.h, score_operand), with the rests of the states' roundings, which a run's tokens share: registers
// go to memory for it (310 us would be 650).
template <int DT, int DKP, bool DIRECT, bool ONE, bool FINE>
__global__ __launch_bounds__(512) void grad_kernel(const Grad p) {
  using T = typename Ty<DT>::T;
  using O = Op<DT>;
  using TK = Tile<DT, DKP>;
  using TV = Tile<DT, kVBlock>;
  constexpr int ND = DKP / 16, NU = kVBlock / O::kStep;
  constexpr int64_t kEs = sizeof(T);
  constexpr int kState = DIRECT ? kVBlock * DKP : 0, kRows = kRun * TV::kLd;  // elements of a buffer's parts
  __shared__ __attribute__((aligned(16))) T s_qk[2][kRun * TK::kLd];  // q, k
  __shared__ __attribute__((aligned(16))) T s_b0[2 * kState + 2 * kRows];  // S, dS, dy, v
  __shared__ __attribute__((aligned(16))) T s_b1[DIRECT ? 2 * kState + 2 * kRows : 8];
  __shared__ Decays s_d[2];
  __shared__ float s_sum[2][2][kRun], s_inter[2][2][kRun];  // M's row and column sums; the states' parts
  int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15;
  const int role = wave >> 2, blk = wave & 3;  // 0: dq, 1: dk

  uint32_t id = blockIdx.x;
  const int set = static_cast<int>(id % p.sets);
  id /= p.sets;
  const int64_t group = id % static_cast<uint32_t>(p.groups);
  id /= static_cast<uint32_t>(p.groups);
  const int64_t run = id % static_cast<uint32_t>(p.runs), b = id / static_cast<uint32_t>(p.runs);
  const int64_t len = length_of(p, b), t0 = run * kRun;
  const int rows = static_cast<int>(len - t0 < 0 ? 0 : len - t0 < kRun ? len - t0 : kRun);
  const int h0 = set * p.set_heads, h1 = h0 + p.set_heads < p.per ? h0 + p.set_heads : static_cast<int>(p.per);
  const int dk = static_cast<int>(p.dk), vblocks = ONE ? 1 : p.vblocks;

  f32x4 out[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) out[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (rows > 0) {
    {
      Staged<DT, DKP, 512> r;
      const char* const q = static_cast<const char*>(p.q) + (b * p.q_stride[0] + t0 * p.q_stride[1] + group * p.q_stride[2]) * kEs;
      const char* const k = static_cast<const char*>(p.k) + (b * p.k_stride[0] + t0 * p.k_stride[1] + group * p.k_stride[2]) * kEs;
      if (p.vec) {
        Staged<DT, DKP, 512> r2;
        r.load(q, static_cast<uint32_t>((r.row() * p.q_stride[1] + r.elem()) * kEs), r.kRows * p.q_stride[1] * kEs, rows, dk);
        r2.load(k, static_cast<uint32_t>((r.row() * p.k_stride[1] + r.elem()) * kEs), r.kRows * p.k_stride[1] * kEs, rows, dk);
        r.store(s_qk[0], static_cast<int>(threadIdx.x));
        r2.store(s_qk[1], static_cast<int>(threadIdx.x));
      } else {
        r.load_any(q, p.q_stride[1], rows, dk);
        r.store(s_qk[0], static_cast<int>(threadIdx.x));
        r.load_any(k, p.k_stride[1], rows, dk);
        r.store(s_qk[1], static_cast<int>(threadIdx.x));
      }
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
        A[ot] = mma<DT>(TK::row(s_other, 16 * ot, u * O::kStep, lane), TK::row(s_own, 16 * blk, u * O::kStep, lane), A[ot]);
    }

    // the own rows of q (or k) as the accumulators of the states' parts hold them (fp32: too many registers)
    uint32_t held[ND][2];
    if (p.dg && !O::kWide) {
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        T e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = s_own[TK::at(16 * blk + 4 * g + r, 16 * t + i)];
        __builtin_memcpy(held[t], e, 8);
      }
    }

    // A step is a head's block of value channels.
    const char* const dy0 = static_cast<const char*>(p.dy) + (b * p.dy_stride[0] + t0 * p.dy_stride[1]) * kEs;
    const char* const v0 = static_cast<const char*>(p.v) + (b * p.v_stride[0] + t0 * p.v_stride[1]) * kEs;
    Staged<DT, kVBlock, 512> ry, rv;
    // Where a lane's direct loads come from.  A state's row of DKP channels is DKP / 8 chunks of 16 bytes, and place c of it
    // holds chunk c ^ turn(row) (the 8 KB that the waves load at once are whole multiples of 16 rows, so that it is the same
    // for all); a row of 64 value channels is 8 chunks.
    const int unit = wave * 64 + lane;
    const uint32_t state_off = static_cast<uint32_t>(unit / (DKP / 8) * DKP * 2 + (unit % (DKP / 8) ^ TK::turn(unit / (DKP / 8))) * 16);
    const int row_here = unit / 8, chunk_here = unit % 8 ^ TV::turn(unit / 8);
    const uint32_t dy_off = static_cast<uint32_t>(row_here * p.dy_stride[1] * kEs) + chunk_here * 16;
    const uint32_t v_off = static_cast<uint32_t>(row_here * p.v_stride[1] * kEs) + chunk_here * 16;
    auto fetch = [&](T* buf, int h, int vb) __attribute__((always_inline)) {
      const int64_t head = group * p.per + h;
      const int vw = static_cast<int>(p.dv - vb * kVBlock < kVBlock ? p.dv - vb * kVBlock : kVBlock);
      const char* const dy = dy0 + (head * p.dy_stride[2] + vb * kVBlock) * kEs;
      const char* const v = v0 + (head * p.v_stride[2] + vb * kVBlock) * kEs;
      if constexpr (DIRECT) {
        char* const to = reinterpret_cast<char*>(buf);
        constexpr int kBytes = kState * static_cast<int>(kEs);
        const int64_t block = ((b * p.heads + head) * p.runs + run) * vblocks + vb;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
          const char* const from = static_cast<const char*>(which ? p.dstates : p.states) + block * kBytes;
#pragma unroll
          for (int q = 0; q < kBytes / 8192; ++q) load_direct(from, q * 8192 + state_off, to + which * kBytes + (q * 8 + wave) * 1024);
        }
        char* const dy_to = to + 2 * kBytes + wave * 1024;
        const bool in = row_here < rows && chunk_here * 8 < vw;
        load_direct(dy, in ? dy_off : kNowhere, dy_to);
        load_direct(v, in ? v_off : kNowhere, dy_to + kRows * kEs);
      } else {
        if (p.vec) {
          ry.load(dy, static_cast<uint32_t>((ry.row() * p.dy_stride[1] + ry.elem()) * kEs), ry.kRows * p.dy_stride[1] * kEs, rows, vw);
          rv.load(v, static_cast<uint32_t>((rv.row() * p.v_stride[1] + rv.elem()) * kEs), rv.kRows * p.v_stride[1] * kEs, rows, vw);
        } else {
          ry.load_any(dy, p.dy_stride[1], rows, vw);
          rv.load_any(v, p.v_stride[1], rows, vw);
        }
      }
    };
    auto gate = [&](int h) {
      return lane < rows ? load_gate(p, b * p.g_stride[0] + (t0 + lane) * p.g_stride[1] + (group * p.per + h) * p.g_stride[2]) : 0u;
    };
    // what the head needs of its states' product and (fp16) powers of two, a step ahead
    auto dot_of = [&](int h) {
      const float* const from = p.dot + ((b * p.heads + group * p.per + h) * p.runs + run) * vblocks;
      float dot = from[0];
      for (int vb = 1; vb < vblocks; ++vb) dot += from[vb];
      return dot;
    };
    auto factor_of = [&](int h, int vb) {
      return (role ? p.dfactors : p.factors)[((b * p.heads + group * p.per + h) * p.runs + run) * vblocks + vb];
    };
    uint32_t g_ahead = 0;  // the next head's log decays
    if (wave == 7 && h0 + 1 < h1) g_ahead = gate(h0 + 1);
    float dot_here = 0.0f, dot_before = 0.0f, factor_here = 1.0f;
    if (p.dg && wave == 0) dot_here = dot_of(h0);
    if (DT == MM_F16) factor_here = factor_of(h0, 0);
    // dg of a head whose parts all waves have left
    auto finish_dg = [&](int h, float dot) __attribute__((always_inline)) {
      const int64_t head = group * p.per + h;
      const float* const sum = &s_sum[(h - h0) & 1][0][0];
      const float* const inter = &s_inter[(h - h0) & 1][0][0];
      const double u = static_cast<double>(sum[lane]) - sum[kRun + lane] + inter[lane];
      const double kv = inter[kRun + lane];
      const double up = prefix_sum(u), all = __shfl(up, 63, 64);
      const double dg = all - up + u + prefix_sum(kv) - kv + dot;
      if (lane < rows) p.dg[(b * p.seqlen + t0 + lane) * p.heads + head] = static_cast<float>(dg);
    };

    f32x4 acc[4], tmp[ND];
    float factor = 1.0f;
    auto step = [&](T* cur, T* other, int h, int vb) __attribute__((always_inline)) {
      asm volatile("" : "+v"(lane));
      const int64_t head = group * p.per + h, bh = b * p.heads + head;
      const bool last_block = vb + 1 == vblocks, more = !last_block || h + 1 < h1;
      const int h_next = last_block ? h + 1 : h, vb_next = last_block ? 0 : vb + 1;
      if constexpr (!DIRECT) {
        __syncthreads();
        ry.store(cur + 2 * kState, static_cast<int>(threadIdx.x));
        rv.store(cur + 2 * kState + kRows, static_cast<int>(threadIdx.x));
      }
      if constexpr (DIRECT) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's direct loads of the step
      __syncthreads();
      const bool decays_now = wave == 7 && last_block && h + 1 < h1;
      const uint32_t g_next = g_ahead;
      if (decays_now && h + 2 < h1) g_ahead = gate(h + 2);
      float factor_next = 1.0f;
      if (DT == MM_F16 && more) factor_next = factor_of(h_next, vb_next);
      if (p.dg && wave == 0 && vb == 0) {
        const float dot_next = h + 1 < h1 ? dot_of(h + 1) : 0.0f;
        if (h > h0) finish_dg(h - 1, dot_before);
        dot_before = dot_here;
        dot_here = dot_next;
      }
      if (more) fetch(other, h_next, vb_next);  // (behind the loads that are waited for first)
      const Decays& D = s_d[(h - h0) & 1];
      if (ONE || vb == 0) {
#pragma unroll
        for (int ot = 0; ot < 4; ++ot) acc[ot] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < ND; ++t) tmp[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        factor = DT == MM_F16 ? 0.0f : 1.0f;
      }
      const T* const own_t = cur + 2 * kState + role * kRows;
      const T* const other_t = cur + 2 * kState + (1 - role) * kRows;
      const T* const state = DIRECT ? cur + role * kState
                                    : static_cast<const T*>(role ? p.dstates : p.states) + ((bh * p.runs + run) * vblocks + vb) * kVBlock * DKP;
      // columns d of the state, 16 t on, over its value channels
      auto state_operand = [&](int u, int t) __attribute__((always_inline)) {
        if constexpr (O::kWide) {
          return *reinterpret_cast<const u32x4*>(state + ((u * ND + t) * 64 + lane) * 4);
        } else {
          T e[O::kE];
#pragma unroll
          for (int j = 0; j < O::kE; ++j) e[j] = state[(u * O::kStep + 16 * (j >> 2) + 4 * g + (j & 3)) * DKP + 16 * t + i];
          u32x4 w;
          __builtin_memcpy(&w, e, 16);
          return w;
        }
      };
      u32x4 own[NU];
#pragma unroll
      for (int u = 0; u < NU; ++u) own[u] = TV::row_acc(own_t, 16 * blk, u * O::kStep, lane);
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int ot = 0; ot < 4; ++ot)
          if (role ? ot >= blk : ot <= blk) acc[ot] = mma<DT>(TV::row_acc(other_t, 16 * ot, u * O::kStep, lane), own[u], acc[ot]);
      // fp16: the sum over blocks stands in the largest of their powers of two, to which the other blocks' parts come down.  (Up to
      // a smaller one, of a block whose states have decayed to nearly nothing, finite sums would overflow.)
      constexpr bool kJoin = DT == MM_F16 && !ONE;
      float part = 1.0f;
      if constexpr (DT == MM_F16) {
        if constexpr (kJoin) {
          const float top = fmaxf(factor, factor_here), down = factor / top;
#pragma unroll
          for (int t = 0; t < ND; ++t) tmp[t] *= down;
          part = factor_here / top;
          factor = top;
        } else {
          factor = factor_here;
        }
        factor_here = factor_next;
      }
      auto add_block = [&](u32x4 a, u32x4 o, f32x4& to) __attribute__((always_inline)) {
        if constexpr (kJoin) to += mma<DT>(a, o, f32x4{0.0f, 0.0f, 0.0f, 0.0f}) * part;
        else to = mma<DT>(a, o, to);
      };
      auto add_state = [&](auto first) __attribute__((always_inline)) {
        constexpr int u = decltype(first)::value;
        if constexpr (DIRECT) {
          u32x4 o[ND];
          uint32_t at[ND];
          columns_at<TK>(state, lane, at);
          columns<TK, u * 32>(at, o);
#pragma unroll
          for (int t = 0; t < ND; ++t) add_block(own[u], o[t], tmp[t]);
        } else {
#pragma unroll
          for (int t = 0; t < ND; ++t) add_block(own[u], state_operand(u, t), tmp[t]);
        }
      };
      add_state(std::integral_constant<int, 0>{});
      add_state(std::integral_constant<int, 1>{});
      if constexpr (NU == 4) {
        add_state(std::integral_constant<int, 2>{});
        add_state(std::integral_constant<int, 3>{});
      }
      if constexpr (FINE) {
        const T* const from = static_cast<const T*>(role ? p.drests : p.rests) + ((bh * p.runs + run) * vblocks + vb) * kVBlock * DKP;
#pragma unroll 1
        for (int t = 0; t < ND; ++t) {
          f32x4 more = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            T e[O::kE];
#pragma unroll
            for (int j = 0; j < O::kE; ++j) e[j] = from[(u * O::kStep + 16 * (j >> 2) + 4 * g + (j & 3)) * DKP + 16 * t + i];
            u32x4 w;
            __builtin_memcpy(&w, e, 16);
            more = mma<DT>(own[u], w, more);
          }
#pragma unroll
          for (int k = 0; k < ND; ++k) tmp[k] += k == t ? more * (part / kRestUp) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
      }
      if (!last_block) return;
      // dP and M
      const float hi_r = D.hi[16 * blk + i], lo_r = D.lo[16 * blk + i];
      float sum = 0.0f;
#pragma unroll
      for (int ot = 0; ot < 4; ++ot) {
        if (role ? ot < blk : ot > blk) continue;
        const f32x4 hi = *reinterpret_cast<const f32x4*>(D.hi + 16 * ot + 4 * g);
        const f32x4 lo = *reinterpret_cast<const f32x4*>(D.lo + 16 * ot + 4 * g);
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float decay = between<DT>(hi_r, lo_r, hi[r], lo[r], role != 0);
          acc[ot][r] *= p.scale * decay;
          x[r] = acc[ot][r] * A[ot][r];
        }
        if (ot == blk) {  // the diagonal's tile
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const bool in = role ? 4 * g + r >= i : 4 * g + r <= i;
            acc[ot][r] = in ? acc[ot][r] : 0.0f;
            x[r] = in ? x[r] : 0.0f;
          }
        }
        sum += (x[0] + x[1]) + (x[2] + x[3]);
      }
      constexpr bool kRange = DT == MM_F16;
      float up = 1.0f, down = 1.0f;
      if constexpr (kRange) {
        score_range(largest(acc), up, down);
#pragma unroll
        for (int ot = 0; ot < 4; ++ot) acc[ot] *= up;
      }
      constexpr bool fine = FINE;
      u32x4 dp[kRun / O::kStep], rest[kRun / O::kStep];
#pragma unroll
      for (int u = 0; u < kRun / O::kStep; ++u) score_operand<DT>(acc + u * O::kTiles, fine, dp[u], rest[u]);
      // the states' part, scaled row by row
      const f32x4 w = *reinterpret_cast<const f32x4*>((role ? D.onward : D.into) + 16 * blk + 4 * g) * ((role ? 1.0f : p.scale) * factor);
      f32x4 inter = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if constexpr (!kRange) {
#pragma unroll
        for (int t = 0; t < ND; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) out[t][r] = __builtin_fmaf(tmp[t][r], w[r], out[t][r]);
      }
      if (p.dg) {
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          float x[4];
          if constexpr (O::kWide) {
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = Ty<DT>::f(s_own[TK::at(16 * blk + 4 * g + r, 16 * t + i)]);
          } else {
            unpack2<DT>(held[t][0], x[0], x[1]);
            unpack2<DT>(held[t][1], x[2], x[3]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) inter[r] = __builtin_fmaf(tmp[t][r], x[r], inter[r]);
        }
        inter *= w;
      }
      // fp16: the head's gradients gather in the states' part, in the units of each row's scores
      if constexpr (kRange) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float to = w[r] * __shfl(up, 4 * g + r, 64);
#pragma unroll
          for (int t = 0; t < ND; ++t) tmp[t][r] *= to;
        }
      }
      auto& gather = [&]() -> auto& {
        if constexpr (kRange) return tmp;
        else return out;
      }();
      auto add_rows = [&](auto first) __attribute__((always_inline)) {
        constexpr int u = decltype(first)::value;
        if (role ? (u + 1) * O::kStep <= 16 * blk : u * O::kStep > 16 * blk + 15) return;
        if constexpr (DIRECT) {
          u32x4 o[ND];
          uint32_t at[ND];
          columns_at<TK>(s_other, lane, at);
          columns<TK, u * 32>(at, o);
#pragma unroll
          for (int t = 0; t < ND; ++t) gather[t] = mma<DT>(dp[u], o[t], gather[t]);
          if (fine) {
#pragma unroll
            for (int t = 0; t < ND; ++t) gather[t] = mma_rest<DT>(rest[u], o[t], gather[t]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < ND; ++t) gather[t] = mma<DT>(dp[u], TK::column(s_other, u * O::kStep, 16 * t, lane), gather[t]);
          if (fine) {
#pragma unroll
            for (int t = 0; t < ND; ++t) gather[t] = mma_rest<DT>(rest[u], TK::column(s_other, u * O::kStep, 16 * t, lane), gather[t]);
          }
        }
      };
      add_rows(std::integral_constant<int, 0>{});
      add_rows(std::integral_constant<int, 1>{});
      if constexpr (NU == 4) {
        add_rows(std::integral_constant<int, 2>{});
        add_rows(std::integral_constant<int, 3>{});
      }
      if constexpr (kRange) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float back = __shfl(down, 4 * g + r, 64);
#pragma unroll
          for (int t = 0; t < ND; ++t) out[t][r] = __builtin_fmaf(tmp[t][r], back, out[t][r]);
        }
      }
      if (p.dg) {
        sum += lane_xor(sum, 16);
        sum += lane_xor(sum, 32);
        if (g == 0) s_sum[(h - h0) & 1][role][16 * blk + i] = sum;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int x = 1; x < 16; x *= 2) inter[r] += lane_xor(inter[r], x);
        }
        if (i == 0) *reinterpret_cast<f32x4*>(&s_inter[(h - h0) & 1][role][16 * blk + 4 * g]) = inter;
      }
      if (decays_now) run_decays(s_d[(h + 1 - h0) & 1], gate_value(p, g_next), lane);
    };
    if (wave == 7) run_decays(s_d[0], gate_value(p, gate(h0)), lane);
    fetch(s_b0, h0, 0);
    const int steps = (h1 - h0) * vblocks;
    int h = h0, vb = 0;
    auto advance = [&] {
      if (++vb == vblocks) {
        vb = 0;
        ++h;
      }
    };
    if constexpr (DIRECT) {
      int n = 0;
      for (; n + 1 < steps; n += 2) {
        step(s_b0, s_b1, h, vb);
        advance();
        step(s_b1, s_b0, h, vb);
        advance();
      }
      if (n < steps) step(s_b0, s_b1, h, vb);
    } else {
      for (int n = 0; n < steps; ++n) {
        step(s_b0, s_b0, h, vb);
        advance();
      }
    }
    __syncthreads();
    if (p.dg && wave == 0) finish_dg(h1 - 1, dot_before);
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

template <int DT, int DKP, bool FINE>
static void launch_grad_f(const Grad& p, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(p.batch * p.runs * p.groups * p.sets));
  constexpr bool kDirect = DT != MM_F32;
  if constexpr (kDirect) {
    if (p.vec) {
      if (p.vblocks == 1) hipLaunchKernelGGL((grad_kernel<DT, DKP, kDirect, true, FINE>), grid, dim3(512), 0, s, p);
      else hipLaunchKernelGGL((grad_kernel<DT, DKP, kDirect, false, FINE>), grid, dim3(512), 0, s, p);
      return;
    }
  }
  hipLaunchKernelGGL((grad_kernel<DT, DKP, false, false, FINE>), grid, dim3(512), 0, s, p);
}
template <int DT, int DKP>
static void launch_grad_t(const Grad& p, hipStream_t s) {
  if constexpr (DT != MM_F32) {
    if (p.rests) return launch_grad_f<DT, DKP, true>(p, s);
  }
  launch_grad_f<DT, DKP, false>(p, s);
}
template <int DT>
static void launch_grad_d(const Grad& p, hipStream_t s) {
  if (padded_dk(p.dk) == 64) launch_grad_t<DT, 64>(p, s); else launch_grad_t<DT, 128>(p, s);
}
void launch_grad(const Grad& p, hipStream_t s) {
  switch (p.dtype) {
    case MM_F32: launch_grad_d<MM_F32>(p, s); break;
    case MM_F16: launch_grad_d<MM_F16>(p, s); break;
    default: launch_grad_d<MM_BF16>(p, s); break;
  }
}

}  // namespace dattn
}  // namespace mm
