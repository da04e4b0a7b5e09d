// What the kernels of decaying linear attention are given, and how their workspaces are laid out.
#pragma once

#include "mm_common.h"

#include "decay_shape.h"

namespace mm {
namespace dattn {

// The pass over the tokens (decay_pass.h), forward or mirrored: mirrored, q is k, k is q, v is dy, y is dv, init the
// gradient of the final state and final_state that of the first.
struct Pass {
  const void *q, *k, *v, *g;
  const float* init;      // (batch, heads, dk, dv) or NULL
  float* final_state;     // or NULL
  void* y;                // (batch, seqlen, heads, dv) contiguous
  const void* lengths;
  void* states;           // the state before (mirrored: its gradient after) each run, or NULL
  float* factors;         // fp16: the power of two each of them was divided by
  void* state_rests;      // `fine`: what the 16-bit states leave of the fp32 ones, or NULL
  const void* rests_with; // mirrored, `fine`: the forward pass's, for the products
  const void* dot_with;   // mirrored: the forward pass's states and their factors, and where their products with
  const float* factors_with;  // this pass's go, (batch, heads, runs, vblocks); NULL = not wanted
  float* dot;
  float* seg_states;      // segments: what each adds, then the state before each
  double* seg_decay;
  int64_t q_stride[3], k_stride[3], v_stride[3], g_stride[3];  // batch, time, head
  int64_t batch, seqlen, heads, per, dk, dv, runs, seg_runs;
  int32_t vblocks, segments, vec, dtype, g_dtype, lengths_dtype, fine;
  float scale;
};

// Gradients of q, k and the log decays from the states on both sides of each run (decay_attention_bwd.hip).
struct Grad {
  const void *q, *k, *v, *dy, *g, *lengths;
  const void *states, *dstates, *rests, *drests;  // the last two: `fine`, or NULL
  const float *factors, *dfactors, *dot;
  void *dq, *dk_out;      // (batch, seqlen, groups, dk) contiguous; with sets > 1 fp32 (sets, batch, seqlen, groups, dk)
  float* dg;              // (batch, seqlen, heads) or NULL
  int64_t q_stride[3], k_stride[3], v_stride[3], dy_stride[3], g_stride[3];
  int64_t batch, seqlen, heads, groups, per, dk, dv, runs;
  int32_t vblocks, sets, set_heads, vec, dtype, g_dtype, lengths_dtype;
  float scale;
};

struct Step {
  const float* state;
  float* state_out;
  const void *q, *k, *v, *g;
  void* y;
  int64_t q_stride[2], k_stride[2], v_stride[2], g_stride[2], y_stride[2];  // batch, head
  int64_t batch, heads, per, dk, dv;
  int32_t vblocks, vec;
  float scale;
};

inline int padded_dk(int64_t dk) { return dk <= 64 ? 64 : 128; }

void launch_pass_forward(const Pass& p, hipStream_t s);
void launch_pass_mirrored(const Pass& p, hipStream_t s);
void launch_grad(const Grad& p, hipStream_t s);

template <typename P>
__device__ __forceinline__ int64_t length_of(const P& p, int64_t b) {
  if (!p.lengths) return p.seqlen;
  const int64_t n = p.lengths_dtype ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
  return n < 0 ? 0 : n < p.seqlen ? n : p.seqlen;
}
// A log decay: the load, and what it stands for, apart, so that the load's time can pass between them.
template <typename P>
__device__ __forceinline__ uint32_t load_gate(const P& p, int64_t at) {
  return p.g_dtype == MM_F32 ? static_cast<const uint32_t*>(p.g)[at] : static_cast<const uint16_t*>(p.g)[at];
}
template <typename P>
__device__ __forceinline__ float gate_value(const P& p, uint32_t raw) {
  return p.g_dtype == MM_F32   ? __uint_as_float(raw)
         : p.g_dtype == MM_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(raw)))
                               : __uint_as_float(raw << 16);
}
typedef float seg_f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ seg_f32x4* seg_state(const Pass& p, int64_t bh, int seg, int vb) {
  const int64_t dkp = p.dk <= 64 ? 64 : 128;
  return reinterpret_cast<seg_f32x4*>(p.seg_states) + ((bh * p.segments + seg) * p.vblocks + vb) * 16 * dkp;
}
}  // namespace dattn
}  // namespace mm
