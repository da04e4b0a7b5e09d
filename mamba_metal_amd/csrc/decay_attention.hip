// Linear attention with a decay for each head: the forward pass's launches, the token step and the C entries.
#include "decay_pass.h"
#include "reduce_rows.h"

namespace mm {
namespace dattn {

void launch_pass_forward(const Pass& p, hipStream_t s) { launch_pass<false>(p, s); }

// One token of a head and 64 value channels: 16 rows of the state at a time, 16 lanes of 4 channels each.  The state is
// read and written once, which is all its time: 64 sequences of 80 heads of 128 by 64, 337 MB, in 60 us, 5.6 TB/s; one
// sequence of 24 heads 4.6 us, a chain of three loads (all of a thread's rows ahead of the barrier: no faster).
template <int DT, int GT>
__global__ __launch_bounds__(256) void step_kernel(const Step p) {
  using T = typename Ty<DT>::T;
  __shared__ float s_y[16][kVBlock + 4];
  __shared__ float s_q[kMaxDk], s_k[kMaxDk];
  uint32_t id = blockIdx.x;
  const int vb = static_cast<int>(id % p.vblocks);
  id /= p.vblocks;
  const int64_t head = id % p.heads, b = id / p.heads, group = head / p.per;
  const int row = threadIdx.x >> 4, c = (threadIdx.x & 15) * 4, v0 = vb * kVBlock + c;
  const int dk = static_cast<int>(p.dk);
  if (static_cast<int>(threadIdx.x) < dk) {
    s_q[threadIdx.x] = ld<DT>(p.q, b * p.q_stride[0] + group * p.q_stride[1] + threadIdx.x) * p.scale;
    s_k[threadIdx.x] = ld<DT>(p.k, b * p.k_stride[0] + group * p.k_stride[1] + threadIdx.x);
  }
  float gate = ld<GT>(p.g, b * p.g_stride[0] + head * p.g_stride[1]);
  const float a = gate != gate ? gate : exp2_acc(gate * kLog2e);
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    v[j] = v0 + j < p.dv ? ld<DT>(p.v, b * p.v_stride[0] + head * p.v_stride[1] + v0 + j) : 0.0f;
  __syncthreads();
  const int64_t base = (b * p.heads + head) * p.dk * p.dv;
  float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.vec) {
    if (v0 < p.dv) {
#pragma unroll 4
      for (int d = row; d < dk; d += 16) {
        const int64_t at = base + static_cast<int64_t>(d) * p.dv + v0;
        f32x4 s = *reinterpret_cast<const f32x4*>(p.state + at);
        const float q = s_q[d], k = s_k[d];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[j] = __builtin_fmaf(a, s[j], k * v[j]);
          y[j] = __builtin_fmaf(q, s[j], y[j]);
        }
        *reinterpret_cast<f32x4*>(p.state_out + at) = s;
      }
    }
  } else {
    for (int d = row; d < dk; d += 16) {
      const float q = s_q[d], k = s_k[d];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (v0 + j < p.dv) {
          const int64_t at = base + static_cast<int64_t>(d) * p.dv + v0 + j;
          const float s = __builtin_fmaf(a, p.state[at], k * v[j]);
          p.state_out[at] = s;
          y[j] = __builtin_fmaf(q, s, y[j]);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s_y[row][c + j] = y[j];
  __syncthreads();
  if (threadIdx.x < kVBlock && vb * kVBlock + static_cast<int>(threadIdx.x) < p.dv) {
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) sum += s_y[r][threadIdx.x];
    static_cast<T*>(p.y)[b * p.y_stride[0] + head * p.y_stride[1] + vb * kVBlock + threadIdx.x] = Ty<DT>::from(sum);
  }
}

// Sums of the sets' gradients, in order.
template <int DT>
__global__ __launch_bounds__(256) void sum_sets_kernel(const float* part, void* out, int64_t n, int sets) {
  const int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (e >= n) return;
  float s = part[e];
  for (int k = 1; k < sets; ++k) s += part[k * n + e];
  st<DT>(out, e, s);
}

// The gradient of a decay that all tokens share.
__global__ __launch_bounds__(64 * rows::kGroups) void sum_heads_kernel(const float* part, float* out, int64_t nrows, int64_t heads) {
  rows::sum_columns(part, nrows, heads, blockIdx.x, 0, nrows, [&](int64_t c, double s) { out[c] = static_cast<float>(s); });
}

// ------------------------------------------------------------------------------------------------------------- host
// The regions of a call's workspace.
struct Layout {
  int64_t seg_states, seg_decay, dstates, dfactors, drests, dot, parts, dg, total;
};
static Layout layout_of(const Shape& s, int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t dk, int64_t dv,
                        int32_t dtype, bool backward) {
  Layout l{};
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += round_up(bytes, 256);
    return was;
  };
  const int64_t bh = batch * heads, block = static_cast<int64_t>(s.vblocks) * kVBlock * padded_dk(dk);
  if (s.segments > 1) {
    l.seg_states = take(bh * s.segments * block * 4);
    l.seg_decay = take(bh * s.segments * 8);
  }
  if (backward) {
    l.dstates = take(bh * s.runs * block * dtype_size(dtype));
    l.dfactors = take(dtype == MM_F16 ? bh * s.runs * s.vblocks * 4 : 0);
    l.drests = take(fine_scores(batch, seqlen, heads, dtype) ? bh * s.runs * block * dtype_size(dtype) : 0);
    l.dot = take(bh * s.runs * s.vblocks * 4);
    l.parts = take(s.sets > 1 ? 2 * s.sets * batch * seqlen * groups * dk * 4 : 0);
    l.dg = take(rows::floats(batch * seqlen, heads) * 4);
  }
  l.total = at;
  return l;
}

static int64_t states_bytes(const Shape& s, int64_t batch, int64_t heads, int64_t dk, int32_t dtype) {
  return round_up(batch * heads * s.runs * s.vblocks * kVBlock * padded_dk(dk) * dtype_size(dtype), 256);
}

// Behind the states: fp16's powers of two, and the rests of calls with fine scores.
static int64_t rests_at(const Shape& s, int64_t batch, int64_t heads, int64_t dk, int32_t dtype) {
  return states_bytes(s, batch, heads, dk, dtype) + (dtype == MM_F16 ? round_up(batch * heads * s.runs * s.vblocks * 4, 256) : 0);
}

static int check_strides(const int64_t* s, const char* name) {
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0) return fail(MM_ERR_LAYOUT, "%s has a negative stride", name);
  return MM_OK;
}
// 16 bytes at a time: aligned rows of a width that 16 bytes divide, a run of them within 32-bit offsets.
static bool vec_ok(const void* p, const int64_t* s, int64_t width, int32_t dtype) {
  const int64_t e = 16 / dtype_size(dtype);
  bool ok = aligned(p, 16) && width % e == 0 && s[1] < (int64_t{1} << 23);
  for (int i = 0; i < 3; ++i) ok = ok && s[i] % e == 0;
  return ok;
}
// The pass's output, 4 channels at a time.
static bool out_ok(const void* p, int64_t width) { return aligned(p, 16) && width % 4 == 0; }

static int check_common(const mm_decay_attention_params* p) {
  if (!p) return fail(MM_ERR_NULL_POINTER, "params is NULL");
  if (!valid_dtype(p->dtype) || !valid_dtype(p->log_decay_dtype)) return fail(MM_ERR_DTYPE, "dtype %d, log_decay's %d", p->dtype, p->log_decay_dtype);
  if (p->lengths && p->lengths_dtype != 0 && p->lengths_dtype != 1) return fail(MM_ERR_DTYPE, "lengths_dtype %d", p->lengths_dtype);
  if (p->key_dim < 1 || p->key_dim > kMaxDk) return fail(MM_ERR_SHAPE, "key_dim %lld is not 1 to %d", (long long)p->key_dim, kMaxDk);
  if (p->value_dim < 1 || p->value_dim > kMaxDv) return fail(MM_ERR_SHAPE, "value_dim %lld is not 1 to %lld", (long long)p->value_dim, (long long)kMaxDv);
  if (p->heads < 1 || p->groups < 1 || p->heads % p->groups) return fail(MM_ERR_SHAPE, "%lld heads in %lld groups", (long long)p->heads, (long long)p->groups);
  if (!sizes_ok(p->batch, p->seqlen, p->heads, p->groups, p->key_dim, p->value_dim))
    return fail(MM_ERR_SHAPE, "batch %lld, seqlen %lld, heads %lld: negative or too large", (long long)p->batch, (long long)p->seqlen, (long long)p->heads);
  return MM_OK;
}
static int check_inputs(const mm_decay_attention_params* p) {
  if (!p->q || !p->k || !p->v || !p->log_decay) return fail(MM_ERR_NULL_POINTER, "q, k, v and log_decay are required");
  int e;
  if ((e = check_strides(p->q_stride, "q")) != MM_OK || (e = check_strides(p->k_stride, "k")) != MM_OK ||
      (e = check_strides(p->v_stride, "v")) != MM_OK || (e = check_strides(p->log_decay_stride, "log_decay")) != MM_OK)
    return e;
  return MM_OK;
}
static int check_workspace(const mm_decay_attention_params* p, int64_t need) {
  if (need > 0 && (!p->workspace || !aligned(p->workspace, 256) || p->workspace_bytes < static_cast<size_t>(need)))
    return fail(MM_ERR_WORKSPACE, "needs %lld bytes of 256-byte aligned workspace", (long long)need);
  return MM_OK;
}
// Either pass's parameters; q and k, v and dy, states and outputs are filled in by the caller.
static Pass pass_of(const mm_decay_attention_params* p, const Shape& s, const Layout& l) {
  Pass k{};
  char* const ws = static_cast<char*>(p->workspace);
  k.g = p->log_decay;
  k.lengths = p->lengths;
  for (int i = 0; i < 3; ++i) k.g_stride[i] = p->log_decay_stride[i];
  k.batch = p->batch;
  k.seqlen = p->seqlen;
  k.heads = p->heads;
  k.per = p->heads / p->groups;
  k.dk = p->key_dim;
  k.dv = p->value_dim;
  k.runs = s.runs;
  k.seg_runs = s.seg_runs;
  k.vblocks = s.vblocks;
  k.segments = s.segments;
  k.dtype = p->dtype;
  k.g_dtype = p->log_decay_dtype;
  k.lengths_dtype = p->lengths_dtype;
  k.scale = p->scale;
  k.fine = fine_scores(p->batch, p->seqlen, p->heads, p->dtype);
  if (s.segments > 1) {
    k.seg_states = reinterpret_cast<float*>(ws + l.seg_states);
    k.seg_decay = reinterpret_cast<double*>(ws + l.seg_decay);
  }
  return k;
}
static void set(const void*& to, int64_t* to_stride, const void* from, const int64_t* stride) {
  to = from;
  for (int i = 0; i < 3; ++i) to_stride[i] = stride[i];
}

}  // namespace dattn
}  // namespace mm

extern "C" {

size_t mm_decay_attention_states_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t key_dim, int64_t value_dim,
                                      int32_t dtype) {
  using namespace mm;
  using namespace mm::dattn;
  if (!valid_dtype(dtype) || !sizes_ok(batch, seqlen, heads, 1, key_dim, value_dim)) return 0;
  const Shape s = shape_of(batch, seqlen, heads, 1, value_dim, dtype);
  return static_cast<size_t>(rests_at(s, batch, heads, key_dim, dtype) +
                             (fine_scores(batch, seqlen, heads, dtype) ? states_bytes(s, batch, heads, key_dim, dtype) : 0));
}

size_t mm_decay_attention_workspace_size(int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t key_dim,
                                         int64_t value_dim, int32_t dtype, int32_t backward) {
  using namespace mm;
  using namespace mm::dattn;
  if (!valid_dtype(dtype) || !sizes_ok(batch, seqlen, heads, groups, key_dim, value_dim) || batch == 0) return 0;
  const Shape s = shape_of(batch, seqlen, heads, groups, value_dim, dtype);
  return static_cast<size_t>(layout_of(s, batch, seqlen, heads, groups, key_dim, value_dim, dtype, backward != 0).total);
}

int mm_decay_attention_fwd(const mm_decay_attention_params* p, void* stream) {
  using namespace mm;
  using namespace mm::dattn;
  clear_error();
  int e = check_common(p);
  if (e != MM_OK || p->batch == 0) return e;
  if (p->seqlen > 0) {
    if ((e = check_inputs(p)) != MM_OK) return e;
    if (!p->y) return fail(MM_ERR_NULL_POINTER, "y is required");
  }
  if (p->run_states && !aligned(p->run_states, 256)) return fail(MM_ERR_LAYOUT, "run_states must be 256-byte aligned");
  const Shape s = shape_of(p->batch, p->seqlen, p->heads, p->groups, p->value_dim, p->dtype);
  const Layout l = layout_of(s, p->batch, p->seqlen, p->heads, p->groups, p->key_dim, p->value_dim, p->dtype, false);
  if ((e = check_workspace(p, l.total)) != MM_OK) return e;
  Pass k = pass_of(p, s, l);
  set(k.q, k.q_stride, p->q, p->q_stride);
  set(k.k, k.k_stride, p->k, p->k_stride);
  set(k.v, k.v_stride, p->v, p->v_stride);
  k.vec = vec_ok(k.q, k.q_stride, k.dk, k.dtype) && vec_ok(k.k, k.k_stride, k.dk, k.dtype) &&
          vec_ok(k.v, k.v_stride, k.dv, k.dtype) && out_ok(p->y, k.dv);
  k.init = p->h0;
  k.final_state = p->state_out;
  k.y = p->y;
  k.states = p->run_states;
  if (k.states && p->dtype == MM_F16)
    k.factors = reinterpret_cast<float*>(static_cast<char*>(k.states) + states_bytes(s, p->batch, p->heads, p->key_dim, p->dtype));
  if (k.states && k.fine) k.state_rests = static_cast<char*>(k.states) + rests_at(s, p->batch, p->heads, p->key_dim, p->dtype);
  launch_pass_forward(k, static_cast<hipStream_t>(stream));
  return check_launch("decay_attention_fwd");
}

int mm_decay_attention_bwd(const mm_decay_attention_params* p, void* stream) {
  using namespace mm;
  using namespace mm::dattn;
  clear_error();
  int e = check_common(p);
  if (e != MM_OK || p->batch == 0) return e;
  if (p->seqlen > 0) {
    if ((e = check_inputs(p)) != MM_OK) return e;
    if (p->dlog_decay && p->dlog_decay_heads) return fail(MM_ERR_SHAPE, "one of dlog_decay and dlog_decay_heads");
    if (!p->dy || !p->run_states) return fail(MM_ERR_NULL_POINTER, "dy and run_states are required");
    if (!p->dq || !p->dk || !p->dv) return fail(MM_ERR_NULL_POINTER, "dq, dk and dv are required");
    if ((e = check_strides(p->dy_stride, "dy")) != MM_OK) return e;
    if (!aligned(p->run_states, 256)) return fail(MM_ERR_LAYOUT, "run_states must be 256-byte aligned");
  }
  const Shape s = shape_of(p->batch, p->seqlen, p->heads, p->groups, p->value_dim, p->dtype);
  const Layout l = layout_of(s, p->batch, p->seqlen, p->heads, p->groups, p->key_dim, p->value_dim, p->dtype, true);
  if ((e = check_workspace(p, l.total)) != MM_OK) return e;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* const ws = static_cast<char*>(p->workspace);
  Pass k = pass_of(p, s, l);
  set(k.q, k.q_stride, p->k, p->k_stride);
  set(k.k, k.k_stride, p->q, p->q_stride);
  set(k.v, k.v_stride, p->dy, p->dy_stride);
  k.vec = vec_ok(k.q, k.q_stride, k.dk, k.dtype) && vec_ok(k.k, k.k_stride, k.dk, k.dtype) &&
          vec_ok(k.v, k.v_stride, k.dv, k.dtype) && out_ok(p->dv, k.dv);
  k.init = p->dstate;
  k.final_state = p->dh0;
  k.y = p->dv;
  k.states = ws + l.dstates;
  k.factors = reinterpret_cast<float*>(ws + l.dfactors);
  const float* const factors = reinterpret_cast<const float*>(
      static_cast<const char*>(p->run_states) + states_bytes(s, p->batch, p->heads, p->key_dim, p->dtype));
  const char* const rests = static_cast<const char*>(p->run_states) + rests_at(s, p->batch, p->heads, p->key_dim, p->dtype);
  if (k.fine) k.state_rests = ws + l.drests;
  float* const dg = p->dlog_decay_heads ? reinterpret_cast<float*>(ws + l.dg) : p->dlog_decay;
  if (dg) {
    k.dot_with = p->run_states;
    if (k.fine) k.rests_with = rests;
    k.factors_with = factors;
    k.dot = reinterpret_cast<float*>(ws + l.dot);
  }
  launch_pass_mirrored(k, st);
  if (s.runs > 0) {
    Grad d{};
    set(d.q, d.q_stride, p->q, p->q_stride);
    set(d.k, d.k_stride, p->k, p->k_stride);
    set(d.v, d.v_stride, p->v, p->v_stride);
    set(d.dy, d.dy_stride, p->dy, p->dy_stride);
    set(d.g, d.g_stride, p->log_decay, p->log_decay_stride);
    d.lengths = p->lengths;
    d.states = p->run_states;
    d.dstates = k.states;
    if (k.fine) d.rests = rests, d.drests = k.state_rests;
    d.factors = factors;
    d.dfactors = k.factors;
    d.dot = k.dot;
    float* const parts = reinterpret_cast<float*>(ws + l.parts);
    const int64_t n = p->batch * p->seqlen * p->groups * p->key_dim;
    d.dq = s.sets > 1 ? static_cast<void*>(parts) : p->dq;
    d.dk_out = s.sets > 1 ? static_cast<void*>(parts + s.sets * n) : p->dk;
    d.dg = dg;
    d.batch = p->batch;
    d.seqlen = p->seqlen;
    d.heads = p->heads;
    d.groups = p->groups;
    d.per = k.per;
    d.dk = p->key_dim;
    d.dv = p->value_dim;
    d.runs = s.runs;
    d.vblocks = s.vblocks;
    d.sets = s.sets;
    d.set_heads = s.set_heads;
    d.vec = vec_ok(d.q, d.q_stride, d.dk, p->dtype) && vec_ok(d.k, d.k_stride, d.dk, p->dtype) &&
            vec_ok(d.v, d.v_stride, d.dv, p->dtype) && vec_ok(d.dy, d.dy_stride, d.dv, p->dtype);
    d.dtype = p->dtype;
    d.g_dtype = p->log_decay_dtype;
    d.lengths_dtype = p->lengths_dtype;
    d.scale = p->scale;
    launch_grad(d, st);
    if (s.sets > 1) {
      const dim3 grid(static_cast<unsigned>(ceil_div(n, 256)));
      for (int which = 0; which < 2; ++which) {
        const float* const from = parts + which * s.sets * n;
        void* const to = which ? p->dk : p->dq;
        switch (p->dtype) {
          case MM_F32: hipLaunchKernelGGL((sum_sets_kernel<MM_F32>), grid, dim3(256), 0, st, from, to, n, s.sets); break;
          case MM_F16: hipLaunchKernelGGL((sum_sets_kernel<MM_F16>), grid, dim3(256), 0, st, from, to, n, s.sets); break;
          default: hipLaunchKernelGGL((sum_sets_kernel<MM_BF16>), grid, dim3(256), 0, st, from, to, n, s.sets); break;
        }
      }
    }
  }
  if (p->dlog_decay_heads && s.runs > 0) {
    int64_t nrows = p->batch * p->seqlen;
    const float* const from = rows::reduce_first(dg, nrows, p->heads, st);
    hipLaunchKernelGGL(sum_heads_kernel, dim3(static_cast<unsigned>(ceil_div(p->heads, 64))), dim3(64 * rows::kGroups), 0, st, from,
                       p->dlog_decay_heads, nrows, p->heads);
  }
  return check_launch("decay_attention_bwd");
}

int mm_decay_attention_step(const float* state, float* state_out, const void* q, const void* k, const void* v,
                            const void* log_decay, void* y, int64_t batch, int64_t heads, int64_t groups, int64_t key_dim,
                            int64_t value_dim, const int64_t q_stride[2], const int64_t k_stride[2], const int64_t v_stride[2],
                            const int64_t log_decay_stride[2], const int64_t y_stride[2], float scale, int32_t dtype,
                            int32_t log_decay_dtype, void* stream) {
  using namespace mm;
  using namespace mm::dattn;
  clear_error();
  if (!valid_dtype(dtype) || !valid_dtype(log_decay_dtype)) return fail(MM_ERR_DTYPE, "dtype %d, log_decay's %d", dtype, log_decay_dtype);
  if (!sizes_ok(batch, 1, heads, groups, key_dim, value_dim))
    return fail(MM_ERR_SHAPE, "batch %lld, heads %lld in %lld groups, key_dim %lld, value_dim %lld", (long long)batch,
                (long long)heads, (long long)groups, (long long)key_dim, (long long)value_dim);
  if (batch == 0) return MM_OK;
  if (!state || !state_out || !q || !k || !v || !log_decay || !y)
    return fail(MM_ERR_NULL_POINTER, "state, state_out, q, k, v, log_decay and y are required");
  if (!q_stride || !k_stride || !v_stride || !log_decay_stride || !y_stride) return fail(MM_ERR_NULL_POINTER, "strides are required");
  const int64_t* const all[5] = {q_stride, k_stride, v_stride, log_decay_stride, y_stride};
  for (const int64_t* s : all)
    if (s[0] < 0 || s[1] < 0) return fail(MM_ERR_LAYOUT, "negative stride");
  if (rows_overlap(batch, heads, value_dim, y_stride)) return fail(MM_ERR_LAYOUT, "rows of y overlap");
  if (partly_same(state, state_out, batch * heads * key_dim * value_dim * 4)) return fail(MM_ERR_LAYOUT, "state_out overlaps state");
  Step p{};
  p.state = state;
  p.state_out = state_out;
  p.q = q;
  p.k = k;
  p.v = v;
  p.g = log_decay;
  p.y = y;
  for (int i = 0; i < 2; ++i) {
    p.q_stride[i] = q_stride[i];
    p.k_stride[i] = k_stride[i];
    p.v_stride[i] = v_stride[i];
    p.g_stride[i] = log_decay_stride[i];
    p.y_stride[i] = y_stride[i];
  }
  p.batch = batch;
  p.heads = heads;
  p.per = heads / groups;
  p.dk = key_dim;
  p.dv = value_dim;
  p.vblocks = static_cast<int32_t>(ceil_div(value_dim, kVBlock));
  p.vec = value_dim % 4 == 0 && aligned(state, 16) && aligned(state_out, 16);
  p.scale = scale;
  const dim3 grid(static_cast<unsigned>(batch * heads * p.vblocks));
  hipStream_t st = static_cast<hipStream_t>(stream);
#define MM_DA(D, G) hipLaunchKernelGGL((step_kernel<D, G>), grid, dim3(256), 0, st, p)
#define MM_DA_G(D)                                                                                   \
  switch (log_decay_dtype) {                                                                         \
    case MM_F32: MM_DA(D, MM_F32); break;                                                            \
    case MM_F16: MM_DA(D, MM_F16); break;                                                            \
    default: MM_DA(D, MM_BF16); break;                                                               \
  }
  switch (dtype) {
    case MM_F32: MM_DA_G(MM_F32) break;
    case MM_F16: MM_DA_G(MM_F16) break;
    default: MM_DA_G(MM_BF16) break;
  }
#undef MM_DA_G
#undef MM_DA
  return check_launch("decay_attention_step");
}

}  // extern "C"
