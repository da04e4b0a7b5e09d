// Rows of an embedding table, scaled, and the table's gradient by sorted tokens.
//
//   y[i] = scale * weight[ids[i]]          dweight[v] = scale * sum_{i : ids[i] = v} dy[i]
//
// All of it is memory traffic.  The gradient's rows are sums in a fixed order, so that calls repeat bit for bit: the
// tokens are sorted by id (a stable radix sort, least digit first, of up to 9 bits a pass), runs of equal ids are
// summed in fp32 in the order of their positions, and rounded once.  A run may be any length (the commonest token of a
// text takes several percent of it): the sorted tokens are cut into tiles of 32, and what a run leaves in the tiles it
// crosses is joined by a last kernel.  Rows without a token are zeros; the whole table is cleared by workgroups that run
// beside the sort's (whose few workgroups would leave the card idle), at no cost of their own.
#include "mm_common.h"

namespace mm {
namespace embed {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 2048;     // tokens a workgroup of the sort
constexpr int kWaveItems = kBlock / 4;
constexpr int kRounds = kWaveItems / 64;
constexpr int kMaxBits = 9;      // of a digit
constexpr int kTile = 32;        // sorted tokens a wave sums
constexpr int64_t kClear = 64 << 10;  // bytes a clearing workgroup writes

struct Params {
  const void* ids;
  const void* weight;
  const void* dy;
  void* out;            // y, or dweight
  int64_t n, vocab, dim, ld, dy_ld;  // ld: weight's row stride
  int64_t padding;      // an id without a gradient, or -1
  int32_t ids64;
  float scale;
  // workspace of the gradient
  uint32_t *key[2], *pos[2], *hist[2];
  float* part;          // (tiles, 2, dim): what a tile's first and last run leave to be joined
  int64_t tiles, sort_blocks, clear_bytes;
};

__device__ __forceinline__ int64_t id_of(const Params& p, int64_t i) {
  return p.ids64 ? static_cast<const int64_t*>(p.ids)[i] : static_cast<const int32_t*>(p.ids)[i];
}
// The sort's key: the id, or vocab for one without a gradient (the padding's, or none of the table's).
__device__ __forceinline__ uint32_t key_of(const Params& p, int64_t i) {
  const int64_t id = id_of(p, i);
  return id < 0 || id >= p.vocab || id == p.padding ? static_cast<uint32_t>(p.vocab) : static_cast<uint32_t>(id);
}

// kV elements at once: 16 bytes, or single elements where rows are not aligned.
template <int DT, int kV>
__device__ __forceinline__ void load_elems(const void* base, int64_t at, float (&x)[kV]) {
  using T = typename Ty<DT>::T;
  const T* const p = static_cast<const T*>(base) + at;
  if constexpr (kV == 1) {
    x[0] = Ty<DT>::f(*p);
  } else {
    const u32x4 w = *reinterpret_cast<const u32x4*>(p);
    T t[kV];
    __builtin_memcpy(t, &w, 16);
#pragma unroll
    for (int j = 0; j < kV; ++j) x[j] = Ty<DT>::f(t[j]);
  }
}
// (x scale) as an fp32 product, then rounded: the empty asm keeps the two from becoming one mixed-precision instruction in
// some kernels and not in others.
template <int DT>
__device__ __forceinline__ typename Ty<DT>::T scaled(float x, float scale) {
  float t = x * scale;
  asm("" : "+v"(t));
  return Ty<DT>::from(t);
}
template <int DT, int kV>
__device__ __forceinline__ void store_elems(void* base, int64_t at, const float (&x)[kV], float scale) {
  using T = typename Ty<DT>::T;
  T* const p = static_cast<T*>(base) + at;
  if constexpr (kV == 1) {
    *p = scaled<DT>(x[0], scale);
  } else {
    T t[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) t[j] = scaled<DT>(x[j], scale);
    u32x4 w;
    __builtin_memcpy(&w, t, 16);
    *reinterpret_cast<u32x4*>(p) = w;
  }
}

// Forward: `lanes` lanes a row (a power of two), 4 waves a workgroup.
template <int DT, int kV>
__global__ __launch_bounds__(256) void rows_kernel(const Params p, int lanes) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t row = wave * (64 / lanes) + lane / lanes;
  if (row >= p.n) return;
  const int64_t id = id_of(p, row);
  const bool in = id >= 0 && id < p.vocab;
  const int64_t units = p.dim / kV;
  for (int64_t u = lane & (lanes - 1); u < units; u += lanes) {
    float x[kV];
    if (in) {
      load_elems<DT, kV>(p.weight, id * p.ld + u * kV, x);
    } else {
#pragma unroll
      for (int j = 0; j < kV; ++j) x[j] = __builtin_nanf("");
    }
    store_elems<DT, kV>(p.out, row * p.dim + u * kV, x, p.scale);
  }
}

// This launch's share of clearing the table: share `part` of `parts`, by the workgroups from p.sort_blocks on.
__device__ __forceinline__ void clear_share(const Params& p, int64_t bytes0, int64_t bytes1) {
  const int64_t b0 = bytes0 + (blockIdx.x - p.sort_blocks) * kClear;
  const int64_t b1 = b0 + kClear < bytes1 ? b0 + kClear : bytes1;
  char* const base = static_cast<char*>(p.out);
  // 16 bytes at a time; the table's last odd bytes (and an unaligned table) by 2
  if ((reinterpret_cast<uintptr_t>(base) & 15) == 0) {
    int64_t at = b0 + threadIdx.x * 16;
#pragma unroll 4
    for (; at + 16 <= b1; at += 256 * 16) *reinterpret_cast<u32x4*>(base + at) = u32x4{0, 0, 0, 0};
    if (at < b1)
      for (; at < b1; at += 2) *reinterpret_cast<uint16_t*>(base + at) = 0;
  } else {
    for (int64_t at = b0 + threadIdx.x * 2; at < b1; at += 512) *reinterpret_cast<uint16_t*>(base + at) = 0;
  }
}

// First launch: how often each value of the first digit occurs in each block of tokens; clears the second's counts.
__global__ __launch_bounds__(256) void count_kernel(const Params p, int bits, int64_t hist_words, int64_t clear1) {
  if (blockIdx.x >= p.sort_blocks) return clear_share(p, 0, clear1);
  __shared__ uint32_t s_hist[1 << kMaxBits];
  const int digits = 1 << bits;
  for (int d = threadIdx.x; d < digits; d += 256) s_hist[d] = 0;
  __syncthreads();
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kBlock;
#pragma unroll
  for (int k = 0; k < kBlock / 256; ++k) {
    const int64_t i = i0 + k * 256 + threadIdx.x;
    if (i < p.n) atomicAdd(&s_hist[key_of(p, i) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += 256) p.hist[0][static_cast<int64_t>(blockIdx.x) * digits + d] = s_hist[d];
  for (int64_t w = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; w < hist_words; w += p.sort_blocks * 256)
    p.hist[1][w] = 0;
}

// One pass: each block's tokens to their places by one digit, stably, and the counts of the next digit at the new
// places (integer atomics: their order does not matter).  hist `in` belongs to this pass; `out` is cleared for use.
__global__ __launch_bounds__(256) void scatter_kernel(const Params p, int pass, int passes, int bits, int64_t clear0, int64_t clear1) {
  if (blockIdx.x >= p.sort_blocks) return clear_share(p, clear0, clear1);
  __shared__ uint32_t s_base[1 << kMaxBits];
  __shared__ uint32_t s_wave[4][1 << kMaxBits];
  __shared__ uint32_t s_sum[4];
  const int digits = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t mask = digits - 1;
  const uint32_t* const hist = p.hist[pass & 1];
  // where each digit of this block begins: all smaller digits, and this one in the blocks before.  Two digits a thread.
  uint32_t before[2] = {0, 0}, total[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int d = threadIdx.x * 2 + e;
    if (d >= digits) continue;
#pragma unroll 4
    for (int64_t b = 0; b < p.sort_blocks; ++b) {
      const uint32_t c = hist[b * digits + d];
      total[e] += c;
      before[e] += b < blockIdx.x ? c : 0;
    }
  }
  uint32_t incl = total[0] + total[1];
  const uint32_t mine = incl;
#pragma unroll
  for (int x = 1; x < 64; x *= 2) {
    const uint32_t up = __shfl_up(incl, x, 64);
    incl += lane >= x ? up : 0;
  }
  if (lane == 63) s_sum[wave] = incl;
  for (int d = threadIdx.x; d < 4 * digits; d += 256) s_wave[d / digits][d % digits] = 0;
  __syncthreads();
  uint32_t start = incl - mine;
  for (int w = 0; w < wave; ++w) start += s_sum[w];
  if (threadIdx.x * 2 < static_cast<unsigned>(digits)) {
    s_base[threadIdx.x * 2] = start + before[0];
    s_base[threadIdx.x * 2 + 1] = start + total[0] + before[1];
  }
  // a wave's items in order, 64 at a time: rank among the equal digits before it
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kBlock + wave * kWaveItems;
  uint32_t key[kRounds], at[kRounds], pos[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = i0 + r * 64 + lane;
    const bool in = i < p.n;
    key[r] = in ? (pass == 0 ? key_of(p, i) : p.key[(pass - 1) & 1][i]) : 0;
    pos[r] = in ? (pass == 0 ? static_cast<uint32_t>(i) : p.pos[(pass - 1) & 1][i]) : 0;
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool in = i0 + r * 64 + lane < p.n;
    const uint32_t d = key[r] >> (pass * bits) & mask;
    uint64_t same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const uint64_t on = __ballot(d >> b & 1);
      same &= d >> b & 1 ? on : ~on;
    }
    const uint64_t below = same & ((1ull << lane) - 1);
    uint32_t first = 0;
    if (in) first = s_wave[wave][d];
    __builtin_amdgcn_wave_barrier();
    if (in && below == 0) s_wave[wave][d] = first + __popcll(same);
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
    at[r] = first + __popcll(below);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (i0 + r * 64 + lane >= p.n) continue;
    const uint32_t d = key[r] >> (pass * bits) & mask;
    uint32_t to = s_base[d] + at[r];
    for (int w = 0; w < wave; ++w) to += s_wave[w][d];
    p.key[pass & 1][to] = key[r];
    p.pos[pass & 1][to] = pos[r];
    if (pass + 1 < passes)
      atomicAdd(&p.hist[(pass + 1) & 1][static_cast<int64_t>(to / kBlock) * digits + (key[r] >> ((pass + 1) * bits) & mask)], 1u);
  }
}

// Between passes where there are more than two: the counts that the pass after the next adds to.
__global__ __launch_bounds__(256) void clear_counts_kernel(uint32_t* hist, int64_t words) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < words) hist[i] = 0;
}

// A wave sums 32 sorted tokens over 64 kV columns: whole runs go to the table, the parts of runs that reach over an
// edge of the tile to the workspace (first: one that began before; last: one that goes on, if it is not the first).
template <int DT, int kV>
__global__ __launch_bounds__(256) void sum_kernel(const Params p, int last, int64_t chunks) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t tile = wave / chunks, c0 = (wave % chunks) * 64 * kV + lane * kV;
  if (tile >= p.tiles) return;
  const uint32_t* const key = p.key[last];
  const uint32_t* const pos = p.pos[last];
  const int64_t i0 = tile * kTile, i1 = i0 + kTile < p.n ? i0 + kTile : p.n;
  const bool on = c0 < p.dim;
  float sum[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) sum[j] = 0.0f;
  uint32_t run = key[i0];
  bool began = i0 == 0 || key[i0 - 1] != run;  // in this tile
  for (int64_t i = i0; i < i1; i += 8) {
    uint32_t k[8];
    float x[8][kV];
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = i + e < i1 ? key[i + e] : static_cast<uint32_t>(p.vocab);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int j = 0; j < kV; ++j) x[e][j] = 0.0f;
      if (k[e] < p.vocab && on) load_elems<DT, kV>(p.dy, static_cast<int64_t>(pos[i + e]) * p.dy_ld + c0, x[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (i + e < i1 && k[e] != run) {
        if (run < p.vocab && on) {
          if (began) {
            store_elems<DT, kV>(p.out, run * p.dim + c0, sum, p.scale);
          } else {
#pragma unroll
            for (int j = 0; j < kV; ++j) p.part[(tile * 2) * p.dim + c0 + j] = sum[j];
          }
        }
        run = k[e];
        began = true;
#pragma unroll
        for (int j = 0; j < kV; ++j) sum[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kV; ++j) sum[j] += x[e][j];
    }
  }
  if (run >= p.vocab || !on) return;
  const bool ends = i1 == p.n || key[i1] != run;
  if (began && ends) {
    store_elems<DT, kV>(p.out, run * p.dim + c0, sum, p.scale);
  } else {
#pragma unroll
    for (int j = 0; j < kV; ++j) p.part[(tile * 2 + (began ? 1 : 0)) * p.dim + c0 + j] = sum[j];
  }
}

// Joins the run that begins in a tile and goes on behind it.
template <int DT, int kV>
__global__ __launch_bounds__(256) void join_kernel(const Params p, int last, int64_t chunks) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t tile = wave / chunks, c0 = (wave % chunks) * 64 * kV + lane * kV;
  const uint32_t* const key = p.key[last];
  const int64_t next = (tile + 1) * kTile;
  if (next >= p.n) return;
  const uint32_t run = key[next - 1];
  if (run >= p.vocab || key[next] != run) return;
  if (key[tile * kTile] == run && tile > 0 && key[tile * kTile - 1] == run) return;  // began before this tile
  if (c0 >= p.dim) return;
  float sum[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) sum[j] = p.part[(tile * 2 + 1) * p.dim + c0 + j];
  // tiles wholly of this run, and the last one, whose first run it is
  int64_t t = tile + 1;
  for (bool more = true; more;) {
    int64_t t1 = t;
    // as far as the next eight tiles go on
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      ++t1;
      if (t1 * kTile >= p.n || key[t1 * kTile - 1] != run || key[t1 * kTile] != run) {
        more = false;
        break;
      }
    }
#pragma unroll 8
    for (; t < t1; ++t)
#pragma unroll
      for (int j = 0; j < kV; ++j) sum[j] += p.part[(t * 2) * p.dim + c0 + j];
  }
  store_elems<DT, kV>(p.out, run * p.dim + c0, sum, p.scale);
}

// ------------------------------------------------------------------------------------------------------------- host
constexpr int64_t kMaxTokens = int64_t{1} << 31, kMaxVocab = int64_t{1} << 30, kMaxDim = int64_t{1} << 20;

struct Plan {
  int64_t blocks, tiles, hist_words, key_at[2], pos_at[2], hist_at[2], part_at, total;
  int bits, passes;
};
// The digits of the keys 0 .. vocab: as few passes as digits of 9 bits allow, of equal widths.
static Plan plan_of(int64_t n, int64_t vocab, int64_t dim) {
  Plan s{};
  int width = 1;
  while ((vocab >> width) != 0) ++width;
  s.passes = (width + kMaxBits - 1) / kMaxBits;
  s.bits = (width + s.passes - 1) / s.passes;
  s.blocks = ceil_div(n, kBlock);
  s.tiles = ceil_div(n, kTile);
  s.hist_words = s.blocks << s.bits;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += round_up(bytes, 256);
    return was;
  };
  for (int k = 0; k < 2; ++k) {
    s.key_at[k] = take(n * 4);
    s.pos_at[k] = take(n * 4);
    s.hist_at[k] = take(s.hist_words * 4);
  }
  s.part_at = take(s.tiles * 2 * dim * 4);
  s.total = at;
  return s;
}
static bool sizes_ok(int64_t n, int64_t vocab, int64_t dim) {
  return n >= 0 && vocab >= 1 && dim >= 1 && n < kMaxTokens && vocab <= kMaxVocab && dim <= kMaxDim && n * dim < (int64_t{1} << 40) &&
         vocab * dim < (int64_t{1} << 42);
}
static int check(const void* ids, int32_t ids_dtype, int64_t n, int64_t vocab, int64_t dim, int32_t dtype) {
  if (!valid_dtype(dtype)) return fail(MM_ERR_DTYPE, "dtype %d", dtype);
  if (ids_dtype != 0 && ids_dtype != 1) return fail(MM_ERR_DTYPE, "ids_dtype %d", ids_dtype);
  if (!sizes_ok(n, vocab, dim))
    return fail(MM_ERR_SHAPE, "%lld tokens, vocab %lld, dim %lld: empty, negative or too large", (long long)n, (long long)vocab, (long long)dim);
  if (n > 0 && !ids) return fail(MM_ERR_NULL_POINTER, "ids is required");
  return MM_OK;
}

template <int DT, int kV>
static void launch_rows(const Params& p, hipStream_t s) {
  const int64_t units = p.dim / kV;
  int lanes = 1;
  while (lanes < 64 && lanes < units) lanes *= 2;
  const int64_t waves = ceil_div(p.n, 64 / lanes);
  hipLaunchKernelGGL((rows_kernel<DT, kV>), dim3(static_cast<unsigned>(ceil_div(waves, 4))), dim3(256), 0, s, p, lanes);
}
template <int DT, int kV>
static void launch_sums(const Params& p, int last, hipStream_t s) {
  const int64_t chunks = ceil_div(p.dim, 64 * kV);
  const dim3 grid(static_cast<unsigned>(ceil_div(p.tiles * chunks, 4)));
  hipLaunchKernelGGL((sum_kernel<DT, kV>), grid, dim3(256), 0, s, p, last, chunks);
  if (p.tiles > 1) hipLaunchKernelGGL((join_kernel<DT, kV>), grid, dim3(256), 0, s, p, last, chunks);
}

}  // namespace embed
}  // namespace mm

#define MM_EMBED(FN, ...)                                                     \
  switch (dtype) {                                                            \
    case MM_F32:                                                              \
      if (vec) FN<MM_F32, 4>(__VA_ARGS__); else FN<MM_F32, 1>(__VA_ARGS__);   \
      break;                                                                  \
    case MM_F16:                                                              \
      if (vec) FN<MM_F16, 8>(__VA_ARGS__); else FN<MM_F16, 1>(__VA_ARGS__);   \
      break;                                                                  \
    default:                                                                  \
      if (vec) FN<MM_BF16, 8>(__VA_ARGS__); else FN<MM_BF16, 1>(__VA_ARGS__); \
      break;                                                                  \
  }

extern "C" {

int mm_embedding_fwd(const void* ids, const void* weight, void* y, int64_t n, int64_t vocab, int64_t dim,
                     int64_t weight_stride, float scale, int32_t ids_dtype, int32_t dtype, void* stream) {
  using namespace mm;
  using namespace mm::embed;
  clear_error();
  int e = check(ids, ids_dtype, n, vocab, dim, dtype);
  if (e != MM_OK || n == 0) return e;
  if (!weight || !y) return fail(MM_ERR_NULL_POINTER, "weight and y are required");
  if (weight_stride < 0) return fail(MM_ERR_LAYOUT, "weight has a negative stride");
  Params p{};
  p.ids = ids;
  p.weight = weight;
  p.out = y;
  p.n = n;
  p.vocab = vocab;
  p.dim = dim;
  p.ld = weight_stride;
  p.ids64 = ids_dtype;
  p.scale = scale;
  const int64_t per = 16 / dtype_size(dtype);
  const bool vec = dim % per == 0 && weight_stride % per == 0 && aligned(weight, 16) && aligned(y, 16);
  MM_EMBED(launch_rows, p, static_cast<hipStream_t>(stream));
  return check_launch("embedding_fwd");
}

size_t mm_embedding_bwd_workspace_size(int64_t n, int64_t vocab, int64_t dim) {
  using namespace mm::embed;
  if (!sizes_ok(n, vocab, dim) || n == 0) return 0;
  return static_cast<size_t>(plan_of(n, vocab, dim).total);
}

int mm_embedding_bwd(const void* ids, const void* dy, void* dweight, int64_t n, int64_t vocab, int64_t dim, int64_t dy_stride,
                     float scale, int64_t padding, int32_t ids_dtype, int32_t dtype, void* workspace, size_t workspace_bytes,
                     void* stream) {
  using namespace mm;
  using namespace mm::embed;
  clear_error();
  int e = check(ids, ids_dtype, n, vocab, dim, dtype);
  if (e != MM_OK) return e;
  if (!dweight || (n > 0 && !dy)) return fail(MM_ERR_NULL_POINTER, "dy and dweight are required");
  if (dy_stride < 0) return fail(MM_ERR_LAYOUT, "dy has a negative stride");
  const Plan s = plan_of(n, vocab, dim);
  if (n > 0 && (!workspace || !aligned(workspace, 256) || workspace_bytes < static_cast<size_t>(s.total)))
    return fail(MM_ERR_WORKSPACE, "needs %lld bytes of 256-byte aligned workspace", (long long)s.total);
  Params p{};
  p.ids = ids;
  p.dy = dy;
  p.out = dweight;
  p.n = n;
  p.vocab = vocab;
  p.dim = dim;
  p.dy_ld = dy_stride;
  p.padding = padding;
  p.ids64 = ids_dtype;
  p.scale = scale;
  char* const ws = static_cast<char*>(workspace);
  for (int k = 0; k < 2; ++k) {
    p.key[k] = reinterpret_cast<uint32_t*>(ws + s.key_at[k]);
    p.pos[k] = reinterpret_cast<uint32_t*>(ws + s.pos_at[k]);
    p.hist[k] = reinterpret_cast<uint32_t*>(ws + s.hist_at[k]);
  }
  p.part = reinterpret_cast<float*>(ws + s.part_at);
  p.tiles = s.tiles;
  p.sort_blocks = s.blocks;
  p.clear_bytes = vocab * dim * dtype_size(dtype);
  hipStream_t st = static_cast<hipStream_t>(stream);
  // the launches of the sort share the clearing, in whole pieces
  const int launches = n > 0 ? s.passes + 1 : 1;
  auto upto = [&](int k) {
    const int64_t pieces = ceil_div(p.clear_bytes, kClear);
    const int64_t b = pieces * k / launches * kClear;
    return b < p.clear_bytes ? b : p.clear_bytes;
  };
  auto grid = [&](int k) { return dim3(static_cast<unsigned>(s.blocks + ceil_div(upto(k + 1) - upto(k), kClear))); };
  if (grid(0).x) hipLaunchKernelGGL(count_kernel, grid(0), dim3(256), 0, st, p, s.bits, s.hist_words, upto(1));
  if (n > 0) {
    for (int k = 0; k < s.passes; ++k) {
      hipLaunchKernelGGL(scatter_kernel, grid(k + 1), dim3(256), 0, st, p, k, s.passes, s.bits, upto(k + 1), upto(k + 2));
      if (k + 2 < s.passes)
        hipLaunchKernelGGL(clear_counts_kernel, dim3(static_cast<unsigned>(ceil_div(s.hist_words, 256))), dim3(256), 0, st, p.hist[k & 1],
                           s.hist_words);
    }
    const int last = (s.passes - 1) & 1;
    const int64_t per = 16 / dtype_size(dtype);
    const bool vec = dim % per == 0 && dy_stride % per == 0 && aligned(dy, 16) && aligned(dweight, 16);
    MM_EMBED(launch_sums, p, last, st);
  }
  return check_launch("embedding_bwd");
}

}  // extern "C"
