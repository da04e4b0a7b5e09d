// Rows of an embedding table, scaled, and the table's gradient by sorted tokens.
//
//   y[i] = scale * weight[ids[i]]          dweight[v] = scale * sum_{i : ids[i] = v} dy[i]
//
// All of it is memory traffic.  Forward, 16384 rows of 2560 in bf16: 33 us, 5.1 TB/s.  The gradient's rows are sums in a fixed order, so that calls repeat bit for bit: the
// tokens are sorted by id (a stable radix sort, least digit first, of up to 9 bits a pass), runs of equal ids are
// summed in fp32 in the order of their positions, and rounded once.  A run may be any length (the commonest token of a
// text takes several percent of it): the sorted tokens are cut into tiles of 16, and what a run leaves in the tiles it
// crosses is joined by a last kernel.  Rows without a token are zeros; the whole table is cleared by workgroups that run
// beside the sort's (whose few workgroups would leave the card idle), at no cost of their own.  Up to 16384 tokens are
// sorted by one workgroup in its LDS, in one launch; more by counting and scattering, a launch for each digit.
#include <type_traits>

#include "mm_common.h"

namespace mm {
namespace embed {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 2048;     // tokens a workgroup of the sort
constexpr int kWaveItems = kBlock / 4;
constexpr int kRounds = kWaveItems / 64;
constexpr int kMaxBits = 9;      // of a digit
constexpr int kTile = 16;        // sorted tokens a wave sums
// Tokens that one workgroup sorts: a key and a place of 14 bits in a word.  (Lookup and gradient in bf16, us in one workgroup and
// by counting: 50280 rows of 2560, 512 tokens 57 and 66, 8192 101 and 115, 16384 138 and 154; 32000 of 512, 512 tokens 30 and
// 41, 8192 46 and 52, 16384 64 and 60.)
constexpr int kOne = 16384, kOneThreads = 1024;
constexpr int64_t kOneVocab = int64_t{1} << 18;
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
using Raw = std::conditional_t<kV == 1, typename Ty<DT>::T, u32x4>;
template <int DT, int kV>
__device__ __forceinline__ Raw<DT, kV> load_raw(const void* base, int64_t at) {
  return *reinterpret_cast<const Raw<DT, kV>*>(static_cast<const typename Ty<DT>::T*>(base) + at);
}
template <int DT, int kV>
__device__ __forceinline__ void elems_of(const Raw<DT, kV>& w, float (&x)[kV]) {
  typename Ty<DT>::T t[kV];
  __builtin_memcpy(t, &w, sizeof(t));
#pragma unroll
  for (int j = 0; j < kV; ++j) x[j] = Ty<DT>::f(t[j]);
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
      elems_of<DT, kV>(load_raw<DT, kV>(p.weight, id * p.ld + u * kV), x);
    } else {
#pragma unroll
      for (int j = 0; j < kV; ++j) x[j] = __builtin_nanf("");
    }
    store_elems<DT, kV>(p.out, row * p.dim + u * kV, x, p.scale);
  }
}

// This launch's share of clearing the table: share `part` of `parts`, by the workgroups from p.sort_blocks on.
template <int NT>
__device__ __forceinline__ void clear_share(const Params& p, int64_t bytes0, int64_t bytes1) {
  const int64_t b0 = bytes0 + (blockIdx.x - p.sort_blocks) * kClear;
  const int64_t b1 = b0 + kClear < bytes1 ? b0 + kClear : bytes1;
  char* const base = static_cast<char*>(p.out);
  // 16 bytes at a time; the table's last odd bytes (and an unaligned table) by 2
  if ((reinterpret_cast<uintptr_t>(base) & 15) == 0) {
    int64_t at = b0 + threadIdx.x * 16;
#pragma unroll 4
    for (; at + 16 <= b1; at += NT * 16) *reinterpret_cast<u32x4*>(base + at) = u32x4{0, 0, 0, 0};
    if (at < b1)
      for (; at < b1; at += 2) *reinterpret_cast<uint16_t*>(base + at) = 0;
  } else {
    for (int64_t at = b0 + threadIdx.x * 2; at < b1; at += 2 * NT) *reinterpret_cast<uint16_t*>(base + at) = 0;
  }
}

// Lanes of a wave with this lane's digit among those of `in`.
__device__ __forceinline__ uint64_t equals(uint64_t in, uint32_t d, int bits) {
  uint64_t same = in;
#pragma unroll
  for (int b = 0; b < kMaxBits; ++b) {
    if (b >= bits) break;
    const bool one = d >> b & 1;
    const uint64_t on = __ballot(one);
    same &= one ? on : ~on;
  }
  return same;
}

// The whole sort, by workgroup 0; the others clear the table (50280 x 2560 in bf16: 257 MB in 39 us, the sort of 16384
// tokens under it).  A wave holds 64 `rounds` neighbouring tokens in registers; a
// pass ranks them among its own, a round at a time, joins the waves' counts, and sends them through the LDS.
__global__ __launch_bounds__(kOneThreads) void sort_kernel(const Params p, int passes, int bits, int rounds, int64_t clear1) {
  if (blockIdx.x >= p.sort_blocks) return clear_share<kOneThreads>(p, 0, clear1);
  constexpr int kWaves = kOneThreads / 64, kRegs = kOne / kOneThreads;
  __shared__ uint32_t s_item[kOne];
  __shared__ uint32_t s_wave[kWaves][1 << kMaxBits];
  __shared__ uint32_t s_sum[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = static_cast<int>(p.n), digits = 1 << bits, i0 = wave * 64 * rounds + lane;
  const uint32_t mask = digits - 1;
  uint32_t item[kRegs], at[kRegs];
#pragma unroll
  for (int r = 0; r < kRegs; ++r) {
    const int i = i0 + r * 64;
    item[r] = r < rounds && i < n ? key_of(p, i) << 14 | i : 0;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 14 + pass * bits;
    for (int d = lane; d < digits; d += 64) s_wave[wave][d] = 0;
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < kRegs; ++r) {
      if (r >= rounds) break;
      const bool in = i0 + r * 64 < n;
      const uint32_t d = item[r] >> shift & mask;
      const uint64_t same = equals(__ballot(in), d, bits), below = same & ((1ull << lane) - 1);
      const uint32_t first = s_wave[wave][d];
      __builtin_amdgcn_wave_barrier();
      if (in && below == 0) s_wave[wave][d] = first + __popcll(same);
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
      at[r] = first + __popcll(below);
    }
    __syncthreads();
    // where a digit's tokens of a wave begin: behind all smaller digits, and this one's in the waves before
    uint32_t count[kWaves], total = 0;
    if (tid < digits) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        count[w] = s_wave[w][tid];
        total += count[w];
      }
    }
    uint32_t incl = total;
#pragma unroll
    for (int x = 1; x < 64; x *= 2) {
      const uint32_t up = __shfl_up(incl, x, 64);
      incl += lane >= x ? up : 0;
    }
    if (lane == 63) s_sum[wave] = incl;
    __syncthreads();
    if (tid < digits) {
      uint32_t start = incl - total;
      for (int w = 0; w < wave; ++w) start += s_sum[w];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        s_wave[w][tid] = start;
        start += count[w];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRegs; ++r)
      if (r < rounds && i0 + r * 64 < n) s_item[s_wave[wave][item[r] >> shift & mask] + at[r]] = item[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRegs; ++r)
      if (r < rounds && i0 + r * 64 < n) item[r] = s_item[i0 + r * 64];
  }
#pragma unroll
  for (int r = 0; r < kRegs; ++r) {
    const int i = i0 + r * 64;
    if (r >= rounds || i >= n) break;
    p.key[0][i] = item[r] >> 14;
    p.pos[0][i] = item[r] & (kOne - 1);
  }
}

// First launch: how often each value of the first digit occurs in each block of tokens; clears the second's counts.
__global__ __launch_bounds__(256) void count_kernel(const Params p, int bits, int64_t hist_words, int64_t clear1) {
  if (blockIdx.x >= p.sort_blocks) return clear_share<256>(p, 0, clear1);
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
  if (blockIdx.x >= p.sort_blocks) return clear_share<256>(p, clear0, clear1);
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
    const uint64_t same = equals(__ballot(in), d, bits), below = same & ((1ull << lane) - 1);
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

// A wave sums 16 sorted tokens over 64 kV columns, all their rows under way at once: whole runs go to the table, the parts
// of runs that reach over an edge of the tile to the workspace (first: one that began before; last: one that goes on, if it
// is not the first).  16384 tokens of 2560 in bf16: 42 us, 3.1 TB/s (tiles of 32, eight rows at a time: 76).
template <int DT, int kV>
__global__ __launch_bounds__(256) void sum_kernel(const Params p, int last, int64_t chunks) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t tile = wave / chunks, c0 = (wave % chunks) * 64 * kV + lane * kV;
  if (tile >= p.tiles) return;
  const uint32_t vocab = static_cast<uint32_t>(p.vocab);
  const int64_t i0 = tile * kTile;
  const bool on = c0 < p.dim;
  // lanes 0 .. 17: the keys from the token before the tile to the one behind it (beyond the tokens: of none)
  const int64_t in = i0 - 1 + lane;
  const bool there = lane < kTile + 2 && in >= 0 && in < p.n;
  const uint32_t own_key = there ? p.key[last][in] : ~0u, own_pos = there ? p.pos[last][in] : 0;
  uint32_t k[kTile + 2];
  Raw<DT, kV> x[kTile];
#pragma unroll
  for (int e = 0; e < kTile + 2; ++e) k[e] = __builtin_amdgcn_readlane(own_key, e);
#pragma unroll
  for (int e = 0; e < kTile; ++e) {
    const int64_t row = static_cast<uint32_t>(__builtin_amdgcn_readlane(own_pos, e + 1));
    x[e] = Raw<DT, kV>{};
    if (k[e + 1] < vocab && on) x[e] = load_raw<DT, kV>(p.dy, row * p.dy_ld + c0);
  }
  float sum[kV];
#pragma unroll
  for (int j = 0; j < kV; ++j) sum[j] = 0.0f;
  bool began = k[0] != k[1];  // the run, in this tile
#pragma unroll
  for (int e = 0; e < kTile; ++e) {
    float f[kV];
    elems_of<DT, kV>(x[e], f);
#pragma unroll
    for (int j = 0; j < kV; ++j) sum[j] += f[j];
    const bool ends = k[e + 2] != k[e + 1];
    if ((ends || e == kTile - 1) && k[e + 1] < vocab) {
      if (on) {
        if (began && ends) {
          store_elems<DT, kV>(p.out, k[e + 1] * p.dim + c0, sum, p.scale);
        } else {
#pragma unroll
          for (int j = 0; j < kV; ++j) p.part[(tile * 2 + (began ? 1 : 0)) * p.dim + c0 + j] = sum[j];
        }
      }
    }
    if (ends) {
      began = true;
#pragma unroll
      for (int j = 0; j < kV; ++j) sum[j] = 0.0f;
    }
  }
}

// Joins the run that begins in a tile and goes on behind it: a wave for 64 columns (few runs are long, and a long one's
// sum is a chain of loads: narrow waves make many chains; 13 us there, 62 with 512 columns a wave).
template <int DT>
__global__ __launch_bounds__(256) void join_kernel(const Params p, int last, int64_t chunks) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int64_t tile = wave / chunks, c = (wave % chunks) * 64 + lane, next = (tile + 1) * kTile;
  if (next >= p.n) return;
  const uint32_t* const key = p.key[last];
  const uint32_t run = key[next - 1], behind = key[next], first = key[tile * kTile], before = tile > 0 ? key[tile * kTile - 1] : ~0u;
  if (run >= static_cast<uint32_t>(p.vocab) || behind != run || (first == run && before == run)) return;
  const bool on = c < p.dim;
  const float* const part = p.part + (on ? c : 0);
  float sum = part[(tile * 2 + 1) * p.dim];
  // tiles wholly of this run, and the last one, whose first run it is: a lane looks at each edge of the next 64
  for (int64_t t = tile + 1, some = 64; some == 64; t += 64) {
    const int64_t edge = (t + 1 + lane) * kTile;
    const bool in = edge < p.n;
    const uint32_t k0 = key[in ? edge - 1 : 0], k1 = key[in ? edge : 0];
    const uint64_t over = __ballot(in && k0 == run && k1 == run);
    some = over == ~0ull ? 64 : __builtin_ctzll(~over);
    const int64_t upto = some < 64 ? some + 1 : 64;
    for (int64_t e = 0; e < upto; e += 16) {
      float x[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = part[(t + (e + j < upto ? e + j : e)) * 2 * p.dim];
#pragma unroll
      for (int j = 0; j < 16; ++j) sum += e + j < upto ? x[j] : 0.0f;
    }
  }
  if (on) static_cast<typename Ty<DT>::T*>(p.out)[run * p.dim + c] = scaled<DT>(sum, p.scale);
}

// ------------------------------------------------------------------------------------------------------------- host
constexpr int64_t kMaxTokens = int64_t{1} << 31, kMaxVocab = int64_t{1} << 30, kMaxDim = int64_t{1} << 20;

struct Plan {
  int64_t blocks, tiles, hist_words, key_at[2], pos_at[2], hist_at[2], part_at, total;
  int bits, passes;
  bool one;
};
// The digits of the keys 0 .. vocab: as few passes as digits of 9 bits allow, of equal widths.  Without tokens there is nothing
// to sort and one launch clears the table.
static Plan plan_of(int64_t n, int64_t vocab, int64_t dim) {
  Plan s{};
  int width = 1;
  while ((vocab >> width) != 0) ++width;
  s.passes = (width + kMaxBits - 1) / kMaxBits;
  s.bits = (width + s.passes - 1) / s.passes;
  s.one = n == 0 || (n <= kOne && vocab < kOneVocab);
  s.blocks = s.one ? n > 0 : ceil_div(n, kBlock);
  s.tiles = ceil_div(n, kTile);
  s.hist_words = s.one ? 0 : s.blocks << s.bits;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t was = at;
    at += round_up(bytes, 256);
    return was;
  };
  for (int k = 0; k < (s.one ? 1 : 2); ++k) {
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
  const int64_t narrow = ceil_div(p.dim, 64);
  if (p.tiles > 1)
    hipLaunchKernelGGL((join_kernel<DT>), dim3(static_cast<unsigned>(ceil_div((p.tiles - 1) * narrow, 4))), dim3(256), 0, s, p, last, narrow);
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
  const int launches = s.one ? 1 : s.passes + 1;
  auto upto = [&](int k) {
    const int64_t pieces = ceil_div(p.clear_bytes, kClear);
    const int64_t b = pieces * k / launches * kClear;
    return b < p.clear_bytes ? b : p.clear_bytes;
  };
  auto grid = [&](int k) { return dim3(static_cast<unsigned>(s.blocks + ceil_div(upto(k + 1) - upto(k), kClear))); };
  if (s.one) {
    hipLaunchKernelGGL(sort_kernel, grid(0), dim3(kOneThreads), 0, st, p, s.passes, s.bits, static_cast<int>(ceil_div(n, kOneThreads)),
                       upto(1));
  } else {
    hipLaunchKernelGGL(count_kernel, grid(0), dim3(256), 0, st, p, s.bits, s.hist_words, upto(1));
    for (int k = 0; k < s.passes; ++k) {
      hipLaunchKernelGGL(scatter_kernel, grid(k + 1), dim3(256), 0, st, p, k, s.passes, s.bits, upto(k + 1), upto(k + 2));
      if (k + 2 < s.passes)
        hipLaunchKernelGGL(clear_counts_kernel, dim3(static_cast<unsigned>(ceil_div(s.hist_words, 256))), dim3(256), 0, st, p.hist[k & 1],
                           s.hist_words);
    }
  }
  if (n > 0) {
    const int last = s.one ? 0 : (s.passes - 1) & 1;
    const int64_t per = 16 / dtype_size(dtype);
    const bool vec = dim % per == 0 && dy_stride % per == 0 && aligned(dy, 16) && aligned(dweight, 16);
    MM_EMBED(launch_sums, p, last, st);
  }
  return check_launch("embedding_bwd");
}

}  // extern "C"
