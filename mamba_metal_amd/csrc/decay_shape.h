// How a call of decaying linear attention is cut: whole numbers only, so that a host compiler takes this file, too.
// mm::ceil_div is declared before it.
#pragma once

#include <cstdint>

#include "../../include/mamba_mi355x.h"

namespace mm {
namespace dattn {

constexpr int kRun = 64;    // tokens a run
constexpr int kVBlock = 64; // value channels a workgroup
constexpr int kMaxDk = 128;
constexpr int64_t kMaxBatch = 65535, kMaxHeads = 65535, kMaxDv = 1024, kMaxTokens = int64_t{1} << 30;

// Whether a call of 16-bit types is `fine`: its scores take a second term (decay_tiles.h, score_operand), and the states that
// gradients of q, k and the decays read the rests of their roundings.  It costs little where launches and few workgroups are most
// of the time, and much where the work is.  16 to 32 heads of 128 by 64 that share q and k, bf16 (fp16), a forward and backward
// pass in us, as it is here and the other way:
//   tokens x heads      8192         16384        32768          65536          262144
//   fine                83 (87)      85 (91)      122 (142)      167 (199)      508 (654)
//   not                 78 (84)      77 (83)      97 (102)       117 (127)      241 (287)
// (32768 of 32 heads with a q and k each: 109 (112), and 96 (96).)  Off by, in roundings of the output: dq and dk 1.0 and 1.41, the
// decays' gradient 1.0 and 1.3 to 1.5, y and dv 1.22 to 1.27 and 1.41, at every one of the sizes.
inline bool fine_scores(int64_t batch, int64_t seqlen, int64_t heads, int32_t dtype) {
  return dtype != MM_F32 && batch * seqlen * heads <= 32768;
}

struct Shape {
  int64_t runs, seg_runs;
  int32_t vblocks, segments, sets, set_heads;
};

// Segments: with fewer than 256 workgroups (one a compute unit) the tokens are cut so that there are as many as run at once,
// 3 a compute unit in 16 bits, else 2 (80 heads, 8192 tokens in bf16: 161 us in 9 segments, 178 in 6).  Two runs are not cut:
// fp32, 8 heads: 17 us whole, 20 in two segments and three launches; four runs: 30 us in two segments, 20 in four.
// Sets of heads in the gradients of q and k, which have a compute unit each: as many as end first, a set's own work (q, k,
// their scores, its sums written and read once more) counted as four heads of a unit.  (80 heads, 256
// runs of 64 tokens, bf16: 307 us in one set, 310 to 330 and 17 more for the sums in three.)
// A batch of no sequences has a shape, too: its workspaces are asked for.
inline Shape shape_of(int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t dv, int32_t dtype) {
  Shape s;
  s.runs = ceil_div(seqlen, kRun);
  s.vblocks = static_cast<int32_t>(ceil_div(dv, kVBlock));
  const int64_t wgs = batch * heads * s.vblocks, per = heads / groups;
  int64_t segs = wgs > 0 && wgs < 256 ? (dtype == MM_F32 ? 512 : 768) / wgs : 1;
  if (segs > s.runs) segs = s.runs > 2 ? s.runs : 1;
  if (segs < 1) segs = 1;
  s.seg_runs = ceil_div(s.runs > 0 ? s.runs : 1, segs);
  s.segments = static_cast<int32_t>(ceil_div(s.runs > 0 ? s.runs : 1, s.seg_runs));
  const int64_t grads = batch * groups * (s.runs > 0 ? s.runs : 1);
  int64_t sets = 1, least = INT64_MAX;
  for (int64_t n = 1; n <= per && n <= 64; ++n) {
    const int64_t t = ceil_div(grads * n, 256) * (ceil_div(per, n) + 4);
    if (t < least) least = t, sets = n;
  }
  s.set_heads = static_cast<int32_t>(ceil_div(per, sets));
  s.sets = static_cast<int32_t>(ceil_div(per, s.set_heads));
  return s;
}

inline bool sizes_ok(int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t dk, int64_t dv) {
  if (batch < 0 || seqlen < 0 || heads < 1 || groups < 1 || heads % groups || dk < 1 || dv < 1) return false;
  if (batch > kMaxBatch || heads > kMaxHeads || seqlen > kMaxTokens || dk > kMaxDk || dv > kMaxDv) return false;
  const int64_t grid = batch * heads * ceil_div(dv, kVBlock);
  return grid < (int64_t{1} << 22) && batch * heads * (ceil_div(seqlen, kRun) + 1) < (int64_t{1} << 31);
}

}  // namespace dattn
}  // namespace mm
