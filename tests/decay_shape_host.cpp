// How a call of decaying linear attention is cut, built by a host compiler.
#include <cstdint>

namespace mm {
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
}  // namespace mm

#include "../mamba_metal_amd/csrc/decay_shape.h"

extern "C" {

// out: runs, runs a segment, blocks of value channels, segments, sets, heads a set
void decay_shape(int64_t batch, int64_t seqlen, int64_t heads, int64_t groups, int64_t dv, int32_t dtype, int64_t* out) {
  const mm::dattn::Shape s = mm::dattn::shape_of(batch, seqlen, heads, groups, dv, dtype);
  const int64_t v[] = {s.runs, s.seg_runs, s.vblocks, s.segments, s.sets, s.set_heads};
  for (int k = 0; k < 6; ++k) out[k] = v[k];
}

}  // extern "C"
