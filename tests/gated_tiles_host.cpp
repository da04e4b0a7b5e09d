// The tiles of a gated recurrence's call and their mapping onto workgroups, built by a host compiler.
#include <cstdint>
#include <initializer_list>

namespace mm {
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
}  // namespace mm

#include "../mamba_metal_amd/csrc/gated_tiles.h"

extern "C" {

// out: waves, strips, turns, strips a die, span, workgroups
void tiles_shape(int64_t batch, int64_t seqlen, int64_t dim, int backward, int ragged, int64_t* out) {
  const mm::gscan::Shape s = mm::gscan::shape_of(batch, seqlen, dim, backward != 0, ragged != 0);
  const int64_t v[] = {s.waves, s.nstrips, s.nturns, s.per_die, s.span, s.tiles};
  for (int k = 0; k < 6; ++k) out[k] = v[k];
}

static mm::gscan::Spread spread(const int64_t* shape) {
  return {static_cast<uint32_t>(shape[1]), static_cast<uint32_t>(shape[2]), static_cast<uint32_t>(shape[3]),
          static_cast<uint32_t>(shape[4])};
}

// A workgroup's strip, -1 where it has none, as the kernels put it together.
int64_t tiles_strip(const int64_t* shape, int64_t block) {
  using namespace mm::gscan;
  const Spread sp = spread(shape);
  const uint32_t k = static_cast<uint32_t>(block);
  if (!sp.per_die) return k % sp.nstrips;
  const uint32_t j = k / kDies, s = place_of(k % kDies, j, sp);
  return s < sp.span ? int64_t{span_of(j, sp) + s} : -1;
}

// count[strip]: the workgroups of that strip.  Returns the workgroups whose strip is out of range.
int64_t tiles_count(const int64_t* shape, int64_t* count) {
  int64_t bad = 0;
  for (int64_t k = 0; k < shape[5]; ++k) {
    const int64_t strip = tiles_strip(shape, k);
    if (strip >= shape[1]) ++bad;
    else if (strip >= 0) ++count[strip];
  }
  return bad;
}
}
