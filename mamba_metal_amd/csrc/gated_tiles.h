// Which tiles a call of the gated recurrence has, and which workgroup takes which: whole numbers only, so that a host
// compiler takes this file, too.  mm::ceil_div is declared before it.
#pragma once

#include <cstdint>

#include "../../include/mamba_mi355x.h"

#ifdef __HIPCC__
#define MM_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define MM_HOST_DEVICE inline
#endif

namespace mm {
namespace gscan {

constexpr int kBlk = MM_ACT8_BLOCK;  // tokens of a wave
// Waves of a tile.  Forward 16 where they hold the whole sequence (one tile, no hand-off).  Longer ones: 4 from
// kManyStrips strips of channels on, where more and smaller workgroups overlap loads, arithmetic and waits better, else
// 8, since with few strips the chain of tiles counts, which 4 make twice as long (us with 8 and 4; 1 strip of 32768
// tokens 29, 51; 16 102, 105; 32 188, 195; 80 427, 431; 160 of 16384 423, 414; 256 of 2048 96.5, 93; 320 of 8192 with
// codes 640, 600).  5 or 6 load the SIMDs unevenly (a fifth slower).  Backward 4, so that four workgroups share a CU's
// registers and LDS.
constexpr int kMaxWaves = 16, kTileWaves = 8, kManyTileWaves = 4, kManyStrips = 128, kMaxWavesBwd = 4;

constexpr int kControlBytes = 128;   // of a strip's counter: a line each
constexpr int kWordsBytes = 64 * 8;  // of a tile

// A workgroup's strip of channels is fixed.  Workgroups go to the chip's 8 dies in turn: with per_die > 0 each die takes
// per_die neighbouring strips out of every `span`, whose rows share DRAM pages and lines (16-row tiles of 128-byte rows:
// 4.65 -> 5.25 TB/s of plain copying); strips past the span's last have no tile.
constexpr uint32_t kDies = 8;
struct Spread {
  uint32_t nstrips, nturns, per_die, span;
};
// With per_die > 0, of the j-th workgroup of a die: the strip within its span (none from `span` on), and the span's first.
MM_HOST_DEVICE uint32_t place_of(uint32_t die, uint32_t j, const Spread& sp) { return die * sp.per_die + j % sp.per_die; }
MM_HOST_DEVICE uint32_t span_of(uint32_t j, const Spread& sp) { return j / sp.per_die * sp.span % sp.nstrips; }

struct Shape {
  int waves;
  int64_t ncb, per_die, span, tiles, nstrips, nturns, control_bytes, handoff_bytes;
};
// Sequences of up to `most` blocks of 16 tokens are one tile: no hand-off, one launch.
inline Shape shape_of(int64_t batch, int64_t seqlen, int64_t dim, bool backward, bool ragged = false) {
  const int most = backward ? kMaxWavesBwd : kMaxWaves;
  const int64_t nblk = ceil_div(seqlen > 0 ? seqlen : 1, kBlk);
  Shape s;
  s.ncb = ceil_div(dim, 64);
  s.nstrips = batch * s.ncb;
  const int tile = backward ? kMaxWavesBwd : s.nstrips >= kManyStrips ? kManyTileWaves : kTileWaves;
  s.waves = nblk <= most ? static_cast<int>(nblk) : tile;
  s.nturns = ceil_div(nblk, s.waves);
  // Neighbouring strips of every sequence on one die, so that ragged sequences spread over all of them, or, where a
  // sequence's do not divide well and all have one length, of all sequences; either where it leaves no more than an
  // eighth of the workgroups without a tile.
  s.per_die = 0;
  s.span = s.nstrips;
  for (int64_t span : {s.ncb, ragged ? s.ncb : s.nstrips}) {
    const int64_t n = ceil_div(span, int64_t{kDies});
    if (8 * kDies * n > 9 * span) continue;
    s.per_die = n;
    s.span = span;
    break;
  }
  s.tiles = s.nturns * (s.per_die ? s.nstrips / s.span * kDies * s.per_die : s.nstrips);
  s.control_bytes = kControlBytes * (1 + s.nstrips);
  s.handoff_bytes = s.nturns > 1 ? s.control_bytes + s.nturns * s.nstrips * kWordsBytes : 0;
  return s;
}

}  // namespace gscan
}  // namespace mm
