"""gated_tiles.h through a host compiler, and the calls that the placement tests make on the GPU."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent

# (batch, seqlen, dim), several sequences each: strips of every sequence on each die, and how many of them (forward
# tiles of 8 waves, of 4 for 9 x 300 x 1000).  500, 960 and 1000 channels leave no, one and no strip of a span over.
CASES = [((3, 700, 500), 1), ((2, 400, 960), 2), ((3, 700, 1000), 2), ((9, 300, 1000), 2)]


def build(folder):
    """The header's functions as a ctypes library, built in ``folder``."""
    so = Path(folder) / "gated_tiles.so"
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", str(HERE / "gated_tiles_host.cpp"), "-o", str(so)],
                   check=True)
    lib = ctypes.CDLL(str(so))
    lib.tiles_shape.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 2 + [ctypes.c_void_p]
    lib.tiles_strip.argtypes, lib.tiles_strip.restype = [ctypes.c_void_p, ctypes.c_int64], ctypes.c_int64
    lib.tiles_count.argtypes, lib.tiles_count.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int64
    return lib


class Shape:
    def __init__(self, lib, batch, seqlen, dim, backward, ragged):
        self.raw = (ctypes.c_int64 * 6)()
        lib.tiles_shape(batch, seqlen, dim, backward, ragged, self.raw)
        self.waves, self.strips, self.turns, self.per_die, self.span, self.workgroups = self.raw

    def counts(self, lib):
        count = (ctypes.c_int64 * self.strips)()
        bad = lib.tiles_count(self.raw, count)
        return list(count), bad
