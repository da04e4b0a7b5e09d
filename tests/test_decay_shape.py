"""How decaying linear attention cuts a call, for every size its entry points take (no GPU needed: the library's own
function, built by a host compiler without optimisation, which would end the process at a division by zero)."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

HERE = Path(__file__).resolve().parent
PROBE = """
import ctypes, itertools, sys
lib = ctypes.CDLL(sys.argv[1])
out = (ctypes.c_int64 * 6)()
i64 = ctypes.c_int64
for batch, seqlen, (heads, groups), dv, dtype in itertools.product(
        (0, 1, 2, 3, 64, 255, 256, 257), (0, 1, 64, 65, 128, 129, 1000, 8192, 1 << 20),
        ((1, 1), (2, 1), (5, 5), (24, 1), (80, 1), (80, 8), (96, 2), (257, 1)), (1, 64, 65, 1024), (0, 1, 2)):
    lib.decay_shape(i64(batch), i64(seqlen), i64(heads), i64(groups), i64(dv), dtype, out)
    runs, seg_runs, vblocks, segments, sets, set_heads = out
    per = heads // groups
    assert runs == -(-seqlen // 64) and vblocks == -(-dv // 64)
    # every run in one segment, every head in one set, none of either empty
    assert seg_runs >= 1 and segments >= 1 and (segments - 1) * seg_runs < max(runs, 1) <= segments * seg_runs
    assert sets >= 1 and (sets - 1) * set_heads < per <= sets * set_heads
    assert segments == 1 or segments * batch * heads * vblocks <= 768
print("all")
"""


def test_shapes(tmp_path):
    so = tmp_path / "shape.so"
    subprocess.run(["g++", "-O0", "-std=c++17", "-shared", "-fPIC", str(HERE / "decay_shape_host.cpp"), "-o", str(so)], check=True)
    done = subprocess.run([sys.executable, "-c", PROBE, str(so)], capture_output=True, text=True)
    assert done.returncode == 0 and done.stdout == "all\n", (done.returncode, done.stderr[-500:])
