"""The token steps refuse a state_out that shares a part of state's memory (no GPU needed: the C entries' own checks)."""

from __future__ import annotations

import pytest

from mamba_metal_amd import _lib

AT, BYTES = 1 << 32, {"attention": 2 * 4 * 64 * 64 * 4, "scan": 2 * 64 * 4}


def step(which, state, state_out):
    lib, two = _lib.load(), _lib._i64a2
    if which == "scan":
        return lib.mm_gated_scan_step(state, state_out, AT, AT, AT, AT, None, AT, 2, 64, 64, 64, 64, 0, 64, 0, None)
    return lib.mm_decay_attention_step(state, state_out, AT, AT, AT, AT, AT, 2, 4, 2, 64, 64, *[two(256, 64)] * 5, 1.0, 0, 0, None)


@pytest.mark.parametrize("which", ["attention", "scan"])
@pytest.mark.parametrize("side", [1, -1])
def test_refused(which, side):
    for by in (4, 256, BYTES[which] - 4):
        assert step(which, AT, AT + side * by) == _lib.ERR_LAYOUT
        assert "state_out overlaps state" in _lib.load().mm_last_error().decode()
