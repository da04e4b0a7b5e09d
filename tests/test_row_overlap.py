"""Outputs whose rows share elements are refused, and no others: the C entry points' rule against all pairs of rows.
(No GPU needed: a layout that is let through fails at the missing workspace instead.)"""

from __future__ import annotations

import ctypes
import itertools

import pytest

from mamba_metal_amd import _lib
from test_abi import FAKE


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def status(lib, batch, seqlen, dim, s0, s1):
    p = _lib.GatedScanParams()
    for k in ("x", "a_gate", "x_gate", "A", "y"):
        setattr(p, k, FAKE)
    p.batch, p.seqlen, p.dim = batch, seqlen, dim
    for k in ("x", "a_gate", "x_gate"):
        setattr(p, f"{k}_stride", (_lib._i64a2)(0, 0))
    p.y_stride = (_lib._i64a2)(s0, s1)
    assert lib.mm_gated_scan_workspace_size(batch, seqlen, dim, 0) > 0
    return lib.mm_gated_scan_fwd(ctypes.byref(p), None)


def overlap(batch, seqlen, dim, s0, s1):
    starts = sorted(b * s0 + t * s1 for b, t in itertools.product(range(batch), range(seqlen)))
    return any(b - a < dim for a, b in zip(starts, starts[1:]))


DIM, N = 5, 300
STRIDES = [0, 1, 4, 5, 6, 7, 9, 10, 11, 15, 20, 35, 1490, 1494, 1495, 1496, 1499, 1500, 1501, 1505, 2990, 3000, 10 ** 6]


@pytest.mark.parametrize("batch", [1, 2, 3, 7, 400])
@pytest.mark.parametrize("s0", STRIDES)
def test_rule(lib, batch, s0):
    for s1 in STRIDES:
        want = _lib.ERR_LAYOUT if overlap(batch, N, DIM, s0, s1) else _lib.ERR_WORKSPACE
        assert status(lib, batch, N, DIM, s0, s1) == want, (batch, s0, s1)


def test_large(lib):
    big = 1 << 61
    assert status(lib, 65535, 1 << 20, 64, big, big) == _lib.ERR_LAYOUT  # row (0, 1) is row (1, 0)
    assert status(lib, 65535, 1 << 20, 64, 64, 65535 * 64) == _lib.ERR_WORKSPACE  # time outside, batch inside
    assert status(lib, 65535, 1 << 20, 64, 64 << 20, 64) == _lib.ERR_WORKSPACE
    assert status(lib, 65535, 1 << 20, 64, (64 << 20) - 1, 64) == _lib.ERR_LAYOUT


def test_unpack(lib):
    two = _lib._i64a2
    for s0, s1 in ((64, 64), (64, 128), (128, 64), (100, 65), (191, 64)):
        assert lib.mm_act8_unpack(FAKE, FAKE, FAKE, 3, 3, 64, two(s0, s1), 0, None) == _lib.ERR_LAYOUT, (s0, s1)
