"""Several sequences whose strips of channels are placed by sequence, whole and ragged, forward and backward."""

from __future__ import annotations

import pytest
import torch

import gated_ref as ref
from gated_placement import CASES
from mamba_metal_amd import _lib, gated_scan
from mamba_metal_amd.selective_scan import reset_scan_status, scan_status

pytestmark = pytest.mark.gpu

LEAVES = ("x", "a_gate", "x_gate", "A", "z", "h0")


def rand(seed, b, n, d, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    f = {k: torch.randn((b, n, d), generator=g).to(dtype).to(dev) for k in ("x", "a_gate", "x_gate", "z", "dy")}
    f["A"] = (-0.001 * 1000.0 ** torch.rand(d, generator=g)).to(dev)
    f["h0"], f["dstate"] = (torch.randn((b, d), generator=g).to(dev) for _ in range(2))
    return f


def train(f, lengths, checkpoint):
    leaves = {k: f[k].detach().clone().requires_grad_(True) for k in LEAVES}
    y, state = gated_scan(leaves["x"], leaves["a_gate"], leaves["x_gate"], leaves["A"], z=leaves["z"], h0=leaves["h0"],
                          lengths=lengths, return_state=True, checkpoint=checkpoint)
    grads = torch.autograd.grad([y, state], list(leaves.values()), [f["dy"], f["dstate"]])
    return y, state, dict(zip(LEAVES, grads))


@pytest.mark.parametrize("dtype,checkpoint", [(torch.float32, "full"), (torch.bfloat16, "int8"), (torch.float16, "full")])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("size", [size for size, _ in CASES])
def test_placement_by_sequence(dev, size, ragged, dtype, checkpoint):
    b, n, d = size
    f = rand(1, *size, dtype, dev)
    lengths = None
    if ragged:  # an empty one, a whole one, ends in the middle of a block and of a tile
        ends = [0, n, n // 2 + 3, 1, n - 1, 64, 65, n // 3, 17]
        lengths = torch.tensor(ends[:b] if b > 2 else [n // 2 + 3, n], dtype=torch.int32, device=dev)
    reset_scan_status(dev)
    y, state, got = train(f, lengths, checkpoint)
    assert scan_status(dev) == 0
    c = ref.Case(f["x"], f["a_gate"], f["x_gate"], f["A"], f["z"], f["h0"], lengths)
    wy, ey, wh, eh = c.forward()
    ref.close(y, wy, ey, dtype, "y")
    ref.close(state, wh, eh, torch.float32, "state")
    want = c.backward(f["dy"], f["dstate"], checkpoint == "int8")
    for k, v in got.items():
        ref.close(v, *want[k], torch.float32 if k in ("A", "h0") else dtype, "d" + k)
    again = train(f, lengths, checkpoint)
    assert torch.equal(y, again[0]) and torch.equal(state, again[1]) and all(torch.equal(got[k], again[2][k]) for k in got)


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0)])
def test_empty_with_codes(dev, shape):
    f = rand(2, *shape, torch.float16, dev)
    y, state, got = train(f, None, "int8")
    assert y.shape == shape and state.shape == (shape[0], shape[2]) and got["z"].shape == shape
    assert got["A"].shape == (shape[2],) and not got["A"].any()
    if shape[1] == 0:
        assert torch.equal(state, f["h0"]) and torch.equal(got["h0"], f["dstate"])


def test_a_wait_that_must_expire(dev):
    """One strip of 256 tiles, all running at once, whose states are handed on from the first to the last: the chain takes
    tens of microseconds, the wait's bound is one.  The call ends, says so, and the workspace serves the next one."""
    b, n, d = 1, 32768, 64
    f = rand(3, b, n, d, torch.float32, dev)
    want = gated_scan(f["x"], f["a_gate"], f["x_gate"], f["A"])
    lib, p = _lib.load(), _lib.GatedScanParams()
    y, status = torch.empty_like(want), torch.zeros(1, dtype=torch.int32, device=dev)
    for k in ("x", "a_gate", "x_gate"):
        setattr(p, k, f[k].data_ptr())
        setattr(p, f"{k}_stride", (_lib._i64a2)(n * d, d))
    p.A, p.y, p.y_stride, p.status = f["A"].data_ptr(), y.data_ptr(), (_lib._i64a2)(n * d, d), status.data_ptr()
    p.batch, p.seqlen, p.dim = b, n, d
    nbytes = lib.mm_gated_scan_workspace_size(b, n, d, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    for us, expires in ((1, True), (0, False), (1, True), (0, False)):
        p.handoff_timeout_us = us
        status.zero_()
        _lib.check(lib.mm_gated_scan_fwd(p, _lib.stream_of(dev)), "mm_gated_scan_fwd")
        torch.cuda.synchronize()
        assert status.item() == (_lib.SCAN_STATUS_HANDOFF_TIMEOUT if expires else 0)
    assert torch.equal(y, want)
