"""The conv's training kernels on runs of several blocks of tokens: what a block takes from the one before it, odd ends
several blocks into a run, and sums over the run."""

from __future__ import annotations

import pytest
import torch

import gated_ref as ref
from mamba_metal_amd import _lib, causal_conv1d_train
from mamba_metal_amd.conv1d import causal_conv1d

pytestmark = pytest.mark.gpu


def run_of(batch, seqlen, dim, width):
    """Tokens of a backward run, from the workspace: a row of (width + 1) dim partial sums a run, and one more for
    every 512 rows where there are more than 512.  The forward pass with codes halves the same way from 64 on, so its run
    is this one, 64 at most."""
    floats = _lib.load().mm_causal_conv1d_bwd_workspace_size(batch, seqlen, dim, width) // 4
    runs = []
    for run in (128, 64, 32, 16):
        rows = batch * -(-seqlen // run)
        if floats == (rows + (-(-rows // 512) if rows > 512 else 0)) * (width + 1) * dim:
            runs.append(run)
    assert runs
    return runs[0]


def magnitudes(x, weight, bias, dout, apply_silu, width):
    """Sums of |dp x| and |dp|, what float32 sums over a run may be off by a step of."""
    p, _, padded = ref.conv(x, weight, bias, apply_silu)
    s = torch.sigmoid(p)
    dp = (dout * (s * (1 + p * (1 - s)) if apply_silu else 1)).abs()
    n = x.shape[1]
    dw = torch.stack([(dp * padded[:, k:k + n].abs()).sum((0, 1)) for k in range(width)], 1)
    return {"weight": dw.view(weight.shape), "bias": dp.sum((0, 1))}


# run, batch, seqlen, dim: last runs of 1, 3, 29 and 128 tokens (ends in the first token of a block, within its first
# half, in its second half 13 tokens into the second block, none), and several workgroups of channels
CASES = [(128, 1100, 129, 9), (128, 1030, 131, 5), (128, 1100, 157, 9), (128, 1030, 256, 7), (128, 260, 200, 270),
         (64, 700, 157, 9), (32, 450, 157, 9), (32, 180, 75, 260)]


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("width", [3, 4, 8])
@pytest.mark.parametrize("run,batch,seqlen,dim", CASES)
def test_runs(dev, run, batch, seqlen, dim, width, checkpoint):
    assert run_of(batch, seqlen, dim, width) == run
    dtype = torch.float32 if (batch, width) != (260, 4) else torch.bfloat16
    g = torch.Generator().manual_seed(width)
    f = {"x": torch.randn((batch, seqlen, dim), generator=g), "weight": torch.randn((dim, 1, width), generator=g) * width ** -0.5,
         "bias": torch.randn(dim, generator=g), "dy": torch.randn((batch, seqlen, dim), generator=g)}
    f = {k: v.to(dtype).to(dev) for k, v in f.items()}
    apply_silu = seqlen != 131
    leaves = [f[k].clone().requires_grad_(True) for k in ("x", "weight", "bias")]
    y = causal_conv1d_train(*leaves, apply_silu=apply_silu, checkpoint=checkpoint)
    got = dict(zip(("x", "weight", "bias"), torch.autograd.grad(y, leaves, f["dy"])))
    assert torch.equal(y, causal_conv1d(f["x"], f["weight"], f["bias"], apply_silu=apply_silu))
    x, w, b, dy = (f[k].cpu().double() for k in ("x", "weight", "bias", "dy"))
    p, ep, _ = ref.conv(x, w, b, apply_silu)
    s, es = ref.sig(p)
    wy = p * s if apply_silu else p
    # silu' is at most 1.1; the product
    ref.close(y, wy, 1.1 * ep + wy.abs() * (es + 3 * ref.U), dtype, "y")
    x = ref.quantise(x) if checkpoint == "int8" else x
    want = ref.conv_backward(x, w, b, dy, apply_silu)
    mags = magnitudes(x, w, b, dy, apply_silu, width)
    for k, v in got.items():
        value, bound = want[k]
        if k in mags:
            # a thread's multiply-adds over its run in float32, a step each, then sums in double of what float32 holds: one
            # more for the run's own sum and one for a first pass over the rows (the bound has 82 of these steps in it)
            bound = bound + max(0, run + 2 - 82) * ref.U * mags[k]
        ref.close(v, value, bound, v.dtype, "d" + k)
