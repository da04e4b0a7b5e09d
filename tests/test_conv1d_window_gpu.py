"""A token reaches the conv's outputs of its window alone, at every width, whatever keeps the input: a NaN or an
infinity in x leaves every other output as it is, bit for bit."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import causal_conv1d_train
from mamba_metal_amd.conv1d import causal_conv1d

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [512, 64, 70])  # whole waves on a run, vectors of 8 channels, single channels
@pytest.mark.parametrize("width", range(1, 9))
def test_not_finite_stays_in_its_window(dev, width, dim, dtype):
    g = torch.Generator().manual_seed(width)
    b, n = 2, 40
    x = torch.randn((b, n, dim), generator=g).to(dtype).to(dev)
    # (no weight of 0: 0 times an infinity inside the window is a NaN, too, but then by the formula)
    w = (0.5 + torch.rand((dim, 1, width), generator=g)).to(dtype).to(dev)
    bias = torch.randn(dim, generator=g).to(dtype).to(dev)
    outs = lambda x: (causal_conv1d(x, w, bias), causal_conv1d_train(x, w, bias, checkpoint="int8"),
                      causal_conv1d_train(x, w, bias))
    clean = causal_conv1d(x, w, bias)
    bad = [(0, 20, 3, "nan"), (1, 9, 5, "inf"), (1, 11, dim - 1, "-inf"), (0, 0, 7, "nan"), (1, n - 1, 0, "nan")]
    for bb, t, c, v in bad:
        x[bb, t, c] = float(v)
    for y in outs(x):
        keep = torch.ones((b, n, dim), dtype=torch.bool, device=dev)
        for bb, t, c, v in bad:
            keep[bb, t:t + width, c] = False
            assert not torch.isfinite(y[bb, t:t + width, c]).any() or v == "inf"
        assert torch.equal(y[keep], clean[keep])
        assert torch.equal(torch.isinf(y[1, 9:9 + width, 5]), torch.ones(width, dtype=torch.bool, device=dev))
    a, c, d = (y.float().nan_to_num(nan=7e30) for y in outs(x))
    assert torch.equal(a, c) and torch.equal(a, d)
