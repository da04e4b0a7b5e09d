"""causal_conv1d_train's weight is (dim, 1, width) or (dim, width), as its message says (no GPU needed)."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import causal_conv1d_train


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("shape", [(4, 2, 3), (4, 0, 3), (4, 4, 4), (4,), (), (1, 4, 1, 3), (4, 3, 1, 1)])
def test_other_weights_are_refused(shape, checkpoint):
    with pytest.raises(ValueError, match="weight must be"):
        causal_conv1d_train(torch.zeros((2, 5, 4)), torch.zeros(shape), checkpoint=checkpoint)


@pytest.mark.parametrize("shape", [(4, 1, 3), (4, 3), (4, 1, 1), (4, 8)])
def test_these_are_not(shape):
    with pytest.raises(ValueError, match="need GPU"):
        causal_conv1d_train(torch.zeros((2, 5, 4)), torch.zeros(shape))
