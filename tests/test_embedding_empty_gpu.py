"""The embedding of no tokens: an empty output, and a table's gradient of zeros, however many rows it has (vocabularies of
2^18 rows and more are sorted by counting)."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import embedding

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,dim", [(1, 1), (1000, 8), ((1 << 18) - 1, 3), (1 << 18, 4), ((1 << 18) + 5, 1), (1 << 27, 1)])
@pytest.mark.parametrize("shape", [(0,), (2, 0), (0, 5)])
def test_no_tokens(dev, vocab, dim, shape):
    weight = torch.ones((vocab, dim), dtype=torch.bfloat16, device=dev, requires_grad=True)
    ids = torch.zeros(shape, dtype=torch.int64, device=dev)
    y = embedding(ids, weight)
    assert y.shape == (*shape, dim)
    grad, = torch.autograd.grad(y, weight, torch.ones_like(y))
    assert grad.shape == weight.shape and not bool(grad.any())
