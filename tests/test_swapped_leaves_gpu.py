"""Gradients of leaves whose memory was replaced between the passes: those of leaves that stayed, bit for bit."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import decay_attention

pytestmark = pytest.mark.gpu


def attention(dev, g_shape):
    gen = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=gen)
    b, n, heads, d = 2, 200, 3, 64
    q, k, v = (r(b, n, h, d).to(dev, torch.bfloat16) for h in (1, 1, heads))
    g = (-torch.rand(g_shape or (b, n, heads), generator=gen)).to(dev)
    leaves = [t.requires_grad_(True) for t in (q, k, v, g)]
    return decay_attention(*leaves), leaves, r(b, n, heads, d).to(dev, torch.bfloat16)


@pytest.mark.parametrize("g_shape", [(3,), None])
@pytest.mark.parametrize("which", range(4))
def test_replaced_data(dev, g_shape, which):
    y, leaves, dy = attention(dev, g_shape)
    want = torch.autograd.grad(y, leaves, dy)
    y, leaves, dy = attention(dev, g_shape)
    t = leaves[which]
    old = t.data
    wide = torch.empty((*t.shape[:-1], t.shape[-1] + 8), dtype=t.dtype, device=dev)[..., :t.shape[-1]].copy_(old)
    t.data = wide
    old.fill_(float("nan"))  # (kept alive: what a stale address would read)
    got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
