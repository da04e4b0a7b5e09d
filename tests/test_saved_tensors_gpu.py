"""Training through hooks on saved tensors: kept on the CPU, in another layout, in 8 bits; what is not what was saved is
refused before a kernel reads it."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import Act8, act8_pack, act8_unpack, causal_conv1d_train, gated_scan

pytestmark = pytest.mark.gpu


def step(dev, checkpoint, hooks=None):
    g = torch.Generator().manual_seed(1)
    b, n, d = 2, 70, 66
    r = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(dev).requires_grad_(True)
    wide = torch.randn((b, n, 2 * d), generator=g).to(torch.bfloat16).to(dev)
    leaves = [r(b, n, d), r(b, n, d), r(b, n, d), (-torch.rand(d, generator=g)).to(dev).requires_grad_(True), r(d, 1, 4), r(d)]
    x, ag, xg, A, w, bias = leaves

    def forward():
        y = causal_conv1d_train(x, w, bias, checkpoint=checkpoint)
        return gated_scan(y, ag, xg, A, z=wide[..., d:], checkpoint=checkpoint)

    if hooks is None:
        y = forward()
    else:
        with torch.autograd.graph.saved_tensors_hooks(*hooks):
            y = forward()
    return y, leaves


def grads(y, leaves):
    return torch.autograd.grad(y, leaves, torch.ones_like(y))


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_hooks(dev, checkpoint):
    want = grads(*step(dev, checkpoint))
    strided = lambda t: torch.stack([t, t], -1)[..., 0] if t.dim() else t
    for hooks in ((lambda t: t.cpu(), lambda t: t.to(dev)), (lambda t: t, strided), (lambda t: t, lambda t: t.clone())):
        assert all(torch.equal(a, b) for a, b in zip(grads(*step(dev, checkpoint, hooks)), want))


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t[:1], lambda t: t.to(torch.int16),
                                    lambda t: t.half() if t.is_floating_point() else t.half().to(torch.int16)])
def test_refused(dev, checkpoint, change):
    y, leaves = step(dev, checkpoint, (lambda t: t, change))
    with pytest.raises(RuntimeError, match="saved tensor|require gradients"):  # (the latter torch's, of whole numbers)
        grads(y, leaves)


def test_inputs_in_8_bits_by_hooks(dev):
    """checkpoint="full" with hooks that pack the activations: the same codes, so the conv's gradients of "int8"."""
    hooks = (lambda t: act8_pack(t) if t.dim() == 3 and t.shape[1] == 70 else t,
             lambda p: act8_unpack(p) if isinstance(p, Act8) else p)
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn((2, 70, 66), generator=g).to(dev).requires_grad_(True), torch.randn((66, 1, 4), generator=g).to(dev)
    with torch.autograd.graph.saved_tensors_hooks(*hooks):
        y = causal_conv1d_train(x, w)
    want = causal_conv1d_train(x, w, checkpoint="int8")
    dy = torch.randn(y.shape, generator=g).to(dev)
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(want, x, dy)[0])
