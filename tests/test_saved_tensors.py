"""A backward pass reads what autograd saved only if it is what was saved: hooks on saved tensors may hand back
another type, size or device, which the kernels would read past its end (no GPU needed), or another layout."""

from __future__ import annotations

import types

import pytest
import torch

from mamba_metal_amd import _lib
from mamba_metal_amd.conv1d import _CausalConv1d
from mamba_metal_amd.gated_scan import _GatedScan

B, N, D = 2, 20, 4
CPU = types.SimpleNamespace(index=-1)  # as get_device() names it


def saved(function, checkpoint):
    """What the forward passes save for float16 inputs, with lengths and a z."""
    x, i8 = torch.zeros((B, N, D), dtype=torch.float16), lambda *s: torch.zeros(s, dtype=torch.int8)
    if function is _CausalConv1d:
        return [torch.zeros((D, 1, 4)), torch.zeros(D), *((i8(B, 2, D, 16), i8(B, 2, D)) if checkpoint == "int8" else (x,))]
    out = [torch.zeros(D), torch.zeros(B, dtype=torch.int32), torch.zeros((B, 2, D))]
    return out + ([i8(4, B, 2, D, 16), i8(4, B, 2, D)] if checkpoint == "int8" else [x, x.clone(), x.clone(), x.clone()])


CHANGES = [lambda t: t.to(torch.int16), lambda t: t[:1], lambda t: t[..., None], lambda t: t.new_zeros(0), lambda t: None]


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("function", [_GatedScan, _CausalConv1d])
def test_the_backward_passes_refuse(function, checkpoint, monkeypatch):
    """Each saved tensor in turn, changed; the others, and the last of all, only not on the GPU."""
    dy = torch.zeros((B, N, D), dtype=torch.float16)
    dev = torch.device("cuda", 0)
    meta = (dev, dy.dtype, dy.shape, True, (torch.int32,) if function is _GatedScan else
            (torch.float32, torch.Size((D, 1, 4)), True))
    was = saved(function, checkpoint)
    ctx = types.SimpleNamespace(meta=meta, saved_tensors=was, needs_input_grad=(True,) * 10)
    with pytest.raises(RuntimeError, match="saved tensor"):
        function.backward(ctx, dy)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for k, t in enumerate(was):
        for change in CHANGES:
            ctx.saved_tensors = was[:k] + [change(t)] + was[k + 1:]
            with pytest.raises(RuntimeError, match="saved tensor"):
                function.backward(ctx, dy)


def test_layouts():
    wide = torch.arange(2 * 3 * 8).view(2, 3, 8)[..., 2:6]
    args = (wide.dtype, wide.shape, CPU)
    assert _lib.saved(wide, *args, rows=True) is wide and _lib.saved(wide, *args).is_contiguous()
    for other in (wide.transpose(1, 2).contiguous().transpose(1, 2), wide.clone()):
        for rows in (False, True):
            got = _lib.saved(other, *args, rows=rows)
            assert got.is_contiguous() and torch.equal(got, wide)


def test_hooks_are_seen():
    assert not _lib.hooked()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
        assert _lib.hooked()
    with torch.autograd.graph.save_on_cpu():
        assert _lib.hooked()
    assert not _lib.hooked()
