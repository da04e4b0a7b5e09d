"""A program that is recorded (torch.jit.trace, make_fx) would hold an operator's output tensor and not the kernel that
fills it: such calls are refused (no GPU needed: the checks come first)."""

from __future__ import annotations

import warnings

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from mamba_metal_amd import Act8, act8_pack, act8_unpack, causal_conv1d_train, gated_scan, gated_scan_step

X3, X2, A = torch.zeros((2, 5, 4)), torch.zeros((2, 4)), torch.zeros(4)
PACKED = Act8(torch.zeros((2, 1, 4, 16), dtype=torch.int8), torch.zeros((2, 1, 4), dtype=torch.uint8), X3.shape, X3.dtype)
CALLS = [(lambda x: gated_scan(x, x, x, A), X3), (lambda x: gated_scan_step(x.clone(), x, x, x, A), X2),
         (lambda x: act8_pack(x).codes, X3), (lambda x: act8_unpack(PACKED) + x, X3),
         (lambda x: causal_conv1d_train(x, torch.zeros((4, 1, 2))), X3),
         (lambda x: causal_conv1d_train(x, torch.zeros((4, 1, 2)), checkpoint="int8"), X3)]


@pytest.mark.parametrize("call,x", CALLS)
def test_recording_is_refused(call, x):
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(call)(x)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(call, (x,), check_trace=False)


@pytest.mark.parametrize("call,x", CALLS)
def test_other_modes_are_not(call, x):
    """Under a mode that only watches, the call goes on to where it needs a GPU."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Watch(), pytest.raises(ValueError, match="need GPU"):
        call(x)
