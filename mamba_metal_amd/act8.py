"""Activations kept in 8 bits for a backward pass.

``act8_pack(x)`` turns an activation (batch, seqlen, dim) into whole numbers of at most 127 and one
power of two for each block of 16 tokens of a channel: 1.06 bytes an element instead of 2 or 4, off by
at most half a step of the block's power of two, 1/127.5 of the block's largest magnitude at worst.
``act8_unpack`` gives back the values that the codes stand for, which the activation's own dtype holds exactly (but for
float16's largest numbers, whose code stands for 65536: they come back as 65504); another dtype rounds them.
``gated_scan`` and ``causal_conv1d_train`` with ``checkpoint="int8"`` keep their inputs this way and
read the codes in their backward kernels; these two functions are for any other activation.

A block with an infinity or a NaN in it comes back as NaNs, so what was broken stays visible.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from mamba_metal_amd import _lib

BLOCK = _lib.ACT8_BLOCK


@dataclass
class Act8:
    """An activation in 8 bits: ``codes`` (batch, ceil(seqlen / 16), dim, 16) int8, a channel's 16 tokens
    side by side, and ``exps`` (batch, ceil(seqlen / 16), dim) uint8, both contiguous, value =
    codes * 2^(exps - 127); the shape and dtype it had."""

    codes: torch.Tensor
    exps: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.exps.numel()


def channels_last(t, name):
    """t has unit channel stride (or a single channel)."""
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have unit channel stride")


def empty_like(x, shape=None) -> Act8:
    """Uninitialised codes for x (batch, seqlen, dim)."""
    b, n, d = x.shape
    nblk = -(-n // BLOCK)
    return Act8(torch.empty((b, nblk, d, BLOCK), dtype=torch.int8, device=x.device),
                torch.empty((b, nblk, d), dtype=torch.uint8, device=x.device),
                x.shape if shape is None else shape, x.dtype)


def act8_pack(x: torch.Tensor) -> Act8:
    """x (batch, seqlen, dim) or (seqlen, dim), float32 / float16 / bfloat16 with unit channel stride.

    Not differentiable: a tensor that requires a gradient is refused while gradients are on (in the pack hook of
    ``torch.autograd.graph.saved_tensors_hooks`` they are off), and one with a tangent always."""
    if x.dim() not in (2, 3):
        raise ValueError(f"act8_pack takes (batch, seqlen, dim) or (seqlen, dim), got {tuple(x.shape)}")
    code = _lib.dtype_code(x.dtype)
    channels_last(x, "x")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("act8_pack has no gradient: call it under no_grad, or on x.detach()")
    _lib.refuse_transforms("act8_pack", x)
    dev = _lib.require_cuda(x)
    lib = _lib.load()
    x3 = x if x.dim() == 3 else x[None]
    out = empty_like(x3, x.shape)
    with _lib.on_device(dev):
        st = lib.mm_act8_pack(x3.data_ptr(), out.codes.data_ptr(), out.exps.data_ptr(), *x3.shape,
                              (_lib._i64a2)(*x3.stride()[:2]), code, _lib.stream_of(dev))
    _lib.check(st, "mm_act8_pack")
    return out


def act8_unpack(packed: Act8, dtype: torch.dtype | None = None, out: torch.Tensor | None = None):
    """The values that ``packed`` stands for, in its dtype unless another is given (or out's).

    ``out``, when given, has packed's shape, unit channel stride and rows that do not overlap."""
    if out is not None and dtype is not None and out.dtype != dtype:
        raise TypeError(f"out is {out.dtype}, not {dtype}")
    dtype = out.dtype if out is not None else dtype or packed.dtype
    code = _lib.dtype_code(dtype)
    if len(packed.shape) not in (2, 3):
        raise ValueError(f"an activation is (batch, seqlen, dim) or (seqlen, dim), not {tuple(packed.shape)}")
    b, n, d = packed.shape if len(packed.shape) == 3 else (1, *packed.shape)
    nblk = -(-n // BLOCK)
    if packed.codes.dtype != torch.int8 or packed.exps.dtype != torch.uint8 \
            or packed.codes.shape != (b, nblk, d, BLOCK) or packed.exps.shape != (b, nblk, d) \
            or not packed.codes.is_contiguous() or not packed.exps.is_contiguous():
        raise ValueError("codes must be contiguous int8 (batch, ceil(seqlen / 16), dim, 16), exps contiguous "
                         "uint8 (batch, ceil(seqlen / 16), dim)")
    if out is not None:
        if out.shape != packed.shape:
            raise ValueError(f"out is {tuple(out.shape)}, the activation {tuple(packed.shape)}")
        channels_last(out, "out")
    _lib.refuse_transforms("act8_unpack", out)
    dev = _lib.require_cuda(packed.codes, packed.exps, out)
    lib = _lib.load()
    if out is None:
        out = torch.empty(packed.shape, dtype=dtype, device=dev)
    o3 = out if out.dim() == 3 else out[None]
    with _lib.on_device(dev):
        st = lib.mm_act8_unpack(packed.codes.data_ptr(), packed.exps.data_ptr(), o3.data_ptr(), b, n, d,
                                (_lib._i64a2)(*o3.stride()[:2]), code, _lib.stream_of(dev))
    _lib.check(st, "mm_act8_unpack")
    return out
