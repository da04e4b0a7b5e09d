"""Causal depthwise conv1d (prefill) and the decode conv-window step.

``causal_conv1d`` replaces the MLX ``nn.Conv1d(groups=d_inner, padding=d_conv-1)``
+ slice + ``nn.silu`` of mamba_metal/mamba_block.py:45-52,77-78,129-130 and
captures the conv state of mamba_block.py:118-127 in the same pass.
``conv_step`` replaces the window shift / dot / bias / SiLU of
mamba_block.py:170-177, updating the resident conv state in place.
``causal_conv1d_train`` is ``causal_conv1d`` with gradients (the reference has none).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from mamba_metal_amd import _lib
from mamba_metal_amd.act8 import BLOCK, Act8, channels_last, empty_like


def _w2d(weight):
    """(dim, 1, K) torch/HF conv weight, or (dim, K) -> 2-D view and its strides."""
    w = weight[:, 0, :] if weight.dim() == 3 else weight
    return w, (_lib._i64a2)(*w.stride())


def causal_conv1d(x, weight, bias=None, *, apply_silu=True, out=None, conv_state_out=None):
    """x: (batch, seqlen, dim) channels-last (any strides).

    Returns out (batch, seqlen, dim) (allocated contiguous unless given);
    writes the last ``width`` inputs to conv_state_out (batch, dim, width) if given.
    """
    lib = _lib.load()
    dev = _lib.require_cuda(x, weight, bias, out, conv_state_out)
    batch, seqlen, dim = x.shape
    w, ws = _w2d(weight)
    width = w.shape[1]
    if w.shape[0] != dim:
        raise ValueError(f"weight has {w.shape[0]} channels, x has {dim}")
    if bias is not None and (bias.shape != (dim,) or bias.dtype != w.dtype or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous (dim,) tensor of the weight's dtype")
    if out is None:
        out = torch.empty((batch, seqlen, dim), dtype=x.dtype, device=dev)
    if conv_state_out is not None:
        if conv_state_out.shape != (batch, dim, width) or not conv_state_out.is_contiguous() \
                or conv_state_out.dtype != x.dtype:
            raise ValueError("conv_state_out must be contiguous (batch, dim, width) of x's dtype")
    if x.numel() == 0:
        if conv_state_out is not None:
            conv_state_out.zero_()
        return out
    with _lib.on_device(dev):
        st = lib.mm_causal_conv1d_fwd(
            x.data_ptr(), w.data_ptr(), _lib.ptr(bias), out.data_ptr(), _lib.ptr(conv_state_out),
            batch, seqlen, dim, width, (_lib._i64a3)(*x.stride()), (_lib._i64a3)(*out.stride()),
            ws, _lib.dtype_code(x.dtype), _lib.dtype_code(w.dtype), 1 if apply_silu else 0,
            _lib.stream_of(dev))
    _lib.check(st, "mm_causal_conv1d_fwd")
    return out


def conv_step(conv_state, x, weight, bias=None, *, apply_silu=True, out=None):
    """conv_state (batch, dim, width) contiguous, updated in place; x (batch, dim)
    with unit channel stride.  Returns out (batch, dim) in x's dtype."""
    lib = _lib.load()
    dev = _lib.require_cuda(conv_state, x, weight, bias, out)
    batch, dim = x.shape
    w, ws = _w2d(weight)
    width = w.shape[1]
    if conv_state.shape != (batch, dim, width) or not conv_state.is_contiguous():
        raise ValueError(f"conv_state must be contiguous {(batch, dim, width)}")
    if x.stride(1) != 1:
        raise ValueError("x must have unit channel stride")
    if bias is not None and (bias.shape != (dim,) or bias.dtype != w.dtype or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous (dim,) tensor of the weight's dtype")
    if out is None:
        out = torch.empty((batch, dim), dtype=x.dtype, device=dev)
    with _lib.on_device(dev):
        st = lib.mm_decode_conv_step(
            conv_state.data_ptr(), x.data_ptr(), w.data_ptr(), _lib.ptr(bias), out.data_ptr(),
            batch, dim, width, x.stride(0), out.stride(0), ws,
            _lib.dtype_code(conv_state.dtype), _lib.dtype_code(x.dtype), _lib.dtype_code(w.dtype),
            1 if apply_silu else 0, _lib.stream_of(dev))
    _lib.check(st, "mm_decode_conv_step")
    return out


def _conv1d_backward(x, packed, weight, bias, dout, apply_silu, want_dx, want_dw):
    """Gradients of x, weight and bias; x as a tensor, or its 8-bit codes in ``packed``."""
    lib = _lib.load()
    dev = weight.device
    batch, seqlen, dim = dout.shape
    w, ws = _w2d(weight)
    width = w.shape[1]
    dx = torch.empty((batch, seqlen, dim), dtype=dout.dtype, device=dev) if want_dx else None
    dw = torch.empty((dim, width), dtype=w.dtype, device=dev) if want_dw else None
    db = torch.empty((dim,), dtype=w.dtype, device=dev) if want_dw and bias is not None else None
    nbytes = lib.mm_causal_conv1d_bwd_workspace_size(batch, seqlen, dim, width) if want_dw else 0
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    two = _lib._i64a2
    with _lib.on_device(dev):
        st = lib.mm_causal_conv1d_bwd(
            _lib.ptr(x), None if packed is None else packed.codes.data_ptr(),
            None if packed is None else packed.exps.data_ptr(), w.data_ptr(), _lib.ptr(bias), dout.data_ptr(),
            _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), batch, seqlen, dim, width,
            two(*x.stride()[:2]) if x is not None else two(0, 0), two(*dout.stride()[:2]), ws,
            _lib.dtype_code(dout.dtype), _lib.dtype_code(w.dtype), 1 if apply_silu else 0, _lib.ptr(work), nbytes,
            _lib.stream_of(dev))
    _lib.check(st, "mm_causal_conv1d_bwd")
    return dx, None if dw is None else dw.view(weight.shape), db


def _conv1d_act8(x, weight, bias, apply_silu):
    """causal_conv1d's output and x's 8-bit codes, in one pass over x."""
    lib = _lib.load()
    dev = _lib.require_cuda(x, weight, bias)
    w, ws = _w2d(weight)
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    packed = empty_like(x)
    with _lib.on_device(dev):
        st = lib.mm_causal_conv1d_fwd_act8(
            x.data_ptr(), w.data_ptr(), _lib.ptr(bias), out.data_ptr(), packed.codes.data_ptr(),
            packed.exps.data_ptr(), *x.shape, w.shape[1], (_lib._i64a2)(*x.stride()[:2]), ws,
            _lib.dtype_code(x.dtype), _lib.dtype_code(w.dtype), 1 if apply_silu else 0, _lib.stream_of(dev))
    _lib.check(st, "mm_causal_conv1d_fwd_act8")
    return out, packed


def _checked(saved, dev, dtype, shape, w_dtype, w_shape, has_bias):
    """The saved tensors, which hooks or a new ``.data`` may have changed."""
    (b, n, d), (weight, bias, *kept) = shape, saved
    if has_bias:
        bias = _lib.saved(bias, w_dtype, (d,), dev)
    if len(kept) == 1:
        kept = (_lib.saved(kept[0], dtype, shape, dev, rows=True),)
    else:
        nblk = -(-n // BLOCK)
        kept = (_lib.saved(kept[0], torch.int8, (b, nblk, d, BLOCK), dev), _lib.saved(kept[1], torch.uint8, (b, nblk, d), dev))
    return _lib.saved(weight, w_dtype, w_shape, dev, strided=True), bias, *kept


class _CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, apply_silu, checkpoint):
        ctx.meta = (x.device, x.dtype, x.shape, apply_silu,
                    (weight.dtype, weight.shape, bias is not None))
        if checkpoint == "int8":
            out, packed = _conv1d_act8(x, weight, bias, apply_silu)
            ctx.save_for_backward(weight, bias, packed.codes, packed.exps)
        else:
            out = causal_conv1d(x, weight, bias, apply_silu=apply_silu)
            ctx.save_for_backward(weight, bias, x)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        dev, dtype, shape, apply_silu, params = ctx.meta
        weight, bias, *kept = _checked(ctx.saved_tensors, dev, dtype, shape, *params)
        x, packed = (kept[0], None) if len(kept) == 1 else (None, Act8(*kept, shape, dtype))
        if dout.dtype != dtype or (dout.stride(-1) != 1 and shape[2] > 1):
            dout = dout.to(dtype).contiguous()
        need = ctx.needs_input_grad
        dx, dw, db = _conv1d_backward(x, packed, weight, bias, dout, apply_silu, need[0], need[1] or need[2])
        return dx, dw, db, None, None


def causal_conv1d_train(x, weight, bias=None, *, apply_silu=True, checkpoint="full"):
    """``causal_conv1d`` with gradients of x, weight and bias.

    x (batch, seqlen, dim) with unit channel stride, weight (dim, 1, width) or (dim, width), width <= 8.
    ``checkpoint`` says how x is kept for the backward pass: "full", as it is, or "int8", as 8-bit codes
    (``act8_pack``); the gradients are then those at the values that the codes stand for.  Sums over batch
    and time are taken in float32 and wider, in a fixed order."""
    if x.dim() != 3:
        raise ValueError(f"x must be (batch, seqlen, dim), got {tuple(x.shape)}")
    channels_last(x, "x")
    shape = tuple(weight.shape)
    if len(shape) not in (2, 3) or shape[0] != x.shape[2] or shape[1:-1] not in ((), (1,)) or not 1 <= shape[-1] <= 8:
        raise ValueError(f"weight must be ({x.shape[2]}, 1, width) with width 1 to 8, got {tuple(weight.shape)}")
    if checkpoint not in ("full", "int8"):
        raise ValueError(f"checkpoint must be 'full' or 'int8', got {checkpoint!r}")
    _lib.dtype_code(x.dtype)
    _lib.dtype_code(weight.dtype)
    if bias is not None and (bias.shape != (x.shape[2],) or bias.dtype != weight.dtype or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous (dim,) tensor of the weight's dtype")
    _lib.refuse_transforms("causal_conv1d_train", x, weight, bias)
    return _CausalConv1d.apply(x, weight, bias, apply_silu, checkpoint)
