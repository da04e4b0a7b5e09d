"""Softmax cross entropy of the rows before a language model's head, without keeping the logits.

    l = W x          loss = log sum_v exp(l_v) - l[target]

It stands at the end of a model that trains through ``gated_scan``, ``decay_attention`` and ``causal_conv1d_train``;
``MambaModel.loss`` scores text with it.  Where logits of (rows, vocab) would be written, read and kept, this keeps a
float32 number a row; its backward pass computes the logits again, a piece of the vocabulary at a time.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from mamba_metal_amd import _lib
from mamba_metal_amd.act8 import channels_last

REDUCTIONS = ("none", "mean", "sum")


def _params(x, weight, targets, ignore_index, reduction):
    p = _lib.LinearCrossEntropyParams()
    p.x, p.x_stride = x.data_ptr(), x.stride(0)
    p.weight, p.weight_stride = weight.data_ptr(), weight.stride(0)
    p.targets, p.targets_dtype = targets.data_ptr(), 1 if targets.dtype == torch.int64 else 0
    p.rows, p.dim = x.shape
    p.vocab = weight.shape[0]
    p.ignore_index = ignore_index
    p.dtype = _lib.dtype_code(x.dtype)
    p.reduction = REDUCTIONS.index(reduction)
    return p


def _call(name, p, backward, dev):
    lib = _lib.load()
    nbytes = lib.mm_linear_cross_entropy_workspace_size(p, backward)
    if nbytes:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    with _lib.on_device(dev):
        st = getattr(lib, name)(p, _lib.stream_of(dev))
    _lib.check(st, name)


def _forward(dev, x, weight, targets, ignore_index, reduction, train):
    """The loss and, for training, each row's log of the sum of exponentials."""
    p = _params(x, weight, targets, ignore_index, reduction)
    if reduction == "none":
        loss = torch.empty(targets.shape, dtype=torch.float32, device=dev)
    elif x.shape[0]:
        loss = torch.empty((), dtype=torch.float32, device=dev)
    else:  # (no rows: a sum of nothing, a mean of none)
        loss = torch.full((), 0.0 if reduction == "sum" else float("nan"), dtype=torch.float32, device=dev)
    p.loss = loss.data_ptr()
    lse = None
    if train:
        lse = torch.empty((x.shape[0],), dtype=torch.float32, device=dev)
        p.lse = lse.data_ptr()
    _call("mm_linear_cross_entropy_fwd", p, 0, dev)
    return loss, lse


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dev, x, weight, targets, ignore_index, reduction):
        loss, lse = _forward(dev, x, weight, targets, ignore_index, reduction, True)
        ctx.meta = (dev, x.dtype, x.shape, weight.shape, ignore_index, reduction, (targets.dtype, targets.shape))
        ctx.save_for_backward(x, weight, targets, lse)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        dev, dtype, x_shape, w_shape, ignore_index, reduction, kind = ctx.meta
        x, weight, targets, lse = ctx.saved_tensors  # (which hooks or a new .data may have changed)
        x, weight = (_lib.saved(t, dtype, s, dev, rows=True) for t, s in ((x, x_shape), (weight, w_shape)))
        targets, lse = _lib.saved(targets, *kind, dev), _lib.saved(lse, torch.float32, x_shape[:1], dev)
        p = _params(x, weight, targets, ignore_index, reduction)
        p.lse = lse.data_ptr()
        dloss = dloss.float().reshape(-1)
        p.dloss, p.dloss_stride = dloss.data_ptr(), dloss.stride(0)
        dx = dweight = None
        if ctx.needs_input_grad[1]:
            dx = torch.empty(x_shape, dtype=dtype, device=dev)
            p.dx = dx.data_ptr()
        if ctx.needs_input_grad[2]:
            dweight = (torch.empty if x_shape[0] else torch.zeros)(w_shape, dtype=dtype, device=dev)
            p.dweight = dweight.data_ptr()
        _call("mm_linear_cross_entropy_bwd", p, 1, dev)
        return None, dx, dweight, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of softmax(x W^T) against ``targets``, in float32.

    x: (..., dim), weight: (vocab, dim), of one dtype (float32, float16, bfloat16) with unit channel stride; targets:
    int32 or int64 of x's leading shape.  A row whose target is ``ignore_index`` has a loss of 0 and no gradient, whatever
    it holds; any other target outside 0 .. vocab - 1 makes its row's loss (and so its gradients) NaN.  ``reduction``:
    "none", a loss for every row, in targets' shape; "mean" over the rows that are not ignored (NaN if there is none);
    "sum".

    Logits and their sums are float32.  Gradients flow to x and weight (once, not twice, and not in forward mode): the
    gradient of the logits is rounded once to x's dtype (in float16 times a power of two that keeps it in range; of a
    "mean" or "sum" before its one factor), in pieces of at most 512 MB (or of 256 tokens), and sums over the vocabulary and
    the rows are float32, in a fixed order.

    To capture a backward pass into a graph, capture the forward pass with it, and let no eager autograd graph of the
    same leaf tensors be alive at that time."""
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {REDUCTIONS}, got {reduction!r}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., dim), got {tuple(x.shape)}")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise ValueError(f"weight must be (vocab, {x.shape[-1]}), got {tuple(weight.shape)}")
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"targets is {tuple(targets.shape)}, expected {tuple(x.shape[:-1])}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"targets is {targets.dtype}, expected int32 or int64")
    if not -2 ** 63 <= int(ignore_index) < 2 ** 63:
        raise ValueError(f"ignore_index {ignore_index} is no 64-bit integer")
    _lib.dtype_code(x.dtype)
    if weight.dtype != x.dtype:
        raise TypeError(f"weight is {weight.dtype}, x {x.dtype}")
    channels_last(x, "x")
    channels_last(weight, "weight")
    _lib.refuse_transforms("linear_cross_entropy", x, weight, targets)
    dev = _lib.require_cuda(x, weight, targets)
    x2, targets = x.reshape(-1, x.shape[-1]), targets.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(dev, x2, weight, targets, int(ignore_index), reduction)
    return _forward(dev, x2, weight, targets, int(ignore_index), reduction, False)[0]
