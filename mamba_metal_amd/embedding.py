"""Rows of an embedding table, scaled, with the table's gradient by sorted tokens.

    y_i = scale weight[ids_i]          dweight[v] = scale sum_{i : ids_i = v} dy_i

It stands at the front of a model that trains through ``gated_scan``, ``decay_attention`` and ``causal_conv1d_train``, as
``linear_cross_entropy`` stands at its end.  A row's gradient is summed in float32 in the order of its tokens and rounded
once: calls repeat bit for bit.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from mamba_metal_amd import _lib
from mamba_metal_amd.act8 import channels_last


def _forward(dev, ids, weight, scale):
    lib = _lib.load()
    y = weight.new_empty((*ids.shape, weight.shape[1]))
    with _lib.on_device(dev):
        st = lib.mm_embedding_fwd(ids.data_ptr(), weight.data_ptr(), y.data_ptr(), ids.numel(), *weight.shape, weight.stride(0),
                                  scale, 1 if ids.dtype == torch.int64 else 0, _lib.dtype_code(weight.dtype), _lib.stream_of(dev))
    _lib.check(st, "mm_embedding_fwd")
    return y


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, dev, ids, weight, scale, padding_idx):
        ctx.meta = (dev, weight.dtype, weight.shape, scale, padding_idx, (ids.dtype, ids.shape))
        ctx.save_for_backward(ids)
        return _forward(dev, ids, weight, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dev, dtype, (vocab, dim), scale, padding_idx, kind = ctx.meta
        ids = _lib.saved(*ctx.saved_tensors, *kind, dev)  # (which hooks or a new .data may have changed)
        dy = (dy if dy.dtype == dtype else dy.to(dtype)).reshape(-1, dim)
        if dy.stride(1) != 1 and dim > 1:
            dy = dy.contiguous()
        lib = _lib.load()
        n = dy.shape[0]
        dweight = dy.new_empty((vocab, dim))
        nbytes = lib.mm_embedding_bwd_workspace_size(n, vocab, dim)
        work = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        with _lib.on_device(dev):
            st = lib.mm_embedding_bwd(ids.data_ptr(), dy.data_ptr(), dweight.data_ptr(), n, vocab, dim, dy.stride(0), scale,
                                      -1 if padding_idx is None else padding_idx, 1 if ids.dtype == torch.int64 else 0,
                                      _lib.dtype_code(dtype), _lib.ptr(work), nbytes, _lib.stream_of(dev))
        _lib.check(st, "mm_embedding_bwd")
        return None, None, dweight, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """The rows ``ids`` of ``weight``, times ``scale``: (*ids.shape, dim) in weight's dtype, rounded once.

    ids: int32 or int64, any shape; weight: (vocab, dim), float32, float16 or bfloat16, with unit channel stride.  An id
    outside 0 .. vocab - 1 gives a row of NaNs, and no gradient.  ``padding_idx`` (negative: from the end) is an id whose
    row is looked up like any other and gets no gradient.

    The gradient flows to weight (once, not twice, and not in forward mode): a dense (vocab, dim), zeros in the rows that
    no id names.  To capture a backward pass into a graph, capture the forward pass with it, and let no eager autograd
    graph of the same weight be alive at that time."""
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids is {ids.dtype}, expected int32 or int64")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be (vocab, dim), got {tuple(weight.shape)}")
    _lib.dtype_code(weight.dtype)
    channels_last(weight, "weight")
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} is outside a vocabulary of {weight.shape[0]}")
        padding_idx %= weight.shape[0]
    _lib.refuse_transforms("embedding", ids, weight)
    dev = _lib.require_cuda(ids, weight)
    ids = ids.contiguous()
    if torch.is_grad_enabled() and weight.requires_grad:
        return _Embedding.apply(dev, ids, weight, float(scale), padding_idx)
    return _forward(dev, ids, weight, float(scale))
