"""A leaf's memory between its forward and its backward pass: replaced data (parameters moved, flattened, sharded) leaves
autograd's version counter alone.  The backward pass reads the leaf where it then lies, and refuses one that has become
another (no GPU needed: a stand-in for the library notes what the entry points are given)."""

from __future__ import annotations

import contextlib

import pytest
import torch

from mamba_metal_amd import _lib
from mamba_metal_amd.conv1d import _CausalConv1d
from mamba_metal_amd.cross_entropy import _LinearCrossEntropy
from mamba_metal_amd.decay_attention import _DecayAttention
from mamba_metal_amd.embedding import _Embedding
from mamba_metal_amd.gated_scan import _GatedScan

CPU = torch.device("cpu")


class Noted:
    """The library's sizes, and entry points that only note their arguments."""

    def __init__(self, lib):
        self.lib, self.calls = lib, {}

    def __getattr__(self, name):
        if name.endswith("_size"):
            return getattr(self.lib, name)

        def entry(*args):
            self.calls[name] = args
            return _lib.OK

        return entry


@pytest.fixture
def noted(monkeypatch):
    lib = Noted(_lib.load())
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_of", lambda dev: None)
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors: CPU)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: CPU.index if t.device == CPU else 0)
    return lib


def leaf(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype).requires_grad_(True)


def fields(lib, name, names):
    return {k: getattr(lib.calls[name][0], k) for k in names}


# Each: the output, what the backward pass reads of the caller's by name, and the addresses that its entry point was given.
def attention(g_shape):
    leaves = dict(q=leaf(2, 70, 1, 8), k=leaf(2, 70, 1, 8), v=leaf(2, 70, 2, 8), log_decay=leaf(*g_shape, dtype=torch.float32))
    y = _DecayAttention.apply(CPU, *leaves.values(), None, torch.full((2,), 70), 1.0, False)
    return y, leaves, lambda lib: fields(lib, "mm_decay_attention_bwd", leaves)


def scan():
    leaves = {k: leaf(2, 20, 8) for k in ("x", "a_gate", "x_gate")}
    leaves["A"] = leaf(8, dtype=torch.float32)
    y = _GatedScan.apply(CPU, *leaves.values(), None, None, torch.full((2,), 20), False, "full")
    return y, leaves, lambda lib: fields(lib, "mm_gated_scan_bwd", leaves)


def conv():
    leaves = dict(x=leaf(2, 20, 8), weight=leaf(8, 4), bias=leaf(8))
    y = _CausalConv1d.apply(*leaves.values(), True, "full")
    return y, leaves, lambda lib: dict(zip(leaves, (lib.calls["mm_causal_conv1d_bwd"][k] for k in (0, 3, 4))))


def head():
    leaves = dict(x=leaf(6, 8), weight=leaf(11, 8), targets=torch.zeros(6, dtype=torch.int64))
    y = _LinearCrossEntropy.apply(CPU, *leaves.values(), -100, "mean")
    return y, leaves, lambda lib: fields(lib, "mm_linear_cross_entropy_bwd", leaves)


def rows():
    ids, weight = torch.zeros(6, dtype=torch.int64), leaf(11, 8)
    y = _Embedding.apply(CPU, ids, weight, 1.0, None)
    return y, dict(ids=ids), lambda lib: dict(ids=lib.calls["mm_embedding_bwd"][0])


CALLS = dict(decays_of_heads=(lambda: attention((2,)), ("q", "k", "v", "log_decay")),
             decays_of_tokens=(lambda: attention((2, 70, 2)), ("q", "k", "v", "log_decay")),
             scan=(scan, ("x", "a_gate", "x_gate", "A")), conv=(conv, ("x", "weight", "bias")),
             head=(head, ("x", "weight", "targets")), rows=(rows, ("ids",)))
NAMES = [pytest.param(f, n, id=f"{what}-{n}") for what, (f, names) in CALLS.items() for n in names]


def lies_elsewhere(t):
    """The same values, with room between the rows: another address, other strides, and the old memory given back."""
    shape = t.shape if t.dim() == 1 else (*t.shape[:-1], t.shape[-1] + 8)
    wide = torch.zeros(shape, dtype=t.dtype)[..., :t.shape[-1]]
    wide.copy_(t.detach())
    t.data = wide


@pytest.mark.parametrize("call,name", NAMES)
def test_read_where_it_lies(noted, call, name):
    y, leaves, given = call()
    lies_elsewhere(leaves[name])
    y.backward(torch.zeros_like(y))
    assert given(noted) == {k: t.data_ptr() for k, t in leaves.items()}


@pytest.mark.parametrize("call", [f for f, _ in CALLS.values()], ids=list(CALLS))
def test_storage_allocated_again(noted, call):
    """What sharded training does: the storage is emptied behind the forward pass and filled before the backward one."""
    y, leaves, given = call()
    sizes = {k: t.untyped_storage().nbytes() for k, t in leaves.items()}
    for t in leaves.values():
        t.untyped_storage().resize_(0)
    others = [torch.zeros(n, dtype=torch.uint8) for n in sizes.values()]
    for k, t in leaves.items():
        t.untyped_storage().resize_(sizes[k])
    y.backward(torch.zeros_like(y))
    assert given(noted) == {k: t.data_ptr() for k, t in leaves.items()} and len(others) == len(leaves)


@pytest.mark.parametrize("call,name", NAMES)
@pytest.mark.parametrize("change", [lambda t: t[..., :1], lambda t: t.new_zeros(0), lambda t: t.to(torch.float64)])
def test_another_one_is_refused(noted, call, name, change):
    y, leaves, _ = call()
    leaves[name].data = change(leaves[name].data)
    with pytest.raises(RuntimeError, match="saved tensor"):
        y.backward(torch.zeros_like(y))


@pytest.mark.parametrize("call,name", NAMES)
def test_hooks_of_one_saved_tensor(noted, call, name):
    """Hooks on a single saved tensor, set behind the forward pass, as offloading does."""
    y, leaves, given = call()
    was, back = leaves[name].data_ptr(), leaves[name].detach().clone()
    for at in y.grad_fn._raw_saved_tensors:  # (autograd's order; what hooks keep of the others is themselves)
        if at.data is not None:
            at.register_hooks(lambda t: None if t.data_ptr() == was else t, lambda t: back if t is None else t)
    y.backward(torch.zeros_like(y))
    assert given(noted)[name] == back.data_ptr()
