"""A leaf's memory between its forward and its backward pass: replaced data (parameters moved, flattened, sharded) leaves
autograd's version counter alone.  The backward pass reads the leaf where it then lies, and refuses one that has become
another (no GPU needed: a stand-in for the library notes what the entry points are given)."""

from __future__ import annotations

import contextlib

import pytest
import torch

from mamba_metal_amd import _lib
from mamba_metal_amd.decay_attention import _DecayAttention

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
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: CPU.index if t.device == CPU else 0)
    return lib


def leaf(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype).requires_grad_(True)


def attention(g_shape):
    leaves = dict(q=leaf(2, 70, 1, 8), k=leaf(2, 70, 1, 8), v=leaf(2, 70, 2, 8), log_decay=leaf(*g_shape, dtype=torch.float32))
    lengths = torch.full((2,), 70)
    y = _DecayAttention.apply(CPU, *leaves.values(), None, lengths, 1.0, False)
    return y, leaves, lambda lib: {k: getattr(lib.calls["mm_decay_attention_bwd"][0], k) for k in leaves}


ATTENTION = [lambda: attention((2,)), lambda: attention((2, 70, 2))]
NAMES = [(f, n) for f in ATTENTION for n in ("q", "k", "v", "log_decay")]


def lies_elsewhere(t):
    """The same values, with room between the rows: another address, other strides, and the old memory given back."""
    wide = torch.zeros((*t.shape[:-1], t.shape[-1] + 8), dtype=t.dtype)[..., :t.shape[-1]]
    wide.copy_(t.detach())
    t.data = wide


@pytest.mark.parametrize("call,name", NAMES)
def test_read_where_it_lies(noted, call, name):
    y, leaves, given = call()
    lies_elsewhere(leaves[name])
    y.backward(torch.zeros_like(y))
    assert given(noted) == {k: t.data_ptr() for k, t in leaves.items()}


@pytest.mark.parametrize("call", ATTENTION)
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
    assert given(noted) == {k: t.data_ptr() for k, t in leaves.items()} and len(others) == 4


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
    back = leaves[name].detach().clone()
    y.grad_fn._raw_saved_tensors[list(leaves).index(name)].register_hooks(lambda t: None, lambda _: back)
    y.backward(torch.zeros_like(y))
    assert given(noted)[name] == back.data_ptr()
