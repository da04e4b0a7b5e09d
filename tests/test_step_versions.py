"""The token steps write the caller's tensors in place, and autograd hears of it: a backward pass that saved one of them
refuses it (no GPU needed: a stand-in for the library)."""

from __future__ import annotations

import contextlib

import pytest
import torch

from mamba_metal_amd import _lib, decay_attention_step, gated_scan_step


@pytest.fixture(autouse=True)
def stand_in(monkeypatch):
    class Lib:
        def __getattr__(self, name):
            return lambda *args: _lib.OK

    monkeypatch.setattr(_lib, "load", Lib)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_of", lambda dev: None)
    monkeypatch.setattr(_lib, "require_cuda", lambda *tensors: torch.device("cpu"))


def attention(state, **kw):
    q, v = torch.ones((2, 1, 4)), torch.ones((2, 3, 5))
    return decay_attention_step(state, q, q, v, torch.zeros((2, 3)), **kw)


def scan(state, **kw):
    x = torch.ones((2, 4))
    return gated_scan_step(state, x, x, x, torch.zeros(4), **kw)


STEPS = [(attention, (2, 3, 4, 5), (2, 3, 5)), (scan, (2, 4), (2, 4))]


@pytest.mark.parametrize("step,state,out", STEPS, ids=["attention", "scan"])
@pytest.mark.parametrize("given", [(), ("state_out",), ("out",), ("state_out", "out")])
def test_what_is_written_is_counted(step, state, out, given):
    t = dict(state=torch.ones(state), state_out=torch.ones(state), out=torch.ones(out))
    leaf = torch.ones((), requires_grad=True)
    losses = {k: (leaf * x).sum() for k, x in t.items()}  # (saves x)
    step(t["state"], **{k: t[k] for k in given})
    written = {"state" if "state_out" not in given else "state_out"} | ({"out"} & set(given))
    for name, loss in losses.items():
        if name in written:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
        else:
            loss.backward()


@pytest.mark.parametrize("step,state,out", STEPS, ids=["attention", "scan"])
def test_inference_tensors(step, state, out):
    with torch.inference_mode():
        step(torch.ones(state), out=torch.ones(out))
        s = torch.ones(state)
    step(s)
    normal = torch.ones(state)
    with torch.inference_mode():
        step(normal)
    assert normal._version == 1


@pytest.mark.parametrize("step,state,out", STEPS, ids=["attention", "scan"])
@pytest.mark.parametrize("name", ["state_out", "out"])
def test_outputs_that_require_a_gradient(step, state, out, name):
    """Refused while gradients are on, like the inputs: what is written there has none."""
    t = torch.ones(out if name == "out" else state, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        step(torch.ones(state), **{name: t})
    with torch.no_grad():
        step(torch.ones(state), **{name: t})
