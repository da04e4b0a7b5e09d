"""Derivatives that an operator would drop without a word are refused (no GPU needed: the checks come first)."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from mamba_metal_amd import act8_pack, causal_conv1d_train, gated_scan, gated_scan_step

Z3 = torch.zeros((2, 5, 4))
Z2 = torch.zeros((2, 4))


def scan(**kw):
    a = {**dict(x=Z3, a_gate=Z3, x_gate=Z3, A=torch.zeros(4), z=None, h0=None), **kw}
    return gated_scan(a["x"], a["a_gate"], a["x_gate"], a["A"], z=a["z"], h0=a["h0"])


def step(**kw):
    a = {**dict(state=Z2, x=Z2, a_gate=Z2, x_gate=Z2, A=torch.zeros(4), z=None), **kw}
    return gated_scan_step(a["state"].clone() if "state" not in kw else a["state"], a["x"], a["a_gate"], a["x_gate"],
                           a["A"], z=a["z"])


CALLS = [(scan, "x", Z3), (scan, "a_gate", Z3), (scan, "x_gate", Z3), (scan, "A", torch.zeros(4)), (scan, "z", Z3),
         (scan, "h0", Z2), (step, "state", Z2), (step, "x", Z2), (step, "a_gate", Z2), (step, "x_gate", Z2),
         (step, "A", torch.zeros(4)), (step, "z", Z2), (lambda x: act8_pack(x), "x", Z3),
         (lambda x: causal_conv1d_train(x, torch.zeros((4, 1, 2))), "x", Z3),
         (lambda w: causal_conv1d_train(Z3, w, checkpoint="int8"), "w", torch.zeros((4, 1, 2)))]


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("call,name,t", CALLS)
def test_tangents_are_refused(call, name, t, no_grad):
    with fw.dual_level(), torch.set_grad_enabled(not no_grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(**{name: fw.make_dual(t, torch.ones_like(t))})


def test_other_tensors_at_a_level_are_not():
    """No tangent on the call's own tensors: the call goes on to where it needs a GPU."""
    with fw.dual_level():
        fw.make_dual(Z3, torch.ones_like(Z3))
        for call in (scan, step, lambda: act8_pack(Z3)):
            with pytest.raises(ValueError, match="need GPU"):
                call()


def test_jvp_is_refused():
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: scan(x=x), (Z3,), (Z3,))


def test_packing_cuts_no_gradient():
    """A tensor that requires a gradient is refused while gradients are on, and goes on otherwise: under no_grad,
    detached, and in the pack hook of autograd's saved tensors."""
    x = Z3.clone().requires_grad_(True)
    for t in (x, x * 1):
        with pytest.raises(RuntimeError, match="no gradient"):
            act8_pack(t)
        for go in (lambda: act8_pack(t.detach()), torch.no_grad()(lambda: act8_pack(t))):
            with pytest.raises(ValueError, match="need GPU"):
                go()
    with pytest.raises(ValueError, match="need GPU"):
        with torch.autograd.graph.saved_tensors_hooks(act8_pack, lambda p: p):
            x.exp()
