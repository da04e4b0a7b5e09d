"""decay_attention at the ends of its sizes: values of 1024 channels, as many sequences and heads as it takes, long ones.
Tolerances as derived in test_decay_attention_gpu.py and test_decay_attention_16bit_gpu.py."""

from __future__ import annotations

import pytest
import torch

import decay_ref
from mamba_metal_amd import decay_attention_step
from test_decay_attention_16bit_gpu import check
from test_decay_attention_gpu import BF16, F16, F32, half_step, inputs, near, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(2, 130, 1, 2, 128, 1024), (1, 70, 2, 1, 5, 1000), (2, 200, 1, 3, 64, 200), (4, 130, 1, 64, 16, 1021)])
def test_wide_values(dev, dt, shape):
    s = inputs(dev, dt, *shape, h0=True, ragged=True, seed=sum(shape))
    outs, grads = run(s, 0.6)
    check(s, 0.6, outs, grads)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("shape", [(65535, 2, 1, 1, 3, 2), (1, 3, 65535, 1, 2, 3), (1, 3, 1, 65535, 2, 3), (300, 65, 13, 7, 4, 4)])
def test_many(dev, dt, shape):
    """Sequences, groups, and heads that share one."""
    s = inputs(dev, dt, *shape, h0=True, ragged=True, seed=5)
    outs, grads = run(s, 1.0)
    check(s, 1.0, outs, grads)


@pytest.mark.parametrize("dt", [F32, F16])
def test_long(dev, dt):
    s = inputs(dev, dt, 1, 9001, 1, 4, 4, 4)
    outs, grads = run(s, 1.0)
    check(s, 1.0, outs, grads)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(2, 1, 2, 128, 1024), (3, 2, 1, 3, 1021), (1, 65535, 1, 1, 1), (65535, 1, 1, 2, 4), (2, 1, 65535, 1, 3)])
def test_steps(dev, dt, shape):
    """The token step in place, as it is called by default."""
    b, groups, per, dk, dv = shape
    s = inputs(dev, dt, b, 1, groups, per, dk, dv, h0=True)
    y_ref, states = decay_ref.forward(s["q"], s["k"], s["v"], s["g"], 0.9, s["h0"])
    ay, ast = decay_ref.forward(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["g"], 0.9, s["h0"].abs())
    state = s["h0"].clone()
    y = decay_attention_step(state, *(s[k][:, 0] for k in ("q", "k", "v", "g")), scale=0.9)
    near(state, states[:, 1], 8 * 2.0 ** -24 * ast[:, 1], "state")
    least = 2.0 ** -25 if dt == F16 else 0.0
    near(y, y_ref[:, 0], half_step(dt) * y_ref[:, 0].abs() + 160 * 2.0 ** -24 * ay[:, 0] + least, "y")


def test_two_calls_at_once(dev):
    """On two streams, with workspaces of their own: the same bits as one after the other."""
    many = [inputs(dev, BF16, 1, 1500, 1, 4, 64, 64, seed=k) for k in range(2)]
    want = [run(s, 1.0) for s in many]
    streams = [torch.cuda.Stream() for _ in many]
    for _ in range(3):
        torch.cuda.synchronize()
        got = []
        for s, stream in zip(many, streams):
            with torch.cuda.stream(stream):
                got.append(run(s, 1.0))
        torch.cuda.synchronize()
        for (o, g), (wo, wg) in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip([*o, *g], [*wo, *wg]))
