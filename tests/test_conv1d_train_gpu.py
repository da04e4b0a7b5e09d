"""causal_conv1d_train: the forward pass is causal_conv1d's, the gradients those of the 64-bit formulas."""

from __future__ import annotations

import pytest
import torch

import gated_ref as ref
from mamba_metal_amd import causal_conv1d_train
from mamba_metal_amd.conv1d import causal_conv1d

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [(1, 1, 1), (2, 2, 3), (3, 3, 64), (2, 16, 65), (1, 63, 130), (2, 64, 64), (1, 65, 66), (2, 130, 200),
         (1, 700, 96), (40, 20, 8)]


def rand(seed, b, n, d, width, dtype, dev, wdtype=None, bias=True):
    g = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(s, generator=g)
    wd = wdtype or dtype
    return {"x": t(b, n, d).to(dtype).to(dev), "weight": (t(d, 1, width) * width ** -0.5).to(wd).to(dev),
            "bias": t(d).to(wd).to(dev) if bias else None, "dy": t(b, n, d).to(dtype).to(dev)}


def train(f, **kw):
    leaves = {k: f[k].detach().clone().requires_grad_(True) for k in ("x", "weight", "bias") if f[k] is not None}
    y = causal_conv1d_train(leaves["x"], leaves["weight"], leaves.get("bias"), **kw)
    return y, dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), f["dy"])))


def check(f, y, got, apply_silu=True, eight=False):
    assert torch.equal(y, causal_conv1d(f["x"], f["weight"], f["bias"], apply_silu=apply_silu))
    d64 = {k: None if v is None else v.detach().cpu().double() for k, v in f.items()}
    x = ref.quantise(d64["x"]) if eight else d64["x"]
    want = ref.conv_backward(x, d64["weight"], d64["bias"], d64["dy"], apply_silu)
    for k, v in got.items():
        assert v.dtype == f[k].dtype and v.shape == f[k].shape
        ref.close(v, *want[k], v.dtype, "d" + k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_gradients(dev, dtype, size, checkpoint):
    f = rand(1, *size, 4, dtype, dev)
    check(f, *train(f, checkpoint=checkpoint), eight=checkpoint == "int8")


@pytest.mark.parametrize("width", [1, 2, 3, 5, 6, 7, 8])
@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("apply_silu,bias", [(True, False), (False, True)])
def test_widths(dev, width, checkpoint, apply_silu, bias):
    f = rand(2, 2, 75, 70, width, torch.float32, dev, bias=bias)
    check(f, *train(f, checkpoint=checkpoint, apply_silu=apply_silu), apply_silu, checkpoint == "int8")


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
def test_weight_dtype(dev, dtype, wdtype):
    f = rand(3, 2, 100, 130, 4, dtype, dev, wdtype)
    check(f, *train(f))


def test_strides(dev):
    f = rand(4, 3, 70, 66, 4, torch.bfloat16, dev)
    wide = torch.zeros((3, 70, 140), dtype=torch.bfloat16, device=dev)
    wide[..., 3:69] = f["x"]
    x = wide[..., 3:69].requires_grad_(True)
    w = f["weight"].transpose(0, 2).contiguous().transpose(0, 2).requires_grad_(True)
    y = causal_conv1d_train(x, w, f["bias"])
    dx, dw = torch.autograd.grad(y, [x, w], f["dy"].transpose(0, 1).contiguous().transpose(0, 1))
    check(f, y, {"x": dx, "weight": dw})
    # a 2-D weight, and only the input's gradient
    x = f["x"].clone().requires_grad_(True)
    y = causal_conv1d_train(x, f["weight"][:, 0], f["bias"])
    check(f, y, {"x": torch.autograd.grad(y, x, f["dy"])[0]})
    # the gradient of a sum, which has no strides; only the weight's gradient
    w = f["weight"].clone().requires_grad_(True)
    y = causal_conv1d_train(f["x"], w, f["bias"])
    dw, = torch.autograd.grad(y.sum(), w)
    check({**f, "dy": torch.ones_like(f["dy"])}, y, {"weight": dw})


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0)])
@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_empty(dev, shape, checkpoint):
    f = rand(5, *shape, 4, torch.float32, dev)
    y, got = train(f, checkpoint=checkpoint)
    assert y.shape == shape and got["x"].shape == shape and not got["weight"].any() and not got["bias"].any()


def test_many_rows_of_partial_sums(dev):
    """Enough runs that the sums' rows go through two passes."""
    f = rand(10, 700, 17, 9, 4, torch.float32, dev)
    check(f, *train(f))


def test_nan_stays_in_its_channel(dev):
    f = rand(6, 2, 100, 130, 4, torch.float32, dev)
    clean = train(f)
    f["x"][0, 50, 100] = float("nan")
    dirty = train(f)
    for k in ("x", "weight", "bias"):
        same = clean[1][k] == dirty[1][k]
        (same[..., 100] if k == "x" else same[100]).fill_(True)
        assert same.all(), k
    assert torch.isnan(dirty[1]["weight"][100]).all()


def test_against_differences(dev):
    f = rand(7, 2, 40, 20, 4, torch.float32, dev)
    _, got = train(f)
    g = torch.Generator().manual_seed(8)
    d64 = {k: v.cpu().double() for k, v in f.items()}
    for k in ("x", "weight", "bias"):
        v = torch.randn(f[k].shape, generator=g, dtype=torch.float64)

        def loss(s):
            q = {**d64, k: d64[k] + s * v}
            p, _, _ = ref.conv(q["x"], q["weight"], q["bias"], True)
            return (p * torch.sigmoid(p) * d64["dy"]).sum()

        diff = ((loss(1e-6) - loss(-1e-6)) / 2e-6).item()
        parts = got[k].cpu().double() * v
        assert abs(parts.sum().item() - diff) <= 1e-5 * parts.abs().sum().item() + 1e-6, k


def test_repeats_bit_for_bit_and_in_a_graph(dev):
    f = rand(9, 2, 1500, 130, 4, torch.bfloat16, dev)
    first = train(f, checkpoint="int8")
    static = {k: v.clone() for k, v in f.items()}
    for k in ("x", "weight", "bias"):
        static[k].requires_grad_(True)

    def step():
        y = causal_conv1d_train(static["x"], static["weight"], static["bias"], checkpoint="int8")
        return torch.autograd.grad(y, [static[k] for k in ("x", "weight", "bias")], static["dy"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        again = train(f, checkpoint="int8")
        graph.replay()
        torch.cuda.synchronize()
        for k, o in zip(("x", "weight", "bias"), out):
            assert torch.equal(first[1][k], again[1][k]) and torch.equal(first[1][k], o)
