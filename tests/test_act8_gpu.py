"""act8_pack / act8_unpack against the format's definition: whole numbers and powers of two, so exactly."""

from __future__ import annotations

import pytest
import torch

import gated_ref as ref
from mamba_metal_amd import act8_pack, act8_unpack

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(x, packed):
    want = ref.quantise(x.cpu().double().reshape(-1, *x.shape[-2:]) if x.dim() == 3 else x.cpu().double()[None])
    want = want.reshape(x.shape)
    got = act8_unpack(packed)
    assert got.dtype == x.dtype and got.shape == x.shape
    top = torch.finfo(x.dtype).max
    want = want.clamp(-top, top) if x.dtype == torch.float16 else want
    assert torch.equal(got.cpu().double().nan_to_num(nan=1e300), want.nan_to_num(nan=1e300))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 15, 3), (1, 16, 64), (3, 17, 65), (2, 100, 130), (4, 33, 1000),
                                   (1, 5, 4096), (2, 160, 256)])
def test_values(dev, dtype, shape):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(shape, generator=g) * torch.exp(4 * torch.randn(shape[-1], generator=g))).to(dtype).to(dev)
    packed = act8_pack(x)
    got = check(x, packed)
    finite = torch.isfinite(x).cpu()
    b, n, d = shape
    assert packed.codes.abs().max() <= 127 and packed.codes.shape == (b, -(-n // 16), d, 16)
    if n % 16:  # past the sequence
        assert not packed.codes[:, -1, :, n % 16:].any()
    # half a step of the block's power of two; the largest magnitude is at least 63.75 steps (127.5 of the next
    # smaller power of two, which it no longer fits), so half a step is at most 1/127.5 of it
    err = (got.cpu().double() - x.cpu().double()).abs()
    for t in range(0, shape[1], 16):
        top = x[:, t:t + 16].cpu().double().abs().amax(1, keepdim=True)
        ok = (err[:, t:t + 16] <= top / 127.5) | ~torch.isfinite(top) | (top > 32767)
        assert ok[finite[:, t:t + 16]].all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_borders(dev, dtype):
    """Ties between codes, largest magnitudes around the exponent's carry, tiny and huge numbers, zeros."""
    f = torch.finfo(dtype)
    vals = [0.0, -0.0, 1.0, 127.0, 127.5, 128.0, 64.0, 63.5, 0.5, 1.5, 2.5, -2.5, 126.5, f.max, -f.max, f.max / 2,
            f.smallest_normal, f.smallest_normal * f.eps, 3 * f.smallest_normal * f.eps, f.smallest_normal * 127]
    rows = []
    for top in vals:
        for v in vals:
            rows.append([top] + [v] * 3 + [0.0] * 12)
    x = torch.tensor(rows, dtype=torch.float64).t()[None].to(dtype).contiguous().to(dev)
    assert x.shape == (1, 16, len(vals) ** 2)
    check(x, act8_pack(x))


@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_not_finite(dev, bad):
    """Such a block comes back as NaNs; its neighbours in time and channel do not."""
    x = torch.randn((2, 40, 70), generator=torch.Generator().manual_seed(2)).to(dev)
    x[1, 20, 33] = float(bad)
    got = check(x, act8_pack(x))
    nan = torch.isnan(got)
    assert nan[1, 16:32, 33].all() and nan.sum() == 16


def test_shapes_and_strides(dev):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn((3, 50, 200), generator=g).to(torch.bfloat16).to(dev)
    for x in (wide[..., 7:77], wide[:, 3:40], wide.transpose(0, 1), wide[0], wide[:1].expand(4, 50, 200)):
        check(x, act8_pack(x))
    packed = act8_pack(wide)
    out = torch.zeros((3, 60, 300), dtype=torch.float32, device=dev)
    act8_unpack(packed, out=out[:, 5:55, 50:250])
    assert torch.equal(out[:, 5:55, 50:250], act8_unpack(packed, torch.float32))
    assert not out[:, :5].any() and not out[:, 55:].any() and not out[..., :50].any() and not out[..., 250:].any()
    assert packed.nbytes == 3 * 4 * 200 * 17


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0)])
def test_empty(dev, shape):
    packed = act8_pack(torch.zeros(shape, device=dev))
    assert act8_unpack(packed).shape == shape


def test_graph(dev):
    x = torch.randn((2, 100, 130), device=dev)
    act8_unpack(act8_pack(x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = act8_unpack(act8_pack(x))
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, act8_unpack(act8_pack(x)))
