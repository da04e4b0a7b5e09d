"""The codes of a block that holds an infinity or a NaN: zeros, whatever bits the NaN carries."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import act8_pack, act8_unpack
from mamba_metal_amd.conv1d import _conv1d_act8

pytestmark = pytest.mark.gpu

BITS = [0x7FC00000, 0x7FC000FF, 0x7FC00080, -0x400000 + 0x55, 0x7F800001, 0x7F8000AA, 0x7F800000, -0x800000]


@pytest.mark.parametrize("huge", [False, True])  # with and without blocks of the largest exponent in the same wave
def test_codes_of_a_broken_block(dev, huge):
    n, d = 40, 70
    x = torch.randn((1, n, d), generator=torch.Generator().manual_seed(1))
    for k, bits in enumerate(BITS):
        x[0, 16 + k, 5 * k] = torch.tensor(bits, dtype=torch.int32).view(torch.float32)
    if huge:
        x[0, 20, 3] = torch.finfo(torch.float32).max
    x = x.to(dev)
    _, conv = _conv1d_act8(x, torch.ones((d, 1, 2), device=dev), None, True)
    for packed in (act8_pack(x), conv):
        bad = torch.zeros((1, 3, d), dtype=torch.bool, device=dev)
        bad[0, 1, [5 * k for k in range(len(BITS))]] = True
        assert torch.equal(packed.exps == 255, bad)
        assert not packed.codes[bad].any() and packed.codes[~bad].any(-1).all()
        assert packed.codes.min() >= -127
        back = act8_unpack(packed)
        assert torch.isnan(back[0, 16:32, ::5][:, :len(BITS)]).all()
        if huge:  # cut to 127 steps of the largest power of two
            assert packed.codes[0, 1, 3, 4] == 127 and packed.exps[0, 1, 3] == 248


@pytest.mark.parametrize("n,strides", [(20, (70, 210)), (2, (140, 70)), (2, (140, 210)), (3, (331, 90))])
def test_unpack_into_rows_between_others(dev, n, strides):
    """Time outside the batch, inside it, and rows of one sequence between those of another; the rest stays."""
    b, d = 3, 70
    packed = act8_pack(torch.randn((b, n, d), generator=torch.Generator().manual_seed(2)).to(dev))
    store = torch.full(((b - 1) * strides[0] + (n - 1) * strides[1] + d + 5,), 9.0, device=dev)
    out = store.as_strided((b, n, d), (*strides, 1))
    act8_unpack(packed, out=out)
    assert torch.equal(out, act8_unpack(packed))
    covered = torch.zeros_like(store, dtype=torch.bool)
    covered.as_strided((b, n, d), (*strides, 1)).fill_(True)
    assert covered.sum() == b * n * d and (store[~covered] == 9.0).all()


def test_unpack_into_rows_that_overlap(dev):
    packed = act8_pack(torch.ones((3, 4, 70), device=dev))
    store = torch.full((2000,), 9.0, device=dev)
    for strides in ((70, 70), (140, 70), (210, 139), (69, 300)):
        with pytest.raises(RuntimeError, match="overlap"):
            act8_unpack(packed, out=store.as_strided((3, 4, 70), (*strides, 1)))
    assert (store == 9.0).all()
