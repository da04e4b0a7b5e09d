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
