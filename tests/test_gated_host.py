"""Refusals of the gated recurrence, the 8-bit checkpoints and the conv's training form, before any HIP call
(no GPU needed): the Python checks, and the C entry points' own."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mamba_metal_amd import Act8, _lib, act8_pack, act8_unpack, causal_conv1d_train, gated_scan, gated_scan_step
from test_abi import FAKE, test_params_layout_matches_header as layout


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_params_layout(tmp_path):
    layout(tmp_path, "mm_gated_scan_params", _lib.GatedScanParams)


def z3(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def scan(x=None, a=None, g=None, A=None, **kw):
    x = z3(2, 5, 4) if x is None else x
    return gated_scan(x, x if a is None else a, x if g is None else g, z3(x.shape[-1]) if A is None else A, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(x=z3(5, 4)), ValueError),
    (dict(a=z3(2, 5, 3)), ValueError),
    (dict(g=z3(2, 4, 4)), ValueError),
    (dict(z=z3(1, 5, 4)), ValueError),
    (dict(a=z3(2, 5, 4, dtype=torch.float16)), TypeError),
    (dict(z=z3(2, 5, 4, dtype=torch.bfloat16)), TypeError),
    (dict(x=z3(2, 5, 4, dtype=torch.float64)), TypeError),
    (dict(x=z3(2, 4, 5).transpose(1, 2)), ValueError),
    (dict(z=z3(1, 1, 1).expand(2, 5, 4)), ValueError),
    (dict(A=z3(5)), ValueError),
    (dict(A=z3(4, 16)), ValueError),
    (dict(A=torch.zeros(4, dtype=torch.int32)), TypeError),
    (dict(h0=z3(2, 5)), ValueError),
    (dict(h0=torch.zeros((2, 4), dtype=torch.int64)), TypeError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(lengths=torch.zeros(2)), TypeError),
    (dict(checkpoint="int4"), ValueError),
    (dict(), ValueError),  # not on a GPU
])
def test_gated_scan_refuses(kw, err):
    with pytest.raises(err):
        scan(**kw)


@pytest.mark.parametrize("kw,err", [
    (dict(x=z3(2, 5, 4)), ValueError),
    (dict(state=z3(2, 5)), ValueError),
    (dict(state=z3(2, 4, dtype=torch.float16)), ValueError),
    (dict(state=z3(4, 2).t()), ValueError),
    (dict(state_out=z3(3, 4)), ValueError),
    (dict(out=z3(2, 4, dtype=torch.float16)), TypeError),
    (dict(x=z3(4, 2).t()), ValueError),
    (dict(A=z3(2)), ValueError),
    (dict(state=z3(2, 4).requires_grad_(True)), RuntimeError),
    (dict(), ValueError),
])
def test_gated_scan_step_refuses(kw, err):
    a = dict(state=z3(2, 4), x=z3(2, 4), A=z3(4))
    a.update(kw)
    with pytest.raises(err):
        gated_scan_step(a["state"], a["x"], a["x"], a["x"], a["A"], state_out=a.get("state_out"), out=a.get("out"))


def test_act8_refuses():
    for x, err in ((z3(4), ValueError), (z3(1, 2, 3, 4), ValueError), (z3(2, 3, dtype=torch.float64), TypeError),
                   (z3(3, 2).t(), ValueError), (z3(2, 3), ValueError)):
        with pytest.raises(err):
            act8_pack(x)
    codes, exps = torch.zeros((1, 2, 3, 16), dtype=torch.int8), torch.zeros((1, 2, 3), dtype=torch.uint8)
    shape = torch.Size((1, 20, 3))
    good = Act8(codes, exps, shape, torch.float32)
    for packed, kw, err in ((Act8(codes, exps[:, :1], shape, torch.float32), {}, ValueError),
                            (Act8(codes, exps, torch.Size((1, 40, 3)), torch.float32), {}, ValueError),
                            (Act8(codes, exps, torch.Size((20,)), torch.float32), {}, ValueError),
                            (Act8(codes.float(), exps, shape, torch.float32), {}, ValueError),
                            (Act8(codes, exps.char(), shape, torch.float32), {}, ValueError),
                            (good, dict(dtype=torch.int8), TypeError),
                            (good, dict(out=z3(1, 20, 4)), ValueError),
                            (good, dict(out=z3(1, 3, 20).transpose(1, 2)), ValueError),
                            (good, dict(out=z3(1, 20, 3), dtype=torch.float16), TypeError),
                            (good, {}, ValueError)):
        with pytest.raises(err):
            act8_unpack(packed, **kw)


@pytest.mark.parametrize("kw,err", [
    (dict(x=z3(5, 4)), ValueError),
    (dict(x=z3(2, 4, 5).transpose(1, 2), weight=z3(4, 1, 4)), ValueError),
    (dict(weight=z3(5, 1, 4)), ValueError),
    (dict(weight=z3(4, 1, 9)), ValueError),
    (dict(weight=z3(4, 1, 0)), ValueError),
    (dict(checkpoint="half"), ValueError),
    (dict(x=z3(2, 5, 4, dtype=torch.float64)), TypeError),
    (dict(weight=z3(4, 1, 4, dtype=torch.float64)), TypeError),
    (dict(bias=z3(5)), ValueError),
    (dict(bias=z3(4, dtype=torch.float16)), ValueError),
    (dict(bias=z3(8)[::2]), ValueError),
    (dict(), ValueError),
    (dict(checkpoint="int8"), ValueError),
])
def test_conv_refuses(kw, err):
    a = dict(x=z3(2, 5, 4), weight=z3(4, 1, 4), checkpoint="full", bias=None)
    a.update(kw)
    with pytest.raises(err):
        causal_conv1d_train(a["x"], a["weight"], a["bias"], checkpoint=a["checkpoint"])


# ------------------------------------------------------------------------------ the C entry points
def params(**over):
    p = _lib.GatedScanParams()
    for k in ("x", "a_gate", "x_gate", "A", "y", "dy", "dx", "da_gate", "dx_gate", "dA", "block_states", "workspace"):
        setattr(p, k, FAKE)
    p.batch, p.seqlen, p.dim, p.workspace_bytes = 2, 3000, 64, 1 << 40
    for k in ("x", "a_gate", "x_gate", "z", "y", "dy"):
        setattr(p, f"{k}_stride", (_lib._i64a2)(3000 * 64, 64))
    for k, v in over.items():
        if k in ("codes", "exps"):
            getattr(p, k)[v] = FAKE
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,status", [
    (dict(batch=-1), _lib.ERR_SHAPE),
    (dict(seqlen=-1), _lib.ERR_SHAPE),
    (dict(dim=-1), _lib.ERR_SHAPE),
    (dict(batch=1 << 40, seqlen=1 << 30), _lib.ERR_SHAPE),
    (dict(dtype=3), _lib.ERR_DTYPE),
    (dict(lengths=FAKE, lengths_dtype=2), _lib.ERR_DTYPE),
    (dict(handoff_timeout_us=-1), _lib.ERR_SHAPE),
    (dict(A=None), _lib.ERR_NULL_POINTER),
    (dict(x=None), _lib.ERR_NULL_POINTER),
    (dict(x_gate=None), _lib.ERR_NULL_POINTER),
    (dict(a_gate_stride=(_lib._i64a2)(-1, 1)), _lib.ERR_LAYOUT),
    (dict(codes=0), _lib.ERR_NULL_POINTER),
    (dict(exps=1), _lib.ERR_NULL_POINTER),
])
def test_gated_scan_c_refuses(lib, over, status):
    for f in (lib.mm_gated_scan_fwd, lib.mm_gated_scan_bwd):
        assert f(ctypes.byref(params(**over)), None) == status
        assert lib.mm_last_error().decode().startswith(lib.mm_status_name(status).decode())


@pytest.mark.parametrize("name,over,status", [
    ("fwd", dict(y=None), _lib.ERR_NULL_POINTER),
    ("fwd", dict(y_stride=(_lib._i64a2)(0, -64)), _lib.ERR_LAYOUT),
    ("fwd", dict(y_stride=(_lib._i64a2)(0, 64)), _lib.ERR_LAYOUT),
    ("fwd", dict(y_stride=(_lib._i64a2)(64, 0)), _lib.ERR_LAYOUT),
    ("bwd", dict(dy=None), _lib.ERR_NULL_POINTER),
    ("bwd", dict(dx=None), _lib.ERR_NULL_POINTER),
    ("bwd", dict(z=FAKE), _lib.ERR_NULL_POINTER),  # dz missing
    ("bwd", dict(block_states=None), _lib.ERR_NULL_POINTER),
    ("bwd", dict(dA=None), _lib.ERR_NULL_POINTER),
    ("bwd", dict(dy_stride=(_lib._i64a2)(-1, 64)), _lib.ERR_LAYOUT),
    ("bwd", dict(workspace=None), _lib.ERR_WORKSPACE),
    ("bwd", dict(workspace_bytes=16), _lib.ERR_WORKSPACE),
    ("bwd", dict(workspace=FAKE + 16), _lib.ERR_WORKSPACE),
])
def test_gated_scan_c_refuses_outputs(lib, name, over, status):
    assert getattr(lib, f"mm_gated_scan_{name}")(ctypes.byref(params(**over)), None) == status


def test_gated_scan_c_empty(lib):
    for over in (dict(batch=0), dict(dim=0)):
        for f in (lib.mm_gated_scan_fwd, lib.mm_gated_scan_bwd):
            assert f(ctypes.byref(params(**over)), None) == _lib.OK
    assert lib.mm_gated_scan_fwd(None, None) == _lib.ERR_NULL_POINTER


def step(lib, **over):
    a = dict(state=FAKE, state_out=FAKE, x=FAKE, a=FAKE, g=FAKE, A=FAKE, z=None, y=FAKE, batch=2, dim=64, xs=64, as_=64,
             gs=64, zs=0, ys=64, dtype=0)
    a.update(over)
    return lib.mm_gated_scan_step(*a.values(), None)


def test_step_c_refuses(lib):
    for k in ("state", "state_out", "x", "a", "g", "A", "y"):
        assert step(lib, **{k: None}) == _lib.ERR_NULL_POINTER
    assert step(lib, batch=-1) == _lib.ERR_SHAPE
    assert step(lib, dtype=9) == _lib.ERR_DTYPE
    assert step(lib, xs=-1) == _lib.ERR_LAYOUT
    assert step(lib, ys=63) == _lib.ERR_LAYOUT
    assert step(lib, batch=0, x=None) == _lib.OK


def test_act8_c_refuses(lib):
    two = (_lib._i64a2)(64, 64)
    for f in (lib.mm_act8_pack, lib.mm_act8_unpack):
        assert f(FAKE, FAKE, None, 1, 1, 64, two, 0, None) == _lib.ERR_NULL_POINTER
        assert f(FAKE, FAKE, FAKE, -1, 1, 64, two, 0, None) == _lib.ERR_SHAPE
        assert f(FAKE, FAKE, FAKE, 1 << 40, 1 << 40, 64, two, 0, None) == _lib.ERR_SHAPE
        assert f(FAKE, FAKE, FAKE, 1, 1, 64, two, 5, None) == _lib.ERR_DTYPE
        assert f(FAKE, FAKE, FAKE, 1, 1, 64, (_lib._i64a2)(-1, 0), 0, None) == _lib.ERR_LAYOUT
        assert f(None, None, None, 0, 1, 64, two, 0, None) == _lib.OK
    assert lib.mm_act8_unpack(FAKE, FAKE, FAKE, 2, 1, 64, (_lib._i64a2)(0, 64), 0, None) == _lib.ERR_LAYOUT
    assert lib.mm_act8_unpack(FAKE, FAKE, FAKE, 1, 2, 64, (_lib._i64a2)(64, 32), 0, None) == _lib.ERR_LAYOUT


def conv(lib, **over):
    two = _lib._i64a2
    a = dict(x=FAKE, codes=None, exps=None, w=FAKE, b=None, dout=FAKE, dx=FAKE, dw=FAKE, db=None, batch=2, seqlen=100,
             dim=64, width=4, xs=two(6400, 64), ds=two(6400, 64), ws=two(4, 1), xdt=0, wdt=0, silu=1, work=FAKE,
             nbytes=1 << 40)
    a.update(over)
    return lib.mm_causal_conv1d_bwd(*a.values(), None)


@pytest.mark.parametrize("over,status", [
    (dict(batch=-1), _lib.ERR_SHAPE),
    (dict(width=9), _lib.ERR_SHAPE),
    (dict(width=0), _lib.ERR_SHAPE),
    (dict(batch=1 << 40, seqlen=1 << 30), _lib.ERR_SHAPE),
    (dict(xdt=4), _lib.ERR_DTYPE),
    (dict(wdt=-1), _lib.ERR_DTYPE),
    (dict(x=None), _lib.ERR_NULL_POINTER),
    (dict(x=None, codes=FAKE), _lib.ERR_NULL_POINTER),
    (dict(w=None), _lib.ERR_NULL_POINTER),
    (dict(dout=None), _lib.ERR_NULL_POINTER),
    (dict(dw=None, db=FAKE), _lib.ERR_NULL_POINTER),
    (dict(ds=(_lib._i64a2)(0, -1)), _lib.ERR_LAYOUT),
    (dict(nbytes=16), _lib.ERR_WORKSPACE),
    (dict(work=None), _lib.ERR_WORKSPACE),
    (dict(work=FAKE + 8), _lib.ERR_WORKSPACE),
    (dict(dx=None, dw=None), _lib.OK),
])
def test_conv_c_refuses(lib, over, status):
    assert conv(lib, **over) == status


def conv_fwd(lib, **over):
    two = _lib._i64a2
    a = dict(x=FAKE, w=FAKE, b=None, out=FAKE, codes=FAKE, exps=FAKE, batch=2, seqlen=100, dim=64, width=4,
             xs=two(6400, 64), ws=two(4, 1), xdt=0, wdt=0, silu=1)
    a.update(over)
    return lib.mm_causal_conv1d_fwd_act8(*a.values(), None)


def test_conv_fwd_act8_c_refuses(lib):
    for k in ("x", "w", "out", "codes", "exps"):
        assert conv_fwd(lib, **{k: None}) == _lib.ERR_NULL_POINTER, k
    assert conv_fwd(lib, width=9) == _lib.ERR_SHAPE
    assert conv_fwd(lib, dim=-1) == _lib.ERR_SHAPE
    assert conv_fwd(lib, wdt=3) == _lib.ERR_DTYPE
    assert conv_fwd(lib, codes=FAKE + 8) == _lib.ERR_LAYOUT
    assert conv_fwd(lib, xs=(_lib._i64a2)(-1, 64)) == _lib.ERR_LAYOUT
    assert conv_fwd(lib, seqlen=0, x=None) == _lib.OK
