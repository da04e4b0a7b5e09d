"""decay_attention's refusals and its C entries' checks, before any GPU call (no GPU needed)."""

from __future__ import annotations

import ctypes
import subprocess
import types
import warnings
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx

from mamba_metal_amd import _lib, decay_attention, decay_attention_step
from mamba_metal_amd.decay_attention import _DecayAttention

ROOT = Path(__file__).resolve().parents[1]
FAKE = 0x1000
Q, V, G, H = torch.zeros((2, 5, 2, 4)), torch.zeros((2, 5, 4, 3)), torch.zeros((2, 5, 4)), torch.zeros((2, 4, 4, 3))


def full(**kw):
    a = {**dict(q=Q, k=Q, v=V, g=G), **kw}
    return decay_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("g"), **a)


def step(**kw):
    a = {**dict(state=H.clone(), q=Q[:, 0], k=Q[:, 0], v=V[:, 0], g=G[:, 0]), **kw}
    return decay_attention_step(a.pop("state"), a.pop("q"), a.pop("k"), a.pop("v"), a.pop("g"), **a)


@pytest.mark.parametrize("kw,error", [
    (dict(q=Q[0]), ValueError), (dict(k=Q[:, :4]), ValueError), (dict(v=V[:1]), ValueError), (dict(v=V[:, :, :3]), ValueError),
    (dict(q=torch.zeros((2, 5, 2, 129)), k=torch.zeros((2, 5, 2, 129))), ValueError), (dict(v=torch.zeros((2, 5, 4, 1025))), ValueError),
    (dict(v=V[..., :0]), ValueError), (dict(q=Q[:, :, :0], k=Q[:, :, :0]), ValueError),
    (dict(g=G[:, :4]), ValueError), (dict(g=torch.zeros(3)), ValueError), (dict(g=G.long()), TypeError),
    (dict(k=Q.half()), TypeError), (dict(v=V.bfloat16()), TypeError), (dict(q=Q.double(), k=Q.double(), v=V.double()), TypeError),
    (dict(v=torch.zeros((2, 5, 3, 4)).transpose(2, 3)), ValueError), (dict(h0=H[:1]), ValueError), (dict(h0=H.long()), TypeError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(lengths=torch.zeros(2)), TypeError),
])
def test_refusals(kw, error):
    with pytest.raises(error):
        full(**kw)
    with pytest.raises(ValueError, match="need GPU"):
        full()


@pytest.mark.parametrize("kw,error", [
    (dict(q=Q), ValueError), (dict(state=H.half()), ValueError), (dict(state=H[:, :, :, :2]), ValueError),
    (dict(state_out=H.transpose(0, 1).contiguous().transpose(0, 1)), ValueError), (dict(g=G), ValueError), (dict(out=V[:, 0, :3]), ValueError),
    (dict(out=V[:, 0].half()), TypeError), (dict(out=torch.zeros((2, 3, 4)).transpose(1, 2)), ValueError), (dict(v=V[:, 0, :3]), ValueError),
])
def test_step_refusals(kw, error):
    with pytest.raises(error):
        step(**kw)
    with pytest.raises(ValueError, match="need GPU"):
        step()


@pytest.mark.parametrize("name", ["state", "q", "k", "v", "g"])
def test_step_has_no_gradient(name):
    t = dict(state=H, q=Q[:, 0], k=Q[:, 0], v=V[:, 0], g=G[:, 0])[name].clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        step(**{name: t})
    with torch.no_grad(), pytest.raises(ValueError, match="need GPU"):
        step(**{name: t})


@pytest.mark.parametrize("call,name,t", [(full, "q", Q), (full, "k", Q), (full, "v", V), (full, "g", G), (full, "h0", H),
                                         (step, "state", H), (step, "q", Q[:, 0]), (step, "k", Q[:, 0]), (step, "v", V[:, 0]), (step, "g", G[:, 0])])
def test_transforms_are_refused(call, name, t):
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(**{name: fw.make_dual(t, torch.ones_like(t))})
    with pytest.raises(RuntimeError, match="recorded"):
        make_fx(lambda x: call(**{name: x}))(t)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(lambda x: call(**{name: x}), (t,), check_trace=False)


def test_saved_tensors_are_checked(monkeypatch):
    """What hooks hand back for a saved tensor is what was saved, or refused."""
    q, v = torch.zeros((2, 70, 1, 8), dtype=torch.float16), torch.zeros((2, 70, 2, 8), dtype=torch.float16)
    g, lengths = torch.zeros((2, 70, 2)), torch.zeros(2, dtype=torch.int32)
    nbytes = _lib.load().mm_decay_attention_states_size(2, 70, 2, 8, 8, _lib.F16)
    was = [q, q.clone(), v, g, lengths, torch.zeros(nbytes, dtype=torch.uint8)]
    meta = (torch.device("cuda", 0), q.dtype, q.shape, v.shape, g.dtype, g.shape, 1.0, (torch.int32,))
    ctx = types.SimpleNamespace(meta=meta, saved_tensors=was, needs_input_grad=(True,) * 9)
    with pytest.raises(RuntimeError, match="saved tensor"):
        _DecayAttention.backward(ctx, v)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for k, t in enumerate(was):
        for change in (lambda t: t.to(torch.int16), lambda t: t[:1], lambda t: t[..., None], lambda t: None):
            ctx.saved_tensors = was[:k] + [change(t)] + was[k + 1:]
            with pytest.raises(RuntimeError, match="saved tensor"):
                _DecayAttention.backward(ctx, v)


# ------------------------------------------------------------------------------ the C entries
def params(**over):
    p = _lib.DecayAttentionParams()
    for f in ("q", "k", "v", "log_decay", "y", "dy", "dq", "dk", "dv"):
        setattr(p, f, FAKE)
    p.run_states, p.workspace, p.workspace_bytes = 0x1000, 0x1000, 1 << 40
    p.batch, p.seqlen, p.heads, p.groups, p.key_dim, p.value_dim = 2, 100, 4, 2, 64, 64
    for k, v in over.items():
        setattr(p, k, v)
    return p


NEG = _lib._i64a3(-1, 1, 1)


@pytest.mark.parametrize("over,status", [
    (dict(q=None), _lib.ERR_NULL_POINTER), (dict(log_decay=None), _lib.ERR_NULL_POINTER), (dict(dtype=3), _lib.ERR_DTYPE),
    (dict(log_decay_dtype=-1), _lib.ERR_DTYPE), (dict(lengths=FAKE, lengths_dtype=2), _lib.ERR_DTYPE), (dict(key_dim=129), _lib.ERR_SHAPE),
    (dict(key_dim=0), _lib.ERR_SHAPE), (dict(value_dim=1025), _lib.ERR_SHAPE), (dict(groups=3), _lib.ERR_SHAPE), (dict(groups=0), _lib.ERR_SHAPE),
    (dict(batch=-1), _lib.ERR_SHAPE), (dict(batch=65536), _lib.ERR_SHAPE), (dict(seqlen=(1 << 30) + 1), _lib.ERR_SHAPE),
    (dict(heads=65534, batch=65535), _lib.ERR_SHAPE), (dict(q_stride=NEG), _lib.ERR_LAYOUT), (dict(log_decay_stride=NEG), _lib.ERR_LAYOUT),
    (dict(run_states=0x1010), _lib.ERR_LAYOUT), (dict(seqlen=4096, workspace=None), _lib.ERR_WORKSPACE),
    (dict(seqlen=4096, workspace_bytes=16), _lib.ERR_WORKSPACE), (dict(seqlen=4096, workspace=0x1010), _lib.ERR_WORKSPACE),
])
def test_validation(over, status):
    lib = _lib.load()
    for entry in (lib.mm_decay_attention_fwd, lib.mm_decay_attention_bwd):
        assert entry(params(**over), None) == status
    assert lib.mm_last_error().decode().startswith(lib.mm_status_name(status).decode())


def test_validation_of_one_pass():
    lib = _lib.load()
    assert lib.mm_decay_attention_fwd(params(y=None), None) == _lib.ERR_NULL_POINTER
    for over in (dict(dy=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(run_states=None)):
        assert lib.mm_decay_attention_bwd(params(**over), None) == _lib.ERR_NULL_POINTER
    assert lib.mm_decay_attention_bwd(params(dy_stride=NEG), None) == _lib.ERR_LAYOUT
    assert lib.mm_decay_attention_bwd(params(dlog_decay=FAKE, dlog_decay_heads=FAKE), None) == _lib.ERR_SHAPE
    for entry in (lib.mm_decay_attention_fwd, lib.mm_decay_attention_bwd):
        assert entry(None, None) == _lib.ERR_NULL_POINTER
        assert entry(params(batch=0), None) == _lib.OK


def test_step_validation():
    lib, two = _lib.load(), _lib._i64a2
    base = dict(ptrs=[FAKE] * 7, sizes=[2, 4, 2, 64, 64], strides=[two(256, 64)] * 4 + [two(256, 64)], dtypes=[0, 0])

    def call(**over):
        a = {**base, **over}
        return lib.mm_decay_attention_step(*a["ptrs"], *a["sizes"], *a["strides"], 1.0, *a["dtypes"], None)

    for k in range(7):
        assert call(ptrs=[None if j == k else FAKE for j in range(7)]) == _lib.ERR_NULL_POINTER
    assert call(sizes=[2, 4, 3, 64, 64]) == _lib.ERR_SHAPE
    assert call(sizes=[2, 4, 2, 129, 64]) == _lib.ERR_SHAPE
    assert call(dtypes=[5, 0]) == _lib.ERR_DTYPE
    assert call(dtypes=[0, 5]) == _lib.ERR_DTYPE
    assert call(strides=[two(-1, 1)] + [two(256, 64)] * 4) == _lib.ERR_LAYOUT
    assert call(strides=[two(256, 64)] * 4 + [two(256, 63)]) == _lib.ERR_LAYOUT  # rows of y that overlap
    assert call(sizes=[0, 4, 2, 64, 64], ptrs=[None] * 7) == _lib.OK


def test_sizes():
    lib = _lib.load()
    # 2 runs of 4 heads, one value block each of 64 x 64 states; float16 keeps a power of two beside each, and 16-bit calls of
    # few tokens what the states' roundings leave
    assert lib.mm_decay_attention_states_size(2, 100, 4, 64, 64, _lib.F32) == 2 * 4 * 2 * 64 * 64 * 4
    assert lib.mm_decay_attention_states_size(2, 100, 4, 65, 65, _lib.F16) == 2 * 4 * 2 * 2 * (2 * 64 * 128 * 2) + 256
    assert lib.mm_decay_attention_states_size(2, 6400, 4, 64, 64, _lib.BF16) == 2 * 4 * 100 * 64 * 64 * 2
    assert lib.mm_decay_attention_states_size(0, 100, 4, 64, 64, 0) == 0
    assert lib.mm_decay_attention_states_size(2, 100, 4, 129, 64, 0) == 0
    assert lib.mm_decay_attention_workspace_size(64, 100, 4, 4, 64, 64, 0, 0) == 0  # enough heads: no segments
    assert lib.mm_decay_attention_workspace_size(1, 4096, 4, 4, 64, 64, 0, 0) > 0
    assert lib.mm_decay_attention_workspace_size(1, 4096, 4, 3, 64, 64, 0, 1) == 0


def test_params_layout_matches_header(tmp_path):
    cls = _lib.DecayAttentionParams
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "off.c"
    body = "\n".join(f'printf("{f} %zu\\n", offsetof(mm_decay_attention_params, {f}));' for f in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mamba_mi355x.h"\nint main(void){\n' + body +
                   '\nprintf("sizeof %zu\\n", sizeof(mm_decay_attention_params));return 0;}\n')
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert all(int(got[f]) == getattr(cls, f).offset for f in fields) and int(got["sizeof"]) == ctypes.sizeof(cls)
