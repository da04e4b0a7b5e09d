"""embedding's and linear_cross_entropy's refusals and their C entries' checks, before any GPU call (no GPU needed)."""

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

from mamba_metal_amd import _lib, embedding, linear_cross_entropy
from mamba_metal_amd.cross_entropy import _LinearCrossEntropy
from mamba_metal_amd.embedding import _Embedding

ROOT = Path(__file__).resolve().parents[1]
FAKE = 0x1000
X, W, T = torch.zeros((3, 5, 8)), torch.zeros((20, 8)), torch.zeros((3, 5), dtype=torch.int64)


def loss(x=X, w=W, t=T, **kw):
    return linear_cross_entropy(x, w, t, **kw)


def embed(ids=T, w=W, **kw):
    return embedding(ids, w, **kw)


@pytest.mark.parametrize("call,kw,error", [
    (loss, dict(x=X[..., :7]), ValueError), (loss, dict(x=torch.zeros(())), ValueError), (loss, dict(w=W[0]), ValueError),
    (loss, dict(w=W[:0]), ValueError), (loss, dict(t=T[:2]), ValueError), (loss, dict(t=T.float()), TypeError), (loss, dict(t=T.short()), TypeError),
    (loss, dict(w=W.half()), TypeError), (loss, dict(x=X.double(), w=W.double()), TypeError), (loss, dict(reduction="max"), ValueError),
    (loss, dict(w=torch.zeros((8, 20)).t()), ValueError), (loss, dict(x=torch.zeros((3, 8, 5)).transpose(1, 2)), ValueError),
    (embed, dict(ids=T.float()), TypeError), (embed, dict(ids=T.bool()), TypeError), (embed, dict(w=W[0]), ValueError),
    (embed, dict(w=W[:0]), ValueError), (embed, dict(w=W[:, :0]), ValueError), (embed, dict(w=W.long()), TypeError),
    (embed, dict(w=torch.zeros((8, 20)).t()), ValueError), (embed, dict(padding_idx=20), ValueError), (embed, dict(padding_idx=-21), ValueError),
])
def test_refusals(call, kw, error):
    with pytest.raises(error):
        call(**kw)
    with pytest.raises(ValueError, match="need GPU"):
        call()


@pytest.mark.parametrize("call,name,t", [(loss, "x", X), (loss, "w", W), (embed, "w", W)])
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
    dev = torch.device("cuda", 0)
    x2, t2 = X.view(15, 8), T.view(-1)
    cases = [(_LinearCrossEntropy, (dev, x2.dtype, x2.shape, W.shape, -100, "mean", (t2.dtype, t2.shape)), [x2, W, t2, torch.zeros(15)], torch.zeros(())),
             (_Embedding, (dev, W.dtype, W.shape, 1.0, None, (t2.dtype, t2.shape)), [t2], x2)]
    for fn, meta, was, up in cases:
        ctx = types.SimpleNamespace(meta=meta, saved_tensors=was, needs_input_grad=(True,) * 6)
        with pytest.raises(RuntimeError, match="saved tensor"):
            fn.backward(ctx, up)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    for fn, meta, was, up in cases:
        for k, t in enumerate(was):
            for change in (lambda t: t.to(torch.int16), lambda t: t[:1], lambda t: t[..., None], lambda t: None):
                ctx = types.SimpleNamespace(meta=meta, saved_tensors=was[:k] + [change(t)] + was[k + 1:], needs_input_grad=(True,) * 6)
                with pytest.raises(RuntimeError, match="saved tensor"):
                    fn.backward(ctx, up)


# ------------------------------------------------------------------------------ the C entries
def params(**over):
    p = _lib.LinearCrossEntropyParams()
    for f in ("x", "weight", "targets", "loss", "lse", "dloss", "dx", "dweight", "workspace"):
        setattr(p, f, FAKE)
    p.workspace_bytes = 1 << 40
    p.rows, p.dim, p.vocab, p.x_stride, p.weight_stride = 100, 64, 1000, 64, 64
    for k, v in over.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("over,status", [
    (dict(x=None), _lib.ERR_NULL_POINTER), (dict(weight=None), _lib.ERR_NULL_POINTER), (dict(targets=None), _lib.ERR_NULL_POINTER),
    (dict(dtype=3), _lib.ERR_DTYPE), (dict(targets_dtype=2), _lib.ERR_DTYPE), (dict(reduction=3), _lib.ERR_SHAPE), (dict(reduction=-1), _lib.ERR_SHAPE),
    (dict(rows=-1), _lib.ERR_SHAPE), (dict(dim=0), _lib.ERR_SHAPE), (dict(vocab=0), _lib.ERR_SHAPE), (dict(rows=1 << 30, dim=1 << 12), _lib.ERR_SHAPE),
    (dict(rows=1 << 29, dim=1, vocab=1 << 29), _lib.ERR_SHAPE), (dict(x_stride=-1), _lib.ERR_LAYOUT), (dict(weight_stride=-1), _lib.ERR_LAYOUT),
    (dict(dloss_stride=-1), _lib.ERR_LAYOUT), (dict(workspace=None), _lib.ERR_WORKSPACE), (dict(workspace=FAKE + 16), _lib.ERR_WORKSPACE),
    (dict(workspace_bytes=64), _lib.ERR_WORKSPACE),
])
def test_loss_validation(over, status):
    lib = _lib.load()
    for entry in (lib.mm_linear_cross_entropy_fwd, lib.mm_linear_cross_entropy_bwd):
        assert entry(params(**over), None) == status
    assert lib.mm_last_error().decode().startswith(lib.mm_status_name(status).decode())


def test_loss_validation_of_one_pass():
    lib = _lib.load()
    assert lib.mm_linear_cross_entropy_fwd(params(loss=None), None) == _lib.ERR_NULL_POINTER
    for over in (dict(lse=None), dict(dloss=None)):
        assert lib.mm_linear_cross_entropy_bwd(params(**over), None) == _lib.ERR_NULL_POINTER
    assert lib.mm_linear_cross_entropy_bwd(params(dx=None, dweight=None), None) == _lib.OK
    for entry in (lib.mm_linear_cross_entropy_fwd, lib.mm_linear_cross_entropy_bwd):
        assert entry(None, None) == _lib.ERR_NULL_POINTER
        assert entry(params(rows=0), None) == _lib.OK


def test_loss_workspace():
    """Bounded by a piece of the vocabulary, not by all logits."""
    size = _lib.load().mm_linear_cross_entropy_workspace_size
    assert size(params(rows=0), 1) == 0 and size(params(dim=0), 1) == 0
    rows, dim, vocab = 1 << 16, 64, 1 << 17
    p = params(rows=rows, dim=dim, vocab=vocab, dtype=_lib.BF16)
    fixed = rows * (28 + 2 * dim + 4 * dim) + 4096
    assert size(p, 1) <= (512 << 20) + fixed < rows * vocab * 2 // 16
    assert size(p, 0) <= rows * (vocab // 128 * 8 + 28 + 2 * dim) + 4096
    # a table off 16 bytes is laid out anew
    assert size(params(weight=FAKE + 4), 0) - size(params(), 0) == 1000 * 64 * 4


def test_embedding_validation():
    lib = _lib.load()

    def fwd(ids=FAKE, w=FAKE, y=FAKE, n=10, vocab=20, dim=8, ld=8, ids_dtype=0, dtype=0):
        return lib.mm_embedding_fwd(ids, w, y, n, vocab, dim, ld, 1.0, ids_dtype, dtype, None)

    def bwd(ids=FAKE, dy=FAKE, dw=FAKE, n=10, vocab=20, dim=8, ld=8, ids_dtype=0, dtype=0, ws=FAKE, size=1 << 30):
        return lib.mm_embedding_bwd(ids, dy, dw, n, vocab, dim, ld, 1.0, -1, ids_dtype, dtype, ws, size, None)

    for entry in (fwd, bwd):
        assert entry(dtype=4) == _lib.ERR_DTYPE and entry(ids_dtype=2) == _lib.ERR_DTYPE
        for over in (dict(n=-1), dict(vocab=0), dict(dim=0), dict(n=1 << 31), dict(vocab=(1 << 30) + 1), dict(n=1 << 30, dim=1 << 10),
                     dict(vocab=1 << 30, dim=1 << 12)):
            assert entry(**over) == _lib.ERR_SHAPE, over
        assert entry(ids=None) == _lib.ERR_NULL_POINTER and entry(ld=-1) == _lib.ERR_LAYOUT
    assert fwd(w=None) == _lib.ERR_NULL_POINTER and fwd(y=None) == _lib.ERR_NULL_POINTER and fwd(n=0, ids=None, w=None, y=None) == _lib.OK
    assert bwd(dy=None) == _lib.ERR_NULL_POINTER and bwd(dw=None) == _lib.ERR_NULL_POINTER
    assert bwd(ws=None) == _lib.ERR_WORKSPACE and bwd(ws=FAKE + 8) == _lib.ERR_WORKSPACE and bwd(size=100) == _lib.ERR_WORKSPACE
    assert lib.mm_embedding_bwd_workspace_size(0, 20, 8) == 0 and lib.mm_embedding_bwd_workspace_size(10, 0, 8) == 0
    assert 0 < lib.mm_embedding_bwd_workspace_size(10, 20, 8) < 1 << 16


def test_params_layout_matches_header(tmp_path):
    cls = _lib.LinearCrossEntropyParams
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "off.c"
    body = "\n".join(f'printf("{f} %zu\\n", offsetof(mm_linear_cross_entropy_params, {f}));' for f in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mamba_mi355x.h"\nint main(void){\n' + body +
                   '\nprintf("sizeof %zu\\n", sizeof(mm_linear_cross_entropy_params));return 0;}\n')
    exe = tmp_path / "off"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert all(int(got[f]) == getattr(cls, f).offset for f in fields) and int(got["sizeof"]) == ctypes.sizeof(cls)


@pytest.mark.parametrize("value", [1 << 63, -(1 << 63) - 1])
def test_ignore_index_is_64_bit(value):
    with pytest.raises(ValueError, match="64-bit"):
        loss(ignore_index=value)
