"""embedding, decay_attention and linear_cross_entropy at sizes where they change their ways, and all three as one model.

Tolerances of the parts are those of their own tests' checks."""

from __future__ import annotations

import pytest
import torch

import decay_ref
import test_cross_entropy_gpu as ce
import test_decay_attention_gpu as da
import test_embedding_gpu as em
from mamba_metal_amd import decay_attention, embedding, linear_cross_entropy

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("n", [1024, 1025, 16383, 16384, 16385])
@pytest.mark.parametrize("vocab", [511, 262143, 262144])
def test_embedding_sorts(dev, n, vocab):
    """One workgroup's sort and the sort in passes, on both sides of where one takes over, a run across many tiles."""
    ids, w, dy = em.make(dev, BF16, n, vocab, 8)
    em.check(ids, w, dy, 1.0)
    ids[n // 3:n // 2] = vocab - 1
    em.check(ids, w, dy, 0.5, padding=int(ids[0]))


@pytest.mark.parametrize("dt,shape", [(F32, (2100, 1100, 16500)), (F32, (700, 260, 5000)), (F16, (1000, 520, 9000)),
                                      (BF16, (2048, 1024, 8192))])
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_loss_sizes(dev, dt, shape, reduction):
    ce.check(*ce.inputs(dev, dt, *shape), reduction)


@pytest.mark.parametrize("dt,shape", [(F32, (700, 260, 5000)), (BF16, (2048, 1024, 8192)), (BF16, (700, 260, 5000))])
def test_loss_one_gradient(dev, dt, shape):
    """x or the weight frozen: dx is then cut into other splits."""
    x, w, t, d = ce.inputs(dev, dt, *shape)
    (_, wdx, wdw), (_, tdx, tdw) = ce.reference(x, w, t, d)
    for k, (want, tol) in enumerate(((wdx, tdx), (wdw, tdw))):
        leaves = [x.clone().requires_grad_(k == 0), w.clone().requires_grad_(k == 1)]
        got, = torch.autograd.grad(linear_cross_entropy(*leaves, t, reduction="none"), [leaves[k]], d)
        ce.near(got, want, tol, "dx dW".split()[k])


@pytest.mark.parametrize("name", ["q", "k", "v", "dy", "g"])
def test_tokens_far_apart(dev, name):
    """Neighbouring tokens 2^27 elements apart: a run of them spans more than 32 bits."""
    s = da.inputs(dev, BF16, 1, 70, 1, 1, 64, 64)
    outs, grads = da.run(s, 1.0)
    flat = torch.empty(70 << 27, dtype=BF16, device=dev)
    far = flat.as_strided(s[name].shape, (1 << 27, 1 << 27, *([64, 1] if s[name].dim() == 4 else [1])))
    far_outs, far_grads = da.run({**s, name: far.copy_(s[name])}, 1.0)
    for a, b in zip(far_outs + list(far_grads), outs + list(grads)):
        assert torch.equal(a, b)


def parameters(gen, vocab, dim, groups, heads, dk, dv):
    r = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)
    return dict(table=r(vocab, dim) * 0.3, wq=r(groups * dk, dim) * dim ** -0.5, wk=r(groups * dk, dim) * (dim * dk) ** -0.5,
                wv=r(heads * dv, dim) * dim ** -0.5, wg=r(heads, dim) * dim ** -0.5, wo=r(dim, heads * dv) * (heads * dv) ** -0.5)


def model(p, ids, sizes, embed, mixer, loss):
    groups, heads, dk, dv = sizes
    x = embed(ids[:, :-1], p["table"])
    batch, n, _ = x.shape
    rows = x.flatten(0, 1)  # (plain products of matrices)
    part = lambda w, h, d: (rows @ p[w].t()).view(batch, n, h, d)
    y = mixer(part("wq", groups, dk), part("wk", groups, dk), part("wv", heads, dv),
              -torch.nn.functional.softplus(rows @ p["wg"].t()).view(batch, n, heads))
    return loss(rows + y.reshape(batch * n, -1) @ p["wo"].t(), p["table"], ids[:, 1:].flatten())


class Recurrence(torch.autograd.Function):
    """The mixer in 64 bits."""

    @staticmethod
    def forward(ctx, q, k, v, g):
        ctx.save_for_backward(q, k, v, g)
        return decay_ref.forward(q, k, v, g, 1.0, None)[0]

    @staticmethod
    def backward(ctx, dy):
        return tuple(decay_ref.backward(*ctx.saved_tensors, dy, 1.0, None, None, None)[:4])


@pytest.mark.parametrize("dt", [F32, BF16])
def test_a_model_trains(dev, dt):
    """Tokens to loss and back, a tied table at both ends: against the same model in 64 bits."""
    vocab, dim, sizes = 300, 48, (1, 3, 32, 24)
    gen = torch.Generator().manual_seed(5)
    p64 = {k: v.to(dev, dt).double().requires_grad_(True) for k, v in parameters(gen, vocab, dim, *sizes).items()}
    ids = torch.randint(0, vocab, (2, 151), generator=gen).to(dev)
    ids[1, 100:] = 7  # padding: a token like others here, and no target
    targets_off = lambda t: torch.where((t == 7), -100, t)
    loss64 = model(p64, ids, sizes, lambda i, w: w[i], Recurrence.apply,
                   lambda x, w, t: torch.nn.functional.cross_entropy(x @ w.t(), targets_off(t)))
    want = torch.autograd.grad(loss64, list(p64.values()))
    p = {k: v.detach().to(dt).requires_grad_(True) for k, v in p64.items()}
    loss = model(p, ids, sizes, embedding, decay_attention, lambda x, w, t: linear_cross_entropy(x, w, targets_off(t)))
    got = torch.autograd.grad(loss, list(p.values()))
    # A chain of a dozen products and sums of up to 300 parts, each off by at most its parts' 2^-24 (2^-9 in bf16, once a
    # product's output), at random: a gradient's error is a share of the largest of its tensor, 12 sqrt(300) roundings.
    u = 2.0 ** -24 if dt == F32 else 2.0 ** -8
    share = 12 * 300 ** 0.5 * u if dt == F32 else 12 * u
    loss, loss64 = float(loss.detach()), float(loss64.detach())
    assert abs(loss - loss64) <= share * loss64
    for (name, g), w in zip(zip(p, got), want):
        assert g.dtype == dt and float((g.double() - w).abs().max()) <= share * float(w.abs().max()), name
