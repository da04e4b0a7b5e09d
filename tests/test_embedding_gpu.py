"""embedding and its gradient.  y is one product rounded once: equal to torch's.  dW: a row's sum of c tokens in fp32
takes c roundings of 2^-24 of the sum of magnitudes, the scale one more, and one to its type (half a step)."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import embedding, linear_cross_entropy

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(ids, w, dy, scale, padding=None):
    vocab, dim = w.shape
    wg = w.detach().requires_grad_(True)
    y = embedding(ids, wg, scale=scale, padding_idx=padding)
    dw, = torch.autograd.grad(y, wg, dy)
    flat = ids.reshape(-1).long()
    inside = (flat >= 0) & (flat < vocab)
    want_y = (w[flat.clamp(0, vocab - 1)].float() * scale).to(w.dtype)
    got = y.detach().reshape(-1, dim)
    assert y.shape == (*ids.shape, dim) and torch.equal(got[inside], want_y[inside]) and bool(got[~inside].isnan().all())
    counts = inside if padding is None else inside & (flat != padding % vocab)
    d = dy.reshape(-1, dim).double()[counts] * scale
    at = flat[counts].cpu()
    want, mag = (torch.zeros((vocab, dim), dtype=torch.float64).index_add_(0, at, t.cpu()).to(w.device) for t in (d, d.abs()))
    c = torch.bincount(at, minlength=vocab).to(w.device)[:, None].double()
    u = 0.0 if w.dtype == F32 else torch.finfo(w.dtype).eps / 2
    tiny = 0.0 if w.dtype != F16 else 2.0 ** -25
    err = (dw.double() - want).abs()
    assert bool((err <= u * want.abs() + (c + 2) * 2.0 ** -24 * mag + tiny).all()), float(err.max())
    assert not bool(dw[c[:, 0] == 0].any())
    again, = torch.autograd.grad(embedding(ids, wg, scale=scale, padding_idx=padding), wg, dy)
    assert torch.equal(again, dw)


def make(dev, dt, n, vocab, dim, seed=0, zipf=True):
    gen = torch.Generator().manual_seed(seed)
    u = torch.rand(n, generator=gen, dtype=torch.float64)
    ids = (vocab ** u).long().clamp(1, vocab) - 1 if zipf else (u * vocab).long()
    r = lambda *s: torch.randn(s, generator=gen).to(dev, dt)
    return ids.to(dev), r(vocab, dim), r(n, dim)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 5, 8), (31, 3, 64), (33, 7, 40), (64, 511, 17), (2047, 512, 72), (2049, 513, 1001),
                                   (5000, 50280, 64), (9001, 262145, 24), (70, 1 << 19, 8)])
def test_against_index_add(dev, dt, shape):
    ids, w, dy = make(dev, dt, *shape)
    check(ids, w, dy, 1.0)
    check(ids.int(), w, dy, 0.37, padding=-1)
    check(ids, w, dy, 8.0, padding=0)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("n", [32, 64, 4096, 20000])
def test_one_token(dev, dt, n):
    """One id for all, two ids in halves, an id that begins and ends inside tiles."""
    _, w, dy = make(dev, dt, n, 300, 48)
    ids = torch.full((n,), 299, device=dev)
    check(ids, w, dy, 1.0)
    ids[n // 2:] = 4
    check(ids, w, dy, 1.0)
    ids[::7] = 5
    check(ids, w, dy, 1.0, padding=5)
    check(ids, w, dy, 1.0, padding=299)


def test_uniform_and_large(dev):
    check(*make(dev, BF16, 40000, 10007, 264, zipf=False), 1.0)
    check(*make(dev, BF16, 300000, 131, 16), 1.0)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_ids_outside(dev, dt):
    ids, w, dy = make(dev, dt, 500, 40, 24)
    ids[3], ids[77], ids[400] = -1, 40, 1 << 40
    check(ids, w, dy, 2.0)
    bad = ids.clone()
    dy[3] = float("nan")  # not read: the row has no place in the table
    check(bad, w, dy, 2.0)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_layouts(dev, dt):
    ids, w, dy = make(dev, dt, 120, 50, 24)
    for off in (0, 1, 8):
        ws, ds = (torch.zeros((a.shape[0], 40), dtype=dt, device=dev)[:, off:off + 24].copy_(a) for a in (w, dy))
        check(ids, ws, ds, 1.5)
    check(ids.view(4, 30).t(), w, dy.view(30, 4, 24), 1.0)
    check(ids, w, dy[:1].expand(120, 24), 1.0)
    check(ids, w, dy.t().contiguous().t(), 1.0)
    assert embedding(ids[:0], w).shape == (0, 24) and embedding(ids[0], w).shape == (24,)
    wg = w.clone().requires_grad_(True)
    assert not bool(torch.autograd.grad(embedding(ids[:0], wg).sum(), wg)[0].any())


def test_offsets_past_32_bits(dev):
    ids, w, dy = make(dev, BF16, 3, 3, 64, zipf=False)
    flat = torch.empty(1 << 34, dtype=torch.uint8, device=dev).view(BF16)
    far = flat.as_strided((3, 64), ((1 << 31) + 64, 1))
    assert torch.equal(embedding(ids, far.copy_(w)), embedding(ids, w))
    wg = w.requires_grad_(True)
    want, = torch.autograd.grad(embedding(ids, wg), wg, dy)
    assert torch.equal(torch.autograd.grad(embedding(ids, wg), wg, far.copy_(dy))[0], want)
    del flat, far
    big = torch.zeros((70000, 40000), dtype=BF16, device=dev)  # a table of more than 2^31 elements
    last = torch.tensor([69999, 60000], device=dev)
    big[last, -8:] = 3.0
    assert bool((embedding(last, big)[:, -8:] == 3).all())
    big.requires_grad_(True)
    dw, = torch.autograd.grad(embedding(last, big), big, torch.ones((2, 40000), dtype=BF16, device=dev))
    assert bool((dw[last] == 1).all()) and float(dw[60001:69999].abs().amax()) == 0 and float(dw[:60000].abs().amax()) == 0


def test_tied_head_in_a_graph(dev):
    """Both ends of a model on one table, forward and backward pass captured together and replayed on other tokens."""
    gen = torch.Generator().manual_seed(0)
    w = (torch.randn((500, 64), generator=gen) * 0.1).to(dev, BF16).requires_grad_(True)
    draw = lambda s: torch.randint(0, 500, (3, 41), generator=torch.Generator().manual_seed(s)).to(dev)
    ids = draw(0)

    def step(ids, w):
        h = embedding(ids[:, :-1], w, scale=8.0, padding_idx=0)
        loss = linear_cross_entropy(torch.tanh(h), w, ids[:, 1:])
        return loss, *torch.autograd.grad(loss, [w])

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(ids, w)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        captured = [t.detach() for t in step(ids, w)]
    for s in range(4):
        ids.copy_(draw(s))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(draw(s), w.detach().clone().requires_grad_(True))):
            assert torch.equal(a, b.detach())
