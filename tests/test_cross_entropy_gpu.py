"""linear_cross_entropy and its gradients against logits, softmax and products in 64 bits.

Tolerances, element by element; u is the type's half step (0 for float32), e = 2^-24:
  a logit is a sum of dim products in fp32: off by E = dim e sum |x| |w|, at most (its row's largest is taken);
  the loss: two logits' errors, and the sums, exponentials (2^-22 each, hardware) and logarithm of a few units;
  dl = (p - onehot) dloss: p off by a share of 2 E and 2^-20, dl rounded once (u); in float16 times a power of two that
  leaves numbers below 2^-37 of the largest |dloss| to a fixed step;
  dx, dW: sums over the vocabulary and the rows in fp32 (their lengths times e of the sum of magnitudes), rounded (u; a
  float16 below 2^-14 has a fixed step of 2^-24, so half of that besides, and float32's numbers end at 2^-126)."""

from __future__ import annotations

import pytest
import torch

from mamba_metal_amd import MambaConfig, MambaModel, init_weights_, linear_cross_entropy

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
e24 = 2.0 ** -24


def half_step(dt):
    return 0.0 if dt == F32 else torch.finfo(dt).eps / 2


def inputs(dev, dt, rows, dim, vocab, ignored=0.2, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x, w = torch.randn((rows, dim), generator=gen), torch.randn((vocab, dim), generator=gen) * 2 * dim ** -0.5
    t = torch.randint(0, vocab, (rows,), generator=gen)
    t[torch.rand(rows, generator=gen) < ignored] = -100
    t[-1] = vocab - 1
    return x.to(dev, dt), w.to(dev, dt), t.to(dev), torch.rand(rows, generator=gen).to(dev)


def reference(x, w, t, dloss, ignore=-100):
    """Losses, dx, dW for per-row dloss, and the bounds of their errors."""
    dt, (rows, dim), vocab = x.dtype, x.shape, w.shape[0]
    u = half_step(dt)
    x, w, dloss = x.double(), w.double(), dloss.double()
    on = t != ignore
    at = torch.where(on, t.long(), 0)
    logits = x @ w.t()
    E = dim * e24 * (x.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(logits, 1)
    loss = torch.where(on, lse - logits.gather(1, at[:, None])[:, 0], 0.0)
    loss_tol = 2 * E + 2.0 ** -20 * (1 + lse.abs() + logits.abs().amax(1))
    p = torch.exp(logits - lse[:, None])
    g = torch.where(on, dloss, 0.0)
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    dl = (p - hot) * g[:, None]
    lse_tol = (2 * E + 2.0 ** -20 * (1 + lse.abs()))[:, None]
    dl_tol = u * dl.abs() + (p * lse_tol + 2.0 ** -22 * hot) * g[:, None]
    floor = 2.0 ** -37 * g.max() if dt == F16 else 2.0 ** -126  # (fp32 ends there, dl and p alike)
    dl_tol = torch.where(on[:, None], dl_tol + floor + 2.0 ** -126 * g[:, None], 0.0)
    dx, dw = dl @ w, dl.t() @ x
    mx, mw = dl.abs() @ w.abs(), dl.abs().t() @ x.abs()
    least = 2.0 ** -25 if dt == F16 else 2.0 ** -126
    dx_tol = least + u * dx.abs() + dl_tol @ w.abs() + (vocab + 8) * e24 * mx
    dw_tol = least + u * dw.abs() + dl_tol.t() @ x.abs() + (rows + 8) * e24 * mw
    return (loss, dx, dw), (loss_tol, dx_tol, dw_tol)


def near(got, want, tol, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by {float((err / tol.clamp_min(1e-300)).max()):.3g} of the bound"


def check(x, w, t, dloss, reduction, **kw):
    xg, wg = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(xg, wg, t, reduction=reduction, **kw)
    rows, on = t.numel(), t.reshape(-1) != kw.get("ignore_index", -100)
    if reduction == "none":
        up = per_row = dloss.view(t.shape)
    else:
        up = dloss.reshape(-1)[0]
        per_row = up.expand(rows) / (on.sum() if reduction == "mean" else 1)
    dx, dw = torch.autograd.grad(loss, [xg, wg], up)
    (want, wdx, wdw), (tol, tdx, tdw) = reference(x.reshape(-1, x.shape[-1]), w, t.reshape(-1), per_row.reshape(-1), **(
        {"ignore": kw["ignore_index"]} if kw else {}))
    if reduction == "none":
        near(loss.detach().reshape(-1), want, tol, "loss")
    else:
        n = on.sum() if reduction == "mean" else 1
        near(loss.detach(), want.sum() / n, (tol * on).sum() / n + e24 * want.sum() / n, "loss")
    near(dx.reshape(wdx.shape), wdx, tdx, "dx")
    near(dw, wdw, tdw, "dW")
    assert not bool(dx.reshape(wdx.shape)[~on].any())
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(x, w, t, reduction=reduction, **kw), loss)


SHAPES = [  # rows, dim, vocab: tiles' edges, odd widths, one of each, many of each
    (1, 1, 1), (1, 8, 2), (3, 64, 129), (64, 32, 128), (65, 72, 257), (130, 1001, 1000), (255, 63, 511), (300, 2560, 777),
    (1000, 40, 3001), (33, 128, 50280), (2049, 136, 6401),
]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_logits(dev, dt, shape):
    reduction = ("none", "mean", "sum")[sum(shape) % 3]
    check(*inputs(dev, dt, *shape), reduction)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reductions(dev, dt, reduction):
    check(*inputs(dev, dt, 200, 96, 700), reduction)
    x, w, t, d = inputs(dev, dt, 120, 40, 300)
    check(x.view(4, 30, 40), w, t.view(4, 30).int(), d, reduction)


def test_large_tiles(dev):
    """Sizes at which all three products take their largest tiles, and more than one piece of the vocabulary."""
    x, w, t, d = inputs(dev, BF16, 8200, 1544, 40000)
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(xg, wg, t, reduction="none")
    dx, dw = torch.autograd.grad(loss, [xg, wg], d)
    x, w = x.detach(), w.detach()
    # the rows' sums are the whole reference; of the gradients, some rows of dx and some of dW
    logits = x.float() @ w.float().t()
    lse = torch.logsumexp(logits, 1)
    on = t != -100
    some = torch.arange(0, 8200, 41, device=dev)
    p = torch.exp(logits - lse[:, None]).double()
    del logits
    p[torch.arange(8200, device=dev)[on], t[on]] -= 1
    p *= torch.where(on, d, 0.0).double()[:, None]
    u, wd, xd = half_step(BF16), w.double(), x.double()
    ref, mag = p[some] @ wd, p[some].abs() @ wd.abs()
    near(dx[some], ref, u * ref.abs() + (u + 1e-4) * mag, "dx")
    cols = torch.arange(0, 40000, 199, device=dev)
    pc = p[:, cols].t().contiguous()
    ref, mag = pc @ xd, pc.abs() @ xd.abs()
    near(dw[cols], ref, u * ref.abs() + (u + 1e-3) * mag, "dW")  # (8200 rows' fp32 sums: 5e-4)
    want, tol = reference(x[some], w, t[some], d[some])
    near(loss[some].detach(), want[0], tol[0], "loss")


@pytest.mark.parametrize("dt", [F32, BF16])
def test_layouts(dev, dt):
    """Rows with a stride, off 16 bytes, a transposed batch, 32-bit targets: the same bits."""
    x, w, t, d = inputs(dev, dt, 60, 48, 200)

    def run(x, w, t, d):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, w, t, reduction="none")
        return loss.detach(), *torch.autograd.grad(loss, [x, w], d)

    want = run(x, w, t, d)
    for off in (0, 1, 8):
        xs, ws = (torch.zeros((a.shape[0], a.shape[1] + 16), dtype=dt, device=dev)[:, off:off + a.shape[1]].copy_(a) for a in (x, w))
        for a, b in zip(run(xs, ws, t.int(), d), want):
            assert torch.equal(a, b)
    xt = x.view(4, 15, 48).transpose(0, 1)
    got = run(xt, w, t.view(4, 15).t(), d.view(4, 15).t())
    assert torch.equal(got[0].t().reshape(-1), want[0]) and torch.equal(got[1].transpose(0, 1).reshape(60, 48), want[1])
    one = run(x, w, t, torch.ones((), device=dev).expand(60))  # a gradient that all rows share
    for a, b in zip(one, run(x, w, t, torch.ones(60, device=dev))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_ignored_rows_hold_anything(dev, dt, bad):
    x, w, t, d = inputs(dev, dt, 150, 64, 300, ignored=0.5)

    def run(x):
        x, wg = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = linear_cross_entropy(x, wg, t)
        return loss.detach(), *torch.autograd.grad(loss, [x, wg])

    want = run(x)
    x[t == -100] = bad
    for a, b in zip(run(x), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_what_is_broken_stays_visible(dev, dt):
    """A NaN row, a target outside the vocabulary: NaN in that row alone, and in dW."""
    x, w, t, d = inputs(dev, dt, 70, 64, 300, ignored=0.0)
    clean = linear_cross_entropy(x, w, t, reduction="none")
    for change in ("nan", "target", "negative"):
        x2, t2 = x.clone(), t.clone()
        if change == "nan":
            x2[5, 3] = float("nan")
        else:
            t2[5] = 300 if change == "target" else -1
        x2.requires_grad_(True)
        wg = w.clone().requires_grad_(True)
        loss = linear_cross_entropy(x2, wg, t2, reduction="none")
        dx, dw = torch.autograd.grad(loss.sum(), [x2, wg])
        rest = torch.arange(70, device=dev) != 5
        assert bool(loss[5].isnan()) and torch.equal(loss[rest], clean[rest])
        assert bool(dx[5].isnan().all()) and bool(dx[rest].isfinite().all()) and bool(dw.isnan().any())
        assert bool(linear_cross_entropy(x2, wg, t2).isnan())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_extreme_logits(dev, dt):
    """Logits of hundreds, one token far above the rest, and -inf logits (a token that a weight rules out)."""
    x, w, t, d = inputs(dev, dt, 64, 32, 400)
    check(x * 60, w, t, d, "none")
    w2 = w.clone()
    w2[:, 0] = 0
    w2[37, 0] = -float("inf")
    x2 = x.clone()
    x2[:, 0] = 1
    t2 = torch.where(t == 37, 36, t)
    loss = linear_cross_entropy(x2, w2, t2, reduction="none")
    keep = torch.arange(400, device=dev) != 37
    want, tol = reference(x2, w2[keep], torch.where(t2 > 37, t2 - 1, t2), d)
    near(loss, want[0], tol[0], "loss")
    one = w2.clone()
    one[:, 0] = -float("inf")
    assert bool(linear_cross_entropy(x2, one, t2, reduction="none")[t2 != -100].isnan().all())  # every token ruled out


def test_float16_small_gradients(dev):
    """A mean over many rows: gradients of 1e-5 whose parts lie far below float16's range."""
    x, w, t, _ = inputs(dev, F16, 700, 64, 5000)
    check(x, w, t, torch.full((700,), 2.0 ** -6, device=dev), "mean")
    check(x, w, t, torch.full((700,), 2.0 ** 12, device=dev), "sum")


@pytest.mark.parametrize("dt", [F32, BF16])
def test_no_row_counts(dev, dt):
    x, w, t, d = inputs(dev, dt, 10, 16, 50)
    t[:] = 7
    for reduction, want in (("sum", 0.0), ("mean", float("nan")), ("none", 0.0)):
        xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = linear_cross_entropy(xg, wg, t, ignore_index=7, reduction=reduction)
        assert torch.equal(loss.detach(), torch.full_like(loss, want)) or (want != want and bool(loss.isnan()))
        assert not any(bool(g.any()) for g in torch.autograd.grad(loss.sum(), [xg, wg]))
    for reduction in ("sum", "mean", "none"):
        xg, wg = x[:0].clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = linear_cross_entropy(xg, wg, t[:0], reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and bool(loss.isnan().any()) == (reduction == "mean")
        dx, dw = torch.autograd.grad(loss.sum(), [xg, wg])
        assert dx.shape == (0, 16) and not bool(dw.any())


def test_other_ignore_index(dev):
    x, w, t, d = inputs(dev, F32, 90, 24, 60)
    t[t == -100] = 3
    check(x, w, t, d, "mean", ignore_index=3)


def test_partial_gradients_repeat(dev):
    x, w, t, d = inputs(dev, BF16, 300, 200, 1500)
    both = None
    for need in ((True, True), (True, False), (False, True), (True, True)):
        xg, wg = x.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
        got = torch.autograd.grad(linear_cross_entropy(xg, wg, t), [a for a, n in zip((xg, wg), need) if n])
        both = both or got
        for a, b in zip(got, [b for b, n in zip(both, need) if n]):
            assert torch.equal(a, b)


def test_gradients_against_differences(dev):
    x, w, t, d = inputs(dev, F32, 20, 12, 40)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(linear_cross_entropy(xg, wg, t, reduction="none"), [xg, wg], d)
    f = lambda x, w: (torch.nn.functional.cross_entropy(x @ w.t(), t, reduction="none") * d.double()).sum()
    gen = torch.Generator().manual_seed(1)
    for name, got in (("x", dx), ("w", dw)):
        v = torch.randn(got.shape, generator=gen).to(dev).double()
        step = lambda s: f(x.double() + (s * v if name == "x" else 0), w.double() + (s * v if name == "w" else 0))
        diff = float((step(1e-5) - step(-1e-5)) / 2e-5)
        assert abs(float((got.double() * v).sum()) - diff) <= 1e-5 * float((got.double().abs() * v.abs()).sum())


def test_offsets_past_32_bits(dev):
    """Rows of x and of the table more than 2^31 elements apart."""
    x, w, t, d = inputs(dev, BF16, 3, 64, 5, ignored=0.0)
    flat = torch.empty(1 << 34, dtype=torch.uint8, device=dev).view(BF16)
    want = linear_cross_entropy(x, w, t, reduction="none")
    far = flat.as_strided((3, 64), ((1 << 31) + 64, 1)).copy_(x)
    assert torch.equal(linear_cross_entropy(far, w, t, reduction="none"), want)
    far = flat.as_strided((3, 64), ((1 << 31) + 64, 1)).copy_(w[:3])
    assert torch.equal(linear_cross_entropy(x, far, t % 3, reduction="none"), linear_cross_entropy(x, w[:3].contiguous(), t % 3, reduction="none"))


def test_graph(dev):
    x, w, t, d = inputs(dev, BF16, 300, 256, 2000)
    xg, wg = x.requires_grad_(True), w.requires_grad_(True)
    step = lambda x, w, t: (lambda y: (y, *torch.autograd.grad(y, [x, w])))(linear_cross_entropy(x, w, t))
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xg, wg, t)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        captured = [a.detach() for a in step(xg, wg, t)]
    for seed in range(1, 5):
        x2, w2, t2, _ = inputs(dev, BF16, 300, 256, 2000, ignored=0.2 * seed, seed=seed)
        with torch.no_grad():
            xg.copy_(x2), wg.copy_(w2), t.copy_(t2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step(x2.requires_grad_(True), w2.requires_grad_(True), t2)):
            assert torch.equal(a, b.detach())


@pytest.mark.parametrize("dt", [F32, BF16])
def test_model_loss(dev, dt):
    """MambaModel.loss against the cross entropy of its own logits."""
    model = init_weights_(MambaModel(MambaConfig(d_model=64, n_layer=2, vocab_size=300), device=dev, dtype=dt), seed=0)
    ids = torch.randint(0, 300, (2, 50), generator=torch.Generator().manual_seed(0)).to(dev)
    with torch.no_grad():
        logits = model(ids).double()
    want = torch.nn.functional.cross_entropy(logits[:, :-1].reshape(-1, 300), ids[:, 1:].reshape(-1), reduction="none").view(2, 49)
    # the model's logits are rounded to its type: two of them in a loss
    tol = 4 * max(half_step(dt), 2.0 ** -20) * logits.abs().amax()
    got = model.loss(ids, reduction="none")
    assert got.shape == (2, 50) and not bool(got[:, -1].any())
    near(got[:, :-1], want, tol.expand(2, 49), "loss")
    near(model.loss(ids), want.mean(), tol, "mean")
    targets = torch.where(ids < 150, ids, -100)
    near(model.loss(ids, targets), torch.nn.functional.cross_entropy(logits.view(-1, 300), targets.view(-1)), tol, "given")
