"""decay_attention, its gradients and its token step against the recurrence in 64 bits.

Tolerances, element by element.  With |.|-sums (the same formulas on the inputs' magnitudes, ``A`` below) every error
is a share of them.  u is the type's half step (0 where an output is float32 and its sums take no rounded factor).
  16-bit types: the scores of a run, or the state, are rounded once before their product: u A; the output: u |y|.
  fp32 sums: a dot product of 128, one of 64 tokens, one of 128 with the state, which is a sum of 64 tokens that takes
  two more roundings a run: (400 + 2 runs) 2^-24 A, decays' own errors (a few units of 2^-24, 2^-22 for the hardware's
  exp2 of the 16-bit types) among the 400.
  The decays' gradient is a difference of sums over a run, so its fp32 share is of the whole run's sums."""

from __future__ import annotations

import pytest
import torch

import decay_ref
from mamba_metal_amd import decay_attention, decay_attention_step

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
RUN = 64


def half_step(dt):
    return 0.0 if dt == F32 else torch.finfo(dt).eps / 2


def inputs(dev, dt, b, n, groups, per, dk, dv, *, fixed=False, h0=False, ragged=False, g_dtype=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    heads = groups * per
    r = lambda *s: torch.randn(s, generator=gen)
    rate = torch.exp(-6.0 * torch.rand(heads, generator=gen))  # memories of one to 400 tokens
    g = -rate if fixed else -rate * torch.rand((b, n, heads), generator=gen) * 2
    lengths = None
    if ragged:
        lengths = torch.randint(0, n + 1, (b,), generator=gen, dtype=torch.int32)
        lengths[0] = n
        if b > 2:
            lengths[1] = 0
    to = lambda t, d=dt: None if t is None else t.to(dev, d)
    return dict(q=to(r(b, n, groups, dk)), k=to(r(b, n, groups, dk) * dk ** -0.5), v=to(r(b, n, heads, dv)),
                g=to(g, g_dtype or dt), h0=to(r(b, heads, dk, dv), F32) if h0 else None, lengths=to(lengths, torch.int32),
                dy=to(r(b, n, heads, dv)), dstate=to(r(b, heads, dk, dv), F32))


def run(s, scale, with_state=True):
    leaves = [s[k].detach().requires_grad_(True) for k in ("q", "k", "v", "g")]
    h0 = None if s["h0"] is None else s["h0"].detach().requires_grad_(True)
    out = decay_attention(*leaves, scale=scale, h0=h0, lengths=s["lengths"], return_state=with_state)
    leaves += [] if h0 is None else [h0]
    outs, ups = (list(out), [s["dy"], s["dstate"]]) if with_state else ([out], [s["dy"]])
    return [t.detach() for t in outs], torch.autograd.grad(outs, leaves, ups)


def near(got, want, tol, what):
    assert got.shape == want.shape, what
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by {float((err / tol.clamp_min(1e-300)).max()):.3g} of the bound"


def check(s, scale, outs, grads):
    dt = s["q"].dtype
    u, n = half_step(dt), s["q"].shape[1]
    f = (400 + 2 * (-(-n // RUN))) * 2.0 ** -24
    args = (s["q"], s["k"], s["v"], s["g"])
    mags = tuple(t.abs().double() for t in args[:3]) + (s["g"],)
    ah0 = None if s["h0"] is None else s["h0"].abs()
    y, states = decay_ref.forward(*args, scale, s["h0"], s["lengths"])
    ay, astates = decay_ref.forward(*mags, scale, ah0, s["lengths"])
    near(outs[0], y, u * y.abs() + (u + f) * ay, "y")
    if len(outs) > 1:
        near(outs[1], states[:, -1], f * astates[:, -1], "state")
    if grads is None:
        return
    dstate = s["dstate"] if len(outs) > 1 else None
    want = decay_ref.backward(*args, s["dy"], scale, s["h0"], s["lengths"], dstate)
    ab = decay_ref.backward(*mags, s["dy"].abs(), scale, ah0, s["lengths"], None if dstate is None else dstate.abs())
    for k, (name, got) in enumerate(zip(("dq", "dk", "dv"), grads)):
        near(got, want[k], u * want[k].abs() + (u + f) * ab[k], name)
    # the decays': the sums of a run that enter and cancel, on both sides of a token
    b, n, heads, _ = s["v"].shape
    per = heads // s["q"].shape[2]
    crossing = (s["q"].abs().double() * ab[0]).sum(3) + (s["k"].abs().double() * ab[1]).sum(3)  # per group, over its heads
    whole = torch.zeros_like(crossing)
    for t in range(0, n, RUN):
        whole[:, t:t + RUN] = crossing[:, t:t + RUN].sum(1, keepdim=True)
    whole = whole.repeat_interleave(per, 2)
    ug = half_step(s["g"].dtype)
    tol = ug * want[3].abs() + (u + f) * ab[3] + f * whole
    if s["g"].dim() == 1:  # one decay a head: summed in 64 bits over batch and time, rounded twice
        near(grads[3], want[3].sum((0, 1)), (tol + 2.0 ** -22 * want[3].abs()).sum((0, 1)), "dg")
    else:
        near(grads[3], want[3], tol, "dg")
    if s["h0"] is not None:
        near(grads[4], want[4], f * ab[4], "dh0")


SHAPES = [  # batch, seqlen, groups, heads a group, key_dim, value_dim
    (1, 1, 1, 1, 1, 1), (2, 1, 2, 1, 64, 64), (1, 63, 1, 2, 16, 8), (3, 64, 2, 1, 128, 64), (2, 65, 1, 3, 64, 128),
    (3, 130, 2, 2, 48, 80), (1, 200, 3, 1, 5, 7), (2, 129, 1, 1, 127, 130), (1, 700, 1, 2, 128, 64), (4, 257, 1, 5, 33, 65),
]


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["plain", "all", "fixed"])
def test_against_the_recurrence(dev, dt, shape, kind):
    s = inputs(dev, dt, *shape, fixed=kind == "fixed", h0=kind == "all", ragged=kind == "all",
               g_dtype=F32 if kind == "fixed" else None, seed=sum(shape))
    outs, grads = run(s, 0.6, with_state=kind != "plain")
    check(s, 0.6, outs, grads)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_many_heads_share(dev, dt):
    """A workgroup that sums the gradients of several heads, and several workgroups' sums."""
    s = inputs(dev, dt, 2, 150, 1, 24, 32, 16, ragged=True)
    check(s, 1.0, *run(s, 1.0))
    s = inputs(dev, dt, 8, 6500, 1, 2, 8, 8)
    outs, grads = run(s, 1.0)
    check(s, 1.0, outs, grads)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_without_a_gradient(dev, dt):
    s = inputs(dev, dt, 2, 300, 2, 2, 64, 64, h0=True, ragged=True)
    args = dict(scale=0.3, h0=s["h0"], lengths=s["lengths"], return_state=True)
    with torch.no_grad():
        y, h = decay_attention(s["q"], s["k"], s["v"], s["g"], **args)
    check(s, 0.3, [y, h], None)
    again = decay_attention(s["q"], s["k"], s["v"], s["g"], **{**args, "lengths": s["lengths"].long()})
    assert torch.equal(y, again[0]) and torch.equal(h, again[1])


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_forgetting_at_once(dev, dt):
    """-inf forgets all before it, and what comes after it is as exact as ever."""
    s = inputs(dev, dt, 2, 190, 1, 2, 32, 32, h0=True)
    s["g"][:, 5] = -float("inf")
    s["g"][0, 100:110] = -float("inf")
    s["g"][1, 64, 0] = -float("inf")
    s["g"][1, 128:, 1] = -1e30
    outs, grads = run(s, 1.0)
    check(s, 1.0, outs, grads)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_lies_behind_a_sequence(dev, dt, bad):
    s = inputs(dev, dt, 4, 200, 2, 2, 64, 48, h0=True, ragged=True, seed=3)
    clean_outs, clean = run(s, 1.0)
    t = torch.arange(200, device=dev)
    dead = t[None] >= s["lengths"][:, None].long()
    for k in ("q", "k", "v", "g", "dy"):
        s[k][dead] = bad
    outs, grads = run(s, 1.0)
    for a, b in zip(outs + list(grads), clean_outs + list(clean)):
        assert torch.equal(a, b)
    for got in (outs[0], *grads[:4]):
        assert not bool(got[dead].any())
    assert torch.equal(outs[1][1], s["h0"][1])  # a sequence of no tokens


@pytest.mark.parametrize("dt", [F32, BF16])
def test_not_a_number_stays(dev, dt):
    """In its sequence and head, and (but for a run's values) behind its token."""
    s = inputs(dev, dt, 3, 200, 3, 2, 64, 64)
    base, _ = run(s, 1.0)
    for name, at, heads in (("q", (1, 100, 1), [2, 3]), ("v", (1, 100, 3), [3]), ("k", (1, 100, 2), [4, 5]), ("g", (1, 100, 0), [0])):
        t = {**s, name: s[name].clone()}
        t[name][at] = float("nan")
        y = run(t, 1.0)[0][0]
        touched = torch.zeros((3, 200, 6), dtype=torch.bool, device=dev)
        touched[1, 64:, heads] = True
        assert torch.equal(y[~touched], base[0][~touched]), name
        after = [100] if name == "q" else range(100, 200)
        assert all(bool(y[1, t0, h].isnan().all()) for t0 in after for h in heads), name


@pytest.mark.parametrize("dt", [F16, BF16, F32])
def test_layouts(dev, dt):
    """Slices of one projection, time before batch, odd offsets and widths: the same bits as from contiguous tensors."""
    b, n, groups, per, dk, dv = 2, 100, 2, 2, 32, 24
    s = inputs(dev, dt, b, n, groups, per, dk, dv)
    want_outs, want = run(s, 1.0)
    heads = groups * per
    for offset in (0, 1):
        wide = torch.zeros((n, b, 2 * groups * dk + heads * dv + 8), dtype=dt, device=dev).transpose(0, 1)
        parts, at = {}, offset
        for k, h, w in (("q", groups, dk), ("k", groups, dk), ("v", heads, dv)):
            parts[k] = wide[..., at:at + h * w].unflatten(2, (h, w))
            parts[k].copy_(s[k])
            at += h * w
        t = {**s, **parts, "dy": s["dy"].transpose(0, 1).contiguous().transpose(0, 1),
             "g": s["g"].permute(2, 0, 1).contiguous().permute(1, 2, 0)}
        outs, grads = run(t, 1.0)
        for a, c in zip(outs + list(grads), want_outs + list(want)):
            assert torch.equal(a, c)
    one = inputs(dev, dt, b, n, 1, 1, dk, dv)
    one["dy"] = one["dy"][:1, :1].expand(b, n, 1, dv)  # a gradient that all tokens share
    outs, grads = run(one, 1.0)
    check(one, 1.0, outs, grads)


def test_offsets_past_32_bits(dev):
    """Sequences and tokens more than 2^31 elements apart."""
    s = inputs(dev, BF16, 2, 70, 1, 1, 64, 64)
    want_outs, want = run(s, 1.0)
    flat = torch.empty((1 << 32) + (1 << 20), dtype=torch.uint8, device=dev).view(BF16)
    far = flat.as_strided((2, 70, 1, 64), ((1 << 31) + 64, 128, 64, 1))
    for k in ("q", "v", "dy"):
        t = {**s, k: far.copy_(s[k])}
        outs, grads = run(t, 1.0)
        for a, c in zip(outs + list(grads), want_outs + list(want)):
            assert torch.equal(a, c), k


def test_float16_range(dev):
    """A state above 65504, and gradients far below 1: the state passes its product through a power of two."""
    s = inputs(dev, F16, 1, 300, 1, 1, 64, 64, fixed=True, g_dtype=F32)
    s["g"].fill_(-1e-4)
    s["k"], s["v"] = s["k"].abs() * 64, s["v"].abs() * 64
    s["q"], s["dy"] = s["q"] * 2.0 ** -12, s["dy"] * 2.0 ** -6
    outs, grads = run(s, 1.0)
    assert float(outs[1].max()) > 65504
    assert all(bool(t.isfinite().all()) for t in [*outs, *grads])
    check(s, 1.0, outs, [*grads[:3], grads[3]])


@pytest.mark.parametrize("dt", [F32, BF16])
def test_gradients_against_differences(dev, dt):
    """The formula's gradients against differences of the recurrence in 64 bits, on small sizes."""
    s = inputs(dev, dt, 1, 70, 1, 2, 3, 2, h0=True)
    _, grads = run(s, 0.8)
    gen = torch.Generator().manual_seed(5)

    def loss(**over):
        a = {**{k: s[k].double() for k in ("q", "k", "v", "g", "h0")}, **over}
        y, st = decay_ref.forward(a["q"], a["k"], a["v"], a["g"], 0.8, a["h0"])
        return float((y * s["dy"].double()).sum() + (st[:, -1] * s["dstate"].double()).sum())

    for name, got in zip(("q", "k", "v", "g", "h0"), grads):
        d = torch.randn(s[name].shape, generator=gen).to(dev).double()
        eps = 1e-4
        diff = (loss(**{name: s[name].double() + eps * d}) - loss(**{name: s[name].double() - eps * d})) / (2 * eps)
        scale = float((got.double().abs() * d.abs()).sum())
        assert abs(float((got.double() * d).sum()) - diff) <= (4 * half_step(dt) + 1e-4) * scale, name


def test_partial_gradients(dev):
    """Only what is asked for, only the state used, and the same bits each time."""
    s = inputs(dev, BF16, 2, 150, 1, 3, 64, 64, h0=True)
    _, full = run(s, 1.0)
    for k, name in enumerate(("q", "k", "v", "g", "h0")):
        a = {n: s[n].detach().clone().requires_grad_(n == name) for n in ("q", "k", "v", "g", "h0")}
        y, h = decay_attention(a["q"], a["k"], a["v"], a["g"], h0=a["h0"], return_state=True)
        got, = torch.autograd.grad([y, h], [a[name]], [s["dy"], s["dstate"]])
        assert torch.equal(got, full[k]), name
    a = [s[n].detach().requires_grad_(True) for n in ("q", "k", "v", "g")]
    _, h = decay_attention(*a, return_state=True)
    grads = torch.autograd.grad(h, a, s["dstate"])
    t = {**s, "dy": torch.zeros_like(s["dy"]), "h0": None}
    for x, y in zip(grads, run(t, 1.0)[1]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("n", [0, 1])
def test_empty(dev, n):
    """No tokens, no sequences."""
    s = inputs(dev, BF16, 2, 1, 1, 2, 16, 8, h0=True)
    for k in ("q", "k", "v", "g", "dy"):
        s[k] = s[k][:, :n] if n == 0 else s[k][:0]
    if n:
        s["h0"], s["dstate"] = s["h0"][:0], s["dstate"][:0]
    outs, grads = run(s, 1.0)
    assert torch.equal(outs[1], s["h0"]) and torch.equal(grads[4], s["dstate"])
    assert outs[0].shape == s["v"].shape and all(a.shape == s[k].shape for a, k in zip(grads, ("q", "k", "v", "g")))
    heads = torch.full((2,), -0.1, device=dev, requires_grad=True)
    y = decay_attention(s["q"], s["k"], s["v"], heads)
    assert not bool(torch.autograd.grad(y, heads, s["dy"])[0].any())


def test_graph_and_streams(dev):
    """A forward and backward pass captured on a stream of its own and replayed on other inputs."""
    s = inputs(dev, BF16, 1, 2000, 1, 4, 64, 64, ragged=True)  # (few heads: cut into segments)
    names = ("q", "k", "v", "g")
    live = {k: s[k].clone().requires_grad_(True) for k in names}
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    step = lambda: (lambda y: (y, *torch.autograd.grad(y, [live[k] for k in names], s["dy"])))(
        decay_attention(*(live[k] for k in names), lengths=s["lengths"]))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        captured = [t.detach() for t in step()]
    for seed in range(4):
        new = inputs(dev, BF16, 1, 2000, 1, 4, 64, 64, seed=seed)
        with torch.no_grad():
            for k in names:
                live[k].copy_(new[k])
        graph.replay()
        torch.cuda.synchronize()
        outs, grads = run({**new, "lengths": s["lengths"], "dy": s["dy"]}, 1.0, with_state=False)
        for a, b in zip(captured, outs + list(grads)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------ the token step
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 2, 2, 64, 64), (2, 1, 5, 128, 96), (2, 1, 3, 7, 130), (5, 3, 1, 33, 18)])
@pytest.mark.parametrize("fixed", [False, True])
def test_step(dev, dt, shape, fixed):
    b, groups, per, dk, dv = shape
    s = inputs(dev, dt, b, 1, groups, per, dk, dv, fixed=fixed, h0=True, g_dtype=F32 if fixed else None)
    q, k, v = (s[n][:, 0] for n in ("q", "k", "v"))
    g = s["g"] if fixed else s["g"][:, 0]
    y_ref, states = decay_ref.forward(s["q"], s["k"], s["v"], s["g"], 0.9, s["h0"])
    ay, ast = decay_ref.forward(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["g"], 0.9, s["h0"].abs())
    new = torch.empty_like(s["h0"])
    y = decay_attention_step(s["h0"], q, k, v, g, scale=0.9, state_out=new)
    # the decay, the product and their sum: 8 units; y: 128 products, 16 partial sums
    near(new, states[:, 1], 8 * 2.0 ** -24 * ast[:, 1], "state")
    near(y, y_ref[:, 0], half_step(dt) * y_ref[:, 0].abs() + 160 * 2.0 ** -24 * ay[:, 0], "y")
    inplace = s["h0"].clone()
    wide = torch.full((b, groups * per, 2 * dv), 7.0, dtype=dt, device=dev)
    y2 = decay_attention_step(inplace, q, k, v, g, scale=0.9, out=wide[..., dv:])
    assert torch.equal(inplace, new) and torch.equal(y2, y) and bool((wide[..., :dv] == 7).all())
    odd = torch.empty(s["h0"].numel() + 1, device=dev)[1:].view_as(s["h0"]).copy_(s["h0"])  # not on 16 bytes
    assert torch.equal(decay_attention_step(odd, q, k, v, g, scale=0.9), y) and torch.equal(odd, new)


@pytest.mark.parametrize("dt", [F32, BF16])
def test_prompt_then_tokens(dev, dt):
    """A prompt's state and then tokens one by one, as a server runs it, against the whole sequence."""
    n, m = 150, 10
    s = inputs(dev, dt, 2, n + m, 1, 2, 64, 64)
    with torch.no_grad():
        y, h = decay_attention(*(s[k][:, :n] for k in ("q", "k", "v", "g")), return_state=True)
        ys = [y] + [decay_attention_step(h, *(s[k][:, t] for k in ("q", "k", "v", "g")))[:, None] for t in range(n, n + m)]
    check(s, 1.0, [torch.cat(ys, 1), h], None)
