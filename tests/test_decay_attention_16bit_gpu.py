"""decay_attention in 16 bits: both of its variants (calls of up to 32768 tokens, batch * seqlen * heads, and larger ones),
blocks of value channels whose states lie far apart, and float16's small numbers.

Tolerances as derived in test_decay_attention_gpu.py, and one addend: below 2^-14 float16's numbers are 2^-24 apart, so that
an output rounded once is off by up to 2^-25 however small it is."""

from __future__ import annotations

import pytest
import torch

import decay_ref
from test_decay_attention_gpu import BF16, F16, F32, RUN, half_step, inputs, near, run

pytestmark = pytest.mark.gpu
# batch and heads a group at 200 tokens: 400 (batch * seqlen * heads), and 38400
SIZES = [(2, 1), (3, 64)]


def check(s, scale, outs, grads):
    """Outputs and gradients (of log decays in float32, or in the inputs' type) against the recurrence."""
    dt = s["q"].dtype
    u, n = half_step(dt), s["q"].shape[1]
    f = (400 + 2 * (-(-n // RUN))) * 2.0 ** -24
    least = 2.0 ** -25 if dt == F16 else 0.0
    args = (s["q"], s["k"], s["v"], s["g"])
    mags = tuple(t.abs().double() for t in args[:3]) + (s["g"],)
    ah0 = None if s["h0"] is None else s["h0"].abs()
    y, states = decay_ref.forward(*args, scale, s["h0"], s["lengths"])
    ay, astates = decay_ref.forward(*mags, scale, ah0, s["lengths"])
    near(outs[0], y, u * y.abs() + (u + f) * ay + least, "y")
    if len(outs) > 1:
        near(outs[1], states[:, -1], f * astates[:, -1], "state")
    del states, astates
    dstate = s["dstate"] if len(outs) > 1 else None
    want = decay_ref.backward(*args, s["dy"], scale, s["h0"], s["lengths"], dstate)
    ab = decay_ref.backward(*mags, s["dy"].abs(), scale, ah0, s["lengths"], None if dstate is None else dstate.abs())
    for k, (name, got) in enumerate(zip(("dq", "dk", "dv"), grads)):
        near(got, want[k], u * want[k].abs() + (u + f) * ab[k] + least, name)
    per = s["v"].shape[2] // s["q"].shape[2]
    crossing = (s["q"].abs().double() * ab[0]).sum(3) + (s["k"].abs().double() * ab[1]).sum(3)
    whole = torch.zeros_like(crossing)
    for t in range(0, n, RUN):
        whole[:, t:t + RUN] = crossing[:, t:t + RUN].sum(1, keepdim=True)
    whole = whole.repeat_interleave(per, 2)
    tol = half_step(s["g"].dtype) * want[3].abs() + (u + f) * ab[3] + f * whole + (least if s["g"].dtype == F16 else 0.0)
    if s["g"].dim() == 1:
        near(grads[3], want[3].sum((0, 1)), (tol + 2.0 ** -22 * want[3].abs()).sum((0, 1)), "dg")
    else:
        near(grads[3], want[3], tol, "dg")
    if s["h0"] is not None:
        near(grads[4], want[4], f * ab[4], "dh0")


@pytest.mark.parametrize("b,per", SIZES)
@pytest.mark.parametrize("what", ["dq", "dk"])
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("far", [0, 1])
def test_blocks_far_apart(dev, b, per, what, odd, far):
    """Two blocks of value channels, of which one's states (their gradients) have decayed to 1e-34 where the other's are near
    1, with what they are multiplied with in the thousands."""
    n, dv = 200, 127 if odd else 128
    s = inputs(dev, F16, b, n, 1, per, 16, dv, g_dtype=F32)
    s["g"].fill_(-1.2)
    block = slice(64 * far, 64 * far + 64)
    if what == "dq":  # the states before tokens 128 on
        s["v"][:, 64:, :, block] = 0
        s["dy"] = s["dy"] * 1024
    else:             # the gradients of the states behind tokens 0 to 63
        s["dy"][:, :128, :, block] = 0
        s["v"] = s["v"] * 4096  # (the largest true gradient, of 64 heads that share k: 33800)
    outs, grads = run(s, 0.01, with_state=False)
    assert all(bool(t.isfinite().all()) for t in (*outs, *grads))
    check(s, 0.01, outs, grads)


def added(k, g, lengths, mirrored=False):
    """What a state would be if each token added |k|, but decayed by whole runs behind (mirrored: before) its own alone."""
    b, n, heads = g.shape
    live = torch.arange(n, device=g.device)[None] < lengths[:, None]
    k = (k.abs().double() * live[..., None, None]).repeat_interleave(heads // k.shape[2], 2)
    g = g.double() * live[..., None]
    total = k.new_zeros((b, heads, k.shape[3]))
    starts = range(0, n, RUN)
    for t in reversed(starts) if mirrored else starts:
        total = torch.exp(g[:, t:t + RUN].sum(1))[..., None] * total + k[:, t:t + RUN].sum(1)
    return total[..., None]


@pytest.mark.parametrize("b,per", SIZES)
@pytest.mark.parametrize("down", [12, 17, 20])
def test_states_of_small_numbers(dev, b, per, down):
    """float16's values and gradients near 2^-down, below 2^-14 subnormal numbers: the state and its gradient are float32 all the
    same.  A run's values are weighted by their decay to its end, and a sum of two float16 numbers, the second times 2^11, stands
    for each: off by 2^-23 of it (among f's), or by 2^-36 where it is small, which then no decay within the run makes less."""
    s = inputs(dev, F16, b, 200, 1, per, 32, 48, h0=True, ragged=True, g_dtype=F32)
    for k in ("v", "dy"):
        s[k] = s[k] * 2.0 ** -down
    s["h0"], s["dstate"] = s["h0"] * 2.0 ** -down, s["dstate"] * 2.0 ** -down
    outs, grads = run(s, 0.6)
    f = (400 + 2 * 4) * 2.0 ** -24
    mags = [s[k].abs() for k in ("q", "k", "v")] + [s["g"]]
    _, states = decay_ref.forward(s["q"], s["k"], s["v"], s["g"], 0.6, s["h0"], s["lengths"])
    _, a = decay_ref.forward(*mags, 0.6, s["h0"].abs(), s["lengths"])
    near(outs[1], states[:, -1], f * a[:, -1] + 2.0 ** -36 * added(s["k"], s["g"], s["lengths"]), "state")
    want = decay_ref.backward(s["q"], s["k"], s["v"], s["g"], s["dy"], 0.6, s["h0"], s["lengths"], s["dstate"])[4]
    a = decay_ref.backward(*mags, s["dy"].abs(), 0.6, s["h0"].abs(), s["lengths"], s["dstate"].abs())[4]
    near(grads[4], want, f * a + 2.0 ** -36 * added(s["q"], s["g"], s["lengths"], mirrored=True), "dh0")


def test_states_where_products_round_to_ties(dev):
    """A weighted value whose product is next to the middle of two float16 numbers: its two terms belong together.  (So many
    tokens that some are; each of the state's elements is near its sum.)"""
    s = inputs(dev, F16, 4, 250, 1, 64, 16, 64, g_dtype=F32, seed=2)
    outs, _ = run(s, 1.0)
    _, states = decay_ref.forward(s["q"], s["k"], s["v"], s["g"])
    _, a = decay_ref.forward(s["q"].abs(), s["k"].abs(), s["v"].abs(), s["g"])
    near(outs[1], states[:, -1], (400 + 2 * 4) * 2.0 ** -24 * a[:, -1], "state")


@pytest.mark.parametrize("b,per", SIZES)
@pytest.mark.parametrize("dk,dv", [(32, 48), (100, 72)])
@pytest.mark.parametrize("q,k,v,dy", [(0, 0, 0, -14), (0, 0, -14, 0), (-10, -9, 9, 5), (-14, 0, 14, -5), (9, 8, -12, -12), (-14, -14, 8, 14)])
def test_scores_of_any_size(dev, b, per, dk, dv, q, k, v, dy):
    """float16's scores, and dy.v of the gradients, far below 2^-14 and far above 65504, where the outputs are neither."""
    s = inputs(dev, F16, b, 200, 1, per, dk, dv, ragged=True, g_dtype=F32)
    for name, up in (("q", q), ("k", k), ("v", v), ("dy", dy)):
        s[name] = (s[name].clamp(-2, 2) * 2.0 ** up).contiguous()
    outs, grads = run(s, 0.125, with_state=False)
    assert all(bool(t.isfinite().all()) for t in (*outs, *grads))
    check(s, 0.125, outs, grads)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("shape", [  # batch, seqlen, groups, heads a group, key_dim, value_dim: above 32768 tokens
    (4, 300, 2, 16, 128, 64), (3, 350, 1, 32, 96, 96), (3, 350, 1, 32, 72, 130), (3, 351, 2, 16, 33, 65), (2, 130, 64, 2, 127, 32),
    (5, 65, 103, 1, 128, 128), (1, 2100, 1, 16, 128, 24)])
@pytest.mark.parametrize("fixed", [False, True])
def test_large_calls(dev, dt, shape, fixed):
    """The variant of ordinary sizes: wide keys, several blocks of value channels, rows off 16 bytes, shared and single heads."""
    assert shape[0] * shape[1] * shape[2] * shape[3] > 32768
    s = inputs(dev, dt, *shape, fixed=fixed, h0=True, ragged=True, g_dtype=F32 if fixed else None, seed=sum(shape))
    outs, grads = run(s, 0.6)
    check(s, 0.6, outs, grads)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("shape", [(1, 300, 1, 2, 64, 64), (2, 150, 1, 24, 128, 64), (1, 333, 2, 2, 65, 96)])
def test_gradients_of_few_tokens_are_rounded_once(dev, dt, shape):
    """Calls of few tokens: dq, dk and dlog_decay are as far from the truth as its rounding.  What else is rounded there, scores
    and states, is to two terms, 2^-16 of a sum's magnitudes and less, which here are some 20 times the sum's root mean
    square: with a rounding of 2^-9 times 0.58 at the root of the mean square, under 0.1 of it, and 1.005 times it together."""
    s = inputs(dev, dt, *shape, h0=True, seed=sum(shape))
    _, grads = run(s, 0.6)
    want = decay_ref.backward(s["q"], s["k"], s["v"], s["g"], s["dy"], 0.6, s["h0"], None, s["dstate"])
    for name, at in (("dq", 0), ("dk", 1), ("dg", 3)):
        rounding = (want[at].to(dt).double() - want[at]).norm()
        assert float((grads[at].double() - want[at]).norm() / rounding) < 1.05, name


@pytest.mark.parametrize("b,per", [(3, 2), (3, 80)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_broken_stays_in_its_head(dev, b, per, bad):
    """A NaN or an infinity in float16, whose powers of two are taken over many numbers: other sequences, and other heads (for dq
    and dk other groups), are the same bits."""
    s = inputs(dev, F16, b, 200, 2, per, 64, 72, h0=True, g_dtype=F32)
    base, clean = run(s, 1.0)
    for name, at in (("q", (1, 100, 1)), ("k", (1, 100, 1)), ("v", (1, 100, 2 * per - 1)), ("dy", (1, 100, 2 * per - 1))):
        t = {**s, name: s[name].clone()}
        t[name][at] = bad
        outs, grads = run(t, 1.0)
        heads = slice(0, per) if name in ("q", "k") else slice(0, 2 * per - 1)
        for a, c in zip([*outs, grads[2], grads[3], grads[4]], [*base, clean[2], clean[3], clean[4]]):
            at_heads = (slice(None), heads) if a.shape[1] == 2 * per else (slice(None), slice(None), heads)
            assert torch.equal(a[0::2], c[0::2]) and torch.equal(a[at_heads], c[at_heads]), name
        for a, c in zip(grads[:2], clean[:2]):
            assert torch.equal(a[0::2], c[0::2]) and torch.equal(a[:, :, 0], c[:, :, 0]), name
        of = grads[0 if name == "k" else 1]  # (dk = dS v holds no k)
        assert bool(of[1, :, 1].isfinite().logical_not().any()), name
