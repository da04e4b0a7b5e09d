"""gated_scan, gated_scan_step and their gradients against 64-bit definitions (gated_ref.py)."""

from __future__ import annotations

import math

import pytest
import torch

import gated_ref as ref
from mamba_metal_amd import _lib, causal_conv1d_train, gated_scan, gated_scan_step
from mamba_metal_amd.selective_scan import reset_scan_status, scan_status

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# lengths of one token, around a block of 16 tokens, around tiles of time, widths around 64 lanes, many sequences
SIZES = [(1, 1, 1), (2, 2, 3), (3, 16, 64), (2, 17, 65), (1, 33, 130), (2, 129, 66), (1, 600, 200), (1, 1021, 70),
         (2, 2600, 64), (129, 300, 9)]


def rand(seed, b, n, d, dtype, dev, z=True, h0=False, rates=1.0):
    g = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(s, generator=g)
    f = {k: t(b, n, d).to(dtype).to(dev) for k in ("x", "a_gate", "x_gate", "z", "dy")}
    if not z:
        f["z"] = None
    f["A"] = (-rates * torch.exp(torch.rand(d, generator=g) * math.log(1000.0) - math.log(1000.0))).to(dev)
    f["h0"] = t(b, d).to(dev) if h0 else None
    f["dstate"] = t(b, d).to(dev)
    return f


def case(f, lengths=None):
    return ref.Case(f["x"], f["a_gate"], f["x_gate"], f["A"], f["z"], f["h0"], lengths)


def forward(f, **kw):
    return gated_scan(f["x"], f["a_gate"], f["x_gate"], f["A"], z=f["z"], h0=f["h0"], return_state=True, **kw)


LEAVES = ("x", "a_gate", "x_gate", "A", "z", "h0")


def train(f, state_grad=True, **kw):
    leaves = {k: f[k].detach().clone().requires_grad_(True) for k in LEAVES if f[k] is not None}
    f = {**f, **leaves}
    y, state = forward(f, **kw)
    outs, grads = ([y, state], [f["dy"], f["dstate"]]) if state_grad else ([y], [f["dy"]])
    got = torch.autograd.grad(outs, list(leaves.values()), grads)
    return y, state, dict(zip(leaves, got))


def check_forward(c, y, state, dtype):
    wy, ey, wh, eh = c.forward()
    ref.close(y, wy, ey, dtype, "y")
    ref.close(state, wh, eh, torch.float32, "state")


def check_grads(c, f, got, dtype, state_grad=True, eight=False):
    want = c.backward(f["dy"], f["dstate"] if state_grad else None, eight)
    for k, v in got.items():
        ref.close(v, *want[k], torch.float32 if k in ("A", "h0") else dtype, "d" + k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("z,h0", [(False, False), (True, True)])
def test_forward(dev, dtype, size, z, h0):
    f = rand(1, *size, dtype, dev, z, h0)
    y, state = forward(f)
    check_forward(case(f), y, state, dtype)
    assert y.dtype == dtype and y.is_contiguous() and state.dtype == torch.float32


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("z,h0,checkpoint", [(False, False, "full"), (True, True, "full"), (True, False, "int8"),
                                             (False, True, "int8")])
def test_gradients(dev, dtype, size, z, h0, checkpoint):
    f = rand(2, *size, dtype, dev, z, h0)
    y, state, got = train(f, checkpoint=checkpoint)
    check_forward(case(f), y, state, dtype)
    check_grads(case(f), f, got, dtype, eight=checkpoint == "int8")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rates", [1e-3, 8.0, 300.0])
def test_rates(dev, dtype, rates):
    """Channels that forget nothing for thousands of tokens, and ones that forget at once."""
    f = rand(3, 1, 900, 96, dtype, dev, rates=rates)
    y, state, got = train(f)
    check_forward(case(f), y, state, dtype)
    check_grads(case(f), f, got, dtype)


@pytest.mark.parametrize("lengths_dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("checkpoint", ["full", "int8"])
@pytest.mark.parametrize("n", [40, 700, 2900])
def test_lengths(dev, lengths_dtype, checkpoint, n):
    """Padded batches: empty slots, single tokens, ends inside a block and on its border, whole ones, lengths out
    of range; what padding holds (here NaNs and infinities) does not matter."""
    lengths = torch.tensor([0, 1, 15, 16, 17, n // 2, n - 1, n, n + 5, -3], dtype=lengths_dtype, device=dev)
    f = rand(4, len(lengths), n, 70, torch.float32, dev, h0=True)
    live = torch.arange(n, device=dev)[None, :, None] < lengths[:, None, None]
    for k, v in (("x", "nan"), ("a_gate", "inf"), ("x_gate", "nan"), ("z", "-inf"), ("dy", "nan")):
        f[k] = torch.where(live, f[k], torch.full_like(f[k], float(v)))
    y, state, got = train(f, lengths=lengths, checkpoint=checkpoint)
    c = case(f, lengths)
    check_forward(c, y, state, torch.float32)
    check_grads(c, f, got, torch.float32, eight=checkpoint == "int8")
    assert torch.equal(state[0], f["h0"][0]) and torch.equal(got["h0"][0], f["dstate"][0])
    for t in (y, got["x"], got["a_gate"], got["x_gate"], got["z"]):
        assert not torch.where(live, torch.zeros_like(t), t).any()


def test_strides(dev):
    """Inputs as slices of one wide projection, transposed batch and time, broadcast over the batch."""
    b, n, d = 3, 75, 66
    f = rand(5, b, n, d, torch.bfloat16, dev)
    wide = torch.zeros((b, n, 4 * d + 1), dtype=torch.bfloat16, device=dev)
    wide[..., :d], wide[..., d:2 * d] = f["x"], f["a_gate"]
    f["x"], f["a_gate"] = wide[..., :d], wide[..., d:2 * d]
    f["x_gate"] = f["x_gate"].transpose(0, 1).contiguous().transpose(0, 1)
    f["z"] = f["z"][:1].expand(b, n, d)
    y, state = forward(f)
    check_forward(case(f), y, state, torch.bfloat16)
    zl = f["z"][:1].detach().clone().requires_grad_(True)
    xl = f["x"].detach().requires_grad_(True)
    y = gated_scan(xl, f["a_gate"], f["x_gate"], f["A"], z=zl.expand(b, n, d))
    dx, dz = torch.autograd.grad(y, [xl, zl], f["dy"].transpose(0, 1).contiguous().transpose(0, 1))
    want = case(f).backward(f["dy"])
    ref.close(dx, *want["x"], torch.bfloat16, "dx")
    # the sum over the batch that autograd takes of the rounded parts, rounded again
    parts, bounds = want["z"]
    half = ref.half_step(torch.bfloat16)
    ref.close(dz, parts.sum(0, keepdim=True), (bounds + 3 * half * parts.abs()).sum(0, keepdim=True),
              torch.bfloat16, "dz")


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_gradient_of_a_sum(dev, checkpoint):
    """y.sum().backward(): the gradient arrives expanded, with no strides at all."""
    f = rand(6, 2, 50, 64, torch.float32, dev)
    leaves = {k: f[k].clone().requires_grad_(True) for k in ("x", "a_gate", "x_gate", "A", "z")}
    gated_scan(leaves["x"], leaves["a_gate"], leaves["x_gate"], leaves["A"], z=leaves["z"],
               checkpoint=checkpoint).sum().backward()
    f["dy"] = torch.ones_like(f["x"])
    check_grads(case(f), f, {k: v.grad for k, v in leaves.items()}, torch.float32, state_grad=False,
                eight=checkpoint == "int8")


def test_state_gradient_only(dev):
    f = rand(7, 2, 40, 64, torch.float32, dev, z=False, h0=True)
    leaves = {k: f[k].clone().requires_grad_(True) for k in ("x", "A", "h0")}
    _, state = gated_scan(leaves["x"], f["a_gate"], f["x_gate"], leaves["A"], h0=leaves["h0"], return_state=True)
    got = dict(zip(leaves, torch.autograd.grad(state, list(leaves.values()), f["dstate"])))
    f["dy"] = torch.zeros_like(f["x"])
    check_grads(case(f), f, got, torch.float32)


def test_against_differences(dev):
    """The kernel's gradient along a direction against differences of the 64-bit definition."""
    f = rand(8, 2, 60, 48, torch.float32, dev, h0=True)
    f["A"] = f["A"] - 0.05  # away from the root's infinite slope at a = 1
    _, _, got = train(f)
    g = torch.Generator().manual_seed(9)
    cpu = {k: v.cpu().double() for k, v in f.items()}
    for k in LEAVES:
        v = torch.randn(f[k].shape, generator=g, dtype=torch.float64)
        step = 1e-6

        def loss(s):
            p = {**cpu, k: cpu[k] + s * v}
            y, _, h, _ = case(p).forward()
            return (y * cpu["dy"]).sum() + (h * cpu["dstate"]).sum()

        diff = ((loss(step) - loss(-step)) / (2 * step)).item()
        parts = got[k].cpu().double() * v
        # float32 gradients: 1e-5 of the parts' magnitude (their bounds above are far below); the difference's
        # own error: step^2 times third derivatives and 2^-52 / step of the loss's parts
        assert abs(parts.sum().item() - diff) <= 1e-5 * parts.abs().sum().item() + 1e-6, k


def test_extreme_gates(dev):
    """Saturated gates, decay rates of 0 and -inf: no NaN where the definition has none."""
    n, d = 64, 8
    f = rand(10, 1, n, d, torch.float32, dev)
    for k, v in enumerate((float("inf"), -float("inf"), 80.0, -80.0, 200.0, -200.0)):
        f["a_gate"][0, 5 + k], f["x_gate"][0, 20 + k] = v, v
    f["A"] = torch.tensor([0.0, -float("inf"), -1e-30, -1e30, -1.0, -1e-7, -50.0, -1e4], device=dev)
    # -inf times a gate of exactly 0 has no value by the formula; the kernel's is a = 1
    f["a_gate"][0, :, 1] = f["a_gate"][0, :, 1].clamp(-80, 80)
    f["a_gate"][0, :, 3] = f["a_gate"][0, :, 3].clamp(-30, 80)
    y, state, got = train(f)
    for t in (y, state, *got.values()):
        assert torch.isfinite(t).all()
    c = case(f)
    wy, ey, wh, eh = c.forward()
    ref.close(y, wy, ey, torch.float32, "y")
    want = c.backward(f["dy"], f["dstate"])
    for k in ("x", "x_gate", "z"):
        ref.close(got[k], *want[k], torch.float32, "d" + k)
    # A = -inf: h is the gated input alone, and nothing flows back
    assert not got["a_gate"][..., 1].any() and got["A"][1] == 0
    # A = 0: the state stays as it is
    assert not state[:, 0].any()


def test_nan_and_infinity_pass_through(dev):
    f = rand(11, 1, 64, 64, torch.float32, dev)
    f["x"][0, 20, 3] = float("nan")
    f["a_gate"][0, 30, 5] = float("nan")
    f["A"][7] = 0.5
    y, state = forward(f)
    nan = torch.isnan(y[0])
    assert nan[20:, 3].all() and nan[30:, 5].all() and nan[:, 7].all()
    keep = [k for k in range(64) if k not in (3, 5, 7)]
    assert not nan[:, keep].any() and not nan[:20, 3].any() and not nan[:30, 5].any()


def test_channels_and_sequences_are_alone(dev):
    """A NaN in one sequence and channel reaches no other, in gradients either."""
    f = rand(12, 2, 300, 130, torch.bfloat16, dev)
    clean = train(f)
    f["x"][0, 7, 100] = float("nan")
    dirty = train(f)
    for k in ("x", "a_gate", "x_gate", "z"):
        same = clean[2][k] == dirty[2][k]
        same[0, :, 100] = True
        assert same.all(), k
    assert torch.isnan(dirty[2]["A"][100]) and torch.equal(clean[2]["A"][:100], dirty[2]["A"][:100])


@pytest.mark.parametrize("shape", [(0, 5, 4), (2, 0, 4), (2, 5, 0)])
def test_empty(dev, shape):
    b, n, d = shape
    f = rand(13, b, n, d, torch.float16, dev, h0=True)
    y, state, got = train(f)
    assert y.shape == shape and torch.equal(state, f["h0"] if n == 0 else state) and state.shape == (b, d)
    assert got["A"].shape == (d,) and not got["A"].any()
    if n == 0:
        assert torch.equal(got["h0"], f["dstate"])
    y, state = gated_scan(f["x"], f["a_gate"], f["x_gate"], f["A"], return_state=True)
    assert not state.any()


def test_other_dtypes_of_rates_and_states(dev):
    f = rand(14, 2, 30, 64, torch.bfloat16, dev, h0=True)
    A, h0 = f["A"].double().requires_grad_(True), f["h0"].to(torch.bfloat16).requires_grad_(True)
    y = gated_scan(f["x"], f["a_gate"], f["x_gate"], A, h0=h0)
    dA, dh0 = torch.autograd.grad(y, [A, h0], f["dy"])
    assert dA.dtype == torch.float64 and dh0.dtype == torch.bfloat16
    f["h0"], f["z"] = h0.detach().float(), None
    want = case(f).backward(f["dy"])
    ref.close(dA, *want["A"], torch.float32, "dA")
    ref.close(dh0, *want["h0"], torch.bfloat16, "dh0")


def test_repeats_bit_for_bit(dev):
    f = rand(15, 2, 5000, 200, torch.bfloat16, dev, h0=True)
    first = train(f)
    for _ in range(3):
        again = train(f)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        assert all(torch.equal(first[2][k], again[2][k]) for k in first[2])


def test_long_sequence_carries_the_state(dev):
    """A state that decays by nothing (A tiny) travels 20000 tokens; one impulse at the start."""
    n, d = 20000, 64
    z = torch.zeros((1, n, d), device=dev)
    x = z.clone()
    x[0, 0] = 1.0
    A = torch.full((d,), -1e-6, device=dev)
    h0 = torch.ones((1, d), device=dev)
    y, state = gated_scan(x, z, z, A, h0=h0, return_state=True)
    c = ref.Case(x, z, z, A, None, h0)
    l = -0.5e-6
    want = torch.exp(l * torch.arange(1, n + 1, dtype=torch.float64)) \
        + 0.5 * math.sqrt(-math.expm1(2 * l)) * torch.exp(l * torch.arange(n, dtype=torch.float64))
    # a's rounding: at most u a token, and the product's u
    err = (y[0].cpu().double() - want[:, None]).abs()
    assert (err <= 3 * ref.U * torch.arange(1, n + 1)[:, None] + 1e-6).all()
    assert torch.equal(y[:, -1], state)


def test_second_stream_and_status(dev):
    """Calls on two streams at once, each with its own workspace; no wait gave up."""
    reset_scan_status(dev)
    fs = [rand(20 + k, 2, 4000, 300, torch.bfloat16, dev) for k in range(2)]
    want = [train(f) for f in fs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in fs]
    got = []
    for s, f in zip(streams, fs):
        with torch.cuda.stream(s):
            got.append(train(f))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert torch.equal(w[0], g[0]) and all(torch.equal(w[2][k], g[2][k]) for k in w[2])
    assert scan_status(dev) == 0


@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_graph(dev, checkpoint):
    """A captured training step, replayed on new inputs between eager calls."""
    f = rand(30, 2, 700, 130, torch.bfloat16, dev, h0=True)
    static = {k: v.clone() for k, v in f.items()}
    for k in LEAVES:
        static[k].requires_grad_(True)

    def step():
        y, state = forward(static, checkpoint=checkpoint)
        return (y, state, *torch.autograd.grad([y, state], [static[k] for k in LEAVES], [static["dy"], static["dstate"]]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (31, 32, 33):
        new = rand(seed, 2, 700, 130, torch.bfloat16, dev, h0=True)
        with torch.no_grad():
            for k, v in new.items():
                static[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        y, state, got = train(new, checkpoint=checkpoint)
        for a, b in zip(out, (y, state, *got.values())):
            assert torch.equal(a, b)


def test_two_graphs_share_nothing(dev):
    """Two captured passes replayed on two streams at once."""
    fs = [rand(40 + k, 1, 3000, 200, torch.float16, dev) for k in range(2)]
    want = [forward(f) for f in fs]
    graphs, outs = [], []
    for f in fs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(forward(f))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in fs]
    for _ in range(3):
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for w, o in zip(want, outs):
            assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])


def test_offsets_past_32_bits(dev):
    """More than 2^31 outputs; the inputs are one token broadcast over time, so h_t = b (1 - a^t) / (1 - a)."""
    n, d = 530_000, 4096
    g = torch.Generator().manual_seed(45)
    token = {k: torch.randn((1, 1, d), generator=g).to(torch.bfloat16).to(dev) for k in ("x", "a_gate", "x_gate")}
    leaves = {k: v.expand(1, n, d) for k, v in token.items()}
    A = (-0.1 - torch.rand(d, generator=g)).to(dev).requires_grad_(True)
    y, state = gated_scan(leaves["x"], leaves["a_gate"], leaves["x_gate"], A, return_state=True, checkpoint="int8")
    assert y.numel() > 2 ** 31
    c = ref.Case(*(t.expand(1, 400, d) for t in token.values()), A)
    wy, ey, wh, eh = c.forward()
    ref.close(y[:, :400], wy, ey, torch.bfloat16, "first tokens")
    r, i, l, a, beta, u, *_ = c.elements()
    assert (1 - a).min() > 0.009
    limit = (beta * u / (1 - a))[:, :1]
    # a token adds at most 10 u of error to a and the state, the state remembers 1 / (1 - a) < 112 of them, and b has
    # 25 u of its own: 1150 u < 1e-4; bf16 half a step, 2^-8
    assert ((state[:, None].cpu().double() - limit).abs() <= 1e-4 * limit.abs() + 1e-30).all()
    assert torch.equal(y[:, -1], state.to(torch.bfloat16))
    # gradient of the last token alone: 2000 tokens before it a^t < 2e-8 of it is left
    dy = torch.zeros((1, n, d), dtype=torch.bfloat16, device=dev)
    dy[:, -1] = 1.0
    dA, = torch.autograd.grad(y, A, dy)
    tail = ref.Case(*(t.expand(1, 2000, d) for t in token.values()), A, h0=limit[:, 0])
    want, bound = tail.backward(torch.cat([torch.zeros((1, 1999, d)), torch.ones((1, 1, d))], 1), eight=True)["A"]
    # the reference starts from the limit, the kernel from its state: 1e-4 of each token's part
    assert ((dA.cpu().double() - want).abs() <= bound + 2e-4 * want.abs()).all()


def test_expired_waits_end_the_call(dev):
    """A wait bound of a microsecond, from the C interface: the call ends, and says so where it gave up."""
    b, n, d = 2, 6000, 128
    f = rand(46, b, n, d, torch.float32, dev, z=False)
    want, _ = gated_scan(f["x"], f["a_gate"], f["x_gate"], f["A"], return_state=True)
    y, status = torch.empty_like(want), torch.zeros(1, dtype=torch.int32, device=dev)
    lib, p = _lib.load(), _lib.GatedScanParams()
    for k in ("x", "a_gate", "x_gate"):
        setattr(p, k, f[k].data_ptr())
        setattr(p, f"{k}_stride", (_lib._i64a2)(n * d, d))
    p.A, p.y, p.y_stride, p.status = f["A"].data_ptr(), y.data_ptr(), (_lib._i64a2)(n * d, d), status.data_ptr()
    p.batch, p.seqlen, p.dim, p.handoff_timeout_us = b, n, d, 1
    nbytes = lib.mm_gated_scan_workspace_size(b, n, d, 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    _lib.check(lib.mm_gated_scan_fwd(p, _lib.stream_of(dev)), "mm_gated_scan_fwd")
    torch.cuda.synchronize()
    assert status.item() in (0, _lib.SCAN_STATUS_HANDOFF_TIMEOUT)
    if status.item() == 0:
        assert torch.equal(y, want)
    # the next call is a good one again, in the same workspace
    p.handoff_timeout_us = 0
    status.zero_()
    _lib.check(lib.mm_gated_scan_fwd(p, _lib.stream_of(dev)), "mm_gated_scan_fwd")
    torch.cuda.synchronize()
    assert status.item() == 0 and torch.equal(y, want)


def test_many_rows_of_partial_sums(dev):
    """Enough tiles that dA's rows go through two passes."""
    f = rand(47, 40, 900, 10, torch.float32, dev)
    y, state, got = train(f)
    check_grads(case(f), f, got, torch.float32)


def test_no_second_derivative(dev):
    f = rand(48, 1, 20, 64, torch.float32, dev)
    x = f["x"].clone().requires_grad_(True)
    y = gated_scan(x, f["a_gate"], f["x_gate"], f["A"])
    dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_backward_twice_with_a_kept_graph(dev):
    f = rand(49, 2, 300, 70, torch.float16, dev)
    leaves = {k: f[k].clone().requires_grad_(True) for k in ("x", "a_gate", "x_gate", "A", "z")}
    y = gated_scan(leaves["x"], leaves["a_gate"], leaves["x_gate"], leaves["A"], z=leaves["z"], checkpoint="int8")
    first = torch.autograd.grad(y, list(leaves.values()), f["dy"], retain_graph=True)
    again = torch.autograd.grad(y, list(leaves.values()), f["dy"])
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_saved_inputs_are_guarded(dev):
    """An input changed between the passes is an error, as for any torch operator; codes do not care."""
    f = rand(50, 1, 20, 64, torch.float32, dev)
    for checkpoint in ("full", "int8"):
        x = f["x"].clone()
        a = f["a_gate"].clone().requires_grad_(True)
        y = gated_scan(x, a, f["x_gate"], f["A"], checkpoint=checkpoint)
        x.add_(1)
        if checkpoint == "full":
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                y.sum().backward()
        else:
            y.sum().backward()
            assert torch.isfinite(a.grad).all()


# ------------------------------------------------------------------------------ one token
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,d", [(1, 1), (1, 64), (3, 65), (64, 1000), (5, 1536)])
@pytest.mark.parametrize("z,inplace", [(False, True), (True, False)])
def test_step(dev, dtype, b, d, z, inplace):
    f = rand(60, b, 1, d, dtype, dev, z, h0=True)
    state = f["h0"].clone()
    out_state = None if inplace else torch.full_like(state, 7.0)
    y = gated_scan_step(state, f["x"][:, 0], f["a_gate"][:, 0], f["x_gate"][:, 0], f["A"],
                        z=None if f["z"] is None else f["z"][:, 0], state_out=out_state)
    check_forward(case(f), y[:, None], state if inplace else out_state, dtype)
    if not inplace:
        assert torch.equal(state, f["h0"])


def test_step_rows_of_a_projection(dev):
    """Slices of one wide projection of the token; out given; the neighbours stay."""
    b, d = 3, 70
    f = rand(61, b, 1, d, torch.float16, dev, h0=True)
    wide = torch.cat([f[k][:, 0] for k in ("x", "a_gate", "x_gate", "z")], 1)
    out = torch.full((b, 2 * d), 9.0, dtype=torch.float16, device=dev)
    parts = wide.split(d, 1)
    state = f["h0"].clone()
    gated_scan_step(state, parts[0], parts[1], parts[2], f["A"], z=parts[3], out=out[:, :d])
    check_forward(case(f), out[:, None, :d], state, torch.float16)
    assert (out[:, d:] == 9.0).all()


def test_prefill_then_steps(dev):
    """A prompt through gated_scan, then its continuation token by token: the scan over all of it."""
    b, n, m, d = 2, 37, 6, 130
    f = rand(62, b, n + m, d, torch.float32, dev)
    part = lambda lo, hi: {k: f[k][:, lo:hi] for k in ("x", "a_gate", "x_gate", "z")}
    p = part(0, n)
    y0, state = gated_scan(p["x"], p["a_gate"], p["x_gate"], f["A"], z=p["z"], return_state=True)
    ys = [y0]
    for t in range(n, n + m):
        p = {k: v[:, 0] for k, v in part(t, t + 1).items()}
        ys.append(gated_scan_step(state, p["x"], p["a_gate"], p["x_gate"], f["A"], z=p["z"])[:, None])
    check_forward(case(f), torch.cat(ys, 1), state, torch.float32)


# ------------------------------------------------------------------------------ the mixer
@pytest.mark.parametrize("checkpoint", ["full", "int8"])
def test_mixer_trains(dev, checkpoint):
    """conv -> gates -> recurrence -> projection, all parameters' gradients against the same layer in
    64 bits (with whole checkpoints; with 8-bit ones within what a half step of the codes may add)."""
    b, n, d = 2, 90, 48
    g = torch.Generator().manual_seed(70)
    t = lambda *s, std=1.0: torch.randn(s, generator=g) * std
    params = {"conv_w": t(d, 1, 4, std=0.5), "conv_b": t(d, std=0.1), "Wa": t(d, d, std=d ** -0.5),
              "Wx": t(d, d, std=d ** -0.5), "Wz": t(d, d, std=d ** -0.5), "A_log": t(d, std=0.5) - 2.0,
              "out": t(d, d, std=d ** -0.5)}
    u, dy = t(b, n, d), t(b, n, d)

    def layer(p, u, conv, scan):
        x = conv(u, p["conv_w"], p["conv_b"])
        return scan(x, x @ p["Wa"].t(), x @ p["Wx"].t(), -torch.exp(p["A_log"]), u @ p["Wz"].t()) @ p["out"].t()

    def conv64(x, w, b_):
        padded = torch.cat([x.new_zeros((b, 3, d)), x], 1)
        v = b_ + sum(padded[:, k:k + n] * w[:, 0, k] for k in range(4))
        return v * torch.sigmoid(v)

    def scan64(x, ag, xg, A, z):
        h, ys = torch.zeros((b, d), dtype=torch.float64), []
        la = A * torch.sigmoid(ag)
        bu = torch.sqrt(-torch.expm1(2 * la)) * torch.sigmoid(xg) * x
        for k in range(n):
            h = torch.exp(la[:, k]) * h + bu[:, k]
            ys.append(h)
        return torch.stack(ys, 1) * z * torch.sigmoid(z)

    p64 = {k: v.double().requires_grad_(True) for k, v in params.items()}
    y64 = layer(p64, u.double(), conv64, scan64)
    g64 = torch.autograd.grad(y64, list(p64.values()), dy.double())
    pd = {k: v.to(dev).requires_grad_(True) for k, v in params.items()}
    y = layer(pd, u.to(dev), lambda x, w, c: causal_conv1d_train(x, w, c, checkpoint=checkpoint),
              lambda x, ag, xg, A, z: gated_scan(x, ag, xg, A, z=z, checkpoint=checkpoint))
    gd = torch.autograd.grad(y, list(pd.values()), dy.to(dev))
    # float32 sums of up to 180 x 48 products through five stages: 1e-5 of the largest is 170 u
    assert (y.cpu().double() - y64).abs().max() <= 1e-5 * y64.abs().max()
    for k, a, w in zip(params, gd, g64):
        # codes are off by up to 1/128 of a block's largest magnitude, uniformly spread: 0.5% of a unit normal's
        # values, through at most five such factors
        tol = 1e-5 if checkpoint == "full" else 5 / 128
        assert (a.cpu().double() - w).norm() <= tol * w.norm(), k
