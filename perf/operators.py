"""The operators of a gated recurrent mixer: its recurrence over long sequences and token by token,
the 8-bit checkpoints that its backward pass can read, and the causal conv1d's backward pass.

Kinds of case:

  scan   ``gated_scan`` on (batch, seqlen, dim): a prompt's pass, output and final state.
  step   ``gated_scan_step``: one token per sequence, the new states in buffers of their own.
  train  ``gated_scan`` and its gradients.  ``checkpoint`` "int8" keeps the inputs for the backward
         pass as 8-bit codes; the gradients are then those at the values the codes stand for, with
         the states recomputed inside each block of 16 tokens from the state at its start.
  act8   ``act8_pack`` and ``act8_unpack``: an activation kept in 8 bits and taken back.
  conv   ``causal_conv1d_train`` and its gradients, the input kept whole or in 8 bits.

The recurrence, for each channel d:

  r = sigmoid(a_gate)   i = sigmoid(x_gate)   a = exp(A[d] r)
  h_t = a_t h_{t-1} + sqrt(1 - a_t^2) i_t x_t          y = h (silu(z) where there is a z)

An 8-bit block is 16 tokens of one channel (the last one of a sequence may be shorter): whole numbers
of at most 127 times a power of two, the smallest one that holds the block.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16


def listed():
    return [
        # A short prompt through one layer of a small model in full precision: one call's latency.
        dict(name="scan_f32_short", kind="scan", dtype="f32", batch=1, seqlen=200, dim=512, gated=True, ragged=False),
        # One long prompt at a large model's inner width: the latency of its first token.
        dict(name="scan_bf16_prompt", kind="scan", dtype="bf16", batch=1, seqlen=8192, dim=5120, gated=True, ragged=False),
        # Prompts of different lengths in one padded batch, on sizes that no tile divides.
        dict(name="scan_f16_ragged", kind="scan", dtype="f16", batch=7, seqlen=3001, dim=1000, gated=False, ragged=True),
        # One sequence decoding at a small model's inner width: the latency of a token.
        dict(name="step_f16_single", kind="step", dtype="f16", batch=1, dim=1536, gated=True),
        # A full serving batch decoding at a large model's inner width.
        dict(name="step_bf16_batch", kind="step", dtype="bf16", batch=64, dim=5120, gated=True),
        # A training step's share of one layer, the activations kept whole.
        dict(name="train_bf16", kind="train", dtype="bf16", batch=8, seqlen=2048, dim=5120, gated=True, ragged=False, checkpoint="full"),
        # Training in full precision on a padded batch of odd sizes.
        dict(name="train_f32_odd", kind="train", dtype="f32", batch=3, seqlen=1021, dim=1000, gated=False, ragged=True, checkpoint="full"),
        # The largest: long documents at a large model's inner width, the activations kept in 8 bits.
        dict(name="train8_bf16_long", kind="train", dtype="bf16", batch=4, seqlen=8192, dim=5120, gated=True, ragged=False, checkpoint="int8"),
        # A small model's layer with its activations in 8 bits, on an odd length.
        dict(name="train8_f16_odd", kind="train", dtype="f16", batch=2, seqlen=777, dim=1536, gated=False, ragged=False, checkpoint="int8"),
        # Any other activation of such a layer, kept in 8 bits until its backward pass.
        dict(name="act8_bf16", kind="act8", dtype="bf16", batch=8, seqlen=2048, dim=2560),
        # The conv before the recurrence, its input kept in 8 bits.
        dict(name="conv8_bf16", kind="conv", dtype="bf16", batch=8, seqlen=2048, dim=5120, width=4, checkpoint="int8"),
        # The conv in full precision on odd sizes.
        dict(name="conv_f32_odd", kind="conv", dtype="f32", batch=3, seqlen=777, dim=1001, width=3, checkpoint="full"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "step", "train", "train", "train", "act8", "conv", "conv"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    while True:
        case = dict(kind=kind, dtype=dtype, batch=_log_int(rng, 1, 64), dim=_log_int(rng, 64, 8192))
        # widths are multiples of a wave's lanes as often as they are odd
        if rng.random() < 0.5:
            case["dim"] = max(64, case["dim"] // 64 * 64)
        if kind != "step":
            case["seqlen"] = _log_int(rng, 17, 32768)
        if kind in ("scan", "step", "train"):
            case["gated"] = rng.random() < 0.5
        if kind in ("scan", "train"):
            case["ragged"] = rng.random() < 0.4
        if kind == "conv":
            case["width"] = rng.choice([4, 4, 4, 2, 3, 5])
        if kind in ("train", "conv"):
            case["checkpoint"] = rng.choice(["full", "int8"])
        elems = case["batch"] * case["dim"] * case.get("seqlen", 1)
        if elems <= (1 << 27) // (2 if dtype == "f32" else 1):
            return case


# ------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Values as a mixer's layer has them: the conv's inputs and outputs and the gates' projections of unit
    size, decay rates that forget over tens to thousands of tokens, gradients of unit size."""
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt, b, d = DTYPES[case["dtype"]], case["batch"], case["dim"]
    shape = (b, case["seqlen"], d) if "seqlen" in case else (b, d)

    def normal(size, dtype=dt, std=1.0, mean=0.0):
        return (torch.randn(size, generator=g, device=DEVICE) * std + mean).to(dtype)

    s = {"x": normal(shape)}
    if case["kind"] in ("scan", "step", "train"):
        s["a_gate"], s["x_gate"] = normal(shape), normal(shape)
        s["z"] = normal(shape) if case["gated"] else None
        s["A"] = -torch.exp(torch.rand((d,), generator=g, device=DEVICE) * math.log(1000.0) - math.log(1000.0))
        s["h0"] = normal((b, d), torch.float32) if case["kind"] == "step" else None
        s["lengths"] = None
        if case.get("ragged"):
            s["lengths"] = torch.randint(1, case["seqlen"] + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
            s["lengths"][0] = case["seqlen"]
            if b > 1:
                s["lengths"][1] = 0  # a slot of the batch that holds no sequence
    if case["kind"] == "conv":
        s["weight"] = normal((d, 1, case["width"]), std=case["width"] ** -0.5)
        s["bias"] = normal((d,), std=0.1)
    if case["kind"] in ("train", "conv"):
        s["dy"] = normal(shape)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["kind"], s["checkpoint"] = case["kind"], case.get("checkpoint")
    if case["kind"] == "step":
        s["state_out"] = torch.empty_like(s["h0"])
    if case["kind"] in ("train", "conv"):
        s["leaves"] = [k for k in ("x", "a_gate", "x_gate", "A", "z", "weight", "bias") if s.get(k) is not None]
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


def _run_own(s):
    from mamba_metal_amd import act8_pack, act8_unpack, causal_conv1d_train, gated_scan, gated_scan_step

    kind = s["kind"]
    if kind == "scan":
        with torch.no_grad():
            return gated_scan(s["x"], s["a_gate"], s["x_gate"], s["A"], z=s["z"], lengths=s["lengths"], return_state=True)
    if kind == "step":
        y = gated_scan_step(s["h0"], s["x"], s["a_gate"], s["x_gate"], s["A"], z=s["z"], state_out=s["state_out"])
        return y, s["state_out"]
    if kind == "act8":
        return act8_unpack(act8_pack(s["x"]))
    if kind == "train":
        y = gated_scan(s["x"], s["a_gate"], s["x_gate"], s["A"], z=s["z"], lengths=s["lengths"], checkpoint=s["checkpoint"])
    else:
        y = causal_conv1d_train(s["x"], s["weight"], s["bias"], checkpoint=s["checkpoint"])
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(s["leaves"], grads)}}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 with h_{-1} = 0, in log2(length) passes."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _valid(s):
    """(batch, seqlen, 1) truth values of the tokens within their sequence, or None."""
    if s["lengths"] is None:
        return None
    t = torch.arange(s["x"].shape[1], device=DEVICE)
    return (t[None, :] < s["lengths"][:, None])[..., None]


def _masked(t, valid):
    return t if valid is None else torch.where(valid, t, torch.zeros((), device=t.device, dtype=t.dtype))


def _gates(x, a_gate, x_gate, A, valid):
    r, i = torch.sigmoid(a_gate), torch.sigmoid(x_gate)
    log_a = A * r
    beta = torch.sqrt(-torch.expm1(2 * log_a))
    a = 1 + torch.expm1(log_a)  # exp's last-bit errors next to 1 lean one way and add up over a long memory
    if valid is not None:
        a = torch.where(valid, a, torch.ones((), device=DEVICE))
    return r, i, log_a, a, beta, _masked(i * x, valid)


def _eight_bits(x):
    """The values that x's 8-bit codes stand for (x in fp32, (batch, seqlen, dim))."""
    b, n, d = x.shape
    pad = -n % BLOCK
    blocks = torch.cat([x, x.new_zeros((b, pad, d))], 1).view(b, -1, BLOCK, d)
    bits = blocks.abs().amax(2, keepdim=True).view(torch.int32)
    # amax / scale lies in [63.75, 127.5): half a code's step added to the mantissa carries from 127.5 on
    exponent = torch.clamp(((bits + 0x10000) >> 23) - 6, min=1)
    scale = (exponent << 23).view(torch.float32)
    scale = torch.where(bits < 0x7F800000, scale, torch.full_like(scale, float("nan")))
    return (torch.round(blocks / scale) * scale).view(b, -1, d)[:, :n]


def _run_plain(s):
    kind, dt = s["kind"], s["x"].dtype
    f = {k: v.float() for k, v in s.items() if torch.is_tensor(v) and v.is_floating_point()}
    if kind == "act8":
        return _eight_bits(f["x"]).to(dt)
    if kind == "conv":
        return _conv_plain(s, f, dt)
    if kind == "step":
        r, i, log_a, a, beta, u = _gates(f["x"], f["a_gate"], f["x_gate"], f["A"], None)
        h = a * f["h0"] + beta * u
        y = h if s["z"] is None else h * f["z"] * torch.sigmoid(f["z"])
        return y.to(dt), h
    valid = _valid(s)
    r, i, log_a, a, beta, u = _gates(f["x"], f["a_gate"], f["x_gate"], f["A"], valid)
    h = _doubling(a, beta * u if valid is None else torch.where(valid, beta * u, torch.zeros((), device=DEVICE)))
    z = _masked(f["z"], valid) if s["z"] is not None else None
    y = _masked(h if z is None else h * z * torch.sigmoid(z), valid).to(dt)
    if kind == "scan":
        return y, h[:, -1].contiguous()
    # backward
    x = f["x"]
    if s["checkpoint"] == "int8":
        n = x.shape[1]
        starts = torch.cat([torch.zeros_like(h[:, :1]), h[:, BLOCK - 1:n - 1:BLOCK]], 1)  # each block's first state
        x, ag, xg = (_eight_bits(_masked(f[k], valid)) for k in ("x", "a_gate", "x_gate"))
        z = _eight_bits(z) if z is not None else None
        r, i, log_a, a, beta, u = _gates(x, ag, xg, f["A"], valid)
        bu = _masked(beta * u, valid)
        pad = -n % BLOCK
        if pad:
            a_p = torch.cat([a, a.new_ones((a.shape[0], pad, a.shape[2]))], 1)
            b_p = torch.cat([bu, bu.new_zeros((a.shape[0], pad, a.shape[2]))], 1)
        else:
            a_p, b_p = a, bu.clone()
        rows = a_p.shape[0] * (a_p.shape[1] // BLOCK)
        a_p, b_p = a_p.view(rows, BLOCK, -1), b_p.view(rows, BLOCK, -1)
        b_p[:, 0] += a_p[:, 0] * starts.reshape(rows, -1)
        h = _doubling(a_p, b_p).view(h.shape[0], -1, h.shape[2])
        h_prev = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
        h_prev[:, ::BLOCK] = starts
        h, h_prev = h[:, :n], h_prev[:, :n]
    else:
        h_prev = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    dy = _masked(f["dy"], valid)
    out = {"y": y}
    if z is not None:
        sz = torch.sigmoid(z)
        dz = _masked(dy * h * sz * (1 + z * (1 - sz)), valid)
        dy = dy * z * sz
    a_next = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    dh = _doubling(a_next.flip(1), dy.flip(1)).flip(1)
    du = _masked(beta * dh, valid)
    ratio = torch.where(beta > 0, a * a / beta, torch.zeros_like(beta))
    dlog = _masked(dh * (h_prev * a - u * ratio), valid)
    out["dx"] = (i * du).to(dt)
    out["da_gate"] = (dlog * log_a * (1 - r)).to(dt)
    out["dx_gate"] = (du * u * (1 - i)).to(dt)
    out["dA"] = (dlog * r).sum((0, 1), dtype=torch.float64).float()
    if z is not None:
        out["dz"] = dz.to(dt)
    return out


def _shifted(t, k):
    """t moved k tokens later (earlier where k < 0), zeros where there is none."""
    if k == 0:
        return t
    zeros = t.new_zeros((t.shape[0], min(abs(k), t.shape[1]), t.shape[2]))
    return torch.cat([zeros, t[:, :-k]], 1)[:, :t.shape[1]] if k > 0 else torch.cat([t[:, -k:], zeros], 1)[:, :t.shape[1]]


def _conv_plain(s, f, dt):
    w = f["weight"][:, 0]
    width = w.shape[1]

    def pre(x):
        p = f["bias"].expand_as(x)
        for k in range(width):
            p = p + w[:, k] * _shifted(x, width - 1 - k)
        return p

    p = pre(f["x"])
    y = (p * torch.sigmoid(p)).to(dt)
    x = f["x"]
    if s["checkpoint"] == "int8":
        x = _eight_bits(x)
        p = pre(x)
    sp = torch.sigmoid(p)
    dp = f["dy"] * sp * (1 + p * (1 - sp))
    dx = torch.zeros_like(x)
    dw = torch.empty_like(w)
    for k in range(width):
        dx += w[:, k] * _shifted(dp, -(width - 1 - k))
        dw[:, k] = (dp * _shifted(x, width - 1 - k)).sum((0, 1), dtype=torch.float64)
    return {"y": y, "dx": dx.to(dt), "dweight": dw[:, None].to(dt), "dbias": dp.sum((0, 1), dtype=torch.float64).to(dt)}


# ------------------------------------------------------------------------------ in 64 bits
@torch.no_grad()
def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "act8":
        return _exact_eight(s["x"])
    if kind == "conv":
        return _exact_conv(s, case)
    if kind == "step":
        a = torch.exp(s["A"] / (1 + torch.exp(-s["a_gate"])))
        h = a * s["h0"] + torch.sqrt((1 - a) * (1 + a)) * s["x"] / (1 + torch.exp(-s["x_gate"]))
        return (h if s["z"] is None else h * s["z"] / (1 + torch.exp(-s["z"]))), h
    b, n, d = s["x"].shape
    ends = torch.full((b,), n, device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    live = [(ends > t)[:, None] for t in range(n)]

    def token(v, t):
        r, i = 1 / (1 + torch.exp(-v["a_gate"][:, t])), 1 / (1 + torch.exp(-v["x_gate"][:, t]))
        la = s["A"] * r
        return r, i, la, torch.exp(la), torch.sqrt(-torch.expm1(2 * la))

    def forward(v, t, h):
        r, i, la, a, beta = token(v, t)
        return torch.where(live[t], a * h + beta * i * v["x"][:, t], h)

    h, y, before = torch.zeros((b, d), device=DEVICE, dtype=torch.float64), torch.zeros_like(s["x"]), []
    for t in range(n):
        if kind == "train" and (case["checkpoint"] == "full" or t % BLOCK == 0):
            before.append(h)
        h = forward(s, t, h)
        gate = 1 if s["z"] is None else s["z"][:, t] / (1 + torch.exp(-s["z"][:, t]))
        y[:, t] = torch.where(live[t], h * gate, torch.zeros_like(h))
    if kind == "scan":
        return y, h
    v = s
    if case["checkpoint"] == "int8":
        keep = torch.stack(live, 1)
        v = dict(s)
        for k in ("x", "a_gate", "x_gate", "z"):
            if s[k] is not None:
                v[k] = _exact_eight(torch.where(keep, s[k], torch.zeros((), device=DEVICE, dtype=torch.float64)))
        starts, before = before, []
        for t in range(n):
            before.append(starts[t // BLOCK] if t % BLOCK == 0 else forward(v, t - 1, before[-1]))
    grads = {k: torch.zeros_like(s["x"]) for k in ("dx", "da_gate", "dx_gate", "dz")}
    dA, carry = torch.zeros((d,), device=DEVICE, dtype=torch.float64), torch.zeros((b, d), device=DEVICE, dtype=torch.float64)
    none = torch.zeros_like(carry)
    for t in range(n - 1, -1, -1):
        r, i, la, a, beta = token(v, t)
        dy = torch.where(live[t], s["dy"][:, t], none)
        if s["z"] is not None:
            q = 1 / (1 + torch.exp(-v["z"][:, t]))
            ht = a * before[t] + beta * i * v["x"][:, t]
            grads["dz"][:, t] = dy * ht * (q + v["z"][:, t] * q * (1 - q))
            dy = dy * v["z"][:, t] * q
        dh = dy + carry
        dbeta = dh * i * v["x"][:, t]
        dl = dh * before[t] * a - torch.where(beta > 0, dbeta * a * a / beta, none)
        dl = torch.where(live[t], dl, none)
        grads["dx"][:, t] = torch.where(live[t], dh * beta * i, none)
        grads["dx_gate"][:, t] = torch.where(live[t], dh * beta * v["x"][:, t] * i * (1 - i), none)
        grads["da_gate"][:, t] = dl * s["A"] * r * (1 - r)
        dA += (dl * r).sum(0)
        carry = torch.where(live[t], a * dh, carry)
    out = {"y": y, "dx": grads["dx"], "da_gate": grads["da_gate"], "dx_gate": grads["dx_gate"], "dA": dA}
    if s["z"] is not None:
        out["dz"] = grads["dz"]
    return out


def _exact_eight(x):
    out = torch.empty_like(x)
    for t in range(0, x.shape[1], BLOCK):
        part = x[:, t:t + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        _, k = torch.frexp(top)                       # top = m 2^k with m in [1/2, 1)
        scale = ((torch.clamp(k.long() - 7, min=-126) + 1023) << 52).view(torch.float64)  # exactly 2^(k - 7)
        scale = torch.where(top >= 127.5 * scale, 2 * scale, scale)
        scale = torch.where(top > 0, scale, torch.ones_like(scale))
        out[:, t:t + BLOCK] = torch.round(part / scale) * scale
    return out


def _exact_conv(s, case):
    import torch.nn.functional as F

    w, K = s["weight"][:, 0], case["width"]

    def pre(x):
        padded = F.pad(x, (0, 0, K - 1, 0))
        return s["bias"] + sum(padded[:, k:k + x.shape[1]] * w[:, k] for k in range(K)), padded

    p, _ = pre(s["x"])
    y = p / (1 + torch.exp(-p))
    n = s["x"].shape[1]
    p, padded = pre(s["x"] if case["checkpoint"] == "full" else _exact_eight(s["x"]))
    q = 1 / (1 + torch.exp(-p))
    dp = s["dy"] * (q + p * q * (1 - q))
    after = F.pad(dp, (0, 0, 0, K - 1))
    dx = sum(after[:, K - 1 - k:K - 1 - k + n] * w[:, k] for k in range(K))
    dw = torch.stack([(dp * padded[:, k:k + n]).sum((0, 1)) for k in range(K)], 1)
    return {"y": y, "dx": dx, "dweight": dw[:, None], "dbias": dp.sum((0, 1))}


# ------------------------------------------------------------------------------ what it takes
def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    kind, b, d = case["kind"], case["batch"], case["dim"]
    n = b * d * case.get("seqlen", 1)
    eight = b * d * (case.get("seqlen", 1) + -(-case.get("seqlen", 1) // BLOCK))  # codes and exponents
    inputs = 4 if case.get("gated") else 3
    if kind == "scan":
        # two sigmoids of 4, the decay, its root and the update 8, the gate 6
        return {"bytes": n * es * (inputs + 1) + b * d * 4 + d * 4, "flops": n * (16 + 6 * case["gated"])}
    if kind == "step":
        return {"bytes": n * (es * (inputs + 1) + 8) + d * 4, "flops": n * (16 + 6 * case["gated"])}
    if kind == "act8":
        return {"bytes": 2 * n * es + 2 * eight, "flops": 4 * n}
    if kind == "train":
        # forward: the inputs and the output; backward: the inputs again, the output's gradient, the inputs' gradients
        kept = inputs * n * es if case["checkpoint"] == "full" else 2 * inputs * eight
        return {"bytes": n * es * (2 * inputs + 2) + kept + 8 * d, "flops": n * (50 + 20 * case["gated"])}
    w = case["width"]
    kept = n * es if case["checkpoint"] == "full" else 2 * eight
    return {"bytes": n * es * 4 + kept + 2 * d * (w + 1) * es, "flops": n * (8 * w + 20)}
