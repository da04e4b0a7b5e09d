"""The operators at the two ends of a language model, and a mixer whose heads decay.

Kinds of case:

  attn   ``decay_attention`` on (batch, seqlen, heads): a prompt's pass, output and final state.
  step   ``decay_attention_step``: one token per sequence, the new states in buffers of their own.
  train  ``decay_attention`` and its gradients.
  loss   ``linear_cross_entropy``: an evaluation's loss of every row, without a gradient.
  head   ``linear_cross_entropy`` and its gradients.
  embed  ``embedding`` and its gradient.

Linear attention with a decay for each head, q and k shared by neighbouring heads (groups of them):

  S_t = exp(g_t) S_{t-1} + k_t v_t^T          o_t = scale S_t^T q_t

The loss of a row x with target t, over a vocabulary of rows of W:

  l = W x          loss = log sum_v exp(l_v) - l_t          (0 where the target is the ignored one)

The embedding: y_i = scale W[id_i], without a gradient for the padding's id.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100
RUN = 64  # tokens that the plain form takes at a time


def listed():
    return [
        # A short prompt through a small layer in full precision: one call's latency.
        dict(name="attn_f32_short", kind="attn", dtype="f32", batch=1, seqlen=200, heads=8, groups=8, dk=64, dv=64, ragged=False, fixed=False),
        # One long prompt at a large model's inner width, q and k shared by all heads: the latency of its first token.
        dict(name="attn_bf16_prompt", kind="attn", dtype="bf16", batch=1, seqlen=8192, heads=80, groups=1, dk=128, dv=64, ragged=False, fixed=False),
        # Prompts of different lengths in one padded batch, every head with its own q and k and a constant decay.
        dict(name="attn_f16_ragged", kind="attn", dtype="f16", batch=7, seqlen=1501, heads=12, groups=12, dk=96, dv=96, ragged=True, fixed=True),
        # One sequence decoding at a small model's inner width: the latency of a token.
        dict(name="step_f16_single", kind="step", dtype="f16", batch=1, heads=24, groups=1, dk=128, dv=64, fixed=False),
        # A full serving batch decoding at a large model's inner width.
        dict(name="step_bf16_batch", kind="step", dtype="bf16", batch=64, heads=80, groups=1, dk=128, dv=64, fixed=False),
        # A training step's share of one layer of a large model.
        dict(name="train_bf16", kind="train", dtype="bf16", batch=8, seqlen=2048, heads=80, groups=1, dk=128, dv=64, ragged=False, fixed=False),
        # Training in full precision on a padded batch of odd sizes.
        dict(name="train_f32_odd", kind="train", dtype="f32", batch=3, seqlen=777, heads=6, groups=2, dk=48, dv=80, ragged=True, fixed=False),
        # A long text scored under a small model.
        dict(name="loss_bf16_eval", kind="loss", dtype="bf16", rows=2048, dim=768, vocab=50280),
        # The largest: the head of a large model in a training step.
        dict(name="head_bf16", kind="head", dtype="bf16", rows=8192, dim=2560, vocab=50280, reduction="mean"),
        # The head in full precision on sizes that no tile divides, a weight of its own for every row's loss.
        dict(name="head_f32_odd", kind="head", dtype="f32", rows=999, dim=1001, vocab=10007, reduction="none"),
        # The tokens of that training step, as often as they occur in text.
        dict(name="embed_bf16", kind="embed", dtype="bf16", rows=16384, dim=2560, vocab=50280, padded=False),
        # A padded batch of a small model in full precision.
        dict(name="embed_f32_odd", kind="embed", dtype="f32", rows=1777, dim=1001, vocab=5003, padded=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "step", "train", "train", "loss", "head", "head", "embed"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    while True:
        case = dict(kind=kind, dtype=dtype)
        if kind in ("attn", "step", "train"):
            per = rng.choice([1, 1, 2, 4, 8])
            case.update(batch=_log_int(rng, 1, 64), groups=_log_int(rng, 1, 32), fixed=rng.random() < 0.3)
            case["heads"] = case["groups"] * (per if rng.random() < 0.7 else _log_int(rng, 1, 80))
            for k in ("dk", "dv"):
                case[k] = rng.choice([64, 128, 64, 128, 16, 32, 96, rng.randint(5, 128)])
            if kind != "step":
                case.update(seqlen=_log_int(rng, 1, 32768), ragged=rng.random() < 0.4)
            tokens = case["batch"] * case["heads"] * case.get("seqlen", 1)
            states = case["batch"] * case["heads"] * -(-case.get("seqlen", 1) // RUN)
            cost = tokens * (case["dk"] + case["dv"]) + states * case["dk"] * case["dv"]
            if cost <= (1 << 28) // (2 if dtype == "f32" else 1) and tokens <= 1 << 21 and case["heads"] <= 128:
                return case
        else:
            case.update(rows=_log_int(rng, 1, 32768), dim=_log_int(rng, 64, 8192), vocab=_log_int(rng, 500, 160000))
            # widths are multiples of a wave's lanes as often as they are odd
            if rng.random() < 0.6:
                case["dim"] = max(64, case["dim"] // 64 * 64)
            if kind == "head":
                case["reduction"] = rng.choice(["mean", "mean", "sum", "none"])
            if kind == "embed":
                case["padded"] = rng.random() < 0.3
                if (case["rows"] + case["vocab"]) * case["dim"] <= 1 << 28:
                    return case
            elif case["rows"] * case["dim"] * case["vocab"] <= (1 << 40) // (4 if dtype == "f32" else 1) \
                    and case["rows"] * case["vocab"] <= 1 << 29 and case["vocab"] * case["dim"] <= 1 << 28:
                return case


# ------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """Values as a model has them: projections of unit size (keys scaled as after a norm), decays that forget over a
    few to thousands of tokens, logits of a few units, tokens by Zipf's law, one target in ten ignored."""
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(size, std=1.0, dtype=dt):
        return (torch.randn(size, generator=g, device=DEVICE) * std).to(dtype)

    def zipf(n, vocab):
        u = torch.rand((n,), generator=g, device=DEVICE, dtype=torch.float64)
        return torch.clamp(torch.exp(u * math.log(vocab + 1)).long() - 1, 0, vocab - 1)

    s = {}
    if case["kind"] in ("attn", "step", "train"):
        b, h, gr, dk, dv = (case[k] for k in ("batch", "heads", "groups", "dk", "dv"))
        lead = (b, case["seqlen"]) if "seqlen" in case else (b,)
        s["q"], s["k"], s["v"] = normal((*lead, gr, dk)), normal((*lead, gr, dk), dk ** -0.5), normal((*lead, h, dv))
        rate = torch.exp(torch.rand((h,), generator=g, device=DEVICE) * math.log(2000.0) - math.log(4000.0))
        if case["fixed"]:  # constants of the layer
            s["decay"] = -rate
        else:  # a projection of the token: a step width, as softplus of a unit normal gives it
            s["g"] = (-rate * torch.log1p(torch.exp(torch.randn((*lead, h), generator=g, device=DEVICE)))).to(dt)
        s["scale"] = 1.0
        s["h0"] = normal((b, h, dk, dv), 1.0, torch.float32) if case["kind"] == "step" else None
        s["lengths"] = None
        if case.get("ragged"):
            s["lengths"] = torch.randint(1, case["seqlen"] + 1, (b,), generator=g, device=DEVICE, dtype=torch.int32)
            s["lengths"][0] = case["seqlen"]
            if b > 1:
                s["lengths"][1] = 0  # a slot of the batch that holds no sequence
        if case["kind"] == "train":
            s["dy"] = normal((*lead, h, dv))
        return s
    rows, dim, vocab = case["rows"], case["dim"], case["vocab"]
    if case["kind"] == "embed":
        s["ids"] = zipf(rows, vocab)
        s["padding"] = 0 if case["padded"] else None
        if case["padded"]:
            s["ids"][rows - rows // 4:] = 0
        s["weight"], s["scale"] = normal((vocab, dim), 0.02), math.sqrt(dim)
        s["dy"] = normal((rows, dim))
        return s
    s["x"], s["weight"] = normal((rows, dim)), normal((vocab, dim), 2.0 * dim ** -0.5)
    s["targets"] = zipf(rows, vocab)
    s["targets"][torch.rand((rows,), generator=g, device=DEVICE) < 0.1] = IGNORE
    s["targets"][0] = vocab - 1  # one row at least counts
    s["reduction"] = case.get("reduction", "none")
    if case["kind"] == "head":
        # what float16 training scales its loss by, so that its gradients stay in range
        up = 1024.0 if case["dtype"] == "f16" else 1.0
        if s["reduction"] == "none":
            s["dy"] = torch.rand((rows,), generator=g, device=DEVICE) * (2 * up / rows)
        else:
            s["dy"] = torch.tensor(up if s["reduction"] == "mean" else up / rows, device=DEVICE)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["kind"] = case["kind"]
    if case["kind"] == "step":
        s["state_out"] = torch.empty_like(s["h0"])
    if case["kind"] in ("train", "head", "embed"):
        s["leaves"] = [k for k in ("q", "k", "v", "g", "x", "weight") if s.get(k) is not None]
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
    from mamba_metal_amd import decay_attention, decay_attention_step, embedding, linear_cross_entropy

    kind, g = s["kind"], s.get("g", s.get("decay"))
    if kind == "attn":
        with torch.no_grad():
            return decay_attention(s["q"], s["k"], s["v"], g, scale=s["scale"], lengths=s["lengths"], return_state=True)
    if kind == "step":
        y = decay_attention_step(s["h0"], s["q"], s["k"], s["v"], g, scale=s["scale"], state_out=s["state_out"])
        return y, s["state_out"]
    if kind == "loss":
        with torch.no_grad():
            return linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORE, reduction="none")
    if kind == "train":
        y = decay_attention(s["q"], s["k"], s["v"], g, scale=s["scale"], lengths=s["lengths"])
    elif kind == "head":
        y = linear_cross_entropy(s["x"], s["weight"], s["targets"], ignore_index=IGNORE, reduction=s["reduction"])
    else:
        y = embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["padding"])
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(s["leaves"], grads)}}


def _run_plain(s):
    kind = s["kind"]
    if kind == "embed":
        return _embed_plain(s)
    if kind in ("loss", "head"):
        return _head_plain(s)
    if kind == "step":
        per = s["v"].shape[1] // s["q"].shape[1]
        q, k = (s[n].float().repeat_interleave(per, 1) for n in ("q", "k"))
        h = torch.exp(s.get("g", s.get("decay")).float())[..., None, None] * s["h0"] + k[..., None] * s["v"].float()[..., None, :]
        return (s["scale"] * (q[..., None] * h).sum(2)).to(s["v"].dtype), h
    return _attention_plain(s)


def _attention_plain(s):
    """Runs of tokens: a product with a decay mask within a run, the state from one run to the next."""
    dt, dev = s["v"].dtype, s["v"].device
    b, n, heads, dv = s["v"].shape
    groups, dk = s["q"].shape[2:]
    per, runs = heads // groups, -(-n // RUN)
    live = torch.ones((b, n), dtype=torch.bool, device=dev)
    if s["lengths"] is not None:
        live = torch.arange(n, device=dev)[None] < s["lengths"][:, None]

    def laid_out(t):  # (batch, n, heads, d) -> (batch, heads, runs, RUN, d), zeros behind a sequence
        t = torch.where(live[..., None, None], t.float(), torch.zeros((), device=dev))
        if t.shape[2] != heads:
            t = t.repeat_interleave(per, 2)
        t = torch.cat([t, t.new_zeros((b, runs * RUN - n, *t.shape[2:]))], 1)
        return t.view(b, runs, RUN, heads, -1).permute(0, 3, 1, 2, 4).contiguous()

    def back(t):  # the other way
        return t.permute(0, 2, 3, 1, 4).reshape(b, runs * RUN, heads, -1)[:, :n]

    q, k, v = laid_out(s["q"]), laid_out(s["k"]), laid_out(s["v"])
    g = laid_out(s.get("g", s.get("decay")).expand(b, n, heads)[..., None])[..., 0]
    c = torch.cumsum(g.double(), 3)                                           # differences of long sums
    causal = torch.ones((RUN, RUN), dtype=torch.bool, device=dev).tril()
    decay = torch.where(causal, torch.exp(c[..., :, None] - c[..., None, :]), torch.zeros((), device=dev, dtype=torch.float64)).float()
    into, onward, whole = torch.exp(c).float()[..., None], torch.exp(c[..., -1:] - c).float()[..., None], torch.exp(c[..., -1]).float()
    scale = s["scale"]
    add = (k * onward).transpose(3, 4) @ v
    state, before = torch.zeros((b, heads, dk, dv), device=dev), []
    for r in range(runs):
        before.append(state)
        state = whole[:, :, r, None, None] * state + add[:, :, r]
    before = torch.stack(before, 2)
    p = (q @ k.transpose(3, 4)) * decay
    y = back(scale * (p @ v + into * (q @ before))).to(dt)
    if s["kind"] == "attn":
        return y, state
    do = laid_out(s["dy"]) * scale
    add = (q * into).transpose(3, 4) @ do
    dstate, after = torch.zeros_like(state), [None] * runs
    for r in range(runs - 1, -1, -1):
        after[r] = dstate
        dstate = whole[:, :, r, None, None] * dstate + add[:, :, r]
    after = torch.stack(after, 2)
    dp = (do @ v.transpose(3, 4)) * decay
    from_before, to_after = into * (do @ before.transpose(3, 4)), onward * (v @ after.transpose(3, 4))
    dq, dk_ = dp @ k + from_before, dp.transpose(3, 4) @ q + to_after
    dv_ = p.transpose(3, 4) @ do + onward * (k @ after)

    def summed(t):
        return back(t).reshape(b, n, groups, per, dk).sum(3).to(dt)

    out = {"y": y, "dq": summed(dq), "dk": summed(dk_), "dv": back(dv_).to(dt)}
    if "g" not in s:
        return out
    # a decay at t scales what tokens from t on take from tokens before t, inside the run and across its ends
    m = (dp * (q @ k.transpose(3, 4))).double()
    inside = (m.sum(4) - m.sum(3)).flip(3).cumsum(3).flip(3)
    later = (q * from_before).sum(4, dtype=torch.float64).flip(3).cumsum(3).flip(3)
    kv = (k * to_after).sum(4, dtype=torch.float64)
    dg = inside + later + (kv.cumsum(3) - kv) + (whole * (before * after).sum((3, 4), dtype=torch.float64))[..., None]
    dg = torch.where(live[..., None], back(dg[..., None])[..., 0], torch.zeros((), device=dev, dtype=torch.float64))
    out["dg"] = dg.to(dt)
    return out


def _head_plain(s):
    x, w, t = s["x"].float(), s["weight"].float(), s["targets"]
    counts = t != IGNORE
    at = torch.where(counts, t, torch.zeros_like(t))[:, None]
    logits = x @ w.t()
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(1, keepdim=True)
    loss = torch.where(counts, (torch.log(total) + top - logits.gather(1, at))[:, 0], torch.zeros((), device=x.device))
    if s["kind"] == "loss":
        return loss
    share = counts.float()
    if s["reduction"] == "mean":
        share = share / counts.sum()
    y = loss if s["reduction"] == "none" else (loss.double() * share).sum().float()
    dl = e.div_(total)
    dl.scatter_add_(1, at, torch.full_like(total, -1.0))
    dl.mul_((s["dy"] * share)[:, None])
    return {"y": y, "dx": (dl @ w).to(s["x"].dtype), "dweight": (dl.t() @ x).to(s["weight"].dtype)}


def _embed_plain(s):
    w = s["weight"]
    y = (w[s["ids"]].float() * s["scale"]).to(w.dtype)
    dy = s["dy"].float() * s["scale"]
    if s["padding"] is not None:
        dy = torch.where((s["ids"] == s["padding"])[:, None], torch.zeros((), device=dy.device), dy)
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, s["ids"], dy)
    return {"y": y, "dweight": dw.to(w.dtype)}


# ------------------------------------------------------------------------------ in 64 bits
@torch.no_grad()
def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in _inputs(case, seed).items()}
    kind = case["kind"]
    if kind == "embed":
        return _exact_embed(s)
    if kind in ("loss", "head"):
        return _exact_head(s, case)
    per = case["heads"] // case["groups"]
    if kind == "step":
        q, k = s["q"].repeat_interleave(per, 1), s["k"].repeat_interleave(per, 1)
        h = s["h0"] * torch.exp(s.get("g", s.get("decay")))[..., None, None] + torch.einsum("bhk,bhv->bhkv", k, s["v"])
        return torch.einsum("bhk,bhkv->bhv", q, h) * s["scale"], h
    b, n, heads, dv = s["v"].shape
    dk, groups, scale = case["dk"], case["groups"], s["scale"]
    ends = torch.full((b,), n, device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    g = s.get("g", s.get("decay")).expand(b, n, heads)
    y, dq = torch.zeros_like(s["v"]), torch.zeros((b, n, heads, dk), device=DEVICE, dtype=torch.float64)
    h = torch.zeros((b, heads, dk, dv), device=DEVICE, dtype=torch.float64)

    def token(t):
        on = (ends > t)[:, None, None]
        q, k = s["q"][:, t].repeat_interleave(per, 1), s["k"][:, t].repeat_interleave(per, 1)
        a = torch.where(on[..., 0], torch.exp(g[:, t]), torch.ones((), device=DEVICE, dtype=torch.float64))
        return on, q * on, k * on, a[..., None, None]

    for t in range(n):
        on, q, k, a = token(t)
        h = torch.addcmul(h.mul_(a), k[..., None], s["v"][:, t, :, None])
        y[:, t] = scale * (q[:, :, None] @ h)[:, :, 0]
        if kind == "train":
            dq[:, t] = scale * on * (h @ s["dy"][:, t, :, :, None])[..., 0]
    if kind == "attn":
        return y, h
    dk_, dv_ = torch.zeros_like(dq), torch.zeros_like(y)
    dh, dg = torch.zeros_like(h), torch.zeros_like(y[..., 0])
    carry = torch.zeros_like(dg[:, 0])
    for t in range(n - 1, -1, -1):
        on, q, k, a = token(t)
        dh = torch.addcmul(dh, q[..., None], scale * s["dy"][:, t, :, None])
        dk_[:, t] = on * (dh @ s["v"][:, t, :, :, None])[..., 0]
        dv_[:, t] = (k[:, :, None] @ dh)[:, :, 0]
        # the decays' running sum c enters o_t as exp(c_t) and key t as exp(-c_t); dg is the sum of dc from t on
        carry = carry + (q * dq[:, t]).sum(2) - (k * dk_[:, t]).sum(2)
        dg[:, t] = carry * on[..., 0]
        dh = dh.mul_(a)
    shared = lambda t: t.view(b, n, groups, per, dk).sum(3)
    out = {"y": y, "dq": shared(dq), "dk": shared(dk_), "dv": dv_}
    return {**out, "dg": dg} if "g" in s else out


def _exact_embed(s):
    """Tokens in order and running sums: the difference at a token's ends is its sum."""
    w, dy = torch.zeros_like(s["weight"]), s["dy"] * s["scale"]
    if s["padding"] is not None:
        dy[s["ids"] == s["padding"]] = 0
    order = torch.sort(s["ids"], stable=True)
    ends = torch.searchsorted(order.values, torch.arange(w.shape[0] + 1, device=DEVICE))
    for c in range(0, w.shape[1], 512):
        run = torch.cumsum(dy[:, c:c + 512][order.indices], 0)
        run = torch.cat([torch.zeros_like(run[:1]), run])
        w[:, c:c + 512] = run[ends[1:]] - run[ends[:-1]]
    return {"y": s["weight"][s["ids"]] * s["scale"], "dweight": w}


def _exact_head(s, case):
    rows = case["rows"]
    counts = s["targets"] != IGNORE
    loss, dx, dw = torch.zeros((rows,), device=DEVICE, dtype=torch.float64), torch.zeros_like(s["x"]), torch.zeros_like(s["weight"])
    weight = counts.double() * (s["dy"] if case["kind"] == "head" else 1.0)
    if s["reduction"] == "mean":
        weight = weight / counts.sum()
    some = max(1, (1 << 27) // case["vocab"])
    for r in range(0, rows, some):
        part, on = slice(r, r + some), counts[r:r + some]
        logits = s["x"][part] @ s["weight"].t()
        lse = torch.logsumexp(logits, 1)
        t = torch.where(on, s["targets"][part], 0)
        at = torch.arange(t.shape[0], device=DEVICE)
        loss[part] = torch.where(on, lse - logits[at, t], 0.0)
        if case["kind"] == "head":
            dl = torch.exp(logits - lse[:, None])
            dl[at, t] -= 1
            dl *= weight[part, None]
            dx[part] = dl @ s["weight"]
            dw += dl.t() @ s["x"][part]
    if case["kind"] == "loss":
        return loss
    y = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / counts.sum()}[s["reduction"]]
    return {"y": y, "dx": dx, "dweight": dw}


# ------------------------------------------------------------------------------ what it takes
def work(case):
    es, kind = 4 if case["dtype"] == "f32" else 2, case["kind"]
    if kind in ("attn", "step", "train"):
        tokens = case["batch"] * case.get("seqlen", 1)
        h, gr, dk, dv = (case[k] for k in ("heads", "groups", "dk", "dv"))
        state = case["batch"] * h * dk * dv
        qk, v, g = tokens * gr * dk * es, tokens * h * dv * es, h * 4 if case["fixed"] else tokens * h * es
        once = tokens * h * dk * dv  # a state's elements, once a token: decayed and added to, then read
        if kind == "train":
            # forward: q, k, v and the output; backward: the inputs again, the output's gradient, the inputs' gradients
            return {"bytes": 6 * qk + 5 * v + 3 * g, "flops": 17 * once}
        return {"bytes": 2 * qk + 2 * v + g + state * (8 if kind == "step" else 4), "flops": 5 * once}
    rows, dim, vocab = case["rows"], case["dim"], case["vocab"]
    if kind == "embed":
        used = min(rows, vocab)
        return {"bytes": (2 * rows + used + vocab) * dim * es + 2 * rows * 8, "flops": 2 * rows * dim}
    tables = (rows + vocab) * dim * es
    if kind == "loss":
        return {"bytes": tables + rows * 12, "flops": 2 * rows * dim * vocab}
    return {"bytes": 3 * tables + rows * 24, "flops": 6 * rows * dim * vocab}
