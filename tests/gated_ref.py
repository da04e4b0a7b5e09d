"""The gated recurrence, its gradients, the 8-bit checkpoints and the conv's gradients in 64 bits on the
CPU, each with a bound on what float32 arithmetic in the kernels' order of operations may add.

Bounds are running error bounds: with u = 2^-24, v_exp_f32, v_rcp_f32, v_sqrt_f32 and v_rsq_f32 off by at
most one unit in the last place (2u), every other operation by half of one (u):

  sigmoid(v)   argument v log2(e): 2u |v|; exp2 2u, sum u, reciprocal 2u    -> (2|v| + 5) u relative
  l = A r      that of r and u
  a = exp(l)   |l| a times that of l; next to 1 the rounding of 1 - q (u) and q's own (4u of q <= 0.25),
               else exp2's 2u and its argument's 2u |l|                     -> at most (2|l| + 3) u a more
  sqrt(1-a^2)  half of l's relative error (|l| a^2 / (1 - a^2) <= 1/2), the series or 1 - a (4u and 2.5
               times exp2's), the product, the root                          -> 14u more
"""

from __future__ import annotations

import torch

U = 2.0 ** -24
BLOCK = 16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the smallest numbers, where a rounding is not relative."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps


def sig(v):
    return torch.sigmoid(v), (2 * v.abs() + 5) * U  # (relative error; sigmoid's value at +-inf has none)


def quantise(x):
    """What the 8-bit codes of x (batch, seqlen, dim), float64, stand for."""
    out = torch.empty_like(x)
    for t in range(0, x.shape[1], BLOCK):
        part = x[:, t:t + BLOCK]
        top = part.abs().amax(1, keepdim=True)
        ok = torch.isfinite(top)
        _, k = torch.frexp(torch.where(ok, top, torch.zeros_like(top)))
        e = (k.long() - 7).clamp(-126, 121)
        scale = torch.ldexp(torch.ones_like(top), e)
        up = (top >= 127.5 * scale) & (e < 121)
        scale = torch.where(up, 2 * scale, scale)
        scale = torch.where(ok, scale, torch.full_like(scale, float("nan")))
        out[:, t:t + BLOCK] = torch.round(part / scale).clamp(-127, 127) * scale
    return out


def _live(shape, lengths):
    t = torch.arange(shape[1])[None, :, None]
    return (t < lengths.clamp(0, shape[1])[:, None, None]).expand(shape)


class Case:
    """Inputs of any dtype on any device; everything here is float64 on the CPU."""

    def __init__(self, x, a_gate, x_gate, A, z=None, h0=None, lengths=None):
        f = lambda t: None if t is None else t.detach().cpu().double()
        self.x, self.ag, self.xg, self.A, self.z, self.h0 = (f(t) for t in (x, a_gate, x_gate, A, z, h0))
        b, n, d = self.x.shape
        lengths = torch.full((b,), n) if lengths is None else lengths.detach().cpu().long()
        self.live = _live((b, n, d), lengths)
        zero = torch.zeros((), dtype=torch.float64)
        for k in ("x", "ag", "xg", "z"):
            if getattr(self, k) is not None:
                setattr(self, k, torch.where(self.live, getattr(self, k), zero))
        self.h0 = torch.zeros((b, d), dtype=torch.float64) if self.h0 is None else self.h0

    def elements(self):
        """r, i, l, a, beta, u = i x and the relative (r, i, l, beta) or absolute (a) errors."""
        r, er = sig(self.ag)
        i, ei = sig(self.xg)
        r, i = torch.where(r.isnan(), r, r), i
        l = torch.clamp(self.A * r, min=-1e30)
        el = er + U
        a = torch.exp(l)
        beta = torch.sqrt(-torch.expm1(2 * l))
        ea = a * l.abs() * el + (2 * l.abs() + 3) * U * a + U
        ea = ea + 2.0 ** -126  # below the smallest normal number errors are not relative, results may be 0
        ebeta = el / 2 + 14 * U
        # A r below the smallest normal number may be taken as 0, and the root with it
        ebeta = torch.where(l.abs() < 2.0 ** -125, torch.ones_like(l), ebeta)
        for e in (er, ei, el, ea, ebeta):
            e[~torch.isfinite(e)] = 0.0  # saturated gates: sigmoid is 0 or 1
        a = torch.where(self.live, a, torch.ones_like(a))
        ea = torch.where(self.live, ea, torch.zeros_like(ea))
        u = torch.where(self.live, i * self.x, torch.zeros_like(a))
        return r, i, l, a, beta, u, er, ei, el, ea, ebeta

    def states(self, starts=None, starts_err=None):
        """h_{t-1}, h_t and a bound of h_t's (and h_{t-1}'s) error; starts, when given, are the states that
        each block of 16 tokens begins from."""
        r, i, l, a, beta, u, er, ei, el, ea, ebeta = self.elements()
        b = torch.where(self.live, beta * u, torch.zeros_like(u))
        eb = b.abs() * (ebeta + ei + 2 * U)
        h, e = self.h0, torch.zeros_like(self.h0)
        before, after, err_before, err = [], [], [], []
        for t in range(a.shape[1]):
            if starts is not None and t % BLOCK == 0:
                h, e = starts[:, t // BLOCK], starts_err[:, t // BLOCK]
            before.append(h)
            err_before.append(e)
            hn = a[:, t] * h + b[:, t]
            # the tile's carry is joined in as well: one more product and sum than the plain recurrence has
            e = (a[:, t] + ea[:, t]) * e + ea[:, t] * h.abs() + eb[:, t] + 3 * U * (hn.abs() + (a[:, t] * h).abs())
            e = torch.where(self.live[:, t], e, err_before[-1])
            h = torch.where(self.live[:, t], hn, h)
            after.append(h)
            err.append(e)
        self.last = (h, e)
        st = lambda v: torch.stack(v, 1) if v else torch.zeros_like(a)
        return st(before), st(after), st(err_before), st(err)

    def forward(self):
        """y and the final state, each with its bound before the last rounding."""
        before, h, eb, e = self.states()
        y, ey = h, e
        if self.z is not None:
            s, es = sig(self.z)
            es = torch.where(torch.isfinite(es), es, torch.zeros_like(es))
            g = self.z * s
            g = torch.where(torch.isneginf(self.z), torch.zeros_like(g), g)
            y = h * g
            ey = e * g.abs() + y.abs() * (es + 3 * U)
        zero = torch.zeros_like(y)
        return torch.where(self.live, y, zero), torch.where(self.live, ey, zero), *self.last

    def backward(self, dy, dstate=None, eight=False):
        """{name: (gradient, bound)}."""
        before, h, eb, e = self.states()
        v = self
        if eight:
            starts, starts_err = before[:, ::BLOCK], eb[:, ::BLOCK]
            v = Case(*(quantise(t) for t in (self.x, self.ag, self.xg)), self.A,
                     None if self.z is None else quantise(self.z), self.h0)
            v.live = self.live
            before, h, eb, e = v.states(starts, starts_err)
        r, i, l, a, beta, u, er, ei, el, ea, ebeta = v.elements()
        zero = torch.zeros_like(a)
        g = torch.where(self.live, dy.detach().cpu().double(), zero)
        eg = zero
        out = {}
        if v.z is not None:
            s, es = sig(v.z)
            slope = s + v.z * s * (1 - s)
            mag = s + (v.z * s * (1 - s)).abs()
            dz = g * h * slope
            edz = g.abs() * (e * slope.abs() + h.abs() * mag * (2 * es + 6 * U)) + 2 * U * dz.abs()
            # 1 - s of a large z: absolute error u
            edz = edz + (g * h * v.z * s).abs() * (es + 2 * U)
            out["z"] = (dz, edz)
            eg = (g * v.z * s).abs() * (es + 3 * U)
            g = g * v.z * s
        carry = torch.zeros_like(self.h0) if dstate is None else dstate.detach().cpu().double()
        ecarry = torch.zeros_like(self.h0)
        dh, edh = torch.zeros_like(a), torch.zeros_like(a)
        for t in range(a.shape[1] - 1, -1, -1):
            dh[:, t] = g[:, t] + carry
            edh[:, t] = eg[:, t] + ecarry + U * (dh[:, t].abs() + carry.abs())
            nxt = a[:, t] * dh[:, t]
            en = (a[:, t] + ea[:, t]) * edh[:, t] + ea[:, t] * dh[:, t].abs() + 3 * U * (nxt.abs() + (a[:, t] * carry).abs())
            carry = torch.where(self.live[:, t], nxt, carry)
            ecarry = torch.where(self.live[:, t], en, ecarry)
        ratio = torch.where(beta > 0, a * a / beta, zero)
        eratio = ratio * (2 * l.abs() * el + ebeta + 10 * U + 4 * U * l.abs())  # relative of a: ea / a
        # a^2 below the smallest normal number (beta is 1 there) has an absolute error like a's
        eratio = eratio + torch.where(a * a < 2.0 ** -126, torch.full_like(a, 2.0 ** -126), zero)
        f = before * a - u * ratio
        ef = eb * a + before.abs() * (ea + 2 * U * a) + u.abs() * eratio + (u * ratio).abs() * (ei + 3 * U)
        dl = dh * f
        edl = edh * f.abs() + dh.abs() * ef + edh * ef + 2 * U * dl.abs()
        du = dh * beta
        edu = edh * beta + du.abs() * (ebeta + 2 * U)
        out["x"] = (i * du, i * edu + (i * du).abs() * (ei + 2 * U))
        # 1 - i and 1 - r: absolute error that of the sigmoid, i er
        t1 = du * u
        out["x_gate"] = (t1 * (1 - i), edu * u.abs() * (1 - i) + t1.abs() * ((1 - i) * (ei + 4 * U) + i * ei + U))
        t2 = torch.where(torch.isfinite(l), dl * l, zero)
        el_abs = l.abs() * el
        out["a_gate"] = (t2 * (1 - r), edl * l.abs() * (1 - r) + dl.abs() * (el_abs * (1 - r) + 4 * U * l.abs() * (1 - r)
                                                                     + l.abs() * (r * er + U)))
        live = lambda w: torch.where(self.live, w, zero)
        out = {k: (live(p), live(q)) for k, (p, q) in out.items()}
        terms, eterms = live(dl * r), live(edl * r + (dl * r).abs() * (er + 2 * U))
        # dA: a thread sums 16 tokens, a workgroup at most 16 such sums, in float32; the rest is double
        out["A"] = (terms.sum((0, 1)), (eterms + 34 * U * terms.abs()).sum((0, 1)))
        out["h0"] = (carry, ecarry)
        return out


def close(got, want, bound, dtype, what=""):
    """got is want within the bound and one rounding to dtype."""
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} != {tuple(want.shape)}"
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaNs differ"
    half = 0.0 if dtype == torch.float32 else half_step(dtype)
    tol = bound * (1 + half) + half * want.abs() + tiny(dtype) + want.abs() * U
    err = (got - want).abs()
    bad = (err > tol) & ~nan & (got != want)
    if bad.any():
        k = torch.where(bad, err / tol, torch.zeros_like(err)).argmax().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; element {k}: got "
                             f"{got.flatten()[k].item()!r}, want {want.flatten()[k].item()!r}, "
                             f"tolerance {tol.flatten()[k].item():.3e}")


def conv(x, weight, bias, apply_silu):
    """p and out of the causal conv in float64, and p's bound."""
    w = weight.reshape(weight.shape[0], -1)
    width, n = w.shape[1], x.shape[1]
    padded = torch.cat([x.new_zeros((x.shape[0], width - 1, x.shape[2])), x], 1)
    p = torch.zeros_like(x) if bias is None else bias.expand_as(x).clone()
    mag = p.abs()
    for k in range(width):
        p = p + padded[:, k:k + n] * w[:, k]
        mag = mag + (padded[:, k:k + n] * w[:, k]).abs()
    return p, mag * (width + 1) * U, padded


def conv_backward(x, weight, bias, dout, apply_silu):
    """{name: (gradient, bound)}; x, weight, bias, dout float64."""
    w = weight.reshape(weight.shape[0], -1)
    width, n = w.shape[1], x.shape[1]
    p, ep, padded = conv(x, weight, bias, apply_silu)
    if apply_silu:
        s, es = sig(p)
        slope = s * (1 + p * (1 - s))
        mag = s * (1 + p.abs() * (1 - s))
        dp = dout * slope
        # silu'' <= 1/2; 1 - s carries s's error; the products
        edp = dout.abs() * (ep * 0.5 + mag * (es + 4 * U) + p.abs() * s * (s * es + U)) + 2 * U * dp.abs()
    else:
        dp, edp = dout, torch.zeros_like(dout)
    after = lambda t: torch.cat([t, t.new_zeros((t.shape[0], width - 1, t.shape[2]))], 1)
    fd, fe = after(dp), after(edp)
    dx, edx = torch.zeros_like(x), torch.zeros_like(x)
    dw, edw = torch.zeros_like(w), torch.zeros_like(w)
    for k in range(width):
        sl = slice(width - 1 - k, width - 1 - k + n)
        dx += fd[:, sl] * w[:, k]
        edx += (fe[:, sl] + (width + 1) * U * fd[:, sl].abs()) * w[:, k].abs()
        term = dp * padded[:, k:k + n]
        dw[:, k] = term.sum((0, 1))
        # at most 64 products in a thread's sum and 16 threads' sums, in float32; the rest is double
        edw[:, k] = (edp * padded[:, k:k + n].abs() + 82 * U * term.abs()).sum((0, 1))
    db, edb = dp.sum((0, 1)), (edp + 82 * U * dp.abs()).sum((0, 1))
    return {"x": (dx, edx), "weight": (dw.view(weight.shape), edw.view(weight.shape)), "bias": (db, edb)}
