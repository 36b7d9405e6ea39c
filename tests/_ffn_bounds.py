"""The feed-forward operators in 64 bits, with a bound for each element of each output.

The bounds count, with u = 2^-24 (fp32's half step) and r = eps / 2 of the 16-bit type:
  * a sum of n products in fp32: n u times the sum of their magnitudes;
  * the activation from it: its slope times that error, and (16 + 4 |z|) u for the exponential (an argument
    z log2(e) rounded to fp32 has an error of |z| 2^-24 that the exponential multiplies), its reciprocal and
    the products around it;
  * the rounding to 16 bits of dz (or [dg | du]) as an operand, r relative;
  * the rounding of the result, r relative, and half the smallest subnormal of the type.
Errors of errors are covered by a factor of 1.01."""
import math

import torch

U = 2.0 ** -24
# Largest slopes of each activation and of its derivative.
SLOPE = {"none": (1.0, 0.0), "relu": (1.0, 0.0), "silu": (1.1, 0.5), "gelu": (1.13, 0.8)}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _round(v, e, dtype):
    """The bound of ``v`` known within ``e`` after rounding to ``dtype``."""
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2
    return 1.01 * (e + half_step(dtype) * v.abs()) + tiny


def act64(z, name):
    if name == "relu":
        return torch.relu(z), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def unpack64(codes, scales):
    C = codes.shape[-1]
    e = (scales.double() - 127).repeat_interleave(32, dim=-1)[..., :C]
    return codes.float().double() * torch.exp2(e)


def gated(x, wg, wu, dh=None, kept=None):
    """{name: (value, bound)} of h and, with ``dh``, of dx, dw_gate and dw_up at ``kept`` (default x)."""
    dt = wg.dtype
    wg, wu = wg.double(), wu.double()

    def halves(x):
        g, u = x @ wg.t(), x @ wu.t()
        n = (x.shape[1] + 2) * U
        return g, u, n * (x.abs() @ wg.abs().t()), n * (x.abs() @ wu.abs().t())

    x = x.double()
    g, u, eg, eu = halves(x)
    a, da = act64(g, "silu")
    e = 1.1 * eg * u.abs() + a.abs() * eu + (16 + 4 * g.abs()) * U * (a * u).abs()
    out = dict(h=(a * u, _round(a * u, e, dt)))
    if dh is None:
        return out
    if kept is not None:
        x = kept.double()
        g, u, eg, eu = halves(x)
        a, da = act64(g, "silu")
    d = dh.double()
    near = (16 + 4 * g.abs()) * U
    dg, du = d * u * da, d * a
    Eg = _round(dg, d.abs() * (1.1 * eu + 0.5 * u.abs() * eg) + near * (d * u).abs() * 1.1, dt)
    Eu = _round(du, d.abs() * 1.1 * eg + near * du.abs(), dt)
    dx = dg @ wg + du @ wu
    n = 2 * (wg.shape[0] + 8) * U
    out["dx"] = (dx, _round(dx, (Eg + n * dg.abs()) @ wg.abs() + (Eu + n * du.abs()) @ wu.abs(), dt))
    n = (x.shape[0] + 64) * U
    for name, v, E in (("dw_gate", dg, Eg), ("dw_up", du, Eu)):
        dw = v.t() @ x
        out[name] = (dw, _round(dw, (E + n * v.abs()).t() @ x.abs(), dt))
    return out


def linear(x, w, bias=None, act="none", residual=None, gate=None, dy=None, kept=None):
    """{name: (value, bound)} of y and, with ``dy``, of dx, dw, dbias and dgate at ``kept`` (default x)."""
    dt = w.dtype
    w = w.double()
    b = 0 if bias is None else bias.double()
    gt = 1 if gate is None else gate.double()
    slope, slope2 = SLOPE[act]

    def pre(x):
        z = x @ w.t() + b
        return z, (x.shape[1] + 3) * U * (x.abs() @ w.abs().t() + abs(b))

    x = x.double()
    z, ez = pre(x)
    a, _ = act64(z, act)
    near = (16 + 4 * z.abs()) * U
    y, e = a * gt, (slope * ez + near * z.abs()) * abs(gt)
    if residual is not None:
        y, e = y + residual.double(), e + 2 * U * (residual.double().abs() + y.abs())
    out = dict(y=(y, _round(y, e, dt)))
    if dy is None:
        return out
    if kept is not None:
        x = kept.double()
        z, ez = pre(x)
        near = (16 + 4 * z.abs()) * U
    a, da = act64(z, act)
    d = dy.double()
    dz = d * gt * da
    # relu's slope may be either where z's sign is not certain
    eda = (z.abs() <= ez).double() if act == "relu" else slope2 * ez + (near if act in ("silu", "gelu") else 0)
    e32 = (d * gt).abs() * eda + 4 * U * dz.abs()
    E = e32 if act == "none" and gate is None else _round(dz, e32, dt)
    M = x.shape[0]
    dx = dz @ w
    ex = (E + (w.shape[0] + 16) * U * dz.abs()) @ w.abs()
    if act == "none" and gate is not None:      # the gate may be on the weight: gate * w rounded, subnormal or not
        ex = ex + d.abs().sum(1, keepdim=True) * torch.finfo(dt).tiny * half_step(dt)
    out["dx"] = (dx, _round(dx, ex, dt))
    dw = dz.t() @ x
    out["dw"] = (dw, _round(dw, (E + (M + 64) * U * dz.abs()).t() @ x.abs(), dt))
    if bias is not None:
        db = dz.sum(0)
        out["dbias"] = (db, _round(db, (e32 + (M + 64) * U * dz.abs()).sum(0), dt))
    if gate is not None:
        dgt = (d * a).sum(0)
        eg = (d.abs() * (slope * ez + near * z.abs()) + (M + 64) * U * (d * a).abs()).sum(0)
        if act == "none":                       # or <w, dy^T x> + bias * sum(dy): sums of M and of K products
            eg = eg + (M + x.shape[1] + 72) * U * (d.abs() * (x.abs() @ w.abs().t() + abs(b))).sum(0)
        out["dgate"] = (dgt, _round(dgt, eg, dt))
    return out


def check(got, want, what):
    """Every element of ``got`` within its bound of ``want = (value, bound)``."""
    value, bound = want
    g = got.double()
    assert g.shape == value.shape, (what, g.shape, value.shape)
    assert bool(torch.isfinite(g).all()), f"{what}: not finite"
    over = (g - value).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times its bound"
