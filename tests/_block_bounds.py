"""Dropout, the block boundary and token log probabilities in 64 bits, with a bound for each element of each output.

The bounds count, with u = 2^-24 (fp32's half step) and r = eps / 2 of the tensors' type:
  * a sum of n products in fp32: (n + 4) u times the sum of their magnitudes (log probabilities: at least 64 threads
    share a row, so that n is V / 64 and 64 for joining them);
  * 1 / sqrt(S / C + eps): half the relative error of S, and 6 u for the mean, eps and the root;
  * 2^x of an x known within e: ln 2 e relative, and 4 u for the exponential itself; a logarithm: 2 u relative;
  * 3 u for c = log2(e) / T (1 / T, the constant and their product are rounded), and u for l c - R;
  * u for each product and sum on the way, r for the rounding of the result, and half the type's smallest subnormal.
Errors of errors are covered by a factor of 1.05."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(v, e, dtype):
    """The bound of ``v`` known within ``e`` after rounding to ``dtype``."""
    f = torch.finfo(dtype)
    return 1.05 * (e + half_step(dtype) * v.abs()) + f.tiny * f.eps / 2


def check(got, want, name):
    v, bound = want
    assert got.shape == v.shape, (name, got.shape, v.shape)
    g = got.double()
    nan = v.isnan()
    assert torch.equal(g.isnan(), nan), name
    inf = v.isinf()
    assert torch.equal(g[inf], v[inf]), name
    ok = nan | inf | ((g - v).abs() <= bound)
    assert ok.all(), (name, int((~ok).sum()), (g - v).abs()[~ok][:4], bound.expand_as(v)[~ok][:4], v[~ok][:4])


# ----------------------------------------------------------------------------- dropout


def words(rows, cols, seed, stream=0):
    """Philox4x32 with seven rounds by its definition, in whole numbers of Python, for a few elements."""
    out = []
    for r in range(rows):
        line = []
        for b in range(-(-cols // 4)):
            c, k = [b, r % 2 ** 32, r >> 32, stream], [seed % 2 ** 32, seed >> 32]
            for _ in range(7):
                p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
                c = [(q >> 32) ^ c[1] ^ k[0], q % 2 ** 32, (p >> 32) ^ c[3] ^ k[1], p % 2 ** 32]
                k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
            line += c
        out.append(line[:cols])
    return torch.tensor(out)


def kept(x, p, seed, stream=0):
    """The mask of ``x [..., C]`` (from ``common.philox_words``, which has a test of its own against ``words``)."""
    from maba_sparse.kernels.common import philox_words
    rows = x.reshape(-1, x.shape[-1])
    below = round(p * 2 ** 32)
    if below == 0 or p >= 1:
        return torch.full_like(x, below == 0, dtype=torch.bool)
    return (philox_words(*rows.shape, seed.cpu(), stream) >= below).reshape(x.shape).to(x.device)


def dropout(x, p, seed, stream=0):
    y = torch.where(kept(x, p, seed, stream), x.double() / (1 - p) if p < 1 else 0.0, 0.0)
    return y, rounded(y, 2 * U * y.abs(), x.dtype)


# ----------------------------------------------------------------------------- the boundary


def _norm(x, eps):
    """1 / sqrt(mean x^2 + eps) of rows, and its relative error."""
    C = x.shape[-1]
    return torch.rsqrt((x * x).mean(-1, keepdim=True) + eps), ((C + 4) / 2 + 6) * U


def added(x, y, wp, g, scale, keep, p, eps):
    """x_out of x and y in 64 bits, and its error in fp32 before it is rounded."""
    z, rel = y, 0.0
    if wp is not None:
        rp, rel = _norm(y, eps)
        z = y * rp * wp.double()
    if keep is not None:
        z = torch.where(keep, z / (1 - p) if p < 1 else 0.0, 0.0)
    add = scale * z * (1.0 if g is None else g.double())
    x = x + add
    return x, (rel + 7 * U) * add.abs() + U * x.abs()


def boundary(x, y, w=None, wp=None, g=None, scale=1.0, keep=None, p=0.0, eps=1e-6):
    """{name: (value, bound)} of x_out and, with a weight, of h."""
    dt = x.dtype
    x, y = x.double(), None if y is None else y.double()
    e = torch.zeros_like(x)
    out = {}
    if y is not None:
        x, e = added(x, y, wp, g, scale, keep, p, eps)
        out["x_out"] = (x, rounded(x, e, dt))
    if w is not None:
        r, rel = _norm(x, eps)
        rel = rel + (x.abs() * e).sum(-1, keepdim=True) / ((x * x).sum(-1, keepdim=True) + x.shape[-1] * eps)
        h = x * r * w.double()
        out["h"] = (h, rounded(h, (r * w.double()).abs() * e + (rel + 4 * U) * h.abs(), dt))
    return out


def boundary_backward(dxo, dh, x, y=None, w=None, wp=None, g=None, scale=1.0, keep=None, p=0.0, eps=1e-6):
    """{name: (value, bound)} of dx, dy, dweight, dpost_weight and dgate, for the forward's x and y."""
    dt, (R, C) = x.dtype, x.shape
    xo, ex = x.double(), torch.zeros_like(x, dtype=torch.float64)
    if y is not None and dh is not None:                    # x_out and its error in fp32
        xo, ex = added(x.double(), y.double(), wp, g, scale, keep, p, eps)
    d = torch.zeros_like(xo) if dxo is None else dxo.double()
    e = torch.zeros_like(d)
    out, rows, cols = {}, (R + 64) * U, (C + 4) * U
    if dh is not None:
        h, w = dh.double(), w.double()
        r, rel = _norm(xo, eps)
        rel = rel + (xo.abs() * ex).sum(-1, keepdim=True) / ((xo * xo).sum(-1, keepdim=True) + C * eps)
        xh, hw, exh = xo * r, h * w, ex * r
        mean = (hw * xh).mean(-1, keepdim=True)
        em = (hw * xh).abs().mean(-1, keepdim=True) * (cols + rel + 4 * U) + (rel + 3 * U) * mean.abs()
        em = em + (hw.abs() * exh).mean(-1, keepdim=True)
        inner = hw - xh * mean
        ei = 2 * U * hw.abs() + xh.abs() * em + (rel + 3 * U) * (xh * mean).abs() + exh * mean.abs()
        d = d + r * inner
        e = r * ei + (rel + 2 * U) * (r * inner).abs() + 2 * U * d.abs()
        t = h * xh
        dw = t.sum(0)
        out["dweight"] = (dw, rounded(dw, ((rel + 3 * U + rows) * t.abs() + h.abs() * exh).sum(0), dt))
    elif w is not None:
        out["dweight"] = (torch.zeros(C, dtype=d.dtype, device=d.device),) * 2
    out["dx"] = (d, rounded(d, e, dt))
    m, e = d, e
    if keep is not None:
        k = 1 / (1 - p) if p < 1 else 0.0
        m = torch.where(keep, d * k, 0.0)
        e = torch.where(keep, k * e, 0.0) + 2 * U * m.abs()
    rp, rel = (1.0, 0.0) if wp is None else _norm(y.double(), eps)
    if g is not None and y is not None:
        z = y.double() * rp * (1.0 if wp is None else wp.double())
        t = scale * m * z
        dg = t.sum(0)
        out["dgate"] = (dg, rounded(dg, (abs(scale) * z.abs() * e + (rel + 6 * U + rows) * t.abs()).sum(0), dt))
    k = scale * (torch.ones(C, dtype=d.dtype, device=d.device) if g is None else g.double())
    dz, e = m * k, e * k.abs() + 3 * U * (m * k).abs()
    if wp is not None:
        yh, q = y.double() * rp, wp.double()
        t = dz * yh
        dp = t.sum(0)
        out["dpost_weight"] = (dp, rounded(dp, (yh.abs() * e + (rel + 3 * U + rows) * t.abs()).sum(0), dt))
        a = dz * q
        ea = e * q.abs() + U * a.abs()
        mean = (a * yh).mean(-1, keepdim=True)
        em = (ea * yh.abs() + (rel + 2 * U + cols) * (a * yh).abs()).mean(-1, keepdim=True) + 3 * U * mean.abs()
        inner = a - yh * mean
        dz = rp * inner
        e = rp * (ea + yh.abs() * em + (rel + 3 * U) * (yh * mean).abs()) + (rel + 2 * U) * dz.abs()
    out["dy"] = (dz, rounded(dz, e, dt))
    return out


# ----------------------------------------------------------------------------- log probabilities


def _weights(x, T):
    """Of rows x / T: the values, log p, p, p's part in sums, and rows of nothing but -inf."""
    u = x.double() / T
    none = (u == -math.inf).all(-1, keepdim=True)
    m = torch.where(none, 0.0, u.amax(-1, keepdim=True))
    lp = u - m - torch.log(torch.exp(u - m).sum(-1, keepdim=True))
    lp = torch.where(none, -math.inf, lp)
    return u, m, lp, torch.exp(lp), none


def _times(p, v):
    """p v, zero where p is zero."""
    return torch.where(p == 0, 0.0, p * torch.where(p == 0, 0.0, v))


def logprobs(x, t, T=1.0, top=0):
    """{name: (value, bound)} of logp, entropy, lse and top_logp, and top_ids as they are."""
    V = x.shape[-1]
    u, m, lp, p, none = _weights(x, T)
    n = (V / 64 + 64 + 10) * U
    mag = torch.where(p == 0, 0.0, u.abs())
    each = 4 * U * mag + n                                              # relative, of a term of the sum
    es = _times(p, each).sum(-1, keepdim=True) + 30 * U                 # of log S
    lse = torch.where(none, -math.inf, m - torch.where(none, 0.0, lp.amax(-1, keepdim=True)))
    out = {"lse": (lse.squeeze(-1), 1.05 * (es + 4 * U * lse.abs()).squeeze(-1))}

    def of(ids, have):
        v = torch.where(have, lp.gather(-1, ids), 0.0)
        at = u.gather(-1, ids).abs()
        return v, 1.05 * (es + 4 * U * torch.where(at == math.inf, 0.0, at) + 4 * U * torch.where(v.isinf(), 0.0, v.abs()))

    tt = t.unsqueeze(-1)
    v, b = of(tt.clamp(0, V - 1), tt >= 0)
    out["logp"] = (torch.where(tt >= V, math.nan, v).squeeze(-1), b.squeeze(-1))
    far = torch.where(p == 0, 0.0, m - u) + 1                           # |x| ln 2 of an element, from a reference above the largest
    H = -_times(p, lp).sum(-1, keepdim=True)
    eh = 2 * es + _times(p, far * (each + es + 6 * U)).sum(-1, keepdim=True) + _times(p, 8 * U * mag).sum(-1, keepdim=True)
    out["entropy"] = (H.squeeze(-1), 1.05 * (eh + 4 * U * H.abs()).squeeze(-1))
    if top:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top]
        out["top_logp"] = of(ids, torch.ones_like(ids, dtype=torch.bool))
        out["top_ids"] = ids
    return out


def logprobs_backward(gl, gh, gz, x, t, T=1.0):
    """(value, bound) of dlogits; lse and entropy are the 64-bit ones rounded to fp32."""
    V = x.shape[-1]
    u, m, lp, p, none = _weights(x, T)
    zero = torch.zeros(x.shape[:-1], dtype=torch.float64, device=x.device)
    gl, gh, gz = ((zero if g is None else g.double()).unsqueeze(-1) for g in (gl, gh, gz))
    tt = t.unsqueeze(-1)
    gl = torch.where((tt < 0) | none, 0.0, torch.where(tt >= V, math.nan, gl))
    H = -_times(p, lp).sum(-1, keepdim=True)
    lse = torch.where(none, 0.0, m - torch.where(none, 0.0, lp.amax(-1, keepdim=True)))
    base = gz - gl - gh * H
    d = p * base - gh * _times(p, lp)
    hit = torch.arange(V, device=x.device) == tt
    d = torch.where(hit, d + gl, d) / T
    mag = torch.where(p == 0, 0.0, u.abs())
    lpa = torch.where(p == 0, 0.0, lp.abs())
    el = 3 * U * (mag + lse.abs() + lpa) + 1e-300                       # of log p: 1 / T, lse, their difference
    parts = gz.abs() + gl.abs() + gh.abs() * (H.abs() + lpa)
    e = p * ((el + 2 * U * lpa + 12 * U) * parts + gh.abs() * el) / T + torch.where(hit, 3 * U * gl.abs() / T, 0.0)
    # the exponential is zero below fp32's normal range: p is then off by less than 2^-126, and its products with what stands
    # beside it, log p of no more than 88 among them, by that many times
    e = e + 2.0 ** -126 * (gz.abs() + gl.abs() + gh.abs() * (H.abs() + 88)) / T
    return d, rounded(d, e, x.dtype)


def likely_rows(V, lse, below, dtype, seed=0):
    """Rows of one likely token, the target, of logit ``lse``, the others ``below`` to ``below + 8`` below it: whole numbers, exact in
    every type; and the gradients of -logp and of the entropy at the targets in 64 bits with their bounds.

    They are the targets' 1 - p, which is the sum of the others' p: relative to itself it is off by what each p is, and that
    by the forward's lse (its sum's terms, (V / 64 + 74 + 30 + 4 |u|) u, and 4 u |lse|), by log p's three roundings, and by
    4 u for the exponential, then by its own sum and the products behind it.  The entropy's are -p (log p + H), log p being
    log(1 - (1 - p)): as far off as 1 - p for log p, u for H, 3 u for their sum and its product."""
    g = torch.Generator().manual_seed(seed + V)
    x = lse - below - torch.randint(0, 9, (5, V), generator=g).double()
    t = torch.tensor([0, V - 1, V // 2, 1, V // 3])
    x[torch.arange(5), t] = lse
    assert torch.equal(x.to(dtype).double(), x)
    p = torch.softmax(x, -1)
    H = -(p * torch.log(p)).sum(-1)
    p[torch.arange(5), t] = 0
    rest = p.sum(-1)
    rel = 1.05 * U * (2 * (V / 64 + 74) + 40 + 8 * abs(lse) + 3 * (below + 8))
    lp = torch.log1p(-rest)
    dH = -(1 - rest) * (lp + H)
    return x.to(dtype), t, H, (rest, rounded(rest, rel * rest, dtype)), (dH, rounded(dH, rel * lp.abs() + U * H + 3 * U * dH.abs(), dtype))
