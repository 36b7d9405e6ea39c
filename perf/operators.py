"""Workloads of the feed-forward operators: the gated block's two projections with their
activation, the linear layer whose epilogue adds a bias, an activation and a gated residual, and
activation checkpoints held in 8 bits, forward and backward.

Sizes are those of the repository's 101M configuration (width 640, feed-forward width 1248) and
generic ones around it.  ``listed()`` names twelve cases, ``draw(rng)`` makes another of the same
ranges, ``prepare`` builds what the caller has in hand, ``run`` is one pass and ``exact`` the same
outputs in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 32          # elements of a row that share one power of two in a packed activation
E4M3_MAX = 448.0


def listed():
    return [
        # The gated block of the 101M model for one decoded token.
        dict(name="gated_decode_1", kind="gated", M=1, C=640, I=1248, dtype="bf16", train=False, ckpt=""),
        # A serving batch of 16 tokens through a wider block, in the other 16-bit type.
        dict(name="gated_decode_16_wide", kind="gated", M=16, C=1024, I=2816, dtype="fp16", train=False, ckpt=""),
        # One piece of a prompt that is prefilled piece by piece.
        dict(name="gated_piece_1003", kind="gated", M=1003, C=640, I=1248, dtype="bf16", train=False, ckpt=""),
        # The 101M model's block over a training batch of 8 sequences of 2,048 tokens.
        dict(name="gated_train_16k", kind="gated", M=16384, C=640, I=1248, dtype="bf16", train=True, ckpt=""),
        # A packed batch that no tile divides, its input kept in 8 bits until the backward pass.
        dict(name="gated_train_8191_e4m3", kind="gated", M=8191, C=640, I=1248, dtype="fp16", train=True, ckpt="e4m3"),
        # A larger model's block: widths at which the products dominate.
        dict(name="gated_train_wide_4k", kind="gated", M=4096, C=2048, I=5504, dtype="bf16", train=True, ckpt=""),
        # The down projection with the block's gated residual, 16 decoded tokens.
        dict(name="down_decode_16", kind="linear", M=16, K=1248, N=640, dtype="bf16", train=False, ckpt="",
             act="none", bias=False, residual=True, gate=True),
        # The same over a long prompt.
        dict(name="down_prefill_32k", kind="linear", M=32768, K=1248, N=640, dtype="bf16", train=False, ckpt="",
             act="none", bias=False, residual=True, gate=True),
        # The same in training, its input (the widest activation of a block) kept in 8 bits.
        dict(name="down_train_16k_e4m3", kind="linear", M=16384, K=1248, N=640, dtype="bf16", train=True, ckpt="e4m3",
             act="none", bias=False, residual=True, gate=True),
        # A biased layer with an activation, at sizes that no vector width divides.
        dict(name="gelu_train_odd", kind="linear", M=1777, K=555, N=1001, dtype="fp16", train=True, ckpt="",
             act="gelu", bias=True, residual=True, gate=False),
        # The feed-forward activations of a batch of long prompts, packed and read back.
        dict(name="pack_32k", kind="pack", M=32768, C=1248, dtype="bf16"),
        # A few fp32 rows whose last group is not whole.
        dict(name="pack_small_fp32", kind="pack", M=333, C=641, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 32 as models have them, now and then any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(32, n // 32 * 32)


def draw(rng):
    kind = rng.choice(["gated", "gated", "gated", "linear", "linear", "linear", "pack"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "pack":
        return dict(kind="pack", M=_log_int(rng, 1, 32768), C=_log_int(rng, 1, 4096),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]))
    train = rng.random() < 0.6
    n, k = _width(rng, 64, 5504), _width(rng, 64, 2048)
    lo, most = (32, 4096 * 2048 * 5504) if train else (1, 4096 * 2048 * 5504 * 2)
    M = _log_int(rng, lo, max(lo, min(32768, most // (n * k))))
    ckpt = rng.choice(["", "e4m3"]) if train else ""
    if kind == "gated":
        return dict(kind="gated", M=M, C=k, I=n, dtype=dtype, train=train, ckpt=ckpt)
    if rng.random() < 0.5:
        n, k = k, n
    return dict(kind="linear", M=M, K=k, N=n, dtype=dtype, train=train, ckpt=ckpt,
                act=rng.choice(["none", "none", "relu", "silu", "gelu"]), bias=rng.random() < 0.5,
                residual=rng.random() < 0.7, gate=rng.random() < 0.5)


def prepare(case, seed):
    """Normalised activations, weights that keep their scale, gradients as a scaled loss gives them."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    M = case["M"]
    s = dict(case=case)
    if case["kind"] == "pack":
        # rows of very different size and a few large channels, as activations have them
        x = randn(M, case["C"]) * torch.exp2(randn(M, 1))
        s["x"] = torch.where(torch.rand(case["C"], generator=g, device=DEV) < 0.01, x * 30, x).to(dt)
        return s
    train = case["train"]
    if case["kind"] == "gated":
        C, I = case["C"], case["I"]
        s["x"] = randn(M, C).to(dt).requires_grad_(train)
        s["w_gate"] = (randn(I, C) / math.sqrt(C)).to(dt).requires_grad_(train)
        s["w_up"] = (randn(I, C) / math.sqrt(C)).to(dt).requires_grad_(train)
        if train:
            s["dy"] = (0.3 * randn(M, I)).to(dt)
        return s
    K, N = case["K"], case["N"]
    s["x"] = randn(M, K).to(dt).requires_grad_(train)
    s["weight"] = (randn(N, K) / math.sqrt(K)).to(dt).requires_grad_(train)
    s["bias"] = (0.5 * randn(N)).to(dt).requires_grad_(train) if case["bias"] else None
    s["residual"] = randn(M, N).to(dt).requires_grad_(train) if case["residual"] else None
    s["gate"] = torch.sigmoid(2 + 0.5 * randn(N)).to(dt).requires_grad_(train) if case["gate"] else None
    if train:
        s["dy"] = (0.3 * randn(M, N)).to(dt)
    return s


# ----------------------------------------------------------------------------- the plain form


def _pack_plain(x):
    """The values that a packed ``x`` stands for, in 32 bits: every GROUP elements of a row share the
    smallest power of two 2^e, e >= -127, with amax <= 448 * 2^e, and keep x / 2^e as an e4m3."""
    M, C = x.shape
    xf = torch.zeros(M, -(-C // GROUP) * GROUP, dtype=torch.float32, device=x.device)
    xf[:, :C] = x.float()
    xg = xf.view(M, -1, GROUP)
    mant, exp = torch.frexp(xg.abs().amax(dim=-1, keepdim=True))       # amax = mant * 2^exp, mant in [0.5, 1)
    e = exp - 9 + (mant > E4M3_MAX / 512).to(exp.dtype)
    e = torch.where(mant > 0, e, -127).clamp(min=-127)
    codes = torch.ldexp(xg, -e).to(torch.float8_e4m3fn)
    return torch.ldexp(codes.float(), e).reshape(M, -1)[:, :C]


def _act_plain(z, act):
    if act == "relu":
        return z * (z > 0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _dact_plain(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sg = 1 / (1 + torch.exp(-z))
        return sg * (1 + z * (1 - sg))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _gated_plain(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.t(), x @ wu.t()
    out = dict(y=(g / (1 + torch.exp(-g)) * u).to(dt))
    if not case["train"]:
        return out
    if case["ckpt"]:                       # the backward pass sees the input that was kept
        x = _pack_plain(s["x"])
        g, u = x @ wg.t(), x @ wu.t()
    dy = s["dy"].float()
    sg = 1 / (1 + torch.exp(-g))
    dg, du = dy * u * sg * (1 + g * (1 - sg)), dy * g * sg
    out["dx"] = (dg @ wg + du @ wu).to(dt)
    out["dw_gate"], out["dw_up"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
    return out


def _linear_plain(s):
    case, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()

    def pre(x):
        z = x @ w.t()
        return z if s["bias"] is None else z + s["bias"].float()

    z = pre(x)
    y = _act_plain(z, case["act"])
    if s["gate"] is not None:
        y = y * s["gate"].float()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = dict(y=y.to(dt))
    if not case["train"]:
        return out
    if case["ckpt"]:
        x = _pack_plain(s["x"])
        z = pre(x)
    dy = s["dy"].float()
    dz = dy * _dact_plain(z, case["act"])
    if s["gate"] is not None:
        out["dgate"] = (dy * _act_plain(z, case["act"])).sum(0).to(dt)
        dz = dz * s["gate"].float()
    if s["bias"] is not None:
        out["dbias"] = dz.sum(0).to(dt)
    out["dx"], out["dw"] = (dz @ w).to(dt), (dz.t() @ x).to(dt)
    return out


# ----------------------------------------------------------------------------- one pass


def _dispatcher():
    pkg = os.path.join(os.getcwd(), "maba-v2-architecture_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from maba_sparse.kernels import dispatcher
    return dispatcher


def _run_own(s):
    D, case = _dispatcher(), s["case"]
    if case["kind"] == "pack":
        codes, scales = D.checkpoint_pack(s["x"])
        return dict(y=D.checkpoint_unpack(codes, scales, dtype=s["x"].dtype))
    ckpt = case["ckpt"] or None
    if case["kind"] == "gated":
        y = D.gated_ffn(s["x"], s["w_gate"], s["w_up"], checkpoint=ckpt)
        leaves = dict(dx=s["x"], dw_gate=s["w_gate"], dw_up=s["w_up"])
    else:
        y = D.linear_epilogue(s["x"], s["weight"], bias=s["bias"], activation=case["act"], residual=s["residual"],
                              gate=s["gate"], checkpoint=ckpt)
        leaves = {k: t for k, t in (("dx", s["x"]), ("dw", s["weight"]), ("dbias", s["bias"]), ("dgate", s["gate"]))
                  if t is not None}
    if not case["train"]:
        return dict(y=y)
    grads = torch.autograd.grad(y, list(leaves.values()), s["dy"])
    return dict(y=y.detach(), **dict(zip(leaves, grads)))


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["case"]["kind"] == "pack":
            return dict(y=_pack_plain(state["x"]).to(state["x"].dtype))
        return _gated_plain(state) if state["case"]["kind"] == "gated" else _linear_plain(state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    M = case["M"]
    if case["kind"] == "pack":
        C = case["C"]
        return dict(bytes=2 * size * M * C + M * C + M * -(-C // GROUP), flops=2 * M * C)
    if case["kind"] == "gated":
        C, I = case["C"], case["I"]
        b, f = M * C + 2 * I * C + M * I, 4 * M * I * C
        if case["train"]:
            b, f = b + M * I + M * C + 2 * I * C, 3 * f
        return dict(bytes=size * b, flops=f)
    K, N = case["K"], case["N"]
    b, f = M * K + N * K + M * N, 2 * M * N * K
    vecs = N * (bool(case["bias"]) + bool(case["gate"]))
    b += vecs + (M * N if case["residual"] else 0)
    if case["train"]:
        b, f = b + M * N + M * K + N * K + vecs, 3 * f
    return dict(bytes=size * b, flops=f)


# ----------------------------------------------------------------------------- in 64 bits


def _pack_exact(x):
    """As a packed row's definition has it: the scale from log2, then e4m3's steps by arithmetic."""
    M, C = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -C % GROUP)).reshape(M, -1, GROUP)
    amax = v.abs().max(dim=2, keepdim=True).values
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -300) / E4M3_MAX))
    e = torch.where(amax > E4M3_MAX * torch.exp2(e), e + 1, e)          # log2 may round across a power of two
    e = torch.where(amax <= E4M3_MAX * torch.exp2(e - 1), e - 1, e).clamp_min(-127)
    r = v / torch.exp2(e)
    a = r.abs().clamp_min(2.0 ** -40)
    step = torch.exp2(torch.floor(torch.log2(a)).clamp_min(-6) - 3)     # three mantissa bits, subnormals below 2^-6
    q = torch.round(r / step) * step                                     # ties to even
    return (q * torch.exp2(e)).reshape(M, -1)[:, :C]


def _acts64(z, act):
    phi = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    cdf = torch.special.ndtr(z)
    sig = torch.sigmoid(z)
    return {"none": (z, torch.ones_like(z)), "relu": (torch.relu(z), (z > 0).double()),
            "silu": (z * sig, sig + z * sig * (1 - sig)), "gelu": (z * cdf, cdf + z * phi)}[act]


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    x64 = s["x"].double()
    if case["kind"] == "pack":
        return dict(y=_pack_exact(s["x"]))
    kept = _pack_exact(s["x"]) if case["ckpt"] else x64
    if case["kind"] == "gated":
        C = case["C"]
        w = torch.cat([s["w_gate"], s["w_up"]]).double()

        def halves(x):
            return torch.mm(x, w.t()).chunk(2, dim=1)

        g, u = halves(x64)
        out = dict(y=g * torch.sigmoid(g) * u)
        if case["train"]:
            g, u = halves(kept)
            a, da = _acts64(g, "silu")
            dy = s["dy"].double()
            d = torch.cat([dy * u * da, dy * a], dim=1)
            out["dx"] = torch.mm(d, w)
            dw = torch.mm(d.t().contiguous(), kept).reshape(2, -1, C)
            out["dw_gate"], out["dw_up"] = dw[0], dw[1]
        return out
    w = s["weight"].double()
    one = torch.ones(case["N"], dtype=torch.float64, device=DEV)
    bias = s["bias"].double() if s["bias"] is not None else 0 * one
    gate = s["gate"].double() if s["gate"] is not None else one
    a, _ = _acts64(torch.addmm(bias, x64, w.t()), case["act"])
    out = dict(y=a * gate + (s["residual"].double() if s["residual"] is not None else 0))
    if case["train"]:
        a, da = _acts64(torch.addmm(bias, kept, w.t()), case["act"])
        dy = s["dy"].double()
        dz = dy * gate * da
        out["dx"], out["dw"] = torch.mm(dz, w), torch.mm(dz.t().contiguous(), kept)
        if s["gate"] is not None:
            out["dgate"] = torch.sum(dy * a, dim=0)
        if s["bias"] is not None:
            out["dbias"] = torch.sum(dz, dim=0)
    return out
