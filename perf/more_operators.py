"""Workloads of the operators around a model's blocks: the boundary between two sub-layers (a norm
after the one, dropout, gate and scale on its way into the residual stream, the norm before the next),
dropout by itself, and the log probabilities of given tokens with their entropy and the likeliest
alternatives, forward and backward.

Sizes are those of the repository's 101M configuration (width 640, vocabulary 32768) and generic ones
around it.  ``listed()`` names twelve cases, ``draw(rng)`` makes another of the same ranges,
``prepare`` builds what the caller has in hand, ``run`` is one pass and ``exact`` the same outputs in
64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def listed():
    return [
        # The boundary of the 101M model's blocks for one decoded token.
        dict(name="boundary_decode_1", kind="boundary", M=1, C=640, dtype="bf16", train=False,
             pre=True, post=False, gate=True, scale=1.0, p=0.0),
        # A serving batch of 16 tokens of a wider model with a norm on either side, in the other 16-bit type.
        dict(name="boundary_decode_16_post", kind="boundary", M=16, C=2048, dtype="fp16", train=False,
             pre=True, post=True, gate=True, scale=0.5, p=0.0),
        # The 101M model's boundary over a long prompt.
        dict(name="boundary_prefill_32k", kind="boundary", M=32768, C=640, dtype="bf16", train=False,
             pre=True, post=False, gate=True, scale=1.0, p=0.0),
        # The same over a training batch of 8 sequences of 2,048 tokens, with dropout.
        dict(name="boundary_train_16k", kind="boundary", M=16384, C=640, dtype="bf16", train=True,
             pre=True, post=False, gate=True, scale=1.0, p=0.1),
        # A larger model's boundary with everything it can hold.
        dict(name="boundary_train_wide_8k", kind="boundary", M=8192, C=4096, dtype="bf16", train=True,
             pre=True, post=True, gate=True, scale=0.7071, p=0.1),
        # fp32 rows that no vector width divides; the stream goes on without a norm of its own.
        dict(name="boundary_train_odd_fp32", kind="boundary", M=1777, C=555, dtype="fp32", train=True,
             pre=False, post=True, gate=False, scale=0.25, p=0.2),
        # Dropout on the embeddings of the 101M model's training batch.
        dict(name="dropout_train_16k", kind="dropout", M=16384, C=640, dtype="bf16", p=0.1),
        # The same at an odd width and a high rate.
        dict(name="dropout_odd_fp16", kind="dropout", M=3001, C=1001, dtype="fp16", p=0.5),
        # One decoded token of 16 sequences, reported with its 20 likeliest alternatives.
        dict(name="logprobs_decode_16_top20", kind="logprobs", M=16, V=32768, dtype="bf16", train=False,
             top=20, temperature=0.8),
        # Scoring of a prompt of 4,096 tokens, the five likeliest alternatives of each.
        dict(name="logprobs_score_4k_top5", kind="logprobs", M=4096, V=32768, dtype="bf16", train=False,
             top=5, temperature=1.0),
        # The loss of a training batch with an entropy term, and its gradient.
        dict(name="logprobs_train_8k", kind="logprobs", M=8192, V=32768, dtype="bf16", train=True,
             top=0, temperature=1.0),
        # fp32 logits of an odd vocabulary, gradient and alternatives at once.
        dict(name="logprobs_train_odd_fp32", kind="logprobs", M=777, V=50257, dtype="fp32", train=True,
             top=8, temperature=1.3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A width: mostly a multiple of 32 as models have them, now and then any number."""
    n = _log_int(rng, lo, hi)
    return n if n < 32 or rng.random() < 0.3 else n // 32 * 32


def draw(rng):
    kind = rng.choice(["boundary", "boundary", "boundary", "dropout", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    half = 2 if dtype == "fp32" else 1
    if kind == "logprobs":
        V = _width(rng, 100, 131072)
        return dict(kind=kind, M=_log_int(rng, 1, min(16384, 8192 * 32768 // (V * half))), V=V, dtype=dtype,
                    train=rng.random() < 0.5, top=rng.choice([0, 0, 1, 5, 20, 64]),
                    temperature=round(rng.uniform(0.5, 1.5), 2))
    C = _width(rng, 1 if kind == "dropout" else 16, 8192)
    M = _log_int(rng, 1, min(65536, 8192 * 4096 // (C * half)))
    if kind == "dropout":
        return dict(kind=kind, M=M, C=C, dtype=dtype, p=round(rng.uniform(0.0, 0.9), 3))
    return dict(kind=kind, M=M, C=C, dtype=dtype, train=rng.random() < 0.6, pre=rng.random() < 0.8,
                post=rng.random() < 0.5, gate=rng.random() < 0.6, scale=rng.choice([1.0, 0.5, 0.7071]),
                p=rng.choice([0.0, 0.0, 0.1, 0.3]))


def prepare(case, seed):
    """A residual stream and a block's output, parameters near their initial values, gradients as a scaled
    loss gives them; logits of a few likely tokens among many, some of them masked."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    M, s = case["M"], dict(case=case)
    if case["kind"] == "logprobs":
        V, train = case["V"], case["train"]
        x = 1.5 * randn(M, V)
        x[:, :: 97] += 4 * randn(M, 1).abs()                           # likelier tokens, some rows surer than others
        x[:, torch.rand(V, generator=g, device=DEV) < 0.01] = -math.inf  # a vocabulary's unused tokens
        s["targets"] = torch.randint(0, V, (M,), generator=g, device=DEV)
        x.scatter_(1, s["targets"][:, None], 2 * randn(M, 1) + 3)
        s["targets"][torch.rand(M, generator=g, device=DEV) < 0.02] = -100   # padding
        s["logits"] = x.to(dt).requires_grad_(train)
        if train:
            s["dlogp"] = -torch.rand(M, generator=g, device=DEV)
            s["dentropy"] = 0.01 * randn(M)
        return s
    C = case["C"]
    s["seed"] = torch.randint(0, 2 ** 62, (1,), generator=g, device=DEV)
    if case["kind"] == "dropout":
        s["x"] = randn(M, C).to(dt).requires_grad_(True)
        s["dy"] = (0.3 * randn(M, C)).to(dt)
        return s
    train = case["train"]
    s["x"] = (2 * randn(M, C)).to(dt).requires_grad_(train)
    s["y"] = (randn(M, C) * torch.exp2(randn(M, 1))).to(dt).requires_grad_(train)
    s["weight"] = (1 + 0.1 * randn(C)).to(dt).requires_grad_(train) if case["pre"] else None
    s["post_weight"] = (1 + 0.1 * randn(C)).to(dt).requires_grad_(train) if case["post"] else None
    s["gate"] = torch.sigmoid(2 + 0.5 * randn(C)).to(dt).requires_grad_(train) if case["gate"] else None
    if train:
        s["dx_out"] = (0.3 * randn(M, C)).to(dt)
        s["dh"] = (0.3 * randn(M, C)).to(dt) if case["pre"] else None
    return s


# ----------------------------------------------------------------------------- the plain form


def _keep_plain(M, C, seed, p):
    """Which elements of [M, C] dropout keeps: word c % 4 of Philox4x32-7 (Salmon et al., "Parallel random
    numbers: as easy as 1, 2, 3", 2011) with the counter (c // 4, row, 0) and the seed as its key, against
    p * 2^32."""
    low = 0xFFFFFFFF
    rows = torch.arange(M, device=DEV).view(-1, 1)
    c0 = torch.arange(-(-C // 4), device=DEV).view(1, -1).expand(M, -1)
    c1, c2, c3 = (rows & low).expand_as(c0), (rows >> 32).expand_as(c0), torch.zeros_like(c0)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57        # 64-bit products; their upper halves are masked after the shift
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), dim=-1).reshape(M, -1)[:, :C]
    return words >= round(p * 2 ** 32)


def _drop_plain(v, keep, p):
    return torch.where(keep, v * (1 / (1 - p)), torch.zeros((), device=DEV))


def _dropout_plain(s):
    case, dt = s["case"], s["x"].dtype
    keep = _keep_plain(case["M"], case["C"], s["seed"], case["p"])
    return dict(y=_drop_plain(s["x"].float(), keep, case["p"]).to(dt),
                dx=_drop_plain(s["dy"].float(), keep, case["p"]).to(dt))


def _boundary_plain(s):
    case, dt, p = s["case"], s["x"].dtype, s["case"]["p"]
    one = torch.ones((), device=DEV)
    w, wp, gate = (one if s[k] is None else s[k].float() for k in ("weight", "post_weight", "gate"))
    y = s["y"].float()
    rp = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) if case["post"] else one
    keep = _keep_plain(case["M"], case["C"], s["seed"], p) if p > 0 else None

    def drop(v):
        return v if keep is None else _drop_plain(v, keep, p)

    z = drop(y * rp * wp)
    x = s["x"].float() + case["scale"] * (gate * z)
    out = dict(x_out=x.to(dt))
    if case["pre"]:
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        out["h"] = (x * r * w).to(dt)
    if not case["train"]:
        return out
    dx = s["dx_out"].float()
    if case["pre"]:
        dh, xh = s["dh"].float(), x * r
        dx = dx + r * (dh * w - xh * (dh * w * xh).mean(-1, keepdim=True))
        out["dweight"] = (dh * xh).sum(0).to(dt)
    out["dx"] = dx.to(dt)
    if case["gate"]:
        out["dgate"] = (case["scale"] * (dx * z)).sum(0).to(dt)
    dz = drop(case["scale"] * (gate * dx))
    if case["post"]:
        yh = y * rp
        out["dpost_weight"] = (dz * yh).sum(0).to(dt)
        dz = rp * (dz * wp - yh * (dz * wp * yh).mean(-1, keepdim=True))
    out["dy"] = dz.to(dt)
    return out


def _logprobs_plain(s):
    case, t = s["case"], s["targets"]
    M, V, inv = case["M"], case["V"], 1 / case["temperature"]
    logits = s["logits"]
    u = logits.float() * inv
    m = u.amax(-1, keepdim=True)
    e = torch.exp(u - m)
    tot = e.sum(-1, keepdim=True)
    lse = m + torch.log(tot)
    lp = u - lse
    prob = e / tot
    plogp = torch.where(prob > 0, prob * lp, torch.zeros((), device=DEV))
    H = -plogp.sum(-1, keepdim=True)
    have = (t >= 0).view(-1, 1)
    at = t.clamp_min(0).view(-1, 1)
    logp = torch.where(have, lp.gather(1, at), torch.zeros((), device=DEV))
    out = dict(logp=logp.view(-1), entropy=H.view(-1), lse=lse.view(-1))
    if case["top"]:
        # values mapped to whole numbers of the same order, the complement of the index below them: no two alike
        bits = (logits.float() + 0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
        keys = order * 2 ** 31 + (V - torch.arange(V, device=DEV))
        top = torch.topk(keys, case["top"], dim=-1).values
        ids = V - (top & (2 ** 31 - 1))
        out["top_logp"], out["top_ids"] = lp.gather(1, ids), ids
    if case["train"]:
        gl = torch.where(have, s["dlogp"].view(-1, 1), torch.zeros((), device=DEV))
        d = -gl * prob - s["dentropy"].view(-1, 1) * (plogp + prob * H)
        d = d + gl * (torch.arange(V, device=DEV) == t.view(-1, 1))
        out["dlogits"] = (inv * d).to(logits.dtype)
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
    if case["kind"] == "dropout":
        y = D.dropout(s["x"], case["p"], s["seed"])
        return dict(y=y.detach(), dx=torch.autograd.grad(y, s["x"], s["dy"])[0])
    if case["kind"] == "logprobs":
        logp, entropy, lse, top_logp, top_ids = D.token_logprobs(s["logits"], s["targets"],
                                                                 temperature=case["temperature"], top=case["top"])
        out = dict(logp=logp.detach(), entropy=entropy.detach(), lse=lse.detach())
        if case["top"]:
            out["top_logp"], out["top_ids"] = top_logp, top_ids
        if case["train"]:
            out["dlogits"] = torch.autograd.grad([logp, entropy], s["logits"], [s["dlogp"], s["dentropy"]])[0]
        return out
    x_out, h = D.residual_norm(s["x"], s["y"], weight=s["weight"], post_weight=s["post_weight"], gate=s["gate"],
                               scale=case["scale"], p=case["p"], seed=s["seed"], eps=EPS)
    out = dict(x_out=x_out.detach())
    if case["pre"]:
        out["h"] = h.detach()
    if case["train"]:
        leaves = {k: s[n] for k, n in (("dweight", "weight"), ("dx", "x"), ("dgate", "gate"),
                                       ("dpost_weight", "post_weight"), ("dy", "y")) if s[n] is not None}
        made, given = ([x_out, h], [s["dx_out"], s["dh"]]) if case["pre"] else ([x_out], [s["dx_out"]])
        out.update(zip(leaves, torch.autograd.grad(made, list(leaves.values()), given)))
    return out


_PLAIN = {"boundary": _boundary_plain, "dropout": _dropout_plain, "logprobs": _logprobs_plain}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["kind"]](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    M = case["M"]
    if case["kind"] == "logprobs":
        n = M * case["V"]
        b = n * size + M * (8 + 12) + M * case["top"] * 12
        if case["train"]:
            return dict(bytes=b + n * size + 8 * M, flops=12 * n)
        return dict(bytes=b, flops=5 * n)
    n = M * case["C"]
    if case["kind"] == "dropout":
        return dict(bytes=4 * n * size, flops=2 * n)
    vecs = case["C"] * (case["pre"] + case["post"] + case["gate"])
    streams = 3 + case["pre"]                                # x and y in, the stream and its norm out
    flops = 8 * n
    if case["train"]:
        streams, vecs, flops = streams + 3 + case["pre"], 2 * vecs, 30 * n
    return dict(bytes=size * (streams * n + vecs), flops=flops)


# ----------------------------------------------------------------------------- in 64 bits


def _keep_exact(M, C, seed, p):
    """The generator by its definition on words held as two 16-bit halves, one column of a block at a time."""
    def mul(c, x):                                           # (upper, lower) words of the 64-bit product
        lo, hi = (c & 0xFFFF) * x, (c >> 16) * x             # both below 2^48
        mid = hi + (lo >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)

    nb = (C + 3) // 4
    idx = torch.arange(M * nb, dtype=torch.int64, device=DEV)
    row, blk = torch.div(idx, nb, rounding_mode="floor"), idx % nb
    ctr = [blk, row % 2 ** 32, torch.div(row, 2 ** 32, rounding_mode="floor"), torch.zeros_like(idx)]
    value = int(seed.item())
    key = [value % 2 ** 32, value // 2 ** 32]
    for _ in range(7):
        h0, l0 = mul(0xD2511F53, ctr[0])
        h1, l1 = mul(0xCD9E8D57, ctr[2])
        ctr = [torch.bitwise_xor(h1, ctr[1]).bitwise_xor(key[0] * torch.ones_like(h1)), l1,
               torch.bitwise_xor(h0, ctr[3]).bitwise_xor(key[1] * torch.ones_like(h0)), l0]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    u = torch.empty(M, 4 * nb, dtype=torch.int64, device=DEV)
    for j in range(4):
        u[:, j::4] = ctr[j].view(M, nb)
    return torch.logical_not(u[:, :C] < round(p * 2 ** 32))


def _boundary_exact(case, s):
    names = ("x", "y", "weight", "post_weight", "gate")
    v = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names if s[k] is not None}
    z = v["y"]
    if case["post"]:
        z = z / torch.sqrt(z.square().mean(dim=1, keepdim=True) + EPS) * v["post_weight"]
    if case["p"] > 0:
        keep = _keep_exact(case["M"], case["C"], s["seed"], case["p"])
        z = torch.where(keep, z / (1 - case["p"]), 0.0)
    if case["gate"]:
        z = z * v["gate"]
    x = v["x"] + z * case["scale"]
    outs, grads = [x], [s["dx_out"].double()] if case["train"] else None
    if case["pre"]:
        outs.append(x / torch.sqrt(x.square().mean(dim=1, keepdim=True) + EPS) * v["weight"])
    out = dict(zip(("x_out", "h"), (o.detach() for o in outs)))
    if case["train"]:
        if case["pre"]:
            grads.append(s["dh"].double())
        got = dict(zip(v, torch.autograd.grad(outs, list(v.values()), grads)))
        for k in ("weight", "x", "gate", "post_weight", "y"):
            if k in got:
                out["d" + k] = got[k]
    return out


def _logprobs_exact(case, s):
    x = s["logits"].detach().double().requires_grad_(case["train"])
    t = s["targets"]
    u = x / case["temperature"]
    lse = torch.logsumexp(u, dim=1)
    lp = u - lse.unsqueeze(1)
    finite = torch.where(torch.isinf(lp), torch.zeros_like(lp), lp)
    entropy = -(torch.exp(lp) * finite).sum(dim=1)
    logp = torch.where(t < 0, torch.zeros_like(lse), lp[torch.arange(len(t), device=DEV), t.clamp(min=0)])
    out = dict(logp=logp.detach(), entropy=entropy.detach(), lse=lse.detach())
    if case["top"]:
        ids = torch.sort(s["logits"].detach(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
        out["top_logp"], out["top_ids"] = torch.take_along_dim(lp.detach(), ids, dim=1), ids
    if case["train"]:
        loss = (logp * s["dlogp"].double()).sum() + (entropy * s["dentropy"].double()).sum()
        out["dlogits"] = torch.autograd.grad(loss, x)[0]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "dropout":
        keep = _keep_exact(case["M"], case["C"], s["seed"], case["p"])
        return dict(y=torch.where(keep, s["x"].detach().double() / (1 - case["p"]), 0.0),
                    dx=torch.where(keep, s["dy"].double() / (1 - case["p"]), 0.0))
    return _boundary_exact(case, s) if case["kind"] == "boundary" else _logprobs_exact(case, s)
