"""fp16 gradients whose intermediates lie outside fp16's range: gradients of pre-activations past 65,504, gradients, gates
and weights so small that their products are below its smallest step.  What the formulas keep is kept.

Every value here scales with its output's gradient (or gate, or weight) as the formulas do, so the bounds are those of
``_ffn_bounds`` at a scaled call, where their allowance for subnormal intermediates is far below the values, scaled back;
the result's own rounding has half of fp16's smallest step at its true size."""
import pytest
import torch

import _ffn_bounds as B
from maba_sparse.kernels import dispatcher as D

pytestmark = pytest.mark.gpu
DEV, HF = "cuda", torch.float16
STEP = 2.0 ** -24                     # fp16's smallest


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setenv("MABA_STRICT_BACKEND", "1")


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=DEV)


def _at(want, power):
    """A (value, bound) pair of a call scaled by 2^power, at the call's own size."""
    value, bound = want
    return value * 2.0 ** -power, bound * 2.0 ** -power + STEP / 2


# Rows and widths for every kind of call: a few rows, sums that are split and that are not, rows that are copied.
SIZES = [(1, 64, 72), (5, 33, 24), (70, 64, 40), (300, 200, 136), (1000, 130, 72), (3000, 256, 520)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("power", [-9, -13, 12])
@pytest.mark.parametrize("M,Cw,I", SIZES)
def test_gated_gradients_at_every_size_of_the_output_gradient(M, Cw, I, power, packed):
    r = _gen(M)
    x = r(M, Cw).to(HF)
    wg, wu = (r(I, Cw) / Cw ** 0.5).to(HF), (r(I, Cw) / Cw ** 0.5).to(HF)
    if power > 0:                                 # dx and dW stay below 65,504 with weights and inputs this small
        x, wg, wu = x * 2.0 ** -6, wg * 2.0 ** -3, wu * 2.0 ** -3
    dh = (r(M, I).clamp(-4, 4) * 2.0 ** power).to(HF)
    codes, scales = D.checkpoint_pack(x)
    kept = B.unpack64(codes, scales) if packed else None
    up = 16 if power < 0 else 0
    want = B.gated(x, wg, wu, dh.double() * 2.0 ** up, kept=kept)
    got = D.gated_ffn_backward(dh, codes if packed else x, wg, wu, x_scales=scales if packed else None)
    for name, g in zip(("dx", "dw_gate", "dw_up"), got):
        B.check(g, _at(want[name], up), name)


def test_gated_gradients_of_pre_activations_past_the_range():
    """[dg | du] up to several times 65,504, dx and dW well below."""
    M, Cw, I = 40, 1024, 24
    r = _gen(1)
    x, wg, wu = (0.15 * r(M, Cw)).to(HF), (0.4 * r(I, Cw)).to(HF), (0.4 * r(I, Cw)).to(HF)
    dh = torch.zeros(M, I, device=DEV, dtype=HF)
    dh[torch.arange(M), torch.arange(M) % I] = 40000.0                  # one of a row's
    want = B.gated(x, wg, wu, dh)
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    assert float((dh.double() * u * B.act64(g, "silu")[1]).abs().max()) > 65504
    got = dict(zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(dh, x, wg, wu)))
    for name, v in got.items():
        inside = want[name][0].abs() < 65000
        assert float(inside.double().mean()) > 0.5
        value, bound = want[name]
        assert bool(((v.double() - value).abs() <= bound)[inside].all()), name


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("gate,weight,dy", [(-16, 0, 0), (-18, -6, 8), (0, 0, -13), (0, -10, 0), (-10, 0, -8), (0, 0, 11), (6, 3, 5)])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_gradients_at_every_size_of_gate_weight_and_output_gradient(M, K, N, act, gate, weight, dy):
    r = _gen(N)
    x = r(M, K).to(HF)
    w = (r(N, K) / K ** 0.5 * 2.0 ** weight).to(HF)
    b = (0.5 * r(N) * 2.0 ** weight).to(HF)
    gt = ((1 + torch.rand(N, device=DEV)) * 2.0 ** gate).to(HF)
    d = (r(M, N).clamp(-4, 4) * 2.0 ** dy).to(HF)
    if gate + dy > 0:
        x = (x * 2.0 ** -6).to(HF)
        w = (w * 2.0 ** -4).to(HF)
    # every gradient scales with dy, and all but dgate with the gate
    up = max(0, 4 - gate - dy)
    want = B.linear(x, w, b, act, None, gt.double(), d.double() * 2.0 ** up)
    want = {k: _at(v, up) for k, v in want.items()}
    if act == "none":                             # dx scales with the weight too
        full = B.linear(x, (w.float() * 2.0 ** -weight).to(HF), None, act, None, gt.double() * 2.0 ** -gate, d.double() * 2.0 ** -dy)
        want["dx"] = _at(full["dx"], -weight - gate - dy)
    got = dict(zip(("dx", "dw", "dbias", "dgate"), D.linear_epilogue_backward(d, x, w, b, act, gt)))
    for name, v in got.items():
        value, bound = want[name]
        inside = value.abs() < 65000
        assert bool(inside.any())
        over = (v.double() - value).abs() / bound
        assert float(over[inside].max()) <= 1.0, (name, float(over[inside].max()))


def test_a_replayed_graph_scales_by_what_it_finds():
    """The powers of two belong to the values of each replay, in two graphs that share their workspaces' memory."""
    r = _gen(7)
    sets = []
    for M, Cw, I in ((300, 136, 72), (70, 64, 200)):
        sets.append(dict(x=r(M, Cw).to(HF), wg=(r(I, Cw) / Cw ** 0.5).to(HF), wu=(r(I, Cw) / Cw ** 0.5).to(HF), dh=r(M, I).to(HF),
                         gate=torch.rand(I, device=DEV).to(HF)))

    def step(t):
        return [*D.gated_ffn_backward(t["dh"], t["x"], t["wg"], t["wu"]),
                *D.linear_epilogue_backward(t["dh"], t["x"], t["wg"], t["gate"], "silu", t["gate"]),
                *D.linear_epilogue_backward(t["dh"], t["x"], t["wg"], None, "none", t["gate"])[:2]]

    for t in sets:
        step(t)
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for t in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(t))
        pool = g.pool()
        graphs.append(g)
    for turn, power in ((0, 0), (1, -12), (1, 6), (0, -14), (1, 0), (0, 3), (0, -8)):
        t = sets[turn]
        t["dh"].copy_(r(*t["dh"].shape) * 2.0 ** power)
        t["gate"].copy_(torch.rand(t["gate"].shape, device=DEV) * 2.0 ** (power / 2))
        graphs[turn].replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs[turn]]
        assert all(torch.equal(a, b) for a, b in zip(got, step(t))), (turn, power)
        want = B.gated(t["x"], t["wg"], t["wu"], t["dh"].double() * 2.0 ** 16)
        for name, v in zip(("dx", "dw_gate", "dw_up"), got):
            B.check(v, _at(want[name], 16), name)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_bad_element_spoils_only_what_is_made_of_it(bad):
    """Elements that are not finite take no part in the bound: the rest keeps its bits, and small gradients theirs."""
    M, Cw, I = 90, 48, 40
    r = _gen(8)
    x, wg, wu, dh = r(M, Cw).to(HF), (r(I, Cw) / 7).to(HF), (r(I, Cw) / 7).to(HF), (r(M, I) * 2.0 ** -12).to(HF)
    rows = torch.arange(M, device=DEV) != 3
    for where in ("x", "dh"):
        args = dict(x=x.clone(), dh=dh.clone())
        args[where][3, 5] = bad
        want = B.gated(x[rows], wg, wu, dh[rows].double() * 2.0 ** 16)
        dx, dwg, _ = D.gated_ffn_backward(args["dh"], args["x"], wg, wu)
        B.check(dx[rows], _at(want["dx"], 16), where)
        assert not torch.isfinite(dx[3]).any() and not torch.isfinite(dwg).all()
        for act in ("silu", "none"):
            b, g = wu[:, 0].contiguous(), wu[:, 1].abs().contiguous()
            want = B.linear(x[rows], wg, b, act, None, g, dh[rows].double() * 2.0 ** 16)
            dx = D.linear_epilogue_backward(args["dh"], args["x"], wg, b, act, g)[0]
            B.check(dx[rows], _at(want["dx"], 16), (where, act))
