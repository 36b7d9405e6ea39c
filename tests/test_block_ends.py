"""Dropout, the block boundary and token log probabilities on the CPU: the definitions, gradients against differences,
refusals of the dispatcher and of the C entry points, and the model's paths over them."""
import copy
import ctypes
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

import _block_bounds as B
from maba_sparse import _native as N
from maba_sparse.kernels import common as C
from maba_sparse.kernels import dispatcher as D
from maba_sparse.model import MabaBlock, MabaConfig, MabaSparseForCausalLM, get_101m_config

F64, BF, HF = torch.float64, torch.bfloat16, torch.float16
SEED = torch.tensor([2 ** 61 + 12345])


def _rand(*shape, dtype=F64, grad=True, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g, dtype=F64).to(dtype).requires_grad_(grad)


# ----------------------------------------------------------------------------- the generator and dropout


def test_philox_of_the_published_vectors():
    """philox4x32, 7 rounds, of the generator's own known answers (counter and key of zeros, and of ones)."""
    assert C.philox_words(1, 4, torch.tensor([0])).tolist() == [[0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]]


@pytest.mark.parametrize("seed,stream", [(0, 0), (1, 7), (2 ** 63 - 1, 2 ** 32 - 1), (-5, 3), (0x123456789ABCDEF, 1)])
def test_philox_words_follow_their_definition(seed, stream):
    got = C.philox_words(5, 11, torch.tensor([seed]), stream)
    assert torch.equal(got, B.words(5, 11, seed % 2 ** 64, stream))


def test_words_are_a_function_of_row_and_column():
    """Any part of the mask is the same wherever it is made: of fewer rows, of fewer columns."""
    w = C.philox_words(40, 37, SEED, 2)
    assert torch.equal(C.philox_words(40, 9, SEED, 2), w[:, :9]) and torch.equal(C.philox_words(7, 37, SEED, 2), w[:7])
    assert not torch.equal(C.philox_words(40, 37, SEED, 3), w) and not torch.equal(C.philox_words(40, 37, SEED + 1, 2), w)


@pytest.mark.parametrize("p", [0.0, 1e-11, 0.1, 0.5, 0.97, 1.0])
@pytest.mark.parametrize("dtype", [F64, torch.float32, BF, HF])
def test_dropout_keeps_and_scales(p, dtype):
    x = _rand(3, 50, 70, dtype=dtype, grad=False)
    y = D.dropout(x, p, SEED if 0 < p < 1 else None, stream=5)
    B.check(y, B.dropout(x, p, SEED, 5), "y")
    n = x.numel()
    assert abs((y == 0).double().mean() - p) < 5 * math.sqrt(p * (1 - p) / n) + 1e-9      # five standard deviations


def test_a_dropped_element_is_zero_whatever_it_was():
    x = torch.full((20, 30), math.nan)
    x[1::3], x[2::3] = math.inf, 3e38
    y = D.dropout(x, 0.5, SEED)
    keep = B.kept(x, 0.5, SEED)
    assert (y[~keep] == 0).all() and not (y[keep] == 0).any()
    assert (D.dropout(x, 1.0) == 0).all()


def test_dropout_gradient():
    x = _rand(4, 5, 9)
    assert torch.autograd.gradcheck(lambda t: D.dropout(t, 0.3, SEED, 1), (x,))
    seed = SEED.clone()
    y = D.dropout(x, 0.3, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ----------------------------------------------------------------------------- the boundary


def _tensors(M=7, Cw=12, dtype=F64, grad=True):
    t = dict(x=_rand(M, Cw), y=_rand(M, Cw, seed=1), weight=_rand(Cw, seed=2), post_weight=_rand(Cw, seed=3), gate=_rand(Cw, seed=4))
    return {k: v.detach().to(dtype).requires_grad_(grad) for k, v in t.items()}


PARTS = [("y",), ("weight",), ("y", "weight"), ("y", "gate"), ("y", "post_weight"), ("y", "weight", "gate"),
         ("y", "weight", "post_weight"), ("y", "post_weight", "gate"), ("y", "weight", "post_weight", "gate")]


@pytest.mark.parametrize("p", [0.0, 0.4, 1.0])
@pytest.mark.parametrize("parts", PARTS)
def test_boundary_gradients_against_differences(parts, p):
    t = {k: v for k, v in _tensors().items() if k in ("x", *parts)}
    names = list(t)

    def f(*a):
        out = D.residual_norm(scale=0.7, p=p, seed=SEED, stream=3, eps=1e-5, **dict(zip(names, a)))
        return tuple(o for o in out if o is not None)

    assert torch.autograd.gradcheck(f, tuple(t.values()))


@pytest.mark.parametrize("parts", PARTS)
@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
def test_boundary_values_and_backward_op(parts, dtype):
    t = {k: (v.detach() if k in ("x", *parts) else None) for k, v in _tensors(9, 33, dtype).items()}
    p = 0.25 if t["y"] is not None else 0.0
    keep = B.kept(t["x"], p, SEED, 2)
    names = dict(w="weight", wp="post_weight", g="gate")
    kw = dict(scale=0.5, p=p)
    xo, h = D.residual_norm(t["x"], t["y"], **{v: t[v] for v in names.values()}, seed=SEED, stream=2, **kw)
    want = B.boundary(t["x"], t["y"], **{k: t[v] for k, v in names.items()}, keep=keep, **kw)
    if t["y"] is None:
        assert xo is t["x"]
    else:
        B.check(xo, want["x_out"], "x_out")
    assert (h is None) == (t["weight"] is None)
    dh = _rand(9, 33, dtype=dtype, grad=False, seed=8) if h is not None else None
    if h is not None:
        B.check(h, want["h"], "h")
    dxo = _rand(9, 33, dtype=dtype, grad=False, seed=9)
    got = D.residual_norm_backward(dxo, dh, t["x"], t["y"], **{v: t[v] for v in names.values()}, seed=SEED, stream=2, **kw)
    want = B.boundary_backward(dxo, dh, t["x"], t["y"], **{k: t[v] for k, v in names.items()}, keep=keep, **kw)
    for name, v in zip(("dx", "dy", "dweight", "dpost_weight", "dgate"), got):
        if v is not None:
            B.check(v, want[name], name)
        else:
            assert name != "dx" and (name != "dy" or t["y"] is None)


def test_boundary_needs_and_missing_gradients():
    t = {k: v.detach() for k, v in _tensors().items()}
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"])
    g = _rand(7, 12, grad=False, seed=9)
    full = D.residual_norm_backward(g, None, t["x"], t["y"], **kw)
    assert torch.equal(full[0], g) and (full[2] == 0).all()
    for needs in ((1, 0, 0, 0, 0), (0, 1, 0, 1, 0), (0, 0, 0, 0, 1)):
        for a, b, n in zip(D.residual_norm_backward(g, None, t["x"], t["y"], **kw, needs=needs), full, needs):
            assert (a is None) if not n else torch.equal(a, b)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_dropped_elements_have_no_part_in_the_gates_gradient(bad, post):
    """As in the forward's own derivative, where a dropped element is zero whatever it was.  (Its own norm makes a row of one
    infinite element zero elsewhere, and a row of one NaN nothing but NaN.)"""
    if post and math.isnan(bad):
        return
    t = {k: v.detach() for k, v in _tensors().items()}
    kw = dict(post_weight=t["post_weight"] if post else None, scale=0.7, p=0.4, seed=SEED)
    keep, y = B.kept(t["x"], 0.4, SEED), t["y"].clone()
    for r in (1, 4):
        y[r, int((~keep[r]).nonzero()[0])] = bad
    gate = t["gate"].requires_grad_()
    xo, h = C.ref_residual_norm(t["x"], y, t["weight"], gate=gate, **kw)
    want, = torch.autograd.grad((xo * t["x"]).sum() + (h * t["y"]).sum(), gate)
    got = D.residual_norm_backward(t["x"], t["y"], t["x"], y, t["weight"], gate=gate.detach(), **kw)[4]
    assert want.isfinite().all()
    torch.testing.assert_close(got, want)


def test_boundary_is_torchs_modules():
    import torch.nn.functional as F
    t = {k: v.detach() for k, v in _tensors(5, 16).items()}
    xo, h = D.residual_norm(t["x"], t["y"], t["weight"], t["post_weight"], t["gate"], scale=0.3)
    want = torch.addcmul(t["x"], 0.3 * t["gate"], F.rms_norm(t["y"], (16,), t["post_weight"], eps=1e-6))
    torch.testing.assert_close(xo, want)
    torch.testing.assert_close(h, F.rms_norm(want, (16,), t["weight"], eps=1e-6))


# ----------------------------------------------------------------------------- log probabilities


def _logits(rows=6, V=23, dtype=F64, seed=0):
    x = 2 * _rand(rows, V, grad=False, seed=seed)
    t = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(seed))
    return x.to(dtype), t


def test_logprob_gradients_against_differences():
    x, t = _logits()
    t[2] = -100
    x.requires_grad_()
    assert torch.autograd.gradcheck(lambda v: D.token_logprobs(v, t, temperature=0.7, top=3)[:3], (x,))
    assert torch.autograd.gradcheck(lambda v: D.token_logprobs(v, t)[1], (x,))


@pytest.mark.parametrize("dtype", [torch.float32, BF, HF])
@pytest.mark.parametrize("V", [1, 2, 64, 301])
def test_logprobs_and_their_backward_op(V, dtype):
    x, t = _logits(9, V, dtype)
    if V > 4:
        x[0, ::2] = -math.inf
        x[1] = -math.inf
        x[1, 3] = 1.0
    x[2], x[3] = -math.inf, torch.finfo(dtype).min
    x[4] = 0
    t[5] = -1
    k = min(V, 5)
    lead = (3, 3)
    got = D.token_logprobs(x.view(*lead, V), t.view(lead), temperature=0.8, top=k)
    want = B.logprobs(x, t, 0.8, k)
    for name, v in zip(("logp", "entropy", "lse", "top_logp", "top_ids"), got):
        assert v.shape[:2] == lead
        v = v.reshape(9, *v.shape[2:])
        if name == "top_ids":
            assert torch.equal(v, want[name])
        else:
            rows = [i for i in range(9) if name != "lse" or i != 3]          # the lowest value over T leaves fp32's range
            B.check(v[rows], tuple(w[rows] for w in want[name]), name)
    g = [_rand(9, dtype=torch.float32, grad=False, seed=i) for i in range(3)]
    lse, H = (want[n][0].float() for n in ("lse", "entropy"))
    lse[3] = torch.finfo(torch.float32).min
    B.check(D.token_logprobs_backward(*g, x, t, lse, H, 0.8), B.logprobs_backward(*g, x, t, 0.8), "dlogits")


@pytest.mark.parametrize("dt", [torch.float32, BF, HF])
@pytest.mark.parametrize("V,below", [(3, 9), (700, 12), (700, 17)])
@pytest.mark.parametrize("lse", [-200, 0, 30, 120, 240])
def test_gradient_of_a_likely_target_is_the_others_sum(V, below, lse, dt):
    """1 - p from a p near 1, or from an lse far from zero, would keep few of its bits or none."""
    x, t, H, want, wantH = B.likely_rows(V, lse, below, dt)
    x.requires_grad_()
    d, = torch.autograd.grad(-D.token_logprobs(x, t)[0].sum(), x)
    B.check(-d.gather(1, t[:, None])[:, 0], want, "at the target")


def test_rows_without_mass_have_no_gradient_whatever_comes_in():
    """A loss of lse^2 under torch.where sends NaN into such a row."""
    x, t = _logits(12, 300, torch.float32, seed=9)
    x[::3] = -math.inf
    x.requires_grad_()
    logp, ent, lse, _, _ = D.token_logprobs(x, t)
    z = torch.where(lse > -math.inf, lse ** 2, torch.zeros_like(lse))
    (z.sum() + ent.sum() - torch.where(lse > -math.inf, logp, torch.zeros_like(logp)).sum()).backward()
    assert (x.grad[::3] == 0).all() and x.grad.isfinite().all() and (x.grad[1] != 0).any()
    nan = torch.full_like(lse, math.nan)
    d = D.token_logprobs_backward(nan, nan, nan, x.detach(), t, lse.detach(), ent.detach())
    assert (d[::3] == 0).all() and d[1].isnan().all()


def test_rows_of_nan_and_targets_past_the_vocabulary():
    x, t = _logits(4, 10, torch.float32)
    x[1, 4], x[2, 4] = math.nan, math.inf
    t[3] = 10
    x.requires_grad_()
    logp, H, lse, tl, ti = D.token_logprobs(x, t, top=3)
    assert logp.isnan().tolist() == [False, True, True, True] and H.isnan().tolist() == [False, True, True, False]
    assert ti[1, 0] == 4 and ti[2, 0] == 4 and tl[1].isnan().all()
    d, = torch.autograd.grad(logp[0] + logp[3], x)
    assert not d[0].isnan().any() and d[3].isnan().all() and (d[0].sum().abs() < 1e-6)


def test_alternatives_are_ordered_by_value_then_index():
    x = torch.tensor([[1.0, 3.0, -0.0, 3.0, 0.0, -math.inf, 1.0]])
    ids = D.token_logprobs(x, torch.tensor([0]), top=7)[4]
    assert ids.tolist() == [[1, 3, 0, 6, 2, 4, 5]]


def test_logprobs_are_torchs():
    x, t = _logits(8, 40)
    logp, H, lse, _, _ = D.token_logprobs(x, t, temperature=1.3)
    torch.testing.assert_close(logp, torch.log_softmax(x / 1.3, -1).gather(1, t[:, None])[:, 0])
    torch.testing.assert_close(H, torch.distributions.Categorical(logits=x / 1.3).entropy())
    torch.testing.assert_close(lse, torch.logsumexp(x / 1.3, -1))


# ----------------------------------------------------------------------------- what all of them share


def test_double_backward_is_refused():
    x = _rand(4, 8)
    t = torch.zeros(4, dtype=torch.long)
    for y in (D.dropout(x, 0.5, SEED), D.residual_norm(x, x * 2, x.new_ones(8))[1], D.token_logprobs(x, t)[0]):
        g, = torch.autograd.grad((y * y).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()


def test_tangents_are_not_dropped():
    from torch.autograd import forward_ad
    x, t = _rand(4, 8, grad=False), _rand(4, 8, grad=False, seed=5)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        for y in (D.dropout(dual, 0.5, SEED), D.residual_norm(dual, dual, x.new_ones(8))[1],
                  D.token_logprobs(dual, torch.zeros(4, dtype=torch.long))[0]):
            assert forward_ad.unpack_dual(y).tangent is not None


@pytest.mark.parametrize("xt,yt", [(torch.float32, BF), (BF, torch.float32), (HF, HF)])
def test_autocast_takes_the_widest_type(xt, yt):
    t = {k: v.detach() for k, v in _tensors(6, 16).items()}
    x, y = t["x"].to(xt).requires_grad_(), t["y"].to(yt).requires_grad_()
    w = t["weight"].float()
    with torch.autocast("cpu", BF):
        xo, h = D.residual_norm(x, y, weight=w)
    assert xo.dtype == h.dtype == torch.float32
    (xo.sum() + h.sum()).backward()
    assert x.grad.dtype == xt and y.grad.dtype == yt
    B.check(xo.detach(), B.boundary(x.detach().float(), y.detach().float(), w)["x_out"], "x_out")
    if xt != yt:
        with pytest.raises(TypeError, match="dtypes must match"):
            D.residual_norm(x, y)


@pytest.mark.parametrize("kw,error", [
    (dict(p=-0.1), ValueError), (dict(p=1.5), ValueError), (dict(p=math.nan), ValueError), (dict(p=0.5, seed=None), ValueError),
    (dict(p=0.5, seed=torch.tensor([1], dtype=torch.int32)), TypeError), (dict(p=0.5, seed=torch.tensor([1, 2])), ValueError),
    (dict(p=0.5, stream=-1), ValueError), (dict(p=0.5, stream=2 ** 32), ValueError),
    (dict(p=0.5, seed=torch.empty(1, dtype=torch.int64, device="meta")), RuntimeError),
])
def test_dropout_refusals(kw, error):
    x = torch.zeros(3, 4)
    kw = {"seed": SEED, **kw}
    with pytest.raises(error):
        D.dropout(x, **kw)
    with pytest.raises(error):
        D.residual_norm(x, x, **kw)
    with pytest.raises(error):
        D.residual_norm_backward(x, None, x, x, **kw)


@pytest.mark.parametrize("x,error", [(torch.zeros(3, 4, dtype=torch.int32), TypeError), (torch.zeros(()), ValueError),
                                     (torch.zeros(3, 0), ValueError)])
def test_inputs_without_channels_or_of_other_types(x, error):
    with pytest.raises(error):
        D.dropout(x, 0.0)
    with pytest.raises(error):
        D.residual_norm(x, x)
    with pytest.raises(error):
        D.token_logprobs(x, torch.zeros(x.shape[:-1], dtype=torch.long))


@pytest.mark.parametrize("kw,error", [
    (dict(y=torch.zeros(4, 12, dtype=F64)), ValueError), (dict(y=torch.zeros(7, 12)), TypeError),
    (dict(weight=torch.zeros(11, dtype=F64)), ValueError), (dict(gate=torch.zeros(1, 12, dtype=F64)), ValueError),
    (dict(post_weight=torch.zeros(12)), TypeError), (dict(y=None), ValueError),
    (dict(y=torch.zeros(7, 12, dtype=F64, device="meta")), RuntimeError),
])
def test_boundary_refusals(kw, error):
    t = {k: v.detach() for k, v in _tensors().items()}
    with pytest.raises(error):
        D.residual_norm(**{**t, **kw})


def test_boundary_backward_refusals():
    t = {k: v.detach() for k, v in _tensors().items()}
    g, x, y, w = t["x"], t["x"], t["y"], t["weight"]
    for args, kw, error in (((None, None, x), {}, ValueError), ((g, g, x), {}, ValueError), ((g, None, x), dict(post_weight=w), ValueError),
                            ((g, None, x), dict(gate=w), ValueError), ((g[:3], None, x, y), {}, ValueError),
                            ((g.float(), None, x, y), {}, TypeError), ((g, None, x, y), dict(needs=(1, 1)), ValueError)):
        with pytest.raises(error):
            D.residual_norm_backward(*args, **kw)


@pytest.mark.parametrize("kw,error", [
    (dict(targets=torch.zeros(5, dtype=torch.long)), ValueError), (dict(targets=torch.zeros(6, dtype=torch.int32)), TypeError),
    (dict(temperature=0.0), ValueError), (dict(temperature=-1.0), ValueError), (dict(temperature=math.nan), ValueError),
    (dict(temperature=math.inf), ValueError), (dict(top=-1), ValueError), (dict(top=24), ValueError),
    (dict(targets=torch.zeros(6, dtype=torch.long, device="meta")), RuntimeError),
])
def test_logprob_refusals(kw, error):
    x, t = _logits()
    with pytest.raises(error):
        D.token_logprobs(**{"logits": x, "targets": t, **kw})


def test_logprob_backward_refusals():
    x, t = _logits(dtype=torch.float32)
    g = torch.zeros(6)
    for args, error in (((None, None, None, x, t, g, g), ValueError), ((g.double(), None, None, x, t, g, g), TypeError),
                        ((g[:5], None, None, x, t, g, g), ValueError), ((g, None, None, x, t, g, g[:4]), ValueError),
                        ((g, None, None, x, t[:2], g, g), ValueError)):
        with pytest.raises(error):
            D.token_logprobs_backward(*args)


def test_no_rows():
    z = torch.zeros(0, 8, dtype=F64, requires_grad=True)
    w = torch.ones(8, dtype=F64, requires_grad=True)
    xo, h = D.residual_norm(z, z, w, w, w, p=0.5, seed=SEED)
    h.sum().backward()
    assert (w.grad == 0).all() and xo.shape == (0, 8)
    assert D.dropout(z, 0.5, SEED).shape == (0, 8)
    out = D.token_logprobs(z, torch.zeros(0, dtype=torch.long), top=2)
    assert [tuple(t.shape) for t in out] == [(0,)] * 3 + [(0, 2)] * 2


# ----------------------------------------------------------------------------- the C entry points


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.skip("libmaba_hip.so not built (run __graft_entry__.build())")
    return N.load()


def _t(shape, dtype=N.MABA_BF16, strides=None, data=0x10000):
    t = N.MabaTensor()
    t.data, t.dtype, t.ndim = data, dtype, len(shape)
    if strides is None:
        strides, acc = [], 1
        for s in reversed(shape):
            strides.insert(0, acc)
            acc *= s
    for i, (s, st) in enumerate(zip(shape, strides)):
        t.shape[i], t.stride[i] = s, st
    return ctypes.byref(t)


A, Bt, Ct, Dt, Et = (i << 24 for i in range(1, 6))     # far apart; never read
F32 = N.MABA_F32


@pytest.mark.parametrize("x,p,seed,out,rc,text", [
    (None, 0.1, 64, _t([4, 8], data=Bt), 1, b"missing"),
    (_t([4, 8, 1], data=A), 0.1, 64, _t([4, 8], data=Bt), 1, b"2D"),
    (_t([-1, 8], data=A), 0.1, 64, _t([-1, 8], data=Bt), 1, b"negative size"),
    (_t([4, 8], dtype=N.MABA_F64, data=A), 0.1, 64, _t([4, 8], data=Bt), 2, b"f32, f16 or bf16"),
    (_t([4, 8], data=A), 1.1, 64, _t([4, 8], data=Bt), 1, b"[0, 1]"),
    (_t([4, 8], data=A), float("nan"), 64, _t([4, 8], data=Bt), 1, b"[0, 1]"),
    (_t([4, 8], data=A), 0.1, None, _t([4, 8], data=Bt), 1, b"seed"),
    (_t([4, 8], data=A), 0.1, 68, _t([4, 8], data=Bt), 1, b"seed"),
    (_t([4, 8], data=A), 0.1, 64, _t([4, 7], data=Bt), 1, b"expected"),
    (_t([4, 8], data=A), 0.1, 64, _t([4, 8], dtype=F32, data=Bt), 2, b"dtype"),
    (_t([4, 8], data=A), 0.1, 64, _t([4, 8], data=A + 16), 1, b"overlap"),
    (_t([4, 8], data=A), 0.1, 64, _t([4, 8], strides=[4, 1], data=Bt), 1, b"overlap"),
    (_t([4, 8], strides=[1, 4], data=A), 0.1, 64, _t([4, 8], data=Bt), 1, b"unit column stride"),
])
def test_c_dropout_refusals(lib, x, p, seed, out, rc, text):
    assert lib.maba_hip_dropout(x, p, seed, 0, out, None) == rc
    assert text in lib.maba_hip_last_error()


def test_c_no_rows_is_fine(lib):
    none = _t([0, 8], data=0)
    assert lib.maba_hip_dropout(none, 0.1, 64, 0, none, None) == 0
    assert lib.maba_hip_residual_norm(none, none, None, None, None, 1.0, 0.0, None, 0, 1e-6, none, None, None) == 0
    assert lib.maba_hip_residual_norm_backward(none, None, none, None, None, None, None, 1.0, 0.0, None, 0, 1e-6, none, None, None, None,
                                               None, None, 0, None) == 0
    v = _t([0], dtype=F32, data=0)
    assert lib.maba_hip_token_logprobs(none, _t([0], dtype=N.MABA_I64, data=0), 1.0, v, v, v, None, None, None) == 0


def _boundary(lib, x=None, y="y", w="w", wp=None, g=None, p=0.0, seed=None, xo="xo", h="h"):
    pick = dict(y=_t([4, 8], data=Bt), w=_t([8], data=Ct), xo=_t([4, 8], data=Dt), h=_t([4, 8], data=Et))
    y, w, xo, h = (pick.get(v, v) if isinstance(v, str) else v for v in (y, w, xo, h))
    return lib.maba_hip_residual_norm(x or _t([4, 8], data=A), y, w, wp, g, 1.0, p, seed, 0, 1e-6, xo, h, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(y=_t([4, 7], data=Bt)), 1, b"y is"), (dict(y=_t([4, 8], dtype=F32, data=Bt)), 2, b"dtype"),
    (dict(y=None), 1, b"go with y"), (dict(y=None, xo=None, g=_t([8], data=Ct)), 1, b"go with y"),
    (dict(x=_t([-1, 8], data=A)), 1, b"negative size"), (dict(h=None), 1, b"go together"), (dict(w=None), 1, b"go together"), (dict(w=None, h=None, xo=None), 1, b"nothing to compute"),
    (dict(w=_t([7], data=Ct)), 1, b"weight must be"), (dict(wp=_t([8], strides=[2], data=Ct)), 1, b"unit stride"),
    (dict(g=_t([8], dtype=F32, data=Ct)), 2, b"gate"), (dict(p=0.5), 1, b"seed"),
    (dict(xo=_t([4, 8], data=A + 2)), 1, b"overlap"), (dict(xo=_t([4, 8], data=Bt)), 1, b"overlap"), (dict(h=_t([4, 8], data=A)), 1, b"overlap"),
    (dict(h=_t([4, 8], data=Dt)), 1, b"overlap"), (dict(xo=_t([4, 8], strides=[7, 1], data=Dt)), 1, b"overlap"),
])
def test_c_boundary_refusals(lib, kw, rc, text):
    assert _boundary(lib, **kw) == rc
    assert text in lib.maba_hip_last_error()


def test_c_boundary_width(lib):
    wide = [_t([2, 8193], data=d) for d in (A, Bt, Dt)]
    assert lib.maba_hip_residual_norm(wide[0], wide[1], None, None, None, 1.0, 0.0, None, 0, 1e-6, wide[2], None, None) == 3
    assert b"8192" in lib.maba_hip_last_error()
    assert lib.maba_hip_residual_norm_backward_workspace_size(wide[0], 7) == 0


def test_c_boundary_backward_refusals(lib):
    t = {n: _t([4, 8], data=d) for n, d in zip("dhxyo", (A, Bt, Ct, Dt, Et))}
    w, far = _t([8], data=6 << 24), 7 << 24

    def call(dxo=t["d"], dh=t["h"], x=t["x"], y=t["y"], weight=w, wp=None, g=None, p=0.0, seed=None, dx=t["o"], dy=None, dw=None, dwp=None,
             dg=None, ws=None, size=0):
        return lib.maba_hip_residual_norm_backward(dxo, dh, x, y, weight, wp, g, 1.0, p, seed, 0, 1e-6, dx, dy, dw, dwp, dg, ws, size, None)

    for kw, rc, text in ((dict(dxo=None, dh=None), 1, b"required"), (dict(weight=None), 1, b"goes with weight"),
                         (dict(y=None, wp=w), 1, b"go with y"), (dict(y=None, dy=_t([8, 8], data=far)), 1, b"dy"), (dict(y=None, dx=None, dy=t["o"]), 1, b"dy goes with y"), (dict(dg=_t([8], data=far)), 1, b"missing parameter"),
                         (dict(dwp=_t([8], data=far)), 1, b"missing parameter"), (dict(dx=t["d"]), 1, b"overlaps an input"),
                         (dict(dy=t["o"]), 1, b"outputs overlap"), (dict(dw=_t([8], data=far)), 5, b"workspace"),
                         (dict(dw=_t([8], data=far), ws=(8 << 24) + 8, size=1 << 20), 1, b"16-byte aligned"),
                         (dict(p=0.3), 1, b"seed"), (dict(dxo=_t([4, 8], dtype=N.MABA_F16, data=A)), 2, b"dtype"),
                         (dict(dx=_t([4, 8], strides=[0, 1], data=Et)), 1, b"overlap")):
        assert call(**kw) == rc, kw
        assert text in lib.maba_hip_last_error(), (kw, lib.maba_hip_last_error())


def test_c_boundary_backward_takes_x_without_data_where_h_has_no_gradient(lib):
    """The calls stop at the workspace, behind all checks of tensors."""
    d, h, x, y, out = (_t([4, 8], data=p) for p in (A, Bt, 0, Ct, Et))
    w, dg = _t([8], data=6 << 24), _t([8], data=7 << 24)
    call = lambda dh, x, dx: lib.maba_hip_residual_norm_backward(d, dh, x, y, w, None, w, 1.0, 0.0, None, 0, 1e-6, dx, None, None, None, dg,
                                                                 None, 0, None)
    for dh, xx, dx, rc, text in ((None, x, out, 5, b"workspace"), (h, x, out, 1, b"x has no data"),
                                 (None, _t([4, 8], data=Et), out, 5, b"workspace"), (h, _t([4, 8], data=Et), out, 1, b"overlaps an input"),
                                 (None, _t([4, 7], data=0), out, 1, b"expected")):
        assert call(dh, xx, dx) == rc and text in lib.maba_hip_last_error(), lib.maba_hip_last_error()


def test_c_workspace_sizes(lib):
    size = lib.maba_hip_residual_norm_backward_workspace_size
    x = _t([1000, 640], data=A)
    assert size(x, 0) == 0 and size(None, 7) == 0 and size(x, 1) >= 640 * 4
    assert size(x, 7) == 3 * size(x, 1) == 3 * size(x, 4) and size(x, 3) == 2 * size(x, 1)
    assert size(_t([0, 640], data=0), 1) >= 640 * 4


def _logprobs(lib, x=None, t=None, T=1.0, outs=None, tl=None, ti=None):
    outs = outs or [_t([4], dtype=F32, data=d) for d in (Ct, Dt, Et)]
    return lib.maba_hip_token_logprobs(x or _t([4, 8], data=A), t or _t([4], dtype=N.MABA_I64, data=Bt), T, *outs, tl, ti, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(x=_t([8], data=A)), 1, b"[M,V] or [B,L,V]"), (dict(x=_t([4, 8], dtype=N.MABA_F64, data=A)), 2, b"f32, f16 or bf16"),
    (dict(x=_t([4, 0], data=A)), 1, b"empty"), (dict(x=_t([4, 8], strides=[1, 4], data=A)), 1, b"unit column stride"),
    (dict(x=_t([4, 8], strides=[-8, 1], data=A)), 1, b"negative"), (dict(x=_t([4, 8], data=0)), 1, b"no data"),
    (dict(T=0.0), 1, b"temperature"), (dict(T=float("nan")), 1, b"temperature"), (dict(T=1e-40), 1, b"temperature"),
    (dict(t=_t([5], dtype=N.MABA_I64, data=Bt)), 1, b"targets"), (dict(t=_t([4], dtype=N.MABA_I32, data=Bt)), 2, b"targets"),
    (dict(t=_t([4], dtype=N.MABA_I64, strides=[2], data=Bt)), 1, b"targets"),
    (dict(tl=_t([4, 2], dtype=F32, data=6 << 24)), 1, b"go together"),
    (dict(tl=_t([4, 9], dtype=F32, data=6 << 24), ti=_t([4, 9], dtype=N.MABA_I64, data=7 << 24)), 1, b"between 1 and V"),
    (dict(tl=_t([4, 2], dtype=F32, data=6 << 24), ti=_t([4, 2], dtype=N.MABA_I32, data=7 << 24)), 2, b"i64"),
    (dict(tl=_t([4, 3], dtype=F32, data=6 << 24), ti=_t([4, 2], dtype=N.MABA_I64, data=7 << 24)), 1, b"contiguous"),
    (dict(x=_t([1 << 40, 1 << 40, 8], strides=[0, 0, 1], data=A)), 3, b"too many rows"),
    (dict(x=_t([1 << 32, 1 << 32, 8], strides=[0, 0, 1], data=A)), 3, b"too many rows"),
    (dict(x=_t([-1, 8], data=A)), 1, b"negative size"),
    (dict(x=_t([4, 100], data=A), tl=_t([4, 65], dtype=F32, data=6 << 24), ti=_t([4, 65], dtype=N.MABA_I64, data=7 << 24)), 3, b"64"),
])
def test_c_logprob_refusals(lib, kw, rc, text):
    assert _logprobs(lib, **kw) == rc
    assert text in lib.maba_hip_last_error()


def test_c_logprob_backward_refusals(lib):
    x, t, v = _t([4, 8], data=A), _t([4], dtype=N.MABA_I64, data=Bt), _t([4], dtype=F32, data=Ct)
    call = lib.maba_hip_token_logprobs_backward
    out = _t([4, 8], data=Et)
    for args, rc, text in (((v, None, None, x, t, v, v, 1.0, None), 1, b"dlogits"), ((v, None, None, x, t, None, v, 1.0, out), 1, b"lse"),
                           ((v, None, None, x, t, v, v, 1.0, _t([4, 8], dtype=F32, data=Et)), 2, b"type"),
                           ((v, None, None, x, t, v, v, 1.0, _t([4, 7], data=Et)), 1, b"rows"),
                           ((v, None, None, x, t, v, v, 1.0, _t([4, 8], strides=[7, 1], data=Et)), 1, b"overlap"),
                           ((v, None, None, x, t, v, v, 1.0, _t([2, 2, 8], strides=[8, 8, 1], data=Et)), 1, b"overlap"),
                           ((v, None, None, x, t, v, v, 1.0, _t([4, 8], data=A + 2)), 1, b"overlap"),
                           ((_t([3], dtype=F32, data=Ct), None, None, x, t, v, v, 1.0, out), 1, b"dlogp")):
        assert call(*args, None) == rc
        assert text in lib.maba_hip_last_error()


def test_native_binding_declines_what_is_not_on_a_gpu(lib):
    m = N.binding()
    x = torch.randn(3, 8)
    assert m.dropout(x, 0.5, SEED, 0) is None
    assert m.residual_norm(x, x, None, None, None, 1.0, 0.0, None, 0, 1e-6) is None
    assert m.token_logprobs(x, torch.zeros(3, dtype=torch.long), 1.0, 0) is None


# ----------------------------------------------------------------------------- the model


SMALL = dict(dim=128, n_layers=4, n_heads=2, d_head=64, vocab_size=97, d_emb=16, d_c=32, d_idx=16, intermediate_size=96, top_k=4,
             dist_lambda=0.1)


def _model(**kw):
    torch.manual_seed(0)
    return MabaSparseForCausalLM(get_101m_config(**SMALL, **kw)).init_normal(0.1)


def _ids(L=70):
    return torch.randint(0, 97, (2, L), generator=torch.Generator().manual_seed(1))


@pytest.mark.parametrize("fused_ffn", [False, True])
def test_fused_boundaries_train_like_the_plain_model(fused_ffn):
    plain, fused = _model(fused_ffn=fused_ffn).double(), _model(fused_ffn=fused_ffn, fused_boundary=True).double()
    fused.load_state_dict(plain.state_dict())
    ids = _ids()
    losses = [-m.score(ids)[0].mean() for m in (plain, fused)]
    torch.testing.assert_close(losses[0], losses[1], rtol=1e-9, atol=1e-12)
    for loss in losses:
        loss.backward()
    n = 0
    for (name, a), b in zip(plain.named_parameters(), fused.parameters()):
        assert (a.grad is None) == (b.grad is None), name
        if a.grad is not None:
            n += 1
            torch.testing.assert_close(b.grad, a.grad, rtol=1e-6, atol=1e-9)
    assert n > 40


def test_score_is_the_log_softmax_of_the_next_token():
    m, ids = _model().eval(), _ids(30)
    with torch.no_grad():
        logp, H, lse, tl, ti = m.score(ids, temperature=0.9, top=4)
        lp = torch.log_softmax(m(ids)[0][:, :-1].double() / 0.9, -1)
    assert logp.shape == H.shape == (2, 29) and ti.shape == (2, 29, 4)
    torch.testing.assert_close(logp.double(), lp.gather(-1, ids[:, 1:, None])[..., 0], rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(tl.double(), lp.topk(4, -1).values, rtol=1e-5, atol=1e-5)
    with pytest.raises(ValueError, match="two tokens"):
        m.score(ids[:, :1])


def test_post_norm_scale_and_dropout_of_a_block_by_hand():
    import torch.nn.functional as F
    m = _model(post_norm=True, residual_scale=0.5).double().eval()
    blk = m.layers[0]
    x = torch.randn(2, 9, 128, dtype=F64)
    with torch.no_grad():
        for p in (blk.post_norm1.weight, blk.post_norm2.weight):
            p.uniform_(0.5, 1.5)
        norm = lambda t, n: F.rms_norm(t, (128,), n.weight, eps=n.eps)
        mo = blk.mixer(norm(x, blk.norm1))[0]
        a = x + 0.5 * torch.sigmoid(blk.res_gate1) * norm(mo, blk.post_norm1)
        want = a + 0.5 * torch.sigmoid(blk.res_gate2) * norm(blk.ffn(norm(a, blk.norm2)), blk.post_norm2)
        torch.testing.assert_close(blk(x)[0], want)


def test_dropout_of_the_model():
    m, ids = _model(dropout=0.2), _ids()
    assert "dropout_seed" not in m.state_dict()
    start = m.dropout_seed.clone()
    a, b = (m(ids)[0] for _ in range(2))
    assert torch.equal(m.dropout_seed, start + 2) and not torch.equal(a, b)
    m.dropout_seed.copy_(start)
    assert torch.equal(m(ids)[0], a)
    m(ids)[0].sum().backward()                                    # the seed has moved on by then
    m.eval()
    with torch.no_grad():
        seed = m.dropout_seed.clone()
        assert torch.equal(m(ids)[0], m(ids)[0]) and torch.equal(m.dropout_seed, seed)


def test_the_models_seed_moves_with_it():
    m = _model(dropout=0.2)
    assert "dropout_seed" not in dict(m.named_buffers()) and not any("dropout_seed" in k for k in m.state_dict())
    c = copy.deepcopy(m)
    c.dropout_seed += 1
    assert not torch.equal(c.dropout_seed, m.dropout_seed)
    assert m.to("meta").dropout_seed.device.type == "meta" and c.bfloat16().dropout_seed.dtype == torch.int64
    assert "dropout_seed" not in _model().__dict__


def test_a_pass_that_is_run_again_takes_the_seed_it_is_given():
    from torch.utils.checkpoint import checkpoint
    m, ids = _model(dropout=0.4).double(), _ids(40)
    p, grads = m.final_norm.weight, []
    seed = m.next_dropout_seed()
    for run in (lambda: m(ids, drop=seed)[0], lambda: checkpoint(lambda i: m(i, drop=seed)[0], ids, use_reentrant=False)):
        before = m.dropout_seed.clone()
        grads.append(torch.autograd.grad((run() ** 2).sum(), [p, m.layers[0].res_gate1]))
        assert torch.equal(m.dropout_seed, before)
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(ids, drop=seed)[0], m(ids)[0])


DATA_PARALLEL = """
import sys
import torch
import torch.distributed as dist
from maba_sparse.model import MabaSparseForCausalLM, get_101m_config

rank, store = int(sys.argv[1]), sys.argv[2]
dist.init_process_group("gloo", init_method="file://" + store, rank=rank, world_size=2)
torch.manual_seed(0)
m = MabaSparseForCausalLM(get_101m_config(dim=64, n_layers=2, n_heads=1, d_head=64, vocab_size=32, d_emb=16, intermediate_size=48,
                                          dropout=0.5))
m.dropout_seed.fill_(100 + rank)
ddp = torch.nn.parallel.DistributedDataParallel(m, find_unused_parameters=True)
ids = torch.arange(24).view(2, 12)
outs = [ddp(ids)[0] for _ in range(2)]
outs[-1].sum().backward()
assert m.dropout_seed.tolist() == [102 + rank], m.dropout_seed
both = [torch.empty_like(outs[0]) for _ in range(2)]
dist.all_gather(both, outs[0].detach())
assert not torch.equal(*both)                   # each rank by its own masks
g = m.final_norm.weight.grad
grads = [torch.empty_like(g) for _ in range(2)]
dist.all_gather(grads, g)
assert torch.equal(*grads) and g.any()          # and one gradient
dist.destroy_process_group()
"""


def test_ranks_of_a_data_parallel_job_drop_by_their_own_seeds(tmp_path):
    script = tmp_path / "rank.py"
    script.write_text(DATA_PARALLEL)
    package = os.path.dirname(os.path.dirname(os.path.abspath(N.__file__)))
    env = dict(os.environ, PYTHONPATH=package, GLOO_SOCKET_IFNAME="lo", OMP_NUM_THREADS="2")
    ranks = [subprocess.Popen([sys.executable, str(script), str(r), str(tmp_path / "store")], env=env, stdout=subprocess.PIPE,
                              stderr=subprocess.STDOUT, text=True) for r in range(2)]
    try:
        for r in ranks:
            out, _ = r.communicate(timeout=240)
            assert r.returncode == 0, out
    finally:
        for r in ranks:
            r.kill()


def test_generation_with_post_norms_equals_state_passing():
    m, ids = _model(post_norm=True, residual_scale=0.7).eval(), _ids(150)
    with torch.no_grad():
        got = m.generate_greedy(ids, 6)
        logits, states = m(ids)
        tok, ref = logits[:, -1].argmax(-1, keepdim=True), []
        for _ in range(6):
            ref.append(tok)
            logits, states = m.step(tok, past_states=states)
            tok = logits[:, -1].argmax(-1, keepdim=True)
    assert torch.equal(got, torch.cat(ref, dim=1))


@pytest.mark.parametrize("kw,fits", [({}, True), (dict(fused_boundary=True), True), (dict(dropout=0.1), True), (dict(post_norm=True), False),
                                     (dict(residual_scale=0.5), False)])
def test_the_decode_linears_of_a_serving_step_take_plain_boundaries_only(kw, fits):
    """Their input stage has no norm on a half's output and no scale: a step over them would leave both out."""
    from maba_sparse.model import _decode_linear_fits
    m = MabaSparseForCausalLM(get_101m_config(n_layers=4, vocab_size=1024, top_k=4, **kw)).bfloat16()
    assert _decode_linear_fits(m) == fits


def test_generation_drops_nothing():
    m, ids = _model(dropout=0.5), _ids(100)
    seed = m.dropout_seed.clone()
    # the prompt's logits (the layers keep no decode caches while training, so later ones differ for that)
    got, want = (m.train(mode).generate_greedy(ids, 2, return_logits=True)[1][:, 0] for mode in (True, False))
    assert torch.equal(got, want) and torch.equal(m.dropout_seed, seed)
    m.train()
    assert not torch.equal(m(ids)[0], m(ids)[0])


def test_generation_leaves_a_training_step_in_another_thread_its_dropout():
    m, ids = _model(dropout=0.5), _ids(80)
    seeds = []

    def meanwhile(*_):
        t = threading.Thread(target=lambda: seeds.append(m.next_dropout_seed()))
        t.start()
        t.join()

    start = m.dropout_seed.clone()
    hook = m.embeddings.register_forward_hook(meanwhile)             # within the prompt's pass
    m.generate_greedy(ids, 1)
    hook.remove()
    assert len(seeds) == 1 and torch.equal(seeds[0], start)


def test_blocks_of_configs_and_modules_from_before_the_fields():
    from types import SimpleNamespace
    cfg = MabaConfig(dim=64, n_heads=1, intermediate_size=40, n_layers=1)
    new = ("fused_boundary", "post_norm", "residual_scale", "dropout")
    blk = MabaBlock(SimpleNamespace(**{k: v for k, v in vars(cfg).items() if k not in new}), 0)
    x = torch.randn(2, 6, 64)
    want = blk(x)[0]
    for name in ("boundary", "residual_scale", "dropout"):
        del blk.__dict__[name]
    assert torch.equal(blk(x)[0], want)
