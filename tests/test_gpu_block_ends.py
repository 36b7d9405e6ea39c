"""Dropout, the block boundary and token log probabilities on the GPU against 64 bits: values, gradients, masks, strides,
streams, graph replays and refusals.  The bounds of ``_block_bounds`` are elementwise."""
import gc
import math
import threading

import pytest
import torch

import _block_bounds as B
from maba_sparse import _native as N
from maba_sparse.kernels import common as C
from maba_sparse.kernels import dispatcher as D
from maba_sparse.kernels import hip_backend as H

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF, HF, FL]


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    """A kernel that raises fails the test instead of falling back."""
    monkeypatch.setenv("MABA_STRICT_BACKEND", "1")


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=DEV)


SEED = torch.tensor([0x1234567890ABCDE])


def _seed():
    return SEED.to(DEV)


def _inside(t, left, right, rows=0):
    """``t``'s values as a view of a larger tensor of NaN."""
    big = torch.full((t.shape[0] + 2 * rows, t.shape[1] + left + right), math.nan, dtype=t.dtype, device=t.device)
    v = big[rows:rows + t.shape[0], left:left + t.shape[1]]
    v.copy_(t)
    return v


def _around_is_nan(v, left, right):
    base = v._base
    for part in (base[:, :left], base[:, base.shape[1] - right:] if right else base[:, :0]):
        assert part.isnan().all()


# ----------------------------------------------------------------------------- dropout


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (1, 4), (7, 8), (2, 3, 33), (64, 640), (5, 2049), (1000, 77), (9, 8200), (3001, 1001)])
@pytest.mark.parametrize("p", [0.0, 1e-6, 0.1, 0.5, 0.999, 1.0])
def test_dropout_of_all_sizes(shape, p, dt):
    x = _gen(sum(shape))(*shape).to(dt)
    y = D.dropout(x, p, _seed() if 0 < p < 1 else None, stream=3)
    B.check(y, B.dropout(x, p, _seed(), 3), "y")
    assert torch.equal(y == 0, ~B.kept(x, p, _seed(), 3) | (x == 0))


def test_dropout_gradient_is_the_same_mask():
    r = _gen(1)
    x, dy = r(300, 200).to(BF).requires_grad_(), r(300, 200).to(BF)
    y = D.dropout(x, 0.3, _seed())
    d, = torch.autograd.grad(y, x, dy)
    assert torch.equal(d, D.dropout(dy, 0.3, _seed()))
    e, = torch.autograd.grad(D.dropout(x, 0.3, _seed()).sum(), x)             # a broadcast gradient
    assert torch.equal(e != 0, B.kept(x, 0.3, _seed()))


def test_dropped_elements_are_zero_whatever_they_were():
    x = torch.full((40, 72), math.nan, device=DEV, dtype=HF)
    x[1::3], x[2::3] = math.inf, -math.inf
    y = D.dropout(x, 0.5, _seed())
    keep = B.kept(x, 0.5, _seed())
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()
    z = torch.zeros(40, 72, device=DEV, dtype=HF)
    xo, _ = D.residual_norm(z, x, p=0.5, seed=_seed())
    assert torch.equal(xo[~keep], z[~keep]) and not torch.isfinite(xo[keep]).any()
    _, dy, *_ = D.residual_norm_backward(x, None, z, p=0.5, seed=_seed())
    assert (dy[~keep] == 0).all() and not torch.isfinite(dy[keep]).any()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("M,Cw", [(40, 72), (40, 37), (9, 2056)])
def test_dropped_elements_have_no_part_in_the_gates_gradient(M, Cw, post, dt):
    """(Its own norm makes a row of one infinite element zero elsewhere, and a row of one NaN nothing but NaN.)"""
    t = _tensors(M, Cw, dt, PARTS[-1] if post else PARTS[2], seed=12)
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"], p=0.5, seed=_seed())
    drop, x, y = ~B.kept(t["y"], 0.5, _seed()), t["x"], t["y"]
    y[1] = y[2] = y[3] = 0 if post else 1
    clean = y.clone()
    for r, bad in ((1, math.inf), (2, -math.inf), (3, math.inf if post else math.nan)):
        y[r, int(drop[r].nonzero()[-1])] = bad
    got, want = (D.residual_norm_backward(x, y.flip(0).nan_to_num(0, 1, -1), x, v, **kw) for v in (y, clean))
    assert want[4].isfinite().all() and torch.equal(got[4], want[4])
    assert torch.equal(got[0], want[0]) and (post or torch.equal(got[1], want[1]))


def test_dropout_in_place_and_inside_other_rows():
    x = _gen(2)(50, 37).to(BF)
    want = D.dropout(x, 0.4, _seed())
    for left, right in ((0, 3), (8, 16), (1, 2)):
        v = _inside(x, left, right, rows=1)
        assert torch.equal(D.dropout(v, 0.4, _seed()), want)
        seed = _seed()
        N.check(N.load().maba_hip_dropout(N.rows_desc(v), 0.4, seed.data_ptr(), 0, N.rows_desc(v), N.stream_ptr(v.device)), "dropout")
        assert torch.equal(v, want)
        _around_is_nan(v, left, right)


# ----------------------------------------------------------------------------- the boundary


PARTS = [("weight",), ("y",), ("y", "weight", "gate"), ("y", "post_weight"), ("y", "weight", "post_weight", "gate")]
# One size for each number of lanes a row and of chunks a lane, and a few for their edges.
SIZES = [(1, 1), (3, 7), (5, 16), (70, 33), (1, 640), (130, 640), (33, 129), (64, 250), (40, 1024), (21, 1030), (9, 2048), (17, 3333),
         (6, 4096), (5, 4100), (3, 8191), (4, 8192)]
MANY = [(5000, 24), (4500, 640), (9001, 136), (4200, 1001), (16400, 640), (16389, 651), (8200, 33), (3000, 2049)]


def _tensors(M, Cw, dt, parts, seed=0):
    r = _gen(seed)
    t = dict(x=2 * r(M, Cw), y=r(M, Cw) * torch.exp2(r(M, 1)), weight=1 + 0.2 * r(Cw), post_weight=1 + 0.2 * r(Cw), gate=torch.sigmoid(r(Cw)))
    return {k: v.to(dt) if k in ("x", *parts) else None for k, v in t.items()}


def _check_boundary(t, dt, p, seed=0, wrap=lambda v: v):
    names = dict(w="weight", wp="post_weight", g="gate")
    x, y = t["x"], t["y"]
    M, Cw = x.shape
    keep = B.kept(x, p, _seed(), 9) if y is not None else None
    kw = {v: t[v] for v in names.values()}
    ref = {k: t[v] for k, v in names.items()}
    args = dict(scale=0.7, p=p if y is not None else 0.0, seed=_seed(), stream=9)
    xo, h = D.residual_norm(wrap(x), None if y is None else wrap(y), **kw, **args)
    want = B.boundary(x, y, **ref, scale=0.7, keep=keep, p=p)
    if y is not None:
        B.check(xo, want["x_out"], "x_out")
    if t["weight"] is not None:
        B.check(h, want["h"], "h")
    r = _gen(seed + 1)
    dxo, dh = (0.3 * r(M, Cw)).to(dt), (0.3 * r(M, Cw)).to(dt) if t["weight"] is not None else None
    got = D.residual_norm_backward(wrap(dxo), None if dh is None else wrap(dh), wrap(x), None if y is None else wrap(y), **kw, **args)
    want = B.boundary_backward(dxo, dh, x, y, **ref, scale=0.7, keep=keep, p=p)
    for name, v in zip(("dx", "dy", "dweight", "dpost_weight", "dgate"), got):
        if v is not None and (name != "dy" or y is not None):
            B.check(v, want[name], name)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("parts", PARTS)
@pytest.mark.parametrize("M,Cw", SIZES)
def test_boundary_of_all_widths(M, Cw, parts, dt):
    _check_boundary(_tensors(M, Cw, dt, parts), dt, 0.3 if Cw % 3 else 0.0)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("parts", PARTS[2:])
@pytest.mark.parametrize("M,Cw", MANY)
def test_boundary_of_many_rows(M, Cw, parts, dt):
    _check_boundary(_tensors(M, Cw, dt, parts, seed=3), dt, 0.1)


@pytest.mark.parametrize("left,right", [(0, 8), (8, 16), (3, 2), (1, 0), (4, 4)])
@pytest.mark.parametrize("M,Cw", [(5, 40), (70, 72), (64, 21), (9, 2056)])
def test_what_lies_around_the_rows_does_not_count(M, Cw, left, right):
    _check_boundary(_tensors(M, Cw, BF, PARTS[-1], seed=4), BF, 0.2, wrap=lambda v: _inside(v, left, right, rows=2))


@pytest.mark.parametrize("Cw", [40, 33, 2100])
def test_boundary_in_place_over_the_stream(Cw):
    t = _tensors(300, Cw, BF, PARTS[-1], seed=5)
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"])
    xo, h = D.residual_norm(t["x"], t["y"], **kw)
    for left, right in ((0, 0), (8, 8), (1, 2)):
        v = _inside(t["x"], left, right, rows=1)
        got = H.hip_residual_norm(v, t["y"], x_out=v, **kw)
        assert got[0] is v and torch.equal(v, xo) and torch.equal(got[1], h)
        _around_is_nan(v, left, right)


def test_boundary_p_of_one_and_scale_of_zero():
    t = _tensors(50, 100, BF, PARTS[-1], seed=6)
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"])
    for args in (dict(p=1.0), dict(scale=0.0)):
        xo, h = D.residual_norm(t["x"], t["y"], **kw, **args)
        assert torch.equal(xo, t["x"])
        B.check(h, B.boundary(t["x"], None, t["weight"])["h"], "h")
        dx, dy, dw, dpw, dg = D.residual_norm_backward(t["x"], h, t["x"], t["y"], **kw, **args)
        assert not dy.any() and not dpw.any() and not dg.any() and dx.any() and dw.any()


@pytest.mark.parametrize("dt", TYPES)
def test_rows_of_zeros_and_an_eps_of_zero(dt):
    """Rows past the last one take no part in the parameters' sums, whatever eps is."""
    t = _tensors(37, 24, dt, PARTS[-1], seed=7)
    t["x"][3], t["y"][3] = 0, 0
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"])
    xo, h = D.residual_norm(t["x"], t["y"], **kw)
    assert not xo[3].any() and not h[3].any()
    live = [i for i in range(37) if i != 3]
    x, y = t["x"][live], t["y"][live]
    xo, h = D.residual_norm(x, y, **kw, eps=0.0)
    want = B.boundary(x, y, t["weight"], t["post_weight"], t["gate"], eps=0.0)
    B.check(xo, want["x_out"], "x_out")
    B.check(h, want["h"], "h")
    got = D.residual_norm_backward(x, y, x, y, **kw, eps=0.0)
    want = B.boundary_backward(x, y, x, y, t["weight"], t["post_weight"], t["gate"], eps=0.0)
    for name, v in zip(("dx", "dy", "dweight", "dpost_weight", "dgate"), got):
        B.check(v, want[name], name)


@pytest.mark.parametrize("Cw", [64, 50, 3000])
@pytest.mark.parametrize("needs", [(1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 0), (0, 0, 0, 1, 0), (0, 0, 0, 0, 1), (1, 1, 0, 0, 0),
                                   (0, 0, 1, 1, 1), (0, 0, 0, 0, 0)])
def test_boundary_gradients_of_some_inputs(needs, Cw):
    t = _tensors(90, Cw, BF, PARTS[-1], seed=8)
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"], p=0.2, seed=_seed())
    for dh in (t["y"], None):
        want = D.residual_norm_backward(t["x"], dh, t["x"], t["y"], **kw)
        got = D.residual_norm_backward(t["x"], dh, t["x"], t["y"], **kw, needs=tuple(map(bool, needs)))
        for n, g, w in zip(needs, got, want):
            assert torch.equal(g, w) if n else g is None
    xo = D.residual_norm_backward(None, t["y"], t["x"], t["y"], **kw)          # only h has a gradient
    zero = D.residual_norm_backward(torch.zeros_like(t["x"]), t["y"], t["x"], t["y"], **kw)
    assert all(torch.equal(a, b) for a, b in zip(xo, zero))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("M,Cw", [(1, 40), (90, 64), (90, 50), (20, 2056), (300, 640)])
def test_x_is_not_read_where_h_has_no_gradient(M, Cw, post):
    t = _tensors(M, Cw, BF, PARTS[-1] if post else ("y", "gate"), seed=15)
    seed, d = _seed(), t["y"].flip(0).contiguous()
    want = D.residual_norm_backward(d, None, t["x"], t["y"], post_weight=t["post_weight"], gate=t["gate"], p=0.2, seed=seed)
    outs = [torch.full_like(v, math.nan) if v is not None else None for v in want]
    size = N.load().maba_hip_residual_norm_backward_workspace_size(N.rows_desc(d), 7)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    none = bytes(8) + N.rows_desc(t["x"])[8:]                                  # the shape and type alone
    N.check(N.load().maba_hip_residual_norm_backward(N.rows_desc(d), None, none, N.rows_desc(t["y"]), None, N.rows_desc(t["post_weight"]),
                                                     N.rows_desc(t["gate"]), 1.0, 0.2, seed.data_ptr(), 0, 1e-6, *map(N.rows_desc, outs),
                                                     ws.data_ptr(), ws.numel(), N.stream_ptr(d.device)), "residual_norm_backward")
    assert all(torch.equal(a, b) for a, b in zip(outs, want) if b is not None)


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (4,), (0, 2), (1, 4), (2, 3, 4)])
@pytest.mark.parametrize("post", [False, True])
def test_boundary_autograd_of_some_inputs(post, which):
    parts = PARTS[-1] if post else ("y", "weight", "gate")
    t = _tensors(70, 48, BF, parts, seed=9)
    names = ["x", "y", "weight", "post_weight", "gate"]
    if not post:
        which = tuple(i for i in which if i != 3) or (0,)
    g = [_gen(10)(70, 48).to(BF) for _ in range(2)]

    def grads(live):
        a = [None if t[n] is None else t[n].detach().clone().requires_grad_(i in live) for i, n in enumerate(names)]
        out = D.residual_norm(*a, scale=0.5, p=0.1, seed=_seed())
        return dict(zip(live, torch.autograd.grad(out, [a[i] for i in live], g)))

    every = grads([i for i in range(5) if post or i != 3])
    for i, v in grads(which).items():
        assert torch.equal(v, every[i]), names[i]


def test_boundary_bad_rows_stay_in_their_rows():
    for bad in (math.nan, math.inf, 3e38):
        t = _tensors(60, 40, BF, PARTS[-1], seed=11)
        t["y"][3, 5] = bad
        t["x"][7, 9] = bad
        rows = [i for i in range(60) if i not in (3, 7)]
        kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"])
        xo, h = D.residual_norm(t["x"], t["y"], **kw)
        want = B.boundary(t["x"][rows], t["y"][rows], t["weight"], t["post_weight"], t["gate"])
        B.check(xo[rows], want["x_out"], "x_out")
        B.check(h[rows], want["h"], "h")
        dx, dy, *_ = D.residual_norm_backward(t["x"], t["y"], t["x"], t["y"], **kw)
        want = B.boundary_backward(t["x"][rows], t["y"][rows], t["x"][rows], t["y"][rows], t["weight"], t["post_weight"], t["gate"])
        B.check(dx[rows], want["dx"], "dx")
        B.check(dy[rows], want["dy"], "dy")


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes into a tensor, and rows that are that far apart."""
    M, Cw, ld = 70000, 40, 32768
    big = torch.zeros(M, ld, dtype=BF, device=DEV)                            # 4.6 GB
    t = _tensors(M, Cw, BF, PARTS[-1], seed=13)
    view, other = big[:, 64:64 + Cw], big[:, 129:129 + Cw]
    view.copy_(t["x"])
    other.copy_(t["y"])
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"], p=0.1, seed=_seed())
    assert all(torch.equal(a, b) for a, b in zip(D.residual_norm(view, other, **kw), D.residual_norm(t["x"], t["y"], **kw)))
    for a, b in zip(D.residual_norm_backward(other, view, view, other, **kw), D.residual_norm_backward(t["y"], t["x"], t["x"], t["y"], **kw)):
        assert torch.equal(a, b)
    assert torch.equal(D.dropout(other, 0.1, _seed()), D.dropout(t["y"], 0.1, _seed()))
    far = big.view(-1).as_strided((8, Cw), (2 ** 28, 1), 3)                   # 512 MB from row to row
    far.copy_(t["x"][:8])
    want = D.residual_norm(t["x"][:8].contiguous(), t["y"][:8].contiguous(), **kw)
    assert all(torch.equal(a, b) for a, b in zip(D.residual_norm(far, t["y"][:8], **kw), want))
    want = D.residual_norm_backward(t["x"][:8], t["x"][:8], t["x"][:8], t["y"][:8], **kw)
    got = D.residual_norm_backward(far, far, far, t["y"][:8], **kw)
    B_ = dict(zip(("dx", "dy", "dweight", "dpost_weight", "dgate"), got))
    assert torch.equal(B_["dx"], want[0]) and torch.equal(B_["dy"], want[1])
    ref = B.boundary_backward(t["x"][:8], t["x"][:8], t["x"][:8], t["y"][:8], t["weight"], t["post_weight"], t["gate"],
                              keep=B.kept(t["x"][:8], 0.1, _seed()), p=0.1)
    for n in ("dweight", "dpost_weight", "dgate"):
        B.check(B_[n], ref[n], n)                                             # other lanes a row: other sums
    x = big.view(1, M, ld)[:, :, :300]                                        # logits that span 4.6 GB
    tt = torch.randint(0, 300, (1, M), device=DEV)
    got = D.token_logprobs(x, tt, top=2)
    flat = D.token_logprobs(x[0].contiguous(), tt[0], top=2)
    assert all(torch.equal(a[0], b) for a, b in zip(got, flat))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("M,Cw", [(1, 64), (129, 640), (2049, 640), (4097, 128), (16385, 640), (16400, 640), (65537, 96), (8193, 24), (5001, 33),
                                  (1025, 2048), (4099, 1001), (3001, 2049), (513, 4096), (2051, 4095), (770, 8192)])
def test_parameters_sums_have_every_row_once(M, Cw, post, dt):
    """Whole numbers all the way: normalised rows of +-1, gradients without a part along them.  What a row adds to a sum is 1 at
    least or nothing, so that a row lost or taken twice shows against the sums' own magnitude times some 2^-24."""
    r = _gen(M + Cw)
    sign = lambda: torch.where(r(M, Cw) > 0, 1.0, -1.0)
    ints = lambda k: (r(M, Cw) * 1.5).round().clamp(-k, k)
    keep = B.kept(torch.empty(M, Cw, device=DEV), 0.5, _seed(), 4)
    y, xo, dxo, e = sign(), sign(), ints(3), ints(2)
    e = torch.cat([e[:, :Cw // 2], -e[:, :Cw // 2], torch.zeros(M, Cw % 2, device=DEV)], 1)      # rows of sum zero
    z = torch.where(keep, 2 * y, 0.0)
    x, dh, one = xo - z, e * xo, torch.ones(Cw, device=DEV)
    got = D.residual_norm_backward(dxo.to(dt), dh.to(dt), x.to(dt), y.to(dt), one.to(dt), one.to(dt) if post else None, one.to(dt), p=0.5,
                                   seed=_seed(), stream=4, eps=0.0)
    dx = (dxo + dh).double()
    for name, v, t in (("dx", got[0], None), ("dweight", got[2], dh * xo), ("dgate", got[4], dx * z), ("dpost_weight", got[3], dx * z)):
        if t is not None and v is not None:
            t = t.double()
            B.check(v, (t.sum(0), 16 * B.U * t.abs().sum(0) + B.half_step(dt) * t.sum(0).abs()), name)
        elif v is not None:
            B.check(v, (dx, 16 * B.U * (dx.abs() + 1)), name)


@pytest.mark.parametrize("stride", [2 ** 27 + 8, 400_000_000, 2 ** 28, 2 ** 30, 2 ** 31])
@pytest.mark.parametrize("dt", [BF, FL])
@pytest.mark.parametrize("Cw", [16, 64, 120, 33, 640])
def test_a_single_row_has_no_stride(Cw, dt, stride):
    """What a dimension of one element has for a stride is never walked by."""
    t = _tensors(1, Cw, dt, PARTS[-1], seed=14)
    d, dh = t["y"].clone(), t["x"].clone()
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"], p=0.2, seed=_seed())
    far = lambda v: v.as_strided((1, Cw), (stride, 1))
    for a, b in zip(D.residual_norm(far(t["x"]), far(t["y"]), **kw), D.residual_norm(t["x"], t["y"], **kw)):
        assert torch.equal(a, b)
    want = D.residual_norm_backward(d, dh, t["x"], t["y"], **kw)
    for a, b in zip(D.residual_norm_backward(far(d), far(dh), far(t["x"]), far(t["y"]), **kw), want):
        assert torch.equal(a, b)
    outs = [torch.full_like(v, math.nan) for v in want]
    ws = torch.empty(N.load().maba_hip_residual_norm_backward_workspace_size(N.rows_desc(t["x"]), 7), dtype=torch.uint8, device=DEV)
    seed, ins = _seed(), [N.rows_desc(v) for v in (far(d), far(dh), far(t["x"]), far(t["y"]), t["weight"], t["post_weight"], t["gate"])]
    N.check(N.load().maba_hip_residual_norm_backward(*ins, 1.0, 0.2, seed.data_ptr(), 0, 1e-6, N.rows_desc(far(outs[0])),
                                                     N.rows_desc(far(outs[1])), *map(N.rows_desc, outs[2:]), ws.data_ptr(), ws.numel(),
                                                     N.stream_ptr(d.device)), "residual_norm_backward")
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Cw", [1000, 4096, 4095])
def test_post_norm_backward_has_the_same_bits_on_every_call(dt, Cw):
    """Rows of several waves sum three values over the row, then one: sums of different rows or calls share nothing."""
    M, f = 3000, _gen(60)
    d, dh, x, y = (f(M, Cw).to(dt) for _ in range(4))
    w, wp, g = (1 + 0.1 * f(Cw).to(dt) for _ in range(3))
    call = lambda: D.residual_norm_backward(d, dh, x, y, w, wp, g, 0.5, 0.1, _seed(), 1)
    want = call()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(call(), want))


# ----------------------------------------------------------------------------- log probabilities


def _logits(M, V, dt, seed=0):
    r = _gen(seed)
    x = 2 * r(M, V)
    x[:, :: 13] += 3 * r(M, 1).abs()
    return x.to(dt), torch.randint(0, V, (M,), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _check_logprobs(x, t, T, k, seed=0):
    want = B.logprobs(x, t, T, k)
    got = dict(zip(("logp", "entropy", "lse", "top_logp", "top_ids"), D.token_logprobs(x, t, temperature=T, top=k)))
    for name, v in want.items():
        if name == "top_ids":
            assert torch.equal(got[name], v), name
        else:
            B.check(got[name], v, name)
    r = _gen(seed + 1)
    g = [r(x.shape[0]) for _ in range(3)]
    lse, ent = want["lse"][0].float(), want["entropy"][0].float()
    B.check(D.token_logprobs_backward(*g, x, t, lse, ent, T), B.logprobs_backward(*g, x, t, T), "dlogits")


# One size for each number of waves a row, by its length and by the number of rows, and a few for their edges.
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,V", [(1, 1), (5, 2), (3, 63), (4, 64), (9, 100), (5, 511), (7, 513), (3, 1024), (6, 1030), (5, 2050), (3, 4096),
                                 (2, 4099), (9, 9000), (3, 33000), (1, 131073), (1500, 300), (2100, 9001), (1100, 17000), (1030, 33001)])
def test_logprobs_of_all_sizes(M, V, dt):
    x, t = _logits(M, V, dt, seed=V)
    if M > 2:
        t[1] = -100
    _check_logprobs(x, t, 0.8, min(V, 20))


@pytest.mark.parametrize("k", [1, 2, 8, 9, 16, 17, 63, 64])
@pytest.mark.parametrize("M,V", [(3, 64), (5, 300), (2, 700), (3, 5000), (2, 40000), (1200, 9000)])
def test_every_number_of_alternatives(M, V, k):
    x, t = _logits(M, V, BF, seed=k)
    want = B.logprobs(x, t, 1.0, k)
    got = D.token_logprobs(x, t, top=k)
    assert torch.equal(got[4], want["top_ids"])
    B.check(got[3], want["top_logp"], "top_logp")


def _hard_rows(V, dt):
    """Rows with masks that leave nothing, one or a few tokens, ties, order, and far from zero."""
    x, t = _logits(14, V, dt, seed=V + 1)
    low = torch.finfo(dt).min
    x[0] = -math.inf
    x[1], x[2] = 0, 1.5
    x[3, :V // 2] = -math.inf
    x[4] = -math.inf
    x[4, V // 2:V // 2 + 3] = 1
    x[5] = (torch.arange(V, device=DEV) / 64).to(dt)
    x[6] = -x[5]
    x[7] = x[7].round()
    x[8, V // 3] = 60
    x[9, ::2] = low
    x[10, 1:] = low
    x[11] = -math.inf
    x[11, V - 1] = low
    x[12] = (x[12].float() + 500).to(dt)
    x[13] = (x[13].float() - 500).to(dt)
    t[7] = -1
    return x, t


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [3, 64, 100, 700, 4097, 5003, 40000])
@pytest.mark.parametrize("k", [1, 20, 64])
def test_masks_ties_and_far_rows(V, dt, k):
    x, t = _hard_rows(V, dt)
    _check_logprobs(x, t, 1.0, min(V, k))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V", [5, 700, 40000])
def test_rows_of_nothing_but_the_lowest_value(V, dt):
    """They are uniform; lse saturates where the lowest value over T is past fp32's range."""
    x, t = _logits(4, V, dt)
    x[:] = torch.finfo(dt).min
    for T in (1.0, 0.5, 2.0):
        logp, ent, lse, tl, ti = D.token_logprobs(x, t, temperature=T, top=3)
        assert torch.allclose(logp, torch.full_like(logp, -math.log(V)), rtol=1e-5, atol=1e-5)
        assert torch.allclose(ent, torch.full_like(ent, math.log(V)), rtol=1e-5, atol=1e-5)
        assert torch.isfinite(lse).all() and ti.tolist() == [[0, 1, 2]] * 4
        assert torch.allclose(tl, logp[:, None].expand(-1, 3))
        d = D.token_logprobs_backward(torch.ones_like(logp), None, None, x, t, lse, ent, T).float()
        want = torch.full_like(d, -1 / V / T).scatter_(1, t[:, None], (1 - 1 / V) / T)
        assert torch.allclose(d, want, rtol=2 * torch.finfo(dt).eps + 2e-5, atol=1e-7)


@pytest.mark.parametrize("V", [50, 900, 33000])
def test_nan_infinity_and_targets_past_the_vocabulary(V):
    x, t = _logits(8, V, FL, seed=5)
    x[1, V // 2], x[2, V // 2], x[3, V - 1] = math.nan, math.inf, math.nan
    x[3, 0] = -math.nan
    t[4] = V
    x.requires_grad_()
    logp, ent, lse, tl, ti = D.token_logprobs(x, t, top=4)
    ref = C.ref_token_logprobs(x.detach().cpu(), t.cpu(), 1.0, 4)
    for a, b in zip((logp, ent, lse, tl), ref):
        assert torch.equal(a.isnan().cpu(), b.isnan())
    assert torch.equal(ti.cpu(), ref[4])
    d, = torch.autograd.grad(logp[[0, 4, 5]].sum(), x)
    assert d[4].isnan().all() and torch.isfinite(d[[0, 5]]).all()


def test_logits_of_three_dimensions_and_other_strides():
    B_, L, V = 3, 40, 333
    x, _ = _logits(B_ * L, V, BF, seed=6)
    t = torch.randint(0, V, (B_, L), device=DEV)
    want = D.token_logprobs(x, t.view(-1), top=5)
    x3 = x.view(B_, L, V)
    for logits, tt, pick in ((x3, t, lambda w: w.view(B_, L, *w.shape[1:])), (x3[:, :-1], t[:, 1:], None),
                             (x3.transpose(0, 1), t.t(), lambda w: w.view(B_, L, *w.shape[1:]).transpose(0, 1)),
                             (x3[:, -1], t[:, -1], lambda w: w.view(B_, L, *w.shape[1:])[:, -1]),
                             (x3.view(3, 5, 8, V), t.view(3, 5, 8), lambda w: w.view(3, 5, 8, *w.shape[1:])),
                             (x3[0, 0], t[0, 0], lambda w: w[0])):
        got = D.token_logprobs(logits, tt, top=5)
        if pick is None:
            flat = D.token_logprobs(logits.reshape(-1, V), tt.reshape(-1), top=5)
            assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, flat))
        else:
            assert all(torch.equal(a, pick(b)) for a, b in zip(got, want))
    cols = x.t().contiguous().t()                                              # columns first: copied
    assert all(torch.equal(a, b) for a, b in zip(D.token_logprobs(cols, t.view(-1), top=5), want))
    one = x[:1].expand(7, V)                                                   # one row for all
    assert torch.equal(D.token_logprobs(one, t.view(-1)[:7])[2], want[2][:1].expand(7))
    v = _inside(x, 3, 6, rows=1)
    assert all(torch.equal(a, b) for a, b in zip(D.token_logprobs(v, t.view(-1), top=5), want))
    g = torch.ones(B_ * L, device=DEV)
    d = D.token_logprobs_backward(g, g, g, v, t.view(-1), want[2], want[1])
    assert torch.equal(d, D.token_logprobs_backward(g, g, g, x, t.view(-1), want[2], want[1]))
    for logits, tt in ((x3[:, :-1], t[:, 1:]), (x3.transpose(0, 1), t.t())):
        got = D.token_logprobs(logits, tt)
        d = D.token_logprobs_backward(torch.ones_like(got[0]), None, None, logits, tt, got[2], got[1])
        flat = D.token_logprobs_backward(g[:tt.numel()], None, None, logits.reshape(-1, V), tt.reshape(-1), got[2].reshape(-1),
                                         got[1].reshape(-1))
        assert torch.equal(d.reshape(-1, V), flat)


def test_logits_gradient_in_place():
    """The C entry's documented form: dlogits over the logits themselves, other rows left as they were."""
    x, t = _logits(50, 700, BF, seed=7)
    logp, ent, lse, _, _ = D.token_logprobs(x, t)
    g = torch.ones_like(logp)
    want = D.token_logprobs_backward(g, None, None, x, t, lse, ent)
    v = _inside(x, 1, 2, rows=1)
    N.check(N.load().maba_hip_token_logprobs_backward(N.rows_desc(g), None, None, N.desc(v), N.rows_desc(t), N.rows_desc(lse),
                                                      N.rows_desc(ent), 1.0, N.desc(v), N.stream_ptr(v.device)), "token_logprobs_backward")
    assert torch.equal(v, want)
    _around_is_nan(v, 1, 2)


@pytest.mark.parametrize("M,V", [(3, 40000), (300, 9001)])
def test_logits_gradient_in_place_of_rows_far_from_zero(M, V):
    """Such rows are summed again by the backward: all of it before any of the row is written."""
    x, t = _logits(M, V, BF, seed=8)
    x += 600
    g = torch.ones(M, device=DEV)
    _, ent, lse, _, _ = D.token_logprobs(x, t)
    want = D.token_logprobs_backward(g, g, None, x, t, lse, ent)
    N.check(N.load().maba_hip_token_logprobs_backward(N.rows_desc(g), N.rows_desc(g), None, N.desc(x), N.rows_desc(t), N.rows_desc(lse),
                                                      N.rows_desc(ent), 1.0, N.desc(x), N.stream_ptr(x.device)), "token_logprobs_backward")
    assert torch.equal(x, want)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("V,below", [(3, 9), (64, 10), (700, 12), (700, 17), (9001, 14), (40000, 15), (40000, 19)])
@pytest.mark.parametrize("lse", [-200, 0, 30, 120, 240])
def test_gradient_of_a_likely_target_is_the_others_sum(V, below, lse, dt):
    """1 - p from a p near 1, or from an lse far from zero, would keep few of its bits or none."""
    x, t, H, want, wantH = B.likely_rows(V, lse, below, dt)
    x, t = x.to(DEV).requires_grad_(), t.to(DEV)
    logp, ent, z, _, _ = D.token_logprobs(x, t)
    d, = torch.autograd.grad(-logp.sum(), x)
    B.check(-d.gather(1, t[:, None])[:, 0].cpu(), want, "at the target")
    dH = D.token_logprobs_backward(None, torch.ones_like(logp), None, x.detach(), t, z.detach(), H.float().to(DEV))
    B.check(dH.gather(1, t[:, None])[:, 0].cpu(), wantH, "the entropy's")
    x, g = x.detach(), torch.full_like(logp, -1)
    _check_logprobs(x, t, 1.0, 2)
    N.check(N.load().maba_hip_token_logprobs_backward(N.rows_desc(g), None, None, N.desc(x), N.rows_desc(t), N.rows_desc(z.detach()),
                                                      N.rows_desc(ent.detach()), 1.0, N.desc(x), N.stream_ptr(x.device)), "token_logprobs_backward")
    assert torch.equal(x, d)                                                   # over the logits


def test_rows_without_mass_have_no_gradient_whatever_comes_in():
    """A loss of lse^2 under torch.where sends NaN into such a row."""
    x, t = _logits(12, 300, FL, seed=9)
    x[::3] = -math.inf
    x.requires_grad_()
    logp, ent, lse, _, _ = D.token_logprobs(x, t)
    z = torch.where(lse > -math.inf, lse ** 2, torch.zeros_like(lse))
    (z.sum() + ent.sum() - torch.where(lse > -math.inf, logp, torch.zeros_like(logp)).sum()).backward()
    assert (x.grad[::3] == 0).all() and x.grad.isfinite().all() and (x.grad[1] != 0).any()
    nan = torch.full_like(lse, math.nan)
    d = D.token_logprobs_backward(nan, nan, nan, x.detach(), t, lse.detach(), ent.detach())
    assert (d[::3] == 0).all() and d[1].isnan().all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,V,k", [(3, 4000, 7), (5000, 2500, 20), (1100, 12000, 64), (2100, 17000, 3), (4, 40000, 20)])
def test_rows_in_order(M, V, k, dt):
    """All of a row's largest elements are those of a few threads."""
    x = torch.arange(V, device=DEV).expand(M, V) * (20 / V)
    t = torch.full((M,), V // 2, device=DEV)
    for rows in (x.to(dt), x.flip(1).to(dt)):
        _check_logprobs(rows.contiguous(), t, 1.0, k)


def test_more_rows_than_a_launch_takes():
    M, V = (1 << 22) + 5, 3
    x, t = _gen(10)(M, V), torch.arange(M, device=DEV) % V
    x.requires_grad_()
    out = D.token_logprobs(x, t, top=2)
    lp = torch.log_softmax(x.detach().double(), -1)
    assert (out[0].detach().double() - lp.gather(1, t[:, None])[:, 0]).abs().max() < 2e-6
    assert torch.equal(out[4], torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :2])
    out[0].sum().backward()
    d = torch.nn.functional.one_hot(t, V).double() - lp.exp()
    assert (x.grad.double() - d).abs().max() < 2e-6


@pytest.mark.parametrize("use", [(0,), (1,), (2,), (0, 1), (0, 1, 2)])
def test_logprob_autograd_of_some_outputs(use):
    x, t = _logits(40, 300, FL, seed=8)
    x.requires_grad_()
    out = D.token_logprobs(x, t, temperature=1.5, top=3)
    assert not out[3].requires_grad and not out[4].requires_grad
    g = [_gen(9 + i)(40) for i in range(3)]
    d, = torch.autograd.grad([out[i] for i in use], x, [g[i] for i in use])
    want = B.logprobs_backward(*(g[i] if i in use else None for i in range(3)), x.detach(), t, 1.5)
    # lse and entropy are the forward's own, as exact as its bounds say
    w = B.logprobs(x.detach(), t, 1.5)
    p = torch.softmax(x.detach().double() / 1.5, -1)
    lp = torch.log(p).abs()
    slack = p * ((w["lse"][1][:, None]) * (sum(v.abs() for v in g)[:, None] * (3 + lp)) + g[1].abs()[:, None] * w["entropy"][1][:, None])
    B.check(d, (want[0], want[1] + 1.05 * slack), "dlogits")


# ----------------------------------------------------------------------------- together


def test_a_training_step_of_all_of_them():
    """Embeddings, dropout, a gated feed-forward block between two boundaries, a head and the loss, as the model runs them:
    each operator's gradients against its formulas at the values that it saw."""
    M, Cw, I, V = 200, 96, 160, 500
    r = _gen(21)
    seed = _seed()
    x0 = r(M, Cw).to(BF).requires_grad_()
    w1, w2, wp, = ((1 + 0.1 * r(Cw)).to(BF).requires_grad_() for _ in range(3))
    gate = torch.sigmoid(r(Cw)).to(BF).requires_grad_()
    wg, wu, wd, head = ((r(a, b) / b ** 0.5).to(BF).requires_grad_() for a, b in ((I, Cw), (I, Cw), (Cw, I), (V, Cw)))
    t = torch.randint(0, V, (M,), device=DEV)
    x = D.dropout(x0, 0.1, seed, stream=0)
    x, h = D.residual_norm(x, weight=w1)
    f = D.linear_epilogue(D.gated_ffn(h, wg, wu), wd)
    x2, h2 = D.residual_norm(x, f, w2, wp, gate, scale=0.5, p=0.2, seed=seed, stream=1)
    logits = D.linear_epilogue(h2, head)
    logp, ent, lse, _, _ = D.token_logprobs(logits, t)
    for v in (x, h, f, x2, h2, logits):
        v.retain_grad()
    (-logp.mean() + 0.01 * ent.mean() + 1e-3 * (x2.float() ** 2).mean() + 1e-4 * (lse ** 2).mean()).backward()
    with torch.no_grad():
        keep = B.kept(f, 0.2, seed, 1)
        want = B.boundary(x, f, w2, wp, gate, 0.5, keep, 0.2)
        B.check(x2, want["x_out"], "x_out")
        B.check(h2, want["h"], "h")
        dxo = (x2.float() * (2e-3 / x2.numel())).to(BF)
        want = B.boundary_backward(dxo, h2.grad, x, f, w2, wp, gate, 0.5, keep, 0.2)
        for name, v in (("dy", f.grad), ("dweight", w2.grad), ("dpost_weight", wp.grad), ("dgate", gate.grad)):
            B.check(v, want[name], name)
        # x has two gradients, its norm's and the boundary's, each rounded once and their sum again
        one = B.boundary_backward(None, h.grad, x, None, w1)
        total = one["dx"][0] + want["dx"][0]
        B.check(x.grad, (total, one["dx"][1] + want["dx"][1] + 1.05 * B.half_step(BF) * total.abs()), "dx")
        B.check(w1.grad, one["dweight"], "dw1")
        B.check(x0.grad, B.dropout(x.grad, 0.1, seed, 0), "dx0")
        wl = B.logprobs(logits, t)
        B.check(logp, wl["logp"], "logp")
        B.check(ent, wl["entropy"], "entropy")
        g = [torch.full((M,), v, device=DEV) for v in (-1 / M, 0.01 / M)] + [lse * (2e-4 / M)]
        d, b = B.logprobs_backward(*g, logits, t)
        B.check(logits.grad, (d, b + 2e-6 * d.abs().amax()), "dlogits")         # lse and entropy within 1e-6 of 64 bits


@pytest.mark.parametrize("post", [False, True])
def test_the_models_boundaries_and_score(post):
    from maba_sparse.model import MabaSparseForCausalLM, get_101m_config
    torch.manual_seed(0)
    cfg = dict(n_layers=4, vocab_size=1024, top_k=4)
    kw = dict(post_norm=True, residual_scale=0.7) if post else {}
    m = MabaSparseForCausalLM(get_101m_config(**cfg, **kw, fused_boundary=True)).init_normal(0.05).to(DEV, BF).eval()
    ids = torch.randint(0, 1024, (2, 300), device=DEV)
    with torch.no_grad():
        logits = m(ids)[0]
        logp, ent, lse, tl, ti = m.score(ids, top=3)
        want = B.logprobs(logits[:, :-1].reshape(-1, 1024), ids[:, 1:].reshape(-1), 1.0, 3)
        B.check(logp.reshape(-1), want["logp"], "logp")
        assert torch.equal(ti.reshape(-1, 3), want["top_ids"])
        if not post:                                                            # the same blocks through the norms' kernel
            other = MabaSparseForCausalLM(get_101m_config(**cfg)).to(DEV, BF).eval()
            other.load_state_dict(m.state_dict())
            a, b = other(ids)[0].float(), logits.float()
            assert (a - b).norm() / a.norm() < 0.02                             # four blocks of bf16 roundings
        toks, seen = m.generate_greedy(ids, 8, return_logits=True)
        eager, seen2 = m.generate_greedy(ids, 8, return_logits=True, graph=False)
        assert toks.shape == (2, 8) and torch.isfinite(seen.float()).all()
        assert (seen[:, 0].float() - logits[:, -1].float()).abs().max() <= 0.05 * logits.float().abs().max()
        assert (seen[:, :1] - seen2[:, :1]).abs().max() == 0


@pytest.mark.parametrize("kw", [dict(post_norm=True), dict(residual_scale=0.5), dict(post_norm=True, residual_scale=0.7)])
def test_captured_decoding_of_extended_blocks_equals_state_passing(kw):
    """Every step's logits, each path given the same tokens.  They differ by bf16 roundings: some ten a block and three of
    the head, each 2^-9 / sqrt(3) of its values, in four blocks 0.007 of the logits' norm."""
    from maba_sparse.model import MabaSparseForCausalLM, get_101m_config
    torch.manual_seed(1)
    m = MabaSparseForCausalLM(get_101m_config(n_layers=4, vocab_size=1024, top_k=4, **kw)).init_normal(0.05).to(DEV, BF).eval()
    ids = torch.randint(0, 1024, (2, 300), generator=torch.Generator().manual_seed(2)).to(DEV)
    with torch.no_grad():
        toks, seen = m.generate_greedy(ids, 5, return_logits=True, graph=True)
        states = m(ids)[1]
        for i in range(4):
            want, states = m.step(toks[:, i:i + 1], past_states=states)
            a, b = seen[:, i + 1].float(), want[:, -1].float()
            assert (a - b).norm() / b.norm() < 0.02, (i, (a - b).norm() / b.norm())


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_a_model_trains_with_dropout_as_on_the_cpu(monkeypatch):
    """The same masks from the same seed: fp32 against 64 bits, gradients among them (its mixers' come from torch).  Of relative
    roundings of 6e-8 some thousands lie on a way through the model, and another mask changes it by tenths."""
    from maba_sparse.model import MabaSparseForCausalLM, get_101m_config
    monkeypatch.setenv("MABA_STRICT_BACKEND", "0")
    torch.manual_seed(3)
    cfg = get_101m_config(dim=128, n_layers=4, n_heads=2, d_head=64, vocab_size=97, d_emb=16, d_c=32, d_idx=16, intermediate_size=96,
                          top_k=4, post_norm=True, residual_scale=0.7, dropout=0.3)
    ref = MabaSparseForCausalLM(cfg).init_normal(0.1).double()
    m = MabaSparseForCausalLM(cfg)
    m.load_state_dict(ref.state_dict())
    m.to(DEV)
    assert m.dropout_seed.device.type == "cuda"
    m.dropout_seed.copy_(ref.dropout_seed)
    ids = torch.randint(0, 97, (2, 70), generator=torch.Generator().manual_seed(4))
    for i in range(2):
        assert int(m.dropout_seed) == int(ref.dropout_seed)
        a, b = (-n.score(ids.to(n.dropout_seed.device))[0].mean() for n in (m, ref))
        assert abs(a.item() - b.item()) < 1e-4 * abs(b.item())
        a.backward()
        b.backward()
        for (name, p), q in zip(m.named_parameters(), ref.parameters()):
            if q.grad is not None:
                assert (p.grad.cpu().double() - q.grad).norm() <= 1e-3 * q.grad.norm() + 1e-9, (name, i)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
def test_a_seed_on_another_device_than_the_model(monkeypatch):
    """As a replica has it whose model keeps its seed elsewhere."""
    from maba_sparse.model import MabaSparseForCausalLM, get_101m_config
    monkeypatch.setenv("MABA_STRICT_BACKEND", "0")
    torch.manual_seed(5)
    m = MabaSparseForCausalLM(get_101m_config(dim=64, n_layers=1, n_heads=1, d_head=64, vocab_size=32, d_emb=16, intermediate_size=48,
                                              dropout=0.5)).to(DEV)
    ids = torch.randint(0, 32, (2, 20), device=DEV)
    seed = m.dropout_seed.clone()
    want = m(ids)[0]
    m.dropout_seed = seed.cpu()
    assert torch.equal(m(ids)[0], want) and int(m.dropout_seed) == int(seed) + 1


# ----------------------------------------------------------------------------- calls


def _calls(seed=31, M=70, Cw=72, V=900, grad=True):
    """name -> (call, leaves, gradients of its results) of each operator."""
    t = _tensors(M, Cw, BF, PARTS[-1], seed=seed)
    x, tt = _logits(M, V, BF, seed=seed)
    leaves = [t[n].requires_grad_(grad) for n in ("x", "y", "weight", "post_weight", "gate")]
    x.requires_grad_(grad)
    r = _gen(seed + 1)
    dev_seed = _seed()
    return {
        "dropout": (lambda: (D.dropout(leaves[0], 0.3, dev_seed, 2),), leaves[:1], [r(M, Cw).to(BF)]),
        "residual_norm": (lambda: D.residual_norm(*leaves, scale=0.5, p=0.2, seed=dev_seed), leaves, [r(M, Cw).to(BF) for _ in range(2)]),
        "norm_alone": (lambda: D.residual_norm(leaves[0], weight=leaves[2])[1:], [leaves[0], leaves[2]], [r(M, Cw).to(BF)]),
        "token_logprobs": (lambda: D.token_logprobs(x, tt, temperature=0.9, top=4), [x], [r(M) for _ in range(3)]),
    }


def _all_of(call, leaves, grads):
    out = call()
    return [*out, *torch.autograd.grad(out[:len(grads)], leaves, grads)]


OPS = ["dropout", "residual_norm", "norm_alone", "token_logprobs"]


@pytest.mark.parametrize("op", OPS)
def test_the_same_bits_every_time_and_on_two_streams(op):
    c = _calls(M=3000, Cw=640)[op]
    want = _all_of(*c)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(_all_of(*c))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("shape", [(5, 64), (30, 33)])
def test_native_and_python_paths_give_the_same_bits(monkeypatch, op, shape):
    c = _calls(M=shape[0], Cw=shape[1], V=shape[1] * 20)[op]
    native = _all_of(*c)
    used, hip = [], D._KERNEL_REGISTRY["hip"]
    for name in ("dropout", "residual_norm", "residual_norm_backward", "token_logprobs", "token_logprobs_backward"):
        def spy(_f=hip[name], _n=name, **kw):
            used.append(_n)
            return _f(**kw)

        monkeypatch.setitem(hip, name, spy)
    python = _all_of(*c)
    assert used
    assert all(a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(native, python))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(c[0](), native))


@pytest.mark.parametrize("op", OPS)
def test_double_backward_is_refused_and_first_is_not(op):
    call, leaves, grads = _calls()[op]
    plain = torch.autograd.grad(call()[:len(grads)], leaves, grads)
    live = [g.clone().requires_grad_() for g in grads]
    once = torch.autograd.grad(call()[:len(grads)], leaves, live, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, once))
    with pytest.raises(RuntimeError, match="twice"):
        sum(g.float().sum() for g in once).backward()


def test_saved_tensors_follow_their_versions():
    seed = _seed()
    x = _gen(40)(20, 64).to(BF).requires_grad_()
    y = D.dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = x * 2
    xo, h = D.residual_norm(x, y, x.detach()[0].clone())
    y.mul_(2)                                                               # the backward pass reads it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t.cpu(), lambda t: t.to(DEV)):
        out = D.residual_norm(x, x.detach(), x.detach()[0].clone(), p=0.5, seed=seed)
    assert len(seen) == 4                                                   # x, y, the weight and the seed
    assert torch.isfinite(torch.autograd.grad(out, x, [x.detach(), x.detach()])[0].float()).all()


def test_calls_that_the_binding_declines_raise_as_before():
    x, t = _logits(20, 64, BF)
    w = x[0].clone()
    for call, error, text in ((lambda: D.dropout(x, 0.5), ValueError, "seed"), (lambda: D.dropout(x, 0.5, SEED), RuntimeError, "same device"),
                              (lambda: D.dropout(x, 2.0, _seed()), ValueError, "p must be"),
                              (lambda: D.dropout(x, 0.5, _seed(), stream=-1), ValueError, "stream"),
                              (lambda: D.residual_norm(x, x[:, :32]), ValueError, "y must be"),
                              (lambda: D.residual_norm(x, x.half()), TypeError, "dtypes must match"),
                              (lambda: D.residual_norm(x, x, w.cpu()), RuntimeError, "same device"),
                              (lambda: D.residual_norm(x, x, w[:3]), ValueError, "weight must be"),
                              (lambda: D.residual_norm(x, gate=w), ValueError, "go with y"),
                              (lambda: D.token_logprobs(x, t.int()), TypeError, "int64"),
                              (lambda: D.token_logprobs(x, t.cpu()), RuntimeError, "same device"),
                              (lambda: D.token_logprobs(x, t[:3]), ValueError, "targets"),
                              (lambda: D.token_logprobs(x, t, temperature=0.0), ValueError, "temperature"),
                              (lambda: D.token_logprobs(x, t, top=65), ValueError, "top")):
        with pytest.raises(error, match=text):
            call()


def test_what_the_kernels_do_not_take_goes_to_the_reference(monkeypatch):
    x = _gen(41)(3, 8200).to(BF)
    l64, t = _logits(4, 50, torch.float64)
    l32, t2 = _logits(4, 100, FL)
    calls = [lambda: D.residual_norm(x, x, x[0].clone()), lambda: D.token_logprobs(l64, t, top=3), lambda: D.token_logprobs(l32, t2, top=70),
             lambda: D.dropout(l64, 0.5, _seed()), lambda: D.residual_norm(l64, l64)]
    for call in calls:
        with pytest.raises(RuntimeError):                    # strict: a fallback is an error
            call()
    monkeypatch.setenv("MABA_STRICT_BACKEND", "0")
    D.clear_fallback_warnings()
    with pytest.warns(RuntimeWarning):
        outs = [call() for call in calls]
    B.check(outs[0][1], B.boundary(x, x, x[0])["h"], "h")
    assert outs[1][0].dtype == torch.float64 and outs[2][4].shape == (4, 70)


def test_no_rows():
    x, t = _logits(4, 40, BF)
    w = x[0].clone().requires_grad_()
    e = x[:0].requires_grad_()
    xo, h = D.residual_norm(e, e, w, w, w, p=0.5, seed=_seed())
    assert xo.shape == h.shape == (0, 40)
    h.sum().backward()
    assert not w.grad.any()
    assert D.dropout(e, 0.5, _seed()).shape == (0, 40)
    out = D.token_logprobs(e, t[:0], top=2)
    assert [tuple(v.shape) for v in out] == [(0,)] * 3 + [(0, 2)] * 2
    assert torch.autograd.grad(out[0].sum(), e)[0].shape == (0, 40)


def test_two_threads_call_at_once():
    sets = [_calls(seed=80 + i, M=300 + 40 * i) for i in range(2)]
    want = [{op: [v.clone() for v in _all_of(*s[op])] for op in OPS} for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                for op in OPS:
                    got = _all_of(*sets[i][op])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i][op])):
                        bad.append((i, op))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("xt,yt", [(FL, BF), (BF, FL), (BF, BF)])
def test_autocast_takes_the_widest_type(xt, yt):
    r = _gen(50)
    x, y, w = r(30, 64).to(xt).requires_grad_(), r(30, 64).to(yt).requires_grad_(), r(64).requires_grad_()
    with torch.autocast("cuda", BF):
        xo, h = D.residual_norm(x, y, w, p=0.1, seed=_seed())
        (xo.float().sum() + h.float().sum()).backward()
    assert xo.dtype == h.dtype == FL
    assert x.grad.dtype == xt and y.grad.dtype == yt and w.grad.dtype == FL
    B.check(xo.detach(), B.boundary(x.detach().float(), y.detach().float(), w.detach(), keep=B.kept(x, 0.1, _seed()), p=0.1)["x_out"], "x_out")


@pytest.mark.parametrize("op", OPS)
def test_tangents_take_the_reference_path(monkeypatch, op):
    from torch.autograd import forward_ad
    x, t = _logits(20, 64, BF)
    calls = {"dropout": lambda v: D.dropout(v, 0.5, _seed()), "residual_norm": lambda v: D.residual_norm(v, v, x[0])[1],
             "norm_alone": lambda v: D.residual_norm(v, weight=x[0])[1], "token_logprobs": lambda v: D.token_logprobs(v, t)[0]}
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x.flip(0))
        with pytest.raises(RuntimeError):
            calls[op](dual)
        monkeypatch.setenv("MABA_STRICT_BACKEND", "0")
        D.clear_fallback_warnings()
        with pytest.warns(RuntimeWarning, match="tangents"):
            assert forward_ad.unpack_dual(calls[op](dual)).tangent is not None


# ----------------------------------------------------------------------------- graphs


def test_captured_ops_replay_with_new_inputs_and_seeds():
    """Forward and backward ops recorded once, replayed on new data and a seed that the graph itself moves on, between eager
    calls of the same ops."""
    M, Cw, V = 1300, 136, 9000
    t = _tensors(M, Cw, BF, PARTS[-1], seed=60)
    x, tt = _logits(M, V, BF, seed=61)
    seed = _seed()
    kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"], scale=0.5, p=0.2)
    g = torch.ones(M, device=DEV)

    def step(seed):
        a = D.dropout(t["x"], 0.3, seed, 1)
        xo, h = D.residual_norm(a, t["y"], **kw, seed=seed)
        back = D.residual_norm_backward(t["y"], h, xo, t["y"], **kw, seed=seed)
        out = D.token_logprobs(x, tt, top=5)
        return [a, xo, h, *back, *out, D.token_logprobs_backward(g, g, g, x, tt, out[2], out[1])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(seed)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(seed)
        seed += 1
    r, masks = _gen(62), []
    for i in range(4):
        for v in (t["x"], t["y"], x):
            v.copy_(r(*v.shape).to(BF))
        now = seed.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert int(seed) == int(now) + 1
        assert all(torch.equal(a, b) for a, b in zip(out, step(now)))
        masks.append(out[0] == 0)
        torch.cuda.synchronize()
    assert not torch.equal(masks[0], masks[1])


def test_two_graphs_of_one_pool_replayed_by_turns():
    """Their workspaces share memory: each replay must make all that it reads."""
    sets = [_tensors(600 + 90 * i, 72 + 8 * i, BF, PARTS[-1], seed=70 + i) for i in range(2)]

    def step(t):
        kw = dict(weight=t["weight"], post_weight=t["post_weight"], gate=t["gate"])
        return [*D.residual_norm_backward(t["x"], t["y"], t["x"], t["y"], **kw), *D.residual_norm(t["x"], t["y"], **kw)]

    want = [step(s) for s in sets]
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(step(s))
        pool = g.pool()
        graphs.append(g)
    for turn in (0, 1, 1, 0, 1, 0, 0):
        for v in outs[turn]:
            v.zero_()
        graphs[turn].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[turn], want[turn]))
        assert all(torch.equal(a, b) for a, b in zip(step(sets[turn]), want[turn]))


@pytest.mark.parametrize("op", OPS)
def test_captured_autograd_step(op):
    """Recorded through autograd once no eager graph of its leaves lives."""
    c = _calls(seed=90, M=130)[op]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _all_of(*c)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _all_of(*c)
    r = _gen(91)
    for _ in range(3):
        with torch.no_grad():
            c[1][0].copy_(r(*c[1][0].shape).to(BF))
        g.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, _all_of(*c)))


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("path", ["native", "python"])
def test_capture_beside_a_live_eager_graph_is_refused(monkeypatch, op, path):
    """Only forwards are recorded here; once the eager graph is gone the same call is taken."""
    if path == "python":
        hip = D._KERNEL_REGISTRY["hip"]
        for name in ("dropout", "residual_norm", "token_logprobs"):
            monkeypatch.setitem(hip, name, lambda _f=hip[name], **kw: _f(**kw))
    call, leaves, grads = _calls(seed=95)[op]
    call()
    eager = leaves[0] * 2                                     # another op's graph, on the current stream
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call()
    torch.cuda.synchronize()
    del eager
    gc.collect()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, call()))


@pytest.mark.parametrize("env,reference", [("reference", True), ("HIP", False), ("", False)])
def test_the_backend_that_is_asked_for(monkeypatch, env, reference):
    x, t = _logits(20, 64, BF)
    used = []
    for name in ("dropout", "residual_norm", "token_logprobs"):
        def ref(_f=D._KERNEL_REGISTRY["reference"][name], _n=name, **kw):
            used.append(_n)
            return _f(**kw)

        monkeypatch.setitem(D._KERNEL_REGISTRY["reference"], name, ref)
    monkeypatch.setenv("MABA_BACKEND", env)
    B.check(D.dropout(x, 0.5, _seed()), B.dropout(x, 0.5, _seed()), "y")
    B.check(D.residual_norm(x, x, x[0])[1], B.boundary(x, x, x[0])["h"], "h")
    B.check(D.token_logprobs(x, t)[0], B.logprobs(x, t)["logp"], "logp")
    assert len(used) == (3 if reference else 0)
