"""The feed-forward operators on the GPU against 64 bits: values, gradients, packed inputs, strides,
streams, graph replays and refusals.  The bounds of ``_ffn_bounds`` are elementwise."""
import gc

import pytest
import torch

import _ffn_bounds as B
from maba_sparse.kernels import common as C
from maba_sparse.kernels import dispatcher as D

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    """A kernel that raises fails the test instead of falling back."""
    monkeypatch.setenv("MABA_STRICT_BACKEND", "1")


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=g, device=DEV)


def _gated(M, Cw, I, dt, seed=0):
    r = _gen(seed)
    return r(M, Cw).to(dt), (r(I, Cw) / Cw ** 0.5).to(dt), (r(I, Cw) / Cw ** 0.5).to(dt), (0.5 * r(M, I)).to(dt)


def _linear(M, K, N, dt, seed=0):
    r = _gen(seed)
    return dict(x=r(M, K).to(dt), w=(r(N, K) / K ** 0.5).to(dt), bias=(0.5 * r(N)).to(dt), residual=r(M, N).to(dt),
                gate=torch.sigmoid(r(N)).to(dt), dy=(0.5 * r(M, N)).to(dt))


GATED = [(1, 8, 8), (1, 640, 1248), (3, 7, 5), (15, 33, 24), (16, 64, 16), (17, 72, 17), (32, 96, 40), (33, 96, 40), (64, 1, 1),
         (100, 40, 1), (127, 136, 63), (128, 64, 64), (129, 200, 65), (257, 130, 100), (700, 64, 200), (1100, 256, 136)]
# One size for each tile and a few for its edges; sums that are split and that are not.
LARGE = [(2048, 640, 1248), (3001, 200, 776), (5000, 512, 3000), (8192, 128, 1096), (4100, 1000, 264), (16390, 72, 136)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,Cw,I", GATED + LARGE)
def test_gated_forward_and_gradients(M, Cw, I, dt):
    x, wg, wu, dh = _gated(M, Cw, I, dt)
    want = B.gated(x, wg, wu, dh)
    B.check(D.gated_ffn(x, wg, wu), want["h"], "h")
    for name, got in zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(dh, x, wg, wu)):
        B.check(got, want[name], name)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,K,N", GATED + LARGE)
@pytest.mark.parametrize("act,bias,residual,gate", [("none", 0, 0, 0), ("none", 0, 1, 1), ("relu", 1, 0, 0), ("silu", 0, 1, 1),
                                                    ("gelu", 1, 1, 0), ("none", 1, 0, 0), ("none", 1, 1, 1)])
def test_linear_forward_and_gradients(M, K, N, dt, act, bias, residual, gate):
    t = _linear(M, K, N, dt)
    b, r, g = (t[k] if on else None for k, on in (("bias", bias), ("residual", residual), ("gate", gate)))
    want = B.linear(t["x"], t["w"], b, act, r, g, t["dy"])
    B.check(D.linear_epilogue(t["x"], t["w"], b, act, r, g), want["y"], "y")
    got = dict(zip(("dx", "dw", "dbias", "dgate"), D.linear_epilogue_backward(t["dy"], t["x"], t["w"], b, act, g)))
    for name, v in got.items():
        if v is None:
            assert name not in want
        else:
            B.check(v, want[name], name)


# ----------------------------------------------------------------------------- packed activations


@pytest.mark.parametrize("dt", [torch.float32, HF, BF])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (5, 32), (2, 3, 33), (64, 640), (7, 1248), (1000, 77), (333, 641)])
def test_pack_bits_equal_the_reference(shape, dt):
    r = _gen(sum(shape))
    x = (r(*shape) * torch.exp2(4 * r(*shape[:-1], 1))).to(dt)
    x.view(-1)[:: 97] = float("nan")
    x.view(-1)[3:: 89] = float("inf")
    x[-1] = 0
    codes, scales = D.checkpoint_pack(x)
    rc, rs = C.ref_checkpoint_pack(x.cpu())
    assert torch.equal(scales.cpu(), rs)
    nan = torch.isnan(rc.float())
    got = codes.cpu()
    assert torch.equal(torch.isnan(got.float()), nan)
    assert torch.equal(got.view(torch.uint8)[~nan], rc.view(torch.uint8)[~nan])
    for out in (torch.float32, HF, BF):
        torch.testing.assert_close(D.checkpoint_unpack(codes, scales, out).cpu(), C.ref_checkpoint_unpack(rc, rs, out), rtol=0,
                                   atol=0, equal_nan=True)


def test_pack_extremes():
    x = torch.zeros(6, 32, device=DEV)
    x[0, 3], x[1, 3], x[3, 0] = 3.4e38, 1e-40, 2.0 ** -149
    x[2, :2] = torch.tensor([448.0, 464.0])
    x[4] = float("nan")
    x[5] = torch.arange(32, device=DEV) / 512 - 0.03       # e4m3's subnormals
    x[5, 0] = 448
    codes, scales = D.checkpoint_pack(x)
    rc, rs = C.ref_checkpoint_pack(x.cpu())
    assert torch.equal(scales.cpu(), rs)
    for out in (torch.float32, HF, BF):
        torch.testing.assert_close(D.checkpoint_unpack(codes, scales, out).cpu(), C.ref_checkpoint_unpack(rc, rs, out), rtol=0,
                                   atol=0, equal_nan=True)


def test_pack_reads_and_writes_strided_rows():
    r = _gen(5)
    big = r(40, 200).to(BF)
    for cut in (big[:, 8:72], big[:, 3:80], big[::3, 1:34], big.t()[:, :40], big[:, :1]):
        codes, scales = D.checkpoint_pack(cut)
        rc, rs = C.ref_checkpoint_pack(cut.cpu().contiguous())
        assert torch.equal(codes.cpu().view(torch.uint8), rc.view(torch.uint8)) and torch.equal(scales.cpu(), rs)
        assert torch.equal(D.checkpoint_unpack(codes, scales, BF).cpu(), C.ref_checkpoint_unpack(rc, rs, BF))


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,Cw,I", [(1, 8, 8), (33, 96, 40), (129, 200, 65), (257, 130, 100), (1500, 640, 256), (5000, 512, 1500)])
def test_gradients_at_a_packed_input(M, Cw, I, dt):
    x, wg, wu, dh = _gated(M, Cw, I, dt, seed=3)
    codes, scales = D.checkpoint_pack(x)
    kept = B.unpack64(codes, scales)
    want = B.gated(x, wg, wu, dh, kept=kept)
    for name, got in zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(dh, codes, wg, wu, x_scales=scales)):
        B.check(got, want[name], name)
    for act, gate in (("none", True), ("none", False), ("silu", True)):
        t = _linear(M, Cw, I, dt, seed=4)
        codes, scales = D.checkpoint_pack(t["x"])
        g = t["gate"] if gate else None
        want = B.linear(t["x"], t["w"], t["bias"], act, None, g, t["dy"], kept=B.unpack64(codes, scales))
        got = D.linear_epilogue_backward(t["dy"], codes, t["w"], t["bias"], act, g, x_scales=scales)
        for name, v in zip(("dx", "dw", "dbias", "dgate"), got):
            if v is not None:
                B.check(v, want[name], (act, name))


# ----------------------------------------------------------------------------- layouts


def _inside(t, left, right, rows=0, fill=float("nan")):
    """``t`` as a view of a larger tensor that holds ``fill`` around it."""
    big = torch.full((t.shape[0] + 2 * rows, left + t.shape[1] + right), fill, dtype=t.dtype, device=t.device)
    view = big[rows:rows + t.shape[0], left:left + t.shape[1]]
    view.copy_(t)
    return view


@pytest.mark.parametrize("left,right", [(0, 8), (8, 16), (3, 2), (1, 0), (4, 4), (0, 24)])
@pytest.mark.parametrize("M,Cw,I", [(5, 40, 24), (70, 72, 40), (300, 136, 72), (64, 21, 19)])
def test_what_lies_around_the_tensors_does_not_count(M, Cw, I, left, right):
    x, wg, wu, dh = _gated(M, Cw, I, BF, seed=7)
    want = B.gated(x, wg, wu, dh)
    args = [_inside(t, left, right, rows=2) for t in (x, wg, wu)]
    B.check(D.gated_ffn(*args), want["h"], "h")
    for name, got in zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(_inside(dh, left, right, rows=2), *args)):
        B.check(got, want[name], name)
    # the two weights with strides of their own
    args[2] = _inside(wu, left + 8, right, rows=1)
    B.check(D.gated_ffn_backward(dh, *args)[0], want["dx"], "dx")
    t = _linear(M, Cw, I, BF, seed=8)
    v = {k: _inside(t[k], left, right, rows=1) for k in ("x", "w", "residual", "dy")}
    want = B.linear(t["x"], t["w"], t["bias"], "silu", t["residual"], t["gate"], t["dy"])
    B.check(D.linear_epilogue(v["x"], v["w"], t["bias"], "silu", v["residual"], t["gate"]), want["y"], "y")
    for act in ("silu", "none"):
        want = B.linear(t["x"], t["w"], t["bias"], act, t["residual"], t["gate"], t["dy"])
        for name, got in zip(("dx", "dw", "dbias", "dgate"),
                             D.linear_epilogue_backward(v["dy"], v["x"], v["w"], t["bias"], act, t["gate"])):
            B.check(got, want[name], (act, name))


def test_outer_shapes_transposed_and_broadcast_inputs():
    r = _gen(11)
    x = r(3, 40, 64).to(BF)
    wg, wu = (r(64, 24) / 8).to(BF).t(), (r(24, 64) / 8).to(BF)              # a transposed weight
    want = B.gated(x.view(-1, 64), wg, wu)
    got = D.gated_ffn(x, wg, wu)
    assert got.shape == (3, 40, 24)
    B.check(got.view(-1, 24), want["h"], "h")
    xt = x.transpose(0, 1)                                                    # tokens first
    B.check(D.gated_ffn(xt, wg, wu).transpose(0, 1).reshape(-1, 24), want["h"], "h")
    one = r(24).to(BF).requires_grad_()                                       # a broadcast residual, and its gradient
    w = wu.detach().clone().requires_grad_()
    y = D.linear_epilogue(x, w, residual=one.expand(3, 40, 24))
    y.sum().backward()                                                        # a broadcast output gradient
    assert torch.equal(one.grad.float(), torch.full((24,), 120.0, device=DEV))
    want = B.linear(x.view(-1, 64), wu, dy=torch.ones(120, 24, device=DEV, dtype=BF))
    B.check(w.grad, want["dw"], "dw")


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes into x, dh and the outputs' operands."""
    M, Cw, I, ld = 70000, 32, 16, 32768
    big = torch.zeros(M, ld, dtype=BF, device=DEV)                            # 4.6 GB
    x, wg, wu, dh = _gated(M, Cw, I, BF, seed=13)
    view = big[:, 64:64 + Cw]
    view.copy_(x)
    last = slice(M - 300, M)
    want = B.gated(x[last], wg, wu, dh[last])
    B.check(D.gated_ffn(view, wg, wu)[last], want["h"], "h")
    dx, dwg, _ = D.gated_ffn_backward(dh, view, wg, wu)
    B.check(dx[last], want["dx"], "dx")
    B.check(dwg, B.gated(x, wg, wu, dh)["dw_gate"], "dw_gate")
    big[:, 128:128 + I].copy_(dh)
    B.check(D.linear_epilogue(view, wg, residual=big[:, 128:128 + I])[last],
            B.linear(x[last], wg, residual=dh[last])["y"], "y")
    codes, scales = D.checkpoint_pack(big[:, 61:61 + Cw])                     # unaligned rows
    rc, rs = C.ref_checkpoint_pack(big[last, 61:61 + Cw].cpu())
    assert torch.equal(codes[last].cpu().view(torch.uint8), rc.view(torch.uint8)) and torch.equal(scales[last].cpu(), rs)


def test_no_rows():
    x, wg, wu, dh = _gated(4, 40, 24, BF)
    e = x[:0]
    assert D.gated_ffn(e, wg, wu).shape == (0, 24)
    dx, a, b = D.gated_ffn_backward(dh[:0], e, wg, wu)
    assert dx.shape == (0, 40) and not a.any() and not b.any()
    for act in ("none", "gelu"):
        for gate in (None, x.new_ones(24)):
            assert D.linear_epilogue(e, wg, wg[:, 0].contiguous(), act, dh[:0], gate).shape == (0, 24)
            got = D.linear_epilogue_backward(dh[:0], e, wg, x.new_ones(24), act, gate)
            assert got[0].shape == (0, 40) and not any(t.any() for t in got[1:] if t is not None)
    codes, scales = D.checkpoint_pack(e)
    assert codes.shape == (0, 40) and scales.shape == (0, 2) and D.checkpoint_unpack(codes, scales).shape == (0, 40)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 3e38])
@pytest.mark.parametrize("M", [6, 90])
def test_a_bad_row_stays_in_its_row(M, bad):
    x, wg, wu, dh = _gated(M, 48, 40, BF, seed=17)
    t = _linear(M, 48, 40, BF, seed=18)
    rows = torch.arange(M, device=DEV) != 3
    for v in (x, t["x"]):
        v[3, 5] = bad
    want = B.gated(x[rows], wg, wu, dh[rows])
    h = D.gated_ffn(x, wg, wu)
    B.check(h[rows], want["h"], "h")
    assert not torch.isfinite(h[3]).all()
    dx, dwg, _ = D.gated_ffn_backward(dh, x, wg, wu)
    B.check(dx[rows], want["dx"], "dx")
    assert not torch.isfinite(dwg).all()
    want = B.linear(t["x"][rows], t["w"], t["bias"], "gelu", t["residual"][rows], None, t["dy"][rows])
    B.check(D.linear_epilogue(t["x"], t["w"], t["bias"], "gelu", t["residual"])[rows], want["y"], "y")
    B.check(D.linear_epilogue_backward(t["dy"], t["x"], t["w"], t["bias"], "gelu")[0][rows], want["dx"], "dx")


# ----------------------------------------------------------------------------- calls


@pytest.mark.parametrize("needs", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (0, 0, 0)])
def test_gated_gradients_of_some_inputs(needs):
    x, wg, wu, dh = _gated(200, 72, 48, BF, seed=19)
    want = D.gated_ffn_backward(dh, x, wg, wu)
    got = D.gated_ffn_backward(dh, x, wg, wu, needs=tuple(map(bool, needs)))
    for n, g, w in zip(needs, got, want):
        assert torch.equal(g, w) if n else g is None


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("needs", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 0, 1, 1), (1, 0, 0, 1), (0, 0, 0, 0)])
def test_linear_gradients_of_some_inputs(act, needs):
    t = _linear(200, 72, 48, BF, seed=20)
    args = (t["dy"], t["x"], t["w"], t["bias"], act, t["gate"])
    want = D.linear_epilogue_backward(*args)
    got = D.linear_epilogue_backward(*args, needs=tuple(map(bool, needs)))
    for n, g, w in zip(needs, got, want):
        assert torch.equal(g, w) if n else g is None


def test_the_same_bits_every_time_and_on_two_streams():
    x, wg, wu, dh = _gated(3000, 640, 1248, BF, seed=21)
    t = _linear(3000, 1248, 640, BF, seed=22)

    def all_of():
        return [D.gated_ffn(x, wg, wu), *D.gated_ffn_backward(dh, x, wg, wu),
                *D.linear_epilogue_backward(t["dy"], t["x"], t["w"], t["bias"], "silu", t["gate"]),
                *D.linear_epilogue_backward(t["dy"], t["x"], t["w"], t["bias"], "none", t["gate"])]

    want = all_of()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(all_of())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_out_may_be_the_residual():
    """The C entry's documented in-place form: out = the residual's own rows."""
    from maba_sparse import _native as N
    t = _linear(333, 72, 48, BF, seed=23)
    want = D.linear_epilogue(t["x"], t["w"], None, "none", t["residual"], t["gate"])
    y = t["residual"].clone()
    rc = N.load().maba_hip_linear_epilogue(N.desc(t["x"]), N.desc(t["w"]), None, 0, N.desc(y), N.desc(t["gate"]), N.desc(y), None, 0,
                                           N.stream_ptr(y.device))
    N.check(rc, "linear_epilogue")
    assert torch.equal(y, want)


@pytest.mark.parametrize("M,K,N", [(7, 640, 96), (40, 2816, 104), (64, 5504, 130), (300, 70, 47), (2100, 640, 640), (4096, 128, 2504),
                                   (5000, 72, 1100)])
def test_the_residual_is_updated_in_place_by_every_kernel(M, K, N):
    from maba_sparse import _native as N_
    t = _linear(M, K, N, BF, seed=24)
    want = D.linear_epilogue(t["x"], t["w"], t["bias"], "silu", t["residual"], t["gate"])
    y = t["residual"].clone()
    lib = N_.load()
    need = lib.maba_hip_linear_epilogue_workspace_size(N_.rows_desc(t["x"]), N_.rows_desc(t["w"]))
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    N_.check(lib.maba_hip_linear_epilogue(*map(N_.rows_desc, (t["x"], t["w"], t["bias"])), 2, *map(N_.rows_desc, (y, t["gate"], y)),
                                          ws.data_ptr(), ws.numel(), N_.stream_ptr(y.device)), "linear_epilogue")
    assert torch.equal(y, want)


@pytest.mark.parametrize("K", [1, 8, 63, 64, 65, 128, 129, 192, 250, 256, 257, 320, 328, 640, 1000])
@pytest.mark.parametrize("M", [33, 70, 128])
def test_a_few_tiles_of_every_length(M, K):
    """Fewer stages than the small tile holds, as many, and more."""
    x, wg, wu, dh = _gated(M, K, 72, BF, seed=41)
    B.check(D.gated_ffn(x, wg, wu), B.gated(x, wg, wu)["h"], "h")
    t = _linear(M, K, 72, HF, seed=42)
    want = B.linear(t["x"], t["w"], t["bias"], "silu", t["residual"], t["gate"], t["dy"])
    B.check(D.linear_epilogue(t["x"], t["w"], t["bias"], "silu", t["residual"], t["gate"]), want["y"], "y")
    got = D.linear_epilogue_backward(t["dy"], t["x"], t["w"], t["bias"], "silu", t["gate"])
    for name, v in zip(("dx", "dw", "dbias", "dgate"), got):
        B.check(v, want[name], name)


@pytest.mark.parametrize("K", [320, 328, 449, 576, 1000, 1160, 1250])
@pytest.mark.parametrize("M,N", [(600, 640), (2048, 640), (4000, 640), (6100, 640), (8190, 636), (1777, 1000)])
def test_two_groups_of_waves_on_a_tile(M, N, K):
    """Tiles fewer than compute units; odd and even numbers of stages, each group's half."""
    t = _linear(M, K, N, BF, seed=45)
    want = B.linear(t["x"], t["w"], t["bias"], "relu", t["residual"], t["gate"])
    B.check(D.linear_epilogue(t["x"], t["w"], t["bias"], "relu", t["residual"], t["gate"]), want["y"], "y")
    # dx of a layer of K outputs: the sum runs over K
    dy, w = t["x"], t["w"].t().contiguous()
    want = B.linear(t["residual"], w, None, "none", None, None, dy)
    B.check(D.linear_epilogue_backward(dy, t["residual"], w, needs=(True, False, False, False))[0], want["dx"], "dx")
    if M < 3000:
        x, wg, wu, dh = _gated(M, N, K // 2 + 5, HF, seed=46)
        B.check(D.gated_ffn_backward(dh, x, wg, wu, needs=(True, False, False))[0], B.gated(x, wg, wu, dh)["dx"], "dx")


@pytest.mark.parametrize("K", [1528, 1536, 1537, 1544, 2048, 2056])
@pytest.mark.parametrize("M", [16, 17, 32, 33])
def test_where_few_rows_change_kernels(M, K):
    x, wg, wu, _ = _gated(M, K, 40, BF, seed=43)
    B.check(D.gated_ffn(x, wg, wu), B.gated(x, wg, wu)["h"], "h")
    t = _linear(M, K, 40, BF, seed=44)
    B.check(D.linear_epilogue(t["x"], t["w"], None, "gelu", t["residual"]),
            B.linear(t["x"], t["w"], None, "gelu", t["residual"])["y"], "y")


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_activations_over_their_whole_range(act, dt):
    """z and dz themselves, through a unit weight: from where the activation vanishes to where it is z."""
    z = torch.cat([torch.linspace(-16, 16, 8 * 900), torch.linspace(-90, 90, 8 * 99), 2.0 ** torch.arange(-20.0, 12.0),
                   -2.0 ** torch.arange(-20.0, 12.0)])
    x = z.reshape(-1, 8).to(dt).to(DEV)
    w, dy = torch.eye(8, device=DEV, dtype=dt), torch.ones(x.shape, device=DEV, dtype=dt)
    want = B.linear(x, w, None, act, None, None, dy)
    B.check(D.linear_epilogue(x, w, None, act), want["y"], "y")
    B.check(D.linear_epilogue_backward(dy, x, w, None, act)[0], want["dx"], "dx")


@pytest.mark.parametrize("ckpt", [None, "e4m3"])
@pytest.mark.parametrize("M,Cw,I", [(1, 64, 96), (50, 64, 96), (1000, 200, 136)])
def test_a_block_trained_through_autograd(M, Cw, I, ckpt):
    """Both operators in a row, as the model's feed-forward half runs them: each one's gradients against its
    formulas at the values that it saw."""
    r = _gen(M)
    x, res = r(M, Cw).to(BF).requires_grad_(), r(M, Cw).to(BF).requires_grad_()
    wg, wu, wd = ((r(a, b) / b ** 0.5).to(BF).requires_grad_() for a, b in ((I, Cw), (I, Cw), (Cw, I)))
    gate = torch.sigmoid(r(Cw)).to(BF).requires_grad_()
    h = D.gated_ffn(x, wg, wu, checkpoint=ckpt)
    h.retain_grad()
    y = D.linear_epilogue(h, wd, residual=res, gate=gate, checkpoint=ckpt)
    dy = r(M, Cw).to(BF)
    y.backward(dy)

    def kept(t):
        return B.unpack64(*D.checkpoint_pack(t.detach())) if ckpt else None

    with torch.no_grad():
        want = B.linear(h, wd, None, "none", res, gate, dy, kept=kept(h))
        for got, name in ((y, "y"), (h.grad, "dx"), (wd.grad, "dw"), (gate.grad, "dgate")):
            B.check(got, want[name], name)
        assert torch.equal(res.grad, dy)
        want = B.gated(x, wg, wu, h.grad, kept=kept(x))
        for got, name in ((h, "h"), (x.grad, "dx"), (wg.grad, "dw_gate"), (wu.grad, "dw_up")):
            B.check(got, want[name], name)


def test_fp32_takes_the_reference_path(monkeypatch):
    x, wg, wu, dh = _gated(20, 24, 16, torch.float32)
    with pytest.raises(RuntimeError):                        # strict: a fallback is an error
        D.gated_ffn(x, wg, wu)
    monkeypatch.setenv("MABA_STRICT_BACKEND", "0")
    with pytest.warns(RuntimeWarning):
        D.clear_fallback_warnings()
        got = D.gated_ffn(x, wg, wu)
    torch.testing.assert_close(got, C.ref_gated_ffn(x, wg, wu))


def test_model_block_fused_feed_forward():
    from maba_sparse.model import SwiGLUFFN
    torch.manual_seed(3)
    ffn = SwiGLUFFN(640, 1248, fused=True, checkpoint="e4m3").to(DEV, BF)
    x = torch.randn(2, 300, 640, device=DEV).to(BF)
    res, gate = torch.randn_like(x), torch.rand(640, device=DEV).to(BF)
    y = ffn.forward_fused(x, residual=res, gate=gate)
    y.float().square().mean().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in ffn.parameters())
    with torch.no_grad():
        h = D.gated_ffn(x, ffn.w_gate.weight, ffn.w_up.weight)
        assert torch.equal(y, D.linear_epilogue(h, ffn.w_down.weight, residual=res, gate=gate))
        assert torch.equal(ffn(x), ffn.forward_hip(x))


# ----------------------------------------------------------------------------- the native binding and the Python path


def _both_ways(monkeypatch, call):
    """``call`` through the native binding and, with wrapped kernels registered, through Python."""
    native = call()
    hip = D._KERNEL_REGISTRY["hip"]
    used = []
    for name in ("gated_ffn", "gated_ffn_backward", "linear_epilogue", "linear_epilogue_backward", "checkpoint_pack",
                 "checkpoint_unpack"):
        def wrapped(_f=hip[name], _n=name, **kw):
            used.append(_n)
            return _f(**kw)
        monkeypatch.setitem(hip, name, wrapped)
    return native, call(), used


@pytest.mark.parametrize("ckpt", [None, "e4m3"])
@pytest.mark.parametrize("shape", [(5, 64), (3, 50, 72), (200, 33), (64,)])
def test_native_and_python_paths_give_the_same_bits(monkeypatch, shape, ckpt):
    r = _gen(71)
    Cw = shape[-1]
    x, wg, wu, w = (r(*s).to(BF).requires_grad_() for s in (shape, (40, Cw), (40, Cw), (24, 40)))
    b, g, res = (r(*s).to(BF).requires_grad_() for s in ((24,), (24,), (*shape[:-1], 24)))
    dy = r(*shape[:-1], 24).to(BF)

    def call():
        h = D.gated_ffn(x, wg, wu, checkpoint=ckpt)
        y = D.linear_epilogue(h, w, b, "gelu", res, g, checkpoint=ckpt)
        with torch.no_grad():
            plain = D.linear_epilogue(D.gated_ffn(x, wg, wu), w, b, "gelu", res, g)
        codes, scales = D.checkpoint_pack(x)
        grads = torch.autograd.grad(y, (x, wg, wu, w, b, res, g), dy)
        some = torch.autograd.grad(D.linear_epilogue(x.detach(), wg, None, "none", None, None), (wg,), torch.ones_like(h))
        return [y, plain, codes.view(torch.uint8), scales, D.checkpoint_unpack(codes, scales, HF), *grads, *some]

    native, python, used = _both_ways(monkeypatch, call)
    assert set(used) >= {"gated_ffn", "gated_ffn_backward", "linear_epilogue", "linear_epilogue_backward", "checkpoint_pack"}
    assert all(a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(native, python))


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (4,), (0, 2), (2, 3), (1, 4)])
@pytest.mark.parametrize("act,ckpt", [("none", None), ("none", "e4m3"), ("silu", None), ("silu", "e4m3")])
def test_autograd_of_some_inputs(act, ckpt, which):
    """Frozen inputs change nothing for the others, also where x need not be kept."""
    t = _linear(70, 48, 40, BF, seed=75)
    names = ("x", "w", "bias", "residual", "gate")

    def grads(live):
        a = [t[n].detach().clone().requires_grad_(i in live) for i, n in enumerate(names)]
        y = D.linear_epilogue(a[0], a[1], a[2], act, a[3], a[4], checkpoint=ckpt)
        return dict(zip(live, torch.autograd.grad(y, [a[i] for i in live], t["dy"])))

    every = grads(range(5))
    for i, g in grads(which).items():
        assert torch.equal(g, every[i]), names[i]


def test_double_backward_is_refused_and_first_is_not():
    x, wg, wu, dh = _gated(20, 64, 24, BF, seed=72)
    x.requires_grad_()
    w = wg.detach().clone().requires_grad_()
    for call in (lambda: D.gated_ffn(x, w, wu), lambda: D.linear_epilogue(x, w, None, "silu")):
        plain = torch.autograd.grad(call(), (x, w), dh)
        grads = torch.autograd.grad(call(), (x, w), dh, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, grads))
        with pytest.raises(RuntimeError, match="twice"):
            (grads[0].float().sum() + grads[1].float().sum()).backward()


def test_calls_that_the_binding_declines_raise_as_before():
    x, wg, wu, _ = _gated(20, 64, 24, BF, seed=73)
    with pytest.raises(RuntimeError, match="same device"):
        D.gated_ffn(x, wg.cpu(), wu)
    with pytest.raises(TypeError, match="dtypes must match"):
        D.gated_ffn(x, wg.half(), wu)
    with pytest.raises(ValueError, match="w_gate"):
        D.gated_ffn(x[:, :32], wg, wu)
    with pytest.raises(ValueError, match="w_up"):
        D.gated_ffn(x, wg, wu[:-1])
    with pytest.raises(ValueError, match="checkpoint"):
        D.gated_ffn(x, wg, wu, checkpoint="int4")
    with pytest.raises(ValueError, match="residual"):
        D.linear_epilogue(x, wg, None, "none", x)
    with pytest.raises(ValueError, match="gate"):
        D.linear_epilogue(x, wg, gate=wg[0])
    with pytest.raises(ValueError, match="activation"):
        D.linear_epilogue(x, wg, None, "tanh")
    codes, scales = D.checkpoint_pack(x)
    with pytest.raises(ValueError, match="x_scales"):
        D.checkpoint_unpack(codes, scales[:, :1])
    with pytest.raises(TypeError):
        D.checkpoint_unpack(codes, scales, torch.float64)


def test_saved_tensors_follow_their_hooks_and_versions():
    x, wg, wu, dh = _gated(20, 64, 24, BF, seed=74)
    x.requires_grad_()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t.cpu(), lambda t: t.to(DEV)):
        y = D.gated_ffn(x, wg, wu)
    assert len(seen) == 3
    assert torch.equal(torch.autograd.grad(y, x, dh)[0], torch.autograd.grad(D.gated_ffn(x, wg, wu), x, dh)[0])
    w = wg.clone()
    y = D.gated_ffn(x, w, wu)
    w.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dh)


def test_two_threads_call_at_once():
    import threading
    sets = [_gated(300 + 40 * i, 136, 72, BF, seed=80 + i) for i in range(2)]
    want = [torch.autograd.grad(D.gated_ffn(x.requires_grad_(), wg, wu), x, dh)[0] for x, wg, wu, dh in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        x, wg, wu, dh = sets[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = torch.autograd.grad(D.gated_ffn(x, wg, wu, checkpoint=None), x, dh)[0]
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


# ----------------------------------------------------------------------------- graphs


def test_captured_step_replays_with_new_inputs():
    """Forward and backward ops recorded once, replayed on new data between eager calls of the same ops."""
    M, Cw, I = 2050, 128, 264
    x, wg, wu, dh = _gated(M, Cw, I, BF, seed=31)
    t = _linear(M, I, Cw, BF, seed=32)

    def step():
        h = D.gated_ffn(x, wg, wu)
        y = D.linear_epilogue(h, t["w"], t["bias"], "silu", t["residual"], t["gate"])
        codes, scales = D.checkpoint_pack(h)
        down = D.linear_epilogue_backward(t["dy"], codes, t["w"], t["bias"], "silu", t["gate"], x_scales=scales)
        plain = D.linear_epilogue_backward(t["dy"], h, t["w"], t["bias"], "none", t["gate"])
        up = D.gated_ffn_backward(down[0], x, wg, wu)
        return [h, y, *down, *plain, *up, D.checkpoint_unpack(codes, scales, BF)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    r = _gen(33)
    for _ in range(4):
        for v in (x, dh, t["dy"], t["residual"]):
            v.copy_(r(*v.shape).to(BF))
        g.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        torch.cuda.synchronize()


def test_two_graphs_of_one_pool_replayed_by_turns():
    """Their workspaces share memory: each replay must make all that it reads."""
    sets = [(_gated(600 + 90 * i, 72, 104, BF, seed=50 + i), _linear(40 + 30 * i, 2816, 72, BF, seed=60 + i)) for i in range(2)]

    def step(s):
        (x, wg, wu, dh), t = s
        return [*D.gated_ffn_backward(dh, x, wg, wu), D.linear_epilogue(t["x"], t["w"], t["bias"], "relu", t["residual"]),
                *D.linear_epilogue_backward(t["dy"], t["x"], t["w"], t["bias"], "gelu", t["gate"])]

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


def test_captured_autograd_step():
    """A whole training step recorded through autograd once no eager graph of its leaves lives."""
    x, wg, wu, dh = _gated(130, 64, 72, BF, seed=35)
    leaves = [v.requires_grad_() for v in (x, wg, wu)]

    def step():
        return torch.autograd.grad(D.gated_ffn(*leaves, checkpoint="e4m3"), leaves, dh)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    r = _gen(36)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(r(*x.shape).to(BF))
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_capture_beside_a_live_eager_graph_is_refused():
    """The forward of such a capture raises before any backward could reach the eager graph's nodes; the
    backward ops themselves can be captured beside it."""
    x, wg, wu, dh = _gated(70, 64, 40, BF, seed=37)
    w = wg.requires_grad_()
    eager = D.gated_ffn(x, w, wu)                            # keeps the leaf's node on the current stream
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(g):
            D.gated_ffn(x, w, wu)
    torch.cuda.synchronize()
    g2 = torch.cuda.CUDAGraph()
    wd = w.detach()
    with torch.cuda.graph(g2):
        out = D.gated_ffn_backward(dh, x, wd, wu)
    g2.replay()
    torch.cuda.synchronize()
    (want,) = torch.autograd.grad(eager, (w,), dh)
    assert torch.equal(out[1], want)
    del eager
    gc.collect()


@pytest.mark.parametrize("env,reference", [("reference", True), ("HIP", False), ("auto", False), ("", False)])
def test_the_backend_that_is_asked_for(monkeypatch, env, reference):
    x, wg, wu, _ = _gated(20, 64, 24, BF, seed=76)
    used = []

    def ref(_f=D._KERNEL_REGISTRY["reference"]["gated_ffn"], **kw):
        used.append("reference")
        return _f(**kw)

    monkeypatch.setitem(D._KERNEL_REGISTRY["reference"], "gated_ffn", ref)
    monkeypatch.setenv("MABA_BACKEND", env)
    B.check(D.gated_ffn(x, wg, wu), B.gated(x, wg, wu)["h"], "h")
    assert bool(used) == reference
    monkeypatch.setenv("MABA_BACKEND", "rocm")
    with pytest.raises(ValueError):
        D.gated_ffn(x, wg, wu)


def test_outputs_are_ordinary_autograd_tensors():
    """In-place changes of an output are recorded, and refused once a later op has kept it."""
    x, wg, wu, dh = _gated(20, 64, 24, BF, seed=77)
    w = _linear(20, 24, 16, BF, seed=78)["w"]
    x.requires_grad_()
    h = D.gated_ffn(x, wg, wu)
    assert not h.is_leaf and not h.is_inference()
    h.mul_(2)
    want = torch.autograd.grad(D.gated_ffn(x, wg, wu), x, 2 * dh)[0]
    assert torch.equal(torch.autograd.grad(h, x, dh)[0], want)
    h = D.gated_ffn(x, wg, wu)
    w.requires_grad_()
    y = D.linear_epilogue(h, w)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with torch.inference_mode():
        assert D.gated_ffn(x, wg, wu).is_inference()


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("M,Cw,I", [(5, 72, 48), (70, 72, 48), (300, 136, 264)])
@pytest.mark.parametrize("up_first", [False, True])
def test_weights_cut_from_one_tensor_at_unlike_alignments(M, Cw, I, up_first, dt):
    """Two column ranges of one tensor, only one of which starts on a 16-byte boundary: one row stride, one weight read
    in place and one copied by the forward."""
    x, wg, wu, dh = _gated(M, Cw, I, dt, seed=90)
    want = B.gated(x, wg, wu, dh)
    big = torch.full((I, 2 * Cw + 24), float("nan"), dtype=dt, device=DEV)
    a, b = big[:, :Cw], big[:, Cw + 4:2 * Cw + 4]
    vg, vu = (b, a) if up_first else (a, b)
    vg.copy_(wg)
    vu.copy_(wu)
    B.check(D.gated_ffn(x, vg, vu), want["h"], "h")
    for name, got in zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(dh, x, vg, vu)):
        B.check(got, want[name], name)
    codes, scales = D.checkpoint_pack(x)
    want = B.gated(x, wg, wu, dh, kept=B.unpack64(codes, scales))
    B.check(D.gated_ffn_backward(dh, codes, vg, vu, x_scales=scales)[0], want["dx"], "dx")


@pytest.mark.parametrize("M", [1, 5, 64, 100, 1000])
@pytest.mark.parametrize("act,gate", [("none", False), ("none", True), ("silu", True)])
def test_rows_that_are_broadcast_or_overlap(M, act, gate):
    """x, the output's gradient or both as one row repeated (strides (0, 1)) or as windows of a signal (strides (8, 1)):
    no row past the last one counts."""
    t = _linear(M, 64, 72, BF, seed=91)
    r = _gen(92)

    def forms(width):
        yield r(1, width).to(BF).expand(M, width)
        yield r(8 * M + width).to(BF).as_strided((M, width), (8, 1))

    g = t["gate"] if gate else None
    for x in (*forms(64), t["x"]):
        for dy in (*forms(72), t["dy"]):
            want = B.linear(x, t["w"], t["bias"], act, None, g, dy)
            for name, got in zip(("dx", "dw", "dbias", "dgate"), D.linear_epilogue_backward(dy, x, t["w"], t["bias"], act, g)):
                if got is not None:
                    B.check(got, want[name], (act, name))
    w = t["w"].clone().requires_grad_()
    x = r(1, 64).to(BF).expand(M, 64)
    D.linear_epilogue(x, w).sum(0).float().sum().backward()              # autograd hands back one row for all
    B.check(w.grad, B.linear(x, w.detach(), dy=torch.ones(M, 72, dtype=BF, device=DEV))["dw"], "dw")


def test_gated_rows_that_are_broadcast_or_overlap():
    r = _gen(93)
    for M in (1, 100, 1000):
        _, wg, wu, dh = _gated(M, 64, 72, BF, seed=94)
        for x in (r(1, 64).to(BF).expand(M, 64), r(8 * M + 64).to(BF).as_strided((M, 64), (8, 1))):
            for d in (dh, dh[:1].expand(M, 72)):
                want = B.gated(x, wg, wu, d)
                B.check(D.gated_ffn(x, wg, wu), want["h"], "h")
                for name, got in zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(d, x, wg, wu)):
                    B.check(got, want[name], name)
        one = wg[:1].expand(72, 64)                                       # and weights whose rows are one
        want = B.gated(t := r(M, 64).to(BF), one, one, dh)
        for name, got in zip(("dx", "dw_gate", "dw_up"), D.gated_ffn_backward(dh, t, one, one)):
            B.check(got, want[name], name)


def test_tangents_take_the_reference_path(monkeypatch):
    """Forward-mode derivatives of 16-bit calls: the reference ops' with one warning, an error where fallbacks are errors."""
    from torch.autograd import forward_ad
    x, wg, wu, dh = _gated(20, 64, 24, BF, seed=95)
    t = _gen(96)(20, 64).to(BF)
    calls = [(lambda f, x, g: f(x, wg, wu), D.gated_ffn, C.ref_gated_ffn),
             (lambda f, x, g: f(x, wg, None, "silu", None, wu[:, 0]), D.linear_epilogue, C.ref_linear_epilogue),
             (lambda f, x, g: f(g, x, wg, wu)[0], D.gated_ffn_backward, C.ref_gated_ffn_backward)]
    for call, op, ref in calls:
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x, t)
            with pytest.raises(RuntimeError):
                call(op, dual, dh)
            monkeypatch.setenv("MABA_STRICT_BACKEND", "0")
            D.clear_fallback_warnings()
            with pytest.warns(RuntimeWarning, match="tangents"):
                got = forward_ad.unpack_dual(call(op, dual, dh))
            monkeypatch.setenv("MABA_STRICT_BACKEND", "1")
            want = forward_ad.unpack_dual(call(ref, dual, dh))
        assert got.tangent is not None
        assert torch.equal(got.tangent, want.tangent) and torch.equal(got.primal, want.primal)


@pytest.mark.parametrize("ckpt", [None, "e4m3"])
@pytest.mark.parametrize("at", [BF, HF])
@pytest.mark.parametrize("xt", [torch.float32, BF, HF])
def test_fp32_parameters_under_autocast_reach_the_kernels(xt, at, ckpt):
    """The usual mixed-precision recipe: the values and gradients of a call on cast tensors, the gradients in each leaf's
    type.  A fallback would raise (``strict``)."""
    r = _gen(97)
    x, res = r(70, 64).to(xt).requires_grad_(), r(70, 40).requires_grad_()
    wg, wu, w, b, g = (r(*s).requires_grad_() for s in ((72, 64), (72, 64), (40, 72), (40,), (40,)))
    dy = r(70, 40)
    leaves = (x, wg, wu, w, b, res, g)

    def cast(*ts):
        return (t.to(at) for t in ts)

    with torch.autocast("cuda", at):
        h = D.gated_ffn(x, wg, wu, checkpoint=ckpt)
        y = D.linear_epilogue(h, w, b, "silu", res, g, checkpoint=ckpt)
        narrow = D.linear_epilogue(h, w, b, "silu", *cast(res, g), checkpoint=ckpt)
    assert h.dtype == narrow.dtype == at and y.dtype == torch.float32
    h2 = D.gated_ffn(*cast(x, wg, wu), checkpoint=ckpt)
    want = torch.addcmul(res, g, D.linear_epilogue(h2, *cast(w, b), "silu", checkpoint=ckpt).float())
    want_narrow = D.linear_epilogue(h2, *cast(w, b), "silu", *cast(res, g), checkpoint=ckpt)
    assert torch.equal(y, want) and torch.equal(narrow, want_narrow)
    for a, c, d in ((y, want, dy), (narrow, want_narrow, dy.to(at))):
        for got, ref, leaf in zip(torch.autograd.grad(a, leaves, d, retain_graph=True),
                                  torch.autograd.grad(c, leaves, d, retain_graph=True), leaves):
            assert got.dtype == leaf.dtype and torch.equal(got, ref)


def test_the_model_feed_forward_under_autocast():
    from maba_sparse.model import SwiGLUFFN
    torch.manual_seed(4)
    plain, fused = SwiGLUFFN(64, 96).to(DEV), SwiGLUFFN(64, 96, fused=True).to(DEV)
    fused.load_state_dict(plain.state_dict())
    for x in (torch.randn(90, 64, device=DEV), torch.randn(90, 64, device=DEV).to(BF)):
        with torch.autocast("cuda", BF):
            a, b = plain(x), fused(x)
            b.float().square().mean().backward()                       # inside the region
        assert a.dtype == b.dtype == BF
        assert all(p.grad.dtype == torch.float32 and bool(torch.isfinite(p.grad).all()) for p in fused.parameters())


@pytest.mark.parametrize("kind", ["another op", "under autocast", "python path"])
def test_capture_beside_an_eager_graph_of_any_op_is_refused(monkeypatch, kind):
    """The leaf's node is known by the stream that it was made on, whichever op made it and whatever cast lies between.
    Only forwards are recorded here; once the eager graph is gone the same call is taken."""
    x, wg, wu, dh = _gated(70, 64, 40, BF, seed=98)
    if kind == "under autocast":
        x, wg = x.float(), wg.float()
    w = wg.requires_grad_()
    if kind == "python path":
        hip = D._KERNEL_REGISTRY["hip"]
        monkeypatch.setitem(hip, "gated_ffn", lambda _f=hip["gated_ffn"], **kw: _f(**kw))

    def call():
        with torch.autocast("cuda", BF, enabled=kind == "under autocast"):
            return D.gated_ffn(x, w, wu)

    call()
    eager = torch.nn.functional.linear(x, w)                 # another op's graph, on the current stream
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
    assert torch.equal(out, call())
