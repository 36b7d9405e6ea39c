"""The feed-forward operators on the CPU: the reference backend's values and gradients, what a
checkpoint keeps, the packed format against its definition, refusals of the dispatcher and of the C
entry points (which return before any GPU work)."""
import ctypes
import os

import pytest
import torch

import _ffn_bounds as B
from maba_sparse import _native as N
from maba_sparse.kernels import common as C
from maba_sparse.kernels import dispatcher as D
from maba_sparse.model import MabaBlock, MabaConfig, SwiGLUFFN

F64 = torch.float64


def _rand(*shape, dtype=F64, grad=True, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=g, dtype=F64).to(dtype).requires_grad_(grad)


# ----------------------------------------------------------------------------- values and gradients


def test_gated_gradients_against_differences():
    x, wg, wu = _rand(2, 3, 12), _rand(7, 12, seed=1), _rand(7, 12, seed=2)
    assert torch.autograd.gradcheck(D.gated_ffn, (x, wg, wu))


@pytest.mark.parametrize("act", C.ACTIVATIONS)
def test_linear_gradients_against_differences(act):
    x, w, b, r, g = _rand(2, 3, 12), _rand(7, 12, seed=1), _rand(7, seed=2), _rand(2, 3, 7, seed=3), _rand(7, seed=4)
    assert torch.autograd.gradcheck(lambda x, w, b, r, g: D.linear_epilogue(x, w, b, act, r, g), (x, w, b, r, g))
    assert torch.autograd.gradcheck(lambda x, w: D.linear_epilogue(x, w, activation=act), (x, w))


@pytest.mark.parametrize("needs", [(1, 0, 0, 0, 0), (0, 1, 0, 0, 0), (0, 0, 1, 0, 0), (0, 0, 0, 1, 0), (0, 0, 0, 0, 1), (0, 0, 1, 1, 0)])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_linear_gradients_of_some_inputs(act, needs):
    full = [_rand(5, 12), _rand(7, 12, seed=1), _rand(7, seed=2), _rand(5, 7, seed=3), _rand(7, seed=4)]
    y = D.linear_epilogue(*[full[0], full[1], full[2]], act, full[3], full[4])
    want = torch.autograd.grad(y.sum(), full)
    some = [t.detach().requires_grad_(bool(n)) for t, n in zip(full, needs)]
    y = D.linear_epilogue(some[0], some[1], some[2], act, some[3], some[4], checkpoint=None)
    y.sum().backward()
    for t, n, w in zip(some, needs, want):
        assert (t.grad is not None) == bool(n)
        if n:
            torch.testing.assert_close(t.grad, w)


def test_double_backward_is_refused():
    x, wg, wu = _rand(2, 8), _rand(3, 8, seed=1), _rand(3, 8, seed=2)
    (g,) = torch.autograd.grad(D.gated_ffn(x, wg, wu).sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_plain_values_match_torch_modules():
    torch.manual_seed(0)
    ffn = SwiGLUFFN(16, 24).double()
    x = _rand(3, 5, 16, grad=False)
    fused = SwiGLUFFN(16, 24, fused=True).double()
    fused.load_state_dict(ffn.state_dict())
    torch.testing.assert_close(fused(x), ffn(x))


# ----------------------------------------------------------------------------- checkpoints


def _pack_by_definition(row):
    """One row's values, codes and scales from the definition, in Python floats."""
    steps = sorted({s * m * 2.0 ** (e - 3) for s in (1, -1) for e in range(-6, 9) for m in range(8, 16)}
                   | {s * m * 2.0 ** -9 for s in (1, -1) for m in range(8)})
    steps = [v for v in steps if abs(v) <= 448]
    vals, scales = [], []
    for k in range(0, len(row), 32):
        grp = row[k:k + 32]
        amax = max([abs(v) for v in grp if v == v and abs(v) != float("inf")], default=0.0)
        e = -127
        while amax > 448 * 2.0 ** e:
            e += 1
        scales.append(e + 127)
        for v in grp:
            if v != v or abs(v) == float("inf"):
                vals.append(float("nan"))
                continue
            r = v / 2.0 ** e
            near = min(abs(r - s) for s in steps)
            at = [s for s in steps if abs(r - s) == near]
            if len(at) > 1:               # ties: the even code, whose last mantissa bit is zero
                def odd(s):
                    import math
                    m, x = math.frexp(abs(s)) if s else (0.0, 0)
                    return int(abs(s) * 2 ** 9) % 2 if abs(s) < 2.0 ** -6 else int(m * 16) % 2
                at = [s for s in at if not odd(s)] or at
            vals.append(at[0] * 2.0 ** e)
    return vals, scales


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("width", [1, 31, 32, 33, 70])
def test_pack_follows_its_definition(dtype, width):
    g = torch.Generator().manual_seed(width)
    x = (torch.randn(6, width, generator=g) * torch.tensor([1.0, 300.0, 1e-3, 1.0, 0.0, 1.0])[:, None]).to(dtype)
    x[3] = (torch.arange(width) - width // 2).to(dtype) / 16        # exact steps and ties
    x[5, 0] = float("inf")
    x[5, -1] = float("nan")
    codes, scales = D.checkpoint_pack(x)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape
    assert scales.dtype == torch.uint8 and scales.shape == (6, -(-width // 32))
    got = B.unpack64(codes, scales)
    for r in range(6):
        vals, sc = _pack_by_definition([float(v) for v in x[r]])
        assert scales[r].tolist() == sc
        torch.testing.assert_close(got[r], torch.tensor(vals, dtype=F64), rtol=0, atol=0, equal_nan=True)


def test_pack_extremes():
    x = torch.zeros(5, 32)
    x[0, 3] = 3.4e38
    x[1, 3] = 1e-40
    x[2, :2] = torch.tensor([448.0, 464.0])          # 464 needs the next power of two
    x[3, 0] = 2.0 ** -149
    x[4] = float("nan")
    codes, scales = D.checkpoint_pack(x)
    assert scales[:, 0].tolist() == [247, 0, 128, 0, 0]
    y = D.checkpoint_unpack(codes, scales, torch.float32)
    assert float(y[0, 3]) == 2.0 ** 128 * (1 - 2.0 ** -3) or abs(float(y[0, 3]) / 3.4e38 - 1) <= 2.0 ** -4
    assert abs(float(y[1, 3]) / 1e-40 - 1) <= 2.0 ** -4
    assert bool(torch.isnan(y[4]).all())


def test_pack_error_is_half_a_step():
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(1))
    codes, scales = D.checkpoint_pack(x)
    y = B.unpack64(codes, scales)
    amax = x.view(64, 3, 32).abs().amax(-1, keepdim=True).expand(64, 3, 32).reshape(64, 96).double()
    # 2^-4 relative; below the type's normal range half of its smallest step, and the scale is under amax / 224
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, amax / 224 * 2.0 ** -10)
    assert bool(((y - x).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_checkpoint_gradients_are_those_at_the_unpacked_input(dtype):
    x, wg, wu = (_rand(*s, dtype=dtype, seed=i) for i, s in enumerate([(9, 40), (11, 40), (11, 40)]))
    dh = _rand(9, 11, dtype=dtype, grad=False)
    y = D.gated_ffn(x, wg, wu, checkpoint="e4m3")
    assert torch.equal(y, D.gated_ffn(x, wg, wu))                # the forward result is unaffected
    got = torch.autograd.grad(y, (x, wg, wu), dh)
    codes, scales = D.checkpoint_pack(x.detach())
    xh = D.checkpoint_unpack(codes, scales, dtype)
    want = D.gated_ffn_backward(dh, xh.detach(), wg.detach(), wu.detach())
    again = D.gated_ffn_backward(dh, codes, wg.detach(), wu.detach(), x_scales=scales)
    for a, b, c in zip(got, want, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_a_checkpoint_keeps_eight_bits():
    x, wg, wu = _rand(64, 64, dtype=torch.bfloat16), _rand(8, 64, dtype=torch.bfloat16), _rand(8, 64, dtype=torch.bfloat16)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        D.gated_ffn(x, wg, wu, checkpoint="e4m3")
    assert sorted(str(t.dtype) for t in seen) == ["torch.bfloat16"] * 2 + ["torch.float8_e4m3fn", "torch.uint8"]
    assert all(t.data_ptr() != x.data_ptr() for t in seen)


def test_frozen_layer_without_activation_keeps_no_input():
    x, w, g = _rand(6, 8), _rand(5, 8, grad=False), _rand(5, grad=False)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        y = D.linear_epilogue(x, w, gate=g, checkpoint="e4m3")
    assert all(t.shape != x.shape for t in seen)
    (dx,) = torch.autograd.grad(y.sum(), (x,))
    torch.testing.assert_close(dx, (g * torch.ones(6, 5, dtype=F64)) @ w)


# ----------------------------------------------------------------------------- the model's block


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_fused_block_trains_like_the_plain_one(checkpoint):
    cfg = dict(dim=64, n_heads=1, intermediate_size=40, n_layers=1)
    torch.manual_seed(0)
    plain = MabaBlock(MabaConfig(**cfg), 0).double()
    fused = MabaBlock(MabaConfig(**cfg, fused_ffn=True, ffn_checkpoint=checkpoint), 0).double()
    fused.load_state_dict(plain.state_dict())
    x = _rand(2, 6, 64, grad=False)
    ys = [blk(x)[0] for blk in (plain, fused)]
    torch.testing.assert_close(ys[1], ys[0])
    for blk, y in zip((plain, fused), ys):
        (y * y).sum().backward()
    rtol = 1e-7 if checkpoint is None else None
    for (name, a), b in zip(plain.named_parameters(), fused.parameters()):
        assert b.grad is not None, name
        if rtol:
            torch.testing.assert_close(b.grad, a.grad, rtol=rtol, atol=1e-9)


def test_config_rejects_nothing_and_defaults_to_the_plain_path():
    assert MabaConfig().fused_ffn is False and MabaConfig().ffn_checkpoint is None


# ----------------------------------------------------------------------------- refusals


def _ok():
    f = dict(dtype=torch.bfloat16, grad=False)
    return dict(x=_rand(4, 16, **f), w_gate=_rand(6, 16, **f), w_up=_rand(6, 16, **f))


@pytest.mark.parametrize("change,error", [
    (dict(w_up=torch.zeros(5, 16, dtype=torch.bfloat16)), ValueError),
    (dict(w_gate=torch.zeros(6, 15, dtype=torch.bfloat16)), ValueError),
    (dict(w_gate=torch.zeros(0, 16, dtype=torch.bfloat16)), ValueError),
    (dict(w_gate=torch.zeros(16, dtype=torch.bfloat16)), ValueError),
    (dict(x=torch.zeros((), dtype=torch.bfloat16)), ValueError),
    (dict(w_up=torch.zeros(6, 16)), TypeError),
    (dict(x=torch.zeros(4, 16, dtype=torch.int32)), TypeError),
    (dict(checkpoint="int4"), ValueError),
])
def test_gated_refusals(change, error):
    with pytest.raises(error):
        D.gated_ffn(**{**_ok(), **change})


@pytest.mark.parametrize("change,error", [
    (dict(bias=torch.zeros(5, dtype=torch.bfloat16)), ValueError),
    (dict(gate=torch.zeros(1, 6, dtype=torch.bfloat16)), ValueError),
    (dict(residual=torch.zeros(6, dtype=torch.bfloat16)), ValueError),      # not broadcast: expand it
    (dict(residual=torch.zeros(4, 6)), TypeError),
    (dict(activation="tanh"), ValueError),
    (dict(checkpoint="fp8"), ValueError),
])
def test_linear_refusals(change, error):
    o = _ok()
    with pytest.raises(error):
        D.linear_epilogue(**{"x": o["x"], "weight": o["w_gate"], **change})


def test_backward_refusals():
    o = _ok()
    dh = torch.zeros(4, 6, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        D.gated_ffn_backward(dh[:3], **o)
    with pytest.raises(ValueError):
        D.gated_ffn_backward(dh, **o, needs=(True, True))
    with pytest.raises(ValueError):
        D.linear_epilogue_backward(dh, o["x"], o["w_gate"], needs=(True,))
    codes, scales = D.checkpoint_pack(o["x"])
    with pytest.raises(TypeError):
        D.gated_ffn_backward(dh, o["x"], o["w_gate"], o["w_up"], x_scales=scales)
    with pytest.raises(ValueError):
        D.gated_ffn_backward(dh, codes, o["w_gate"], o["w_up"], x_scales=scales[:, :0])


def test_pack_refusals():
    for bad, err in ((torch.zeros(3, 4, dtype=F64), TypeError), (torch.zeros(3, 0), ValueError), (torch.zeros(()), ValueError)):
        with pytest.raises(err):
            D.checkpoint_pack(bad)
    codes, scales = D.checkpoint_pack(torch.zeros(3, 40))
    with pytest.raises(TypeError):
        D.checkpoint_unpack(codes, scales, torch.float64)
    with pytest.raises(ValueError):
        D.checkpoint_unpack(codes, scales[:, :1])
    with pytest.raises(TypeError):
        D.checkpoint_unpack(codes.view(torch.uint8), scales)


# --- the C entry points


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


X, W, H = 0x100000, 0x200000, 0x400000     # far apart; never read


def _gated(lib, x=None, wg=None, wu=None, out=None):
    return lib.maba_hip_gated_ffn(x or _t([64, 32], data=X), wg or _t([48, 32], data=W), wu or _t([48, 32], data=W + 0x10000),
                                  out or _t([64, 48], data=H), None, 0, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(x=_t([64, 32, 1], data=X)), 1, b"2D"),
    (dict(x=_t([64, 31], data=X)), 1, b"w_gate"),
    (dict(wu=_t([47, 32], data=W + 0x10000)), 1, b"w_up"),
    (dict(wg=_t([48, 32], dtype=N.MABA_F32, data=W)), 3, b"16-bit"),
    (dict(wg=_t([48, 32], dtype=N.MABA_I64, data=W)), 2, b"16-bit"),
    (dict(x=_t([64, 32], dtype=N.MABA_F16, data=X)), 2, b"dtype"),
    (dict(x=_t([64, 32], strides=[1, 64], data=X)), 1, b"unit column stride"),
    (dict(out=_t([64, 48], strides=[24, 1], data=H)), 1, b"overlap"),
    (dict(out=_t([64, 48], data=X + 16)), 1, b"overlaps an input"),
    (dict(x=_t([64, 32], data=X + 2)), 5, b"workspace"),                      # unaligned rows need a copy
    (dict(x=_t([64, 32], data=0)), 1, b"no data"),
])
def test_c_gated_refusals(lib, kw, rc, text):
    assert _gated(lib, **kw) == rc
    assert text in lib.maba_hip_last_error()


def test_c_empty_batch_is_fine(lib):
    assert lib.maba_hip_gated_ffn(_t([0, 32], data=0), _t([48, 32], data=W), _t([48, 32], data=W + 0x10000),
                                  _t([0, 48], data=0), None, 0, None) == 0
    assert lib.maba_hip_checkpoint_pack(_t([0, 32], data=0), _t([0, 32], dtype=N.MABA_E4M3, data=0),
                                        _t([0, 1], dtype=N.MABA_U8, data=0), None) == 0


def test_c_workspace_sizes(lib):
    g = lib.maba_hip_gated_ffn_workspace_size
    assert g(_t([64, 32]), _t([48, 32]), _t([48, 32])) == 0                   # all aligned
    assert g(_t([32, 31]), _t([48, 31]), _t([48, 31])) == 0                   # the decode kernel reads any rows
    assert g(_t([64, 31]), _t([48, 31]), _t([48, 31])) >= 2 * 32 * (64 + 96)
    assert g(_t([64, 31]), _t([48, 31]), _t([48, 30])) == 0                   # what the call refuses
    b = lib.maba_hip_gated_ffn_backward_workspace_size
    assert b(_t([0, 32], data=0), None, _t([48, 32]), _t([48, 32]), 3) >= 0    # no rows
    lin = lib.maba_hip_linear_epilogue_backward_workspace_size
    assert lin(_t([0, 48], data=0), _t([0, 32], data=0), None, _t([48, 32]), 2, 1, 1, 15) >= 0
    some = b(_t([64, 32]), None, _t([48, 32]), _t([48, 32]), 1)
    assert some >= 2 * 64 * 96 and b(_t([64, 32]), None, _t([48, 32]), _t([48, 32]), 3) >= some


def test_native_binding_declines_what_is_not_on_a_gpu(lib):
    m = N.binding()
    x, w = torch.randn(3, 8).bfloat16(), torch.randn(5, 8).bfloat16()
    assert m.gated_ffn(x, w, w, False) is None
    assert m.linear_epilogue(x, w, None, 0, None, None, True) is None
    assert m.checkpoint_pack(x) is None
    codes, scales = D.checkpoint_pack(x)
    assert m.checkpoint_unpack(codes, scales, torch.float16) is None


def test_c_workspace_must_be_aligned(lib):
    x, wg, wu, dh = _t([64, 31], data=X), _t([48, 31], data=W), _t([48, 31], data=W + 0x10000), _t([64, 48], data=H)
    far = 0x900000
    assert lib.maba_hip_gated_ffn(x, wg, wu, dh, far + 8, 1 << 20, None) == 1
    assert b"16-byte aligned" in lib.maba_hip_last_error()
    assert lib.maba_hip_gated_ffn_backward(dh, x, None, wg, wu, _t([64, 31], data=far), None, None, 2 * far + 2, 1 << 20, None) == 1
    assert lib.maba_hip_linear_epilogue(x, wg, None, 0, None, None, dh, far + 4, 1 << 20, None) == 1
    assert lib.maba_hip_linear_epilogue_backward(dh, x, None, wg, None, 0, None, _t([64, 31], data=far), None, None, None, 2 * far + 8,
                                                 1 << 20, None) == 1
    assert lib.maba_hip_gated_ffn(x, wg, wu, dh, far, 64, None) == 5


def test_c_backward_refusals(lib):
    x, wg, wu, dh = _t([64, 32], data=X), _t([48, 32], data=W), _t([48, 32], data=W + 0x10000), _t([64, 48], data=H)
    dx, far = _t([64, 32], data=H + 0x100000), 0x900000
    call = lib.maba_hip_gated_ffn_backward
    assert call(dh, x, None, wg, wu, dx, None, None, None, 0, None) == 5
    assert call(dh, x, None, wg, wu, _t([64, 32], data=H), None, None, None, 0, None) == 1      # dx over dh
    assert call(dh, x, None, wg, wu, None, _t([48, 32], data=far), _t([48, 32], data=far + 64), None, 0, None) == 1
    assert b"two gradients" in lib.maba_hip_last_error()
    assert call(dh, x, _t([64, 1], dtype=N.MABA_U8), wg, wu, dx, None, None, None, 0, None) == 2  # x is not codes
    codes = _t([64, 32], dtype=N.MABA_E4M3, data=X)
    assert call(dh, codes, _t([63, 1], dtype=N.MABA_U8), wg, wu, dx, None, None, None, 0, None) == 1


def test_c_linear_refusals(lib):
    x, w, y = _t([64, 32], data=X), _t([48, 32], data=W), _t([64, 48], data=H)
    call = lib.maba_hip_linear_epilogue
    assert call(x, w, _t([47]), 0, None, None, y, None, 0, None) == 1
    assert call(x, w, None, 4, None, None, y, None, 0, None) == 1
    assert call(x, w, None, 0, _t([64, 48], data=H + 2), None, y, None, 0, None) == 1           # shifted residual
    assert b"another place" in lib.maba_hip_last_error()
    assert call(x, w, None, 0, _t([64, 48], dtype=N.MABA_F32, data=H + 0x10000), None, y, None, 0, None) == 2
    back = lib.maba_hip_linear_epilogue_backward
    assert back(y, x, None, w, None, 0, None, None, None, None, _t([48], data=0x900000), None, 0, None) == 1
    assert b"without a gate" in lib.maba_hip_last_error()


def test_c_pack_refusals(lib):
    x = _t([4, 40], data=X)
    codes, scales = _t([4, 40], dtype=N.MABA_E4M3, data=H), _t([4, 2], dtype=N.MABA_U8, data=H + 4096)
    call = lib.maba_hip_checkpoint_pack
    assert call(x, codes, _t([4, 1], dtype=N.MABA_U8, data=H + 4096), None) == 1
    assert call(x, _t([4, 40], dtype=N.MABA_U8, data=H), scales, None) == 2
    assert call(_t([4, 40], dtype=N.MABA_F64, data=X), codes, scales, None) == 2
    assert call(x, codes, _t([4, 2], dtype=N.MABA_U8, data=H + 8), None) == 1                   # scales over codes


def test_c_backward_copies_both_weights_or_neither(lib):
    """dx reads the two weights with one row stride: where one of them has to be copied, so is the other."""
    size = lib.maba_hip_gated_ffn_backward_workspace_size
    x, ld = _t([64, 72], data=X), [160, 1]
    aligned, shifted = _t([48, 72], strides=ld, data=W), _t([48, 72], strides=ld, data=W + 152)
    narrow = _t([48, 72], data=W)
    for needs in (1, 2, 3):
        both = size(x, None, shifted, shifted, needs)
        assert size(x, None, aligned, shifted, needs) == size(x, None, shifted, aligned, needs) == both
        assert size(x, None, aligned, narrow, needs) == size(x, None, narrow, aligned, needs) == both     # strides of their own
        assert size(x, None, aligned, aligned, needs) == size(x, None, narrow, narrow, needs) < both


def test_c_backward_copies_rows_that_overlap(lib):
    """What is read along its columns ends at its last row only if rows lie apart: broadcast and overlapping rows are
    copied, rows that are apart are not."""
    lin, gated = lib.maba_hip_linear_epilogue_backward_workspace_size, lib.maba_hip_gated_ffn_backward_workspace_size
    for rows in (1, 100):
        dense, broadcast, windows = (_t([rows, 64], strides=[s, 1], data=X) for s in (64, 0, 8))
        x_copy, w = rows * 64 * 2, _t([64, 64], data=W)
        for cut in (broadcast, windows):
            assert lin(dense, cut, None, w, 0, 0, 0, 2) >= lin(dense, dense, None, w, 0, 0, 0, 2) + x_copy
            assert lin(cut, dense, None, w, 0, 0, 0, 2) >= lin(dense, dense, None, w, 0, 0, 0, 2) + x_copy
            assert gated(cut, None, w, w, 3) >= gated(dense, None, w, w, 3) + x_copy
            assert lib.maba_hip_linear_epilogue_workspace_size(cut, w) == 0                  # along rows they are read in place


def test_tangents_are_not_dropped():
    """Forward-mode derivatives: the host ops carry them, the HIP wrappers decline what would lose them."""
    from torch.autograd import forward_ad

    from maba_sparse.kernels import hip_backend as hb
    x, w, t = _rand(3, 8, grad=False), _rand(5, 8, grad=False), _rand(3, 8, grad=False, seed=9)
    hb._no_grad_needed("op", x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, t)
        torch.testing.assert_close(forward_ad.unpack_dual(D.linear_epilogue(dual, w)).tangent, t @ w.t())
        assert forward_ad.unpack_dual(D.gated_ffn(dual, w, w)).tangent is not None
        hb._no_grad_needed("op", x, None)
        with pytest.raises(NotImplementedError, match="tangents"):
            hb._no_grad_needed("op", w, None, dual)


@pytest.mark.parametrize("env,loads", [("reference", False), ("cpu", False), ("hip", True), ("", True)])
def test_another_backend_needs_no_built_module(monkeypatch, env, loads):
    """A GPU tensor's call that goes to another backend does not ask for the native binding."""
    class Gpu:
        is_cuda, device = True, torch.device("cuda", 0)

    def missing():
        raise N.HipLibraryMissing("not built")

    monkeypatch.setattr(D, "_NATIVE", {})
    monkeypatch.setattr(D, "_load_native", missing)
    monkeypatch.setattr(torch.version, "hip", "7.0")
    monkeypatch.setenv("MABA_BACKEND", env)
    for op in ("gated_ffn", "linear_epilogue", "checkpoint_pack", "checkpoint_unpack"):
        if loads:
            with pytest.raises(N.HipLibraryMissing):
                D._bound(op, Gpu)
        else:
            assert D._bound(op, Gpu) is None
    monkeypatch.setenv("MABA_BACKEND", "rocm")
    with pytest.raises(ValueError, match="MABA_BACKEND"):
        D._bound("gated_ffn", Gpu)


def test_the_environment_may_change_while_the_binding_is_called(lib):
    """The binding reads MABA_BACKEND under the interpreter's lock, as os.environ is written."""
    import sys
    import threading
    m, x, stop = N.binding(), torch.randn(3, 8).bfloat16(), threading.Event()

    def churn():
        n = 0
        while not stop.is_set():
            os.environ[f"MABA_TEST_{n % 500}"] = "x" * (n % 97)
            n += 1

    t, interval = threading.Thread(target=churn), sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    t.start()
    try:
        for _ in range(5000):
            assert m.checkpoint_pack(x) is None
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        t.join()
        for i in range(500):
            os.environ.pop(f"MABA_TEST_{i}", None)


# ----------------------------------------------------------------------------- autocast


def _cast(dtype):
    return lambda t: t if t is None else t.to(dtype)


@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_autocast_computes_in_its_type(xt, checkpoint):
    """fp32 parameters under autocast: the products' type is autocast's whatever x is, gradients have each leaf's own type, and
    both are those of a call on cast tensors."""
    x, wg, wu = _rand(6, 40, dtype=xt), _rand(24, 40, dtype=torch.float32, seed=1), _rand(24, 40, dtype=torch.float32, seed=2)
    w, b = _rand(10, 24, dtype=torch.float32, seed=3), _rand(10, dtype=torch.float32, seed=4)
    to = _cast(torch.bfloat16)
    with torch.autocast("cpu", torch.bfloat16):
        h = D.gated_ffn(x, wg, wu, checkpoint=checkpoint)
        y = D.linear_epilogue(h, w, b, "gelu", checkpoint=checkpoint)
        torch.manual_seed(0)
        dy = torch.randn(6, 10).bfloat16()
        got = torch.autograd.grad(y, (x, wg, wu, w, b), dy, retain_graph=True)          # inside the region
    outside = torch.autograd.grad(y, (x, wg, wu, w, b), dy)
    want_y = D.linear_epilogue(D.gated_ffn(to(x), to(wg), to(wu), checkpoint=checkpoint), to(w), to(b), "gelu", checkpoint=checkpoint)
    assert y.dtype == torch.bfloat16 and torch.equal(y, want_y)
    want = torch.autograd.grad(want_y, (x, wg, wu, w, b), dy)
    for a, o, c, leaf in zip(got, outside, want, (x, wg, wu, w, b)):
        assert a.dtype == leaf.dtype and torch.equal(a, c) and torch.equal(o, c)


@pytest.mark.parametrize("rt,gt", [(torch.float32, torch.float32), (torch.float32, None), (None, torch.float32),
                                   (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16)])
def test_autocast_keeps_a_wide_residual(rt, gt):
    """The gated residual of a type wider than autocast's stays in it, as torch's own addcmul does under autocast."""
    x, w = _rand(6, 40, dtype=torch.float32), _rand(10, 40, dtype=torch.float32, seed=1)
    res = None if rt is None else _rand(6, 10, dtype=rt, seed=2)
    gate = None if gt is None else _rand(10, dtype=gt, seed=3)
    live = [t for t in (x, w, res, gate) if t is not None]
    with torch.autocast("cpu", torch.bfloat16):
        got = D.linear_epilogue(x, w, None, "silu", res, gate)
    to = _cast(torch.bfloat16)
    wide = [t.dtype for t in (res, gate) if t is not None]
    if all(t == torch.bfloat16 for t in wide):
        want = D.linear_epilogue(to(x), to(w), None, "silu", res, gate)
    else:
        y = D.linear_epilogue(to(x), to(w), None, "silu").float()
        y = y if gate is None else y * gate
        want = y if res is None else torch.addcmul(res.float(), gate.float(), D.linear_epilogue(to(x), to(w), None, "silu").float()) \
            if gate is not None else res + y
    assert got.dtype == want.dtype and torch.equal(got, want)
    dy = torch.ones_like(got)
    for a, b in zip(torch.autograd.grad(got, live, dy), torch.autograd.grad(want, live, dy)):
        assert a.dtype == b.dtype and torch.equal(a, b)


@pytest.mark.parametrize("xt", [torch.float32, torch.bfloat16])
def test_autocast_of_the_model_feed_forward(xt):
    """What fused=True returns under autocast has the type of what fused=False does, and a block keeps its residual's."""
    torch.manual_seed(0)
    plain, fused = SwiGLUFFN(64, 96), SwiGLUFFN(64, 96, fused=True)
    fused.load_state_dict(plain.state_dict())
    x = torch.randn(3, 64).to(xt)
    with torch.autocast("cpu", torch.bfloat16):
        ys = [plain(x), fused(x)]
    assert ys[0].dtype == ys[1].dtype == torch.bfloat16
    for m, y in zip((plain, fused), ys):
        y.float().square().sum().backward()
    assert all(p.grad.dtype == torch.float32 for p in fused.parameters())
    cfg = dict(dim=64, n_heads=1, intermediate_size=40, n_layers=1)
    blocks = [MabaBlock(MabaConfig(**cfg, fused_ffn=f), 0) for f in (False, True)]
    res, mo = torch.randn(3, 5, 64), torch.randn(3, 5, 64)
    with torch.autocast("cpu", torch.bfloat16):
        outs = [b._residual(res, mo) for b in blocks]
    assert outs[0].dtype == outs[1].dtype == torch.float32


def test_autocast_leaves_64_bits_alone():
    x, w = _rand(6, 40), _rand(10, 40, seed=1)
    with torch.autocast("cpu", torch.bfloat16):
        y = D.linear_epilogue(x, w)
        with pytest.raises(TypeError, match="dtypes must match"):
            D.linear_epilogue(x, w.float())
    assert y.dtype == F64 and torch.equal(y, D.linear_epilogue(x, w))


def test_blocks_of_configs_and_modules_from_before_the_switch():
    """A config without the fused fields and a module saved without them run as they did."""
    from types import SimpleNamespace
    cfg = MabaConfig(dim=64, n_heads=1, intermediate_size=40, n_layers=1)
    old = SimpleNamespace(**{k: v for k, v in vars(cfg).items() if k not in ("fused_ffn", "ffn_checkpoint")})
    blk = MabaBlock(old, 0)
    x = torch.randn(2, 6, 64)
    want = blk(x)[0]
    for name in ("fused", "checkpoint"):
        del blk.ffn.__dict__[name]
    assert torch.equal(blk(x)[0], want)
