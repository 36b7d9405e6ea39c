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
