"""Kernel registry and dispatcher -- the drop-in boundary of the hot path.

Mirrors the public contract of the reference dispatcher
(``maba_sparse/kernels/dispatcher.py``): the registry and ``register_kernel`` /
``get_kernel`` (:31-111), ``get_backend`` routing with the ``MABA_BACKEND``
override (:181-238), the five ``dispatch_*`` ops with keyword-only kernel
calls (:258-508) and the once-per-``backend:op`` fallback warning with
``MABA_STRICT_BACKEND`` escalation (:241-255).

Differences, all deliberate:

* The GPU backend is ``"hip"`` (gfx950 kernels in ``libmaba_hip.so``).  A ROCm
  GPU tensor routes to it; ``MABA_BACKEND=hip`` selects it and the reference's
  GPU names ``triton``/``cuda``/``gpu`` map to it.  ``rocm`` stays invalid, as
  the reference's tests require.
* A missing HIP library is never papered over: ``HipLibraryMissing`` propagates
  instead of falling back, so a GPU run cannot silently take a non-HIP path.
* Five ops the reference only has as inline torch code get dispatcher entries:
  ``index_topk_decode`` (layers/indexer.py:101-112), ``hca_pool``
  (layers/sparse_attention.py:206), ``maba_sa_decode``
  (layers/sparse_attention.py:79-219,263-275), ``maba_sa_prefill`` (the three
  prefill streams and their gate, layers/sparse_attention.py:95-219,275) and
  ``dgda_prologue`` (the DGDA layer's conv, gates and key normalisation,
  layers/dgda.py:103-121,186-207).
* The feed-forward operators ``gated_ffn`` and ``linear_epilogue`` (model.py:25-38, 92-128, where
  the reference composes torch modules) carry their own gradients on every backend, through their
  ``*_backward`` ops; ``checkpoint_pack`` and ``checkpoint_unpack`` hold activations in 8 bits.
* So do ``residual_norm`` (the block boundary of model.py:11-22, 92-128, with a norm on the
  sub-layer's output, a scale and dropout), ``dropout`` and ``token_logprobs``.
* ``allow_mixed_dtypes=True`` (keyword) lets ``dgda_prefill``/``dgda_step``
  accept bf16 q/k/v with fp32 gates and state; without it the reference's
  "dtypes must match" ``TypeError`` is kept.
"""
from __future__ import annotations

import logging
import os
import warnings
from typing import Any, Callable, Dict, Optional, Set, Tuple, Union

import torch

from maba_sparse import _native
from maba_sparse._native import HipLibraryMissing
from maba_sparse.kernels import block_ends as _be
from maba_sparse.kernels import common as _c
from maba_sparse.kernels import cpu_dgda as _cpu
from maba_sparse.kernels import feed_forward as _ff

logger = logging.getLogger(__name__)

_KERNEL_REGISTRY: Dict[str, Dict[str, Callable]] = {
    "reference": {
        "dgda_prefill": _c.reference_dgda_prefill,
        "dgda_step": _c.reference_dgda_step,
        "compute_centroids": _c.reference_compute_centroids,
        "index_topk": _c.reference_index_topk,
        "stream_superposition": _c.reference_stream_superposition,
        "index_topk_decode": _c.ref_index_topk_decode,
        "hca_pool": _c.ref_hca_pool,
        "maba_sa_decode": _c.ref_maba_sa_decode,
        "dgda_prologue": _c.ref_dgda_prologue,
        "maba_sa_prefill": _c.ref_maba_sa_prefill,
        "gated_ffn": _c.ref_gated_ffn,
        "gated_ffn_backward": _c.ref_gated_ffn_backward,
        "linear_epilogue": _c.ref_linear_epilogue,
        "linear_epilogue_backward": _c.ref_linear_epilogue_backward,
        "checkpoint_pack": _c.ref_checkpoint_pack,
        "checkpoint_unpack": _c.ref_checkpoint_unpack,
        "dropout": _c.ref_dropout,
        "residual_norm": _c.ref_residual_norm,
        "residual_norm_backward": _c.ref_residual_norm_backward,
        "token_logprobs": _c.ref_token_logprobs,
        "token_logprobs_backward": _c.ref_token_logprobs_backward,
    },
    # host cores: the chunked DGDA of the reference's CPU backend (cpu_dgda.py), the rest as
    # the reference ops in torch
    "cpu": {
        "dgda_prefill": _cpu.cpu_dgda_prefill,
        "dgda_step": _cpu.cpu_dgda_step,
        "compute_centroids": _c.reference_compute_centroids,
        "index_topk": _c.reference_index_topk,
        "stream_superposition": _c.reference_stream_superposition,
        "index_topk_decode": _c.ref_index_topk_decode,
        "hca_pool": _c.ref_hca_pool,
        "maba_sa_decode": _c.ref_maba_sa_decode,
        "dgda_prologue": _c.ref_dgda_prologue,
        "maba_sa_prefill": _c.ref_maba_sa_prefill,
        "gated_ffn": _c.ref_gated_ffn,
        "gated_ffn_backward": _c.ref_gated_ffn_backward,
        "linear_epilogue": _c.ref_linear_epilogue,
        "linear_epilogue_backward": _c.ref_linear_epilogue_backward,
        "checkpoint_pack": _c.ref_checkpoint_pack,
        "checkpoint_unpack": _c.ref_checkpoint_unpack,
        "dropout": _c.ref_dropout,
        "residual_norm": _c.ref_residual_norm,
        "residual_norm_backward": _c.ref_residual_norm_backward,
        "token_logprobs": _c.ref_token_logprobs,
        "token_logprobs_backward": _c.ref_token_logprobs_backward,
    },
    "hip": {},
    "xla": {},
}

_WARNED_FALLBACKS: Set[str] = set()
_BACKEND_CACHE: Dict[Tuple[Optional[str], Optional[int], Optional[str]], str] = {}
_HIP_IMPORTED = False


def clear_dispatcher_cache() -> None:
    _BACKEND_CACHE.clear()


def clear_fallback_warnings() -> None:
    _WARNED_FALLBACKS.clear()
    clear_dispatcher_cache()


def register_kernel(backend: str, op_name: str) -> Callable:
    """Decorator registering ``fn`` as ``op_name`` of ``backend`` (creates both on demand)."""
    def decorator(fn: Callable) -> Callable:
        _KERNEL_REGISTRY.setdefault(backend, {})[op_name] = fn
        return fn
    return decorator


def _ensure_hip_registered() -> None:
    global _HIP_IMPORTED
    if not _HIP_IMPORTED:
        _HIP_IMPORTED = True
        import maba_sparse.kernels.hip_backend  # noqa: F401  (registers on import)


def get_kernel(backend: str, op_name: str) -> Optional[Callable]:
    if backend == "hip":
        _ensure_hip_registered()
    return _KERNEL_REGISTRY.get(backend, {}).get(op_name)


def is_rocm_gpu_available(device: Optional[Union[torch.device, str, int]] = None) -> bool:
    """True when torch is a ROCm build and a GPU is visible."""
    return bool(getattr(torch.version, "hip", None)) and torch.cuda.is_available()


def is_hip_backend_available() -> bool:
    from maba_sparse import _native
    return _native.available()


def is_openmp_available() -> bool:
    try:
        return bool(torch.backends.openmp.is_available())
    except Exception:
        return False


def _parse_device(device) -> Tuple[Optional[str], Optional[int]]:
    if device is None:
        return None, None
    if isinstance(device, int):
        return "cuda", device
    d = torch.device(device) if isinstance(device, str) else device
    return d.type, (d.index if d.index is not None else 0)


def get_backend(device: Union[torch.device, str, None] = None) -> str:
    """Backend name for ``device`` (reference dispatcher.py:181-238, with ``hip``)."""
    try:
        dev_type, dev_idx = _parse_device(device)
    except Exception:
        return "reference"
    env = os.environ.get("MABA_BACKEND")
    key = (dev_type, dev_idx, env)
    hit = _BACKEND_CACHE.get(key)
    if hit is not None:
        return hit
    if env and env.lower() != "auto":
        val = env.lower()
        if val in ("hip", "triton", "cuda", "gpu"):
            res = "hip"
        elif val in ("xla", "tpu"):
            res = "xla"
        elif val in ("cpu", "openmp"):
            res = "cpu"
        elif val in ("reference", "pytorch", "ref"):
            res = "reference"
        else:
            raise ValueError(
                f"Unsupported MABA_BACKEND '{env}'. Supported: ['auto', 'hip', 'triton', 'cpu', 'xla', "
                f"'reference', 'ref']"
            )
    elif dev_type is None:
        res = "hip" if is_rocm_gpu_available() else "cpu"
    elif dev_type == "cuda":
        res = "hip" if getattr(torch.version, "hip", None) else "reference"
    elif dev_type == "cpu":
        res = "cpu"
    else:
        res = "reference"
    _BACKEND_CACHE[key] = res
    return res


def _log_fallback_warning(op_name: str, backend: str, exc: Optional[Exception] = None) -> None:
    strict = os.environ.get("MABA_STRICT_BACKEND", "0").lower() in ("1", "true")
    detail = f" ({type(exc).__name__}: {exc})" if exc is not None else ""
    msg = (f"[Maba Dispatcher Fallback] Native kernel for '{op_name}' on backend '{backend}' "
           f"is unavailable or failed{detail}. Falling back to reference.")
    if strict:
        raise RuntimeError(msg)
    key = f"{backend}:{op_name}"
    if key not in _WARNED_FALLBACKS:
        _WARNED_FALLBACKS.add(key)
        warnings.warn(msg, RuntimeWarning, stacklevel=3)
        logger.debug(msg)


def _run(op_name: str, device, kwargs: Dict[str, Any], backend: Optional[str] = None):
    if backend is None:
        backend = get_backend(device)
    fn = get_kernel(backend, op_name)
    if fn is not None and backend != "reference":
        try:
            return fn(**kwargs)
        except HipLibraryMissing:
            raise
        except Exception as exc:
            _log_fallback_warning(op_name, backend, exc)
    elif backend != "reference" and fn is None:
        _log_fallback_warning(op_name, backend, None)
    ref = get_kernel("reference", op_name)
    kwargs = {k: v for k, v in kwargs.items() if k != "allow_mixed_dtypes"}
    return ref(**kwargs)


def _dgda_precheck(q, k, v, alpha, b, w, log_alpha, extra_name, extra, mixed: bool) -> None:
    """Cheap checks the reference dispatcher runs before routing (dispatcher.py:270-305)."""
    if alpha is None and log_alpha is None:
        raise ValueError("Either alpha or log_alpha must be provided")
    if b is None or w is None:
        raise ValueError("Both b and w gate tensors must be provided")
    if q.dtype not in (torch.float32, torch.float16, torch.bfloat16, torch.float64):
        raise TypeError(f"Unsupported dtype {q.dtype}. Supported: "
                        f"{(torch.float32, torch.float16, torch.bfloat16, torch.float64)}")
    named = [("k", k), ("v", v), ("b", b), ("w", w), ("alpha", alpha), ("log_alpha", log_alpha),
             (extra_name, extra)]
    for name, t in named:
        if t is None:
            continue
        if t.device != q.device:
            raise RuntimeError(
                f"Expected all tensors to be on the same device, but got {q.device} and {t.device} for {name}")
        if not mixed and t.dtype != q.dtype:
            raise TypeError(f"Tensor dtypes must match, but got {q.dtype} for q and {t.dtype} for {name}")


def dispatch_dgda_prefill(q, k, v, alpha=None, b=None, w=None, chunk_size: int = 16, initial_state=None,
                          log_alpha=None, **kwargs: Any) -> Tuple[torch.Tensor, torch.Tensor]:
    _dgda_precheck(q, k, v, alpha, b, w, log_alpha, "initial_state", initial_state,
                   bool(kwargs.get("allow_mixed_dtypes", False)))
    return _run("dgda_prefill", q.device, dict(q=q, k=k, v=v, alpha=alpha, b=b, w=w, chunk_size=chunk_size,
                                               initial_state=initial_state, log_alpha=log_alpha, **kwargs))


def dispatch_dgda_step(q, k, v, alpha=None, b=None, w=None, state=None, log_alpha=None,
                       **kwargs: Any) -> Tuple[torch.Tensor, torch.Tensor]:
    _dgda_precheck(q, k, v, alpha, b, w, log_alpha, "state", state,
                   bool(kwargs.get("allow_mixed_dtypes", False)))
    return _run("dgda_step", q.device, dict(q=q, k=k, v=v, alpha=alpha, b=b, w=w, state=state,
                                            log_alpha=log_alpha, **kwargs))


def dispatch_compute_centroids(k_idx, block_size: int = 64, **kwargs: Any) -> torch.Tensor:
    _c.validate_indexer_inputs(k_idx=k_idx)
    if block_size <= 0:
        raise ValueError(f"block_size must be positive, got {block_size}")
    return _run("compute_centroids", k_idx.device, dict(k_idx=k_idx, block_size=block_size, **kwargs))


def dispatch_index_topk(q_idx, centroids, lambda_dist: float = 0.5, top_k: int = 32, block_size: int = 64,
                        **kwargs: Any):
    if q_idx.device != centroids.device:
        raise RuntimeError(
            f"Expected all tensors to be on the same device, but got {q_idx.device} and {centroids.device}")
    if q_idx.dim() != 3 or centroids.dim() != 3:
        raise ValueError(f"q_idx and centroids must be 3D, got {q_idx.dim()}D and {centroids.dim()}D")
    if q_idx.shape[0] != centroids.shape[0] or q_idx.shape[2] != centroids.shape[2]:
        raise ValueError(
            f"Dimension mismatch between q_idx {list(q_idx.shape)} and centroids {list(centroids.shape)}")
    if top_k <= 0:
        raise ValueError(f"top_k must be positive, got {top_k}")
    if block_size <= 0:
        raise ValueError(f"block_size must be positive, got {block_size}")
    return _run("index_topk", q_idx.device, dict(q_idx=q_idx, centroids=centroids, lambda_dist=lambda_dist,
                                                 top_k=top_k, block_size=block_size, **kwargs))


def dispatch_index_topk_decode(q, centroids, lambda_dist: float = 0.5, top_k: int = 32, **kwargs: Any):
    """Decode-step scoring + top-k; ``q [B, Hq, d]``, ``centroids [B, nb, d]``."""
    if q.device != centroids.device:
        raise RuntimeError(
            f"Expected all tensors to be on the same device, but got {q.device} and {centroids.device}")
    if q.dim() != 3 or centroids.dim() != 3 or q.shape[0] != centroids.shape[0] or q.shape[2] != centroids.shape[2]:
        raise ValueError(f"Dimension mismatch between q {list(q.shape)} and centroids {list(centroids.shape)}")
    if top_k <= 0:
        raise ValueError(f"top_k must be positive, got {top_k}")
    return _run("index_topk_decode", q.device, dict(q=q, centroids=centroids, lambda_dist=lambda_dist,
                                                    top_k=top_k, **kwargs))


def dispatch_stream_superposition(o_local, o_sparse, o_hca, gate_logits=None, **kwargs: Any) -> torch.Tensor:
    dev = o_local.device
    if o_sparse.device != dev or o_hca.device != dev:
        raise RuntimeError(
            f"Expected all tensors to be on the same device, but got {dev}, {o_sparse.device}, {o_hca.device}")
    gate = gate_logits if gate_logits is not None else kwargs.get("gate_weights")
    if gate is not None and gate.device != dev:
        raise RuntimeError(f"Expected all tensors to be on the same device, but got {dev} and {gate.device}")
    _c.validate_superposition_inputs(o_local, o_sparse, o_hca, gate)
    return _run("stream_superposition", dev, dict(o_local=o_local, o_sparse=o_sparse, o_hca=o_hca,
                                                  gate_logits=gate_logits, **kwargs))


def dispatch_hca_pool(c_kv, pool: int = 64, **kwargs: Any) -> torch.Tensor:
    if c_kv.dim() != 3:
        raise ValueError(f"c_kv must be 3D [B, L, d_c], got {list(c_kv.shape)}")
    if pool <= 0:
        raise ValueError(f"pool must be positive, got {pool}")
    return _run("hca_pool", c_kv.device, dict(c_kv=c_kv, pool=pool, **kwargs))


def dispatch_maba_sa_decode(q_lat, c_kv, hca, idx, gate, L: int, scale: float, window: int = 128,
                            n_sink: int = 4, block_size: int = 64, pool: int = 64, **kwargs: Any) -> torch.Tensor:
    """Fused three-stream MABA-SA decode in latent space (see ``common.ref_maba_sa_decode``)."""
    for name, t in (("c_kv", c_kv), ("hca", hca), ("idx", idx), ("gate", gate)):
        if t.device != q_lat.device:
            raise RuntimeError(
                f"Expected all tensors to be on the same device, but got {q_lat.device} and {t.device} for {name}")
    if L <= 0 or L > c_kv.shape[1]:
        raise ValueError(f"L={L} must be in [1, {c_kv.shape[1]}]")
    return _run("maba_sa_decode", q_lat.device, dict(q_lat=q_lat, c_kv=c_kv, hca=hca, idx=idx, gate=gate, L=L,
                                                     scale=scale, window=window, n_sink=n_sink,
                                                     block_size=block_size, pool=pool, **kwargs))


def dispatch_dgda_prologue(projections, conv_weights, history=None, n_heads: int = 10, eps: float = 1e-6,
                           gate_dtype: Optional[torch.dtype] = None, with_alpha: bool = True, **kwargs: Any):
    """The DGDA layer's op inputs from its six projections (see ``common.ref_dgda_prologue``)."""
    if len(projections) != 6 or len(conv_weights) != 3 or (history is not None and len(history) != 3):
        raise ValueError("dgda_prologue takes six projections, three conv weights and three histories or None")
    dev = projections[0].device
    for t in (*projections, *conv_weights, *(history or ())):
        if t.device != dev:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {dev} and {t.device}")
    shape = projections[0].shape
    if len(shape) != 3 or any(p.shape != shape for p in projections):
        raise ValueError(f"projections must share one [B, L, C] shape, got {[list(p.shape) for p in projections]}")
    if shape[2] % n_heads != 0:
        raise ValueError(f"C={shape[2]} is not a multiple of n_heads={n_heads}")
    return _run("dgda_prologue", dev, dict(projections=projections, conv_weights=conv_weights, history=history,
                                           n_heads=n_heads, eps=eps, gate_dtype=gate_dtype, with_alpha=with_alpha,
                                           **kwargs))


def dispatch_maba_sa_prefill(q, k, v, kh, vh, early, idx, gate_logits, scale: float, window: int = 128,
                             n_sink: int = 4, block_size: int = 64, pool: int = 64, **kwargs: Any) -> torch.Tensor:
    """The three MABA-SA prefill streams and their gate (see ``common.ref_maba_sa_prefill``)."""
    dev = q.device
    for name, t in (("k", k), ("v", v), ("kh", kh), ("vh", vh), ("early", early), ("idx", idx),
                    ("gate_logits", gate_logits)):
        if t is not None and t.device != dev:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {dev} and {t.device} for {name}")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"q [B,H,Lq,dh] and k, v [B,H,Lkv,dh] expected, got {list(q.shape)}, {list(k.shape)}")
    if q.shape[2] > k.shape[2]:
        raise ValueError(f"more queries ({q.shape[2]}) than keys ({k.shape[2]})")
    return _run("maba_sa_prefill", dev, dict(q=q, k=k, v=v, kh=kh, vh=vh, early=early, idx=idx,
                                             gate_logits=gate_logits, scale=scale, window=window, n_sink=n_sink,
                                             block_size=block_size, pool=pool, **kwargs))


# ----------------------------------------------------------------------------- feed-forward operators


_FFN_DTYPES = frozenset((torch.float32, torch.float16, torch.bfloat16, torch.float64))


def _ffn_same(first, /, **named) -> None:
    """One floating dtype and one device for all tensors."""
    dtype, device = first.dtype, first.device
    if dtype not in _FFN_DTYPES:
        raise TypeError(f"Unsupported dtype {dtype}. Supported: "
                        f"{(torch.float32, torch.float16, torch.bfloat16, torch.float64)}")
    for name, t in named.items():
        if t is None:
            continue
        if t.device != device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {device} and {t.device} for {name}")
        if t.dtype != dtype:
            raise TypeError(f"Tensor dtypes must match, but got {dtype} and {t.dtype} for {name}")


def _ffn_shape(name, t, shape) -> None:
    if t is not None and t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")


def _ffn_weight(name, w, width) -> None:
    if w.dim() != 2 or w.shape[1] != width or w.shape[0] == 0 or width == 0:
        raise ValueError(f"{name} must be [width, {width}] with positive widths, got {list(w.shape)}")


def _ffn_input(x) -> None:
    if x.dim() < 1:
        raise ValueError("x must have a channel dimension")


def _ffn_checkpoint(checkpoint) -> None:
    if checkpoint not in (None, "e4m3"):
        raise ValueError(f"checkpoint must be None or 'e4m3', got {checkpoint!r}")


def _ffn_activation(activation) -> None:
    if activation not in _c.ACTIVATIONS:
        raise ValueError(f"activation must be one of {_c.ACTIVATIONS}, got {activation!r}")


def _ffn_kept(x, x_scales) -> None:
    """The kept input of a backward op: a tensor, or codes with their scales."""
    if x_scales is None:
        return
    if x.dtype != torch.float8_e4m3fn or x_scales.dtype != torch.uint8:
        raise TypeError(f"a packed input is float8_e4m3fn codes and uint8 scales, got {x.dtype} and {x_scales.dtype}")
    _ffn_shape("x_scales", x_scales, (*x.shape[:-1], -(-x.shape[-1] // _c.PACK_GROUP)))
    if x.device != x_scales.device:
        raise RuntimeError(
            f"Expected all tensors to be on the same device, but got {x.device} and {x_scales.device} for x_scales")


_AUTOCAST_DTYPES = frozenset((torch.float32, torch.float16, torch.bfloat16))      # fp64 stays as it is, as in torch


def _autocast_dtype(x) -> Optional[torch.dtype]:
    """The type that autocast asks for on ``x``'s device, or None."""
    kind = "cuda" if x.is_cuda else x.device.type
    if kind not in ("cuda", "cpu") or not torch.is_autocast_enabled(kind):
        return None
    return torch.get_autocast_dtype(kind)


def _autocast_to(dtype, *tensors):
    return (t if t is None or t.dtype not in _AUTOCAST_DTYPES else t.to(dtype) for t in tensors)


class _FFNOps:
    """The ops that the autograd functions call, through the backend of the tensors' device: a backward pass runs
    where its forward did, and both in their tensors' types whatever autocast says."""

    __slots__ = ("backend", "kind")

    def __init__(self, device):
        self.backend = get_backend(device)
        self.kind = device.type if device.type in ("cuda", "cpu") else None

    def _run(self, op, **kwargs):
        if self.kind is not None and torch.is_autocast_enabled(self.kind):
            with torch.autocast(self.kind, enabled=False):
                return _run(op, None, kwargs, self.backend)
        return _run(op, None, kwargs, self.backend)

    run = _run

    def pack(self, x):
        return self._run("checkpoint_pack", x=x)

    def gated_ffn(self, x, w_gate, w_up):
        return self._run("gated_ffn", x=x, w_gate=w_gate, w_up=w_up)

    def gated_ffn_backward(self, dh, x, w_gate, w_up, x_scales, needs):
        return self._run("gated_ffn_backward", dh=dh, x=x, w_gate=w_gate, w_up=w_up, x_scales=x_scales, needs=tuple(needs))

    def linear_epilogue(self, x, weight, bias, activation, residual, gate):
        return self._run("linear_epilogue", x=x, weight=weight, bias=bias, activation=activation, residual=residual, gate=gate)

    def linear_epilogue_backward(self, dy, x, weight, bias, activation, gate, x_scales, needs):
        return self._run("linear_epilogue_backward", dy=dy, x=x, weight=weight, bias=bias, gate=gate, activation=activation,
                         x_scales=x_scales, needs=tuple(needs))


# op -> the native binding's form of it, and the kernels of this package that it stands for
_NATIVE: Dict[str, Tuple[Callable, Tuple[Tuple[str, Callable], ...]]] = {}


def _load_native() -> None:
    _ensure_hip_registered()
    import maba_sparse.kernels.hip_backend as hb
    binding, ops = _native.binding(), {}
    for op, names in (("gated_ffn", ("gated_ffn", "gated_ffn_backward")), ("checkpoint_pack", ("checkpoint_pack",)),
                      ("linear_epilogue", ("linear_epilogue", "linear_epilogue_backward")),
                      ("checkpoint_unpack", ("checkpoint_unpack",)), ("dropout", ("dropout",)),
                      ("residual_norm", ("residual_norm", "residual_norm_backward")),
                      ("token_logprobs", ("token_logprobs", "token_logprobs_backward"))):
        ops[op] = (getattr(binding, op), tuple((n, getattr(hb, "hip_" + n)) for n in names))
    _NATIVE.update(ops)


def _bound(op: str, x) -> Optional[Callable]:
    """The native binding's form of ``op`` for a GPU tensor ``x``, unless another kernel is registered in place of this
    package's own.  It returns None for a call that is not plain or goes to another backend, which then takes the path
    with the checks, the fallbacks and the errors."""
    if not x.is_cuda or torch.version.hip is None:
        return None
    if not _NATIVE:
        if get_backend(x.device) != "hip":         # later the binding reads the choice by itself
            return None
        _load_native()
    fn, own = _NATIVE[op]
    registered = _KERNEL_REGISTRY["hip"]
    for name, kernel in own:
        if registered.get(name) is not kernel:
            return None
    return fn


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def dispatch_gated_ffn(x, w_gate, w_up, checkpoint: Optional[str] = None) -> torch.Tensor:
    """``silu(x Wg^T) * (x Wu^T)``: the gated feed-forward block up to its down projection.

    x ``[..., C]``, w_gate and w_up ``[I, C]`` of one dtype and device; returns ``[..., I]``, computed in
    fp32 and rounded once.  Differentiable on every backend.  What the backward pass keeps is ``x``; with
    ``checkpoint="e4m3"`` its packed form, half the bytes, and the gradients are those at the unpacked input.  Under
    autocast the tensors are cast to its type first, and gradients come back in each tensor's own."""
    _ffn_checkpoint(checkpoint)
    dtype = _autocast_dtype(x)
    if dtype is not None:
        x, w_gate, w_up = _autocast_to(dtype, x, w_gate, w_up)
    native = _bound("gated_ffn", x)
    if native is not None:
        out = native(x, w_gate, w_up, checkpoint is not None)
        if out is not None:
            return _ff.guard_capture(out)
    _ffn_input(x)
    _ffn_same(x, w_gate=w_gate, w_up=w_up)
    _ffn_weight("w_gate", w_gate, x.shape[-1])
    _ffn_shape("w_up", w_up, w_gate.shape)
    if _wants_grad(x, w_gate, w_up):
        return _ff.guard_capture(_ff.GatedFFN.apply(_FFNOps(x.device), checkpoint, x, w_gate, w_up))
    return _FFNOps(x.device).gated_ffn(x, w_gate, w_up)


def dispatch_gated_ffn_backward(dh, x, w_gate, w_up, x_scales=None, needs=(True, True, True)):
    """``(dx, dw_gate, dw_up)`` of ``gated_ffn`` for its output's gradient ``dh [..., I]``, None where ``needs``
    is false.  ``x`` is the forward's input, or with ``x_scales`` its packed codes.  No autograd takes part.  On the HIP
    backend the gradients of the two pre-activations are rounded to 16 bits once, as operands of the products."""
    _ffn_input(x)
    _ffn_kept(x, x_scales)
    _ffn_same(dh, x=x if x_scales is None else None, w_gate=w_gate, w_up=w_up)
    _ffn_weight("w_gate", w_gate, x.shape[-1])
    _ffn_shape("w_up", w_up, w_gate.shape)
    _ffn_shape("dh", dh, (*x.shape[:-1], w_gate.shape[0]))
    if len(needs) != 3:
        raise ValueError(f"needs takes three flags (dx, dw_gate, dw_up), got {needs!r}")
    with torch.no_grad():
        return _FFNOps(dh.device).gated_ffn_backward(dh, x, w_gate, w_up, x_scales, needs)


def _gated_residual(y, gate, residual):
    """``residual + gate * y`` (both optional) in the widest of their types."""
    _ffn_shape("gate", gate, y.shape[-1:])
    _ffn_shape("residual", residual, y.shape)
    wide = y.dtype
    for t in (gate, residual):
        if t is not None:
            wide = torch.promote_types(wide, t.dtype)
    y = y.to(wide)
    if residual is None:
        return y * gate.to(wide)
    return residual.to(wide) + y if gate is None else torch.addcmul(residual.to(wide), gate.to(wide), y)


def dispatch_linear_epilogue(x, weight, bias=None, activation: str = "none", residual=None, gate=None,
                             checkpoint: Optional[str] = None) -> torch.Tensor:
    """``residual + gate * act(x W^T + bias)``: a linear layer with what follows it in its epilogue.

    x ``[..., K]``, weight ``[N, K]``, bias and gate ``[N]``, residual ``[..., N]`` of one dtype and device; bias,
    gate and residual are optional; activation none, relu, silu or gelu (with the error function).  Computed
    in fp32 and rounded once.  Differentiable on every backend; ``checkpoint`` as for ``gated_ffn``.  Under autocast x,
    weight and bias are cast to its type; a gate or residual of another type is then applied by itself, in the widest of
    them, and the result has that type (torch's addcmul does the same under autocast)."""
    _ffn_activation(activation)
    _ffn_checkpoint(checkpoint)
    dtype = _autocast_dtype(x)
    if dtype is not None:
        x, weight, bias = _autocast_to(dtype, x, weight, bias)
        apart = [t.dtype for t in (gate, residual) if t is not None and t.dtype != x.dtype]
        if apart and _AUTOCAST_DTYPES.issuperset((*apart, x.dtype)):
            return _gated_residual(linear_epilogue(x, weight, bias, activation, checkpoint=checkpoint), gate, residual)
    native = _bound("linear_epilogue", x)
    if native is not None:
        out = native(x, weight, bias, _c.ACTIVATIONS.index(activation), residual, gate, checkpoint is not None)
        if out is not None:
            return _ff.guard_capture(out)
    _ffn_input(x)
    _ffn_same(x, weight=weight, bias=bias, residual=residual, gate=gate)
    _ffn_weight("weight", weight, x.shape[-1])
    n = weight.shape[0]
    _ffn_shape("bias", bias, (n,))
    _ffn_shape("gate", gate, (n,))
    _ffn_shape("residual", residual, (*x.shape[:-1], n))
    if _wants_grad(x, weight, bias, residual, gate):
        return _ff.guard_capture(_ff.LinearEpilogue.apply(_FFNOps(x.device), checkpoint, activation, x, weight, bias, residual, gate))
    return _FFNOps(x.device).linear_epilogue(x, weight, bias, activation, residual, gate)


def dispatch_linear_epilogue_backward(dy, x, weight, bias=None, activation: str = "none", gate=None, x_scales=None,
                                      needs=(True, True, True, True)):
    """``(dx, dw, dbias, dgate)`` of ``linear_epilogue`` for its output's gradient ``dy [..., N]``, None where
    ``needs`` is false or there is no bias or gate; the residual's gradient is ``dy``.  ``x`` as for
    ``gated_ffn_backward``.  No autograd takes part.  On the HIP backend the pre-activation's gradient (without an
    activation, gate times weight) is rounded to 16 bits once, as an operand of the products."""
    _ffn_input(x)
    _ffn_kept(x, x_scales)
    _ffn_same(dy, x=x if x_scales is None else None, weight=weight, bias=bias, gate=gate)
    _ffn_weight("weight", weight, x.shape[-1])
    n = weight.shape[0]
    _ffn_shape("bias", bias, (n,))
    _ffn_shape("gate", gate, (n,))
    _ffn_shape("dy", dy, (*x.shape[:-1], n))
    _ffn_activation(activation)
    if len(needs) != 4:
        raise ValueError(f"needs takes four flags (dx, dw, dbias, dgate), got {needs!r}")
    with torch.no_grad():
        return _FFNOps(dy.device).linear_epilogue_backward(dy, x, weight, bias, activation, gate, x_scales, needs)


def dispatch_checkpoint_pack(x) -> Tuple[torch.Tensor, torch.Tensor]:
    """An activation ``x [..., C]`` in 8 bits: ``(codes, scales)`` (see ``common.ref_checkpoint_pack``), not
    differentiable."""
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a positive channel dimension, got {list(x.shape)}")
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"Unsupported dtype {x.dtype}. Supported: {(torch.float32, torch.float16, torch.bfloat16)}")
    native = _bound("checkpoint_pack", x)
    if native is not None:
        out = native(x)
        if out is not None:
            return out
    return _FFNOps(x.device).pack(x.detach() if x.requires_grad else x)


def dispatch_checkpoint_unpack(codes, scales, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``(codes, scales)`` stand for, in ``dtype``."""
    if codes.dim() < 1 or codes.shape[-1] == 0:
        raise ValueError(f"codes must have a positive channel dimension, got {list(codes.shape)}")
    _ffn_kept(codes, scales)
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"Unsupported dtype {dtype}. Supported: {(torch.float32, torch.float16, torch.bfloat16)}")
    native = _bound("checkpoint_unpack", codes)
    if native is not None:
        out = native(codes, scales, dtype)
        if out is not None:
            return out
    return _run("checkpoint_unpack", codes.device, dict(codes=codes, scales=scales, dtype=dtype))


# ----------------------------------------------------------------------------- the block boundary and dropout


def _drop_args(x, p, seed, stream) -> None:
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not 0 <= stream < 2 ** 32:
        raise ValueError(f"stream must be in [0, 2^32), got {stream}")
    if 0.0 < p < 1.0:
        if seed is None:
            raise ValueError("dropout needs a seed: an int64 tensor of one element")
        if seed.dtype != torch.int64:
            raise TypeError(f"the seed must be int64, got {seed.dtype}")
        if seed.numel() != 1:
            raise ValueError(f"the seed must have one element, got {list(seed.shape)}")
        if seed.device != x.device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {x.device} and {seed.device} for seed")


def _channels(x, name: str = "x") -> None:
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{name} must have a positive channel dimension, got {list(x.shape)}")


def dispatch_dropout(x, p: float, seed=None, stream: int = 0) -> torch.Tensor:
    """Elements of ``x [..., C]`` zeroed with probability ``p``, the others times ``1 / (1 - p)``.

    The mask is never stored: it is a function of ``seed`` (an int64 tensor of one element on x's device, read when the
    kernel runs), ``stream`` (an int in ``[0, 2^32)``: one for each place that drops under the same seed), the row
    (counted over the leading dimensions) and the column; see ``common.philox_words``.  A dropped element is 0 whatever it
    was.  A seed that is advanced in place after the backward pass, also inside a captured graph, gives every step
    masks of its own.  Differentiable on every backend."""
    native = _bound("dropout", x)
    if native is not None:
        out = native(x, p, seed, stream)
        if out is not None:
            return _ff.guard_capture(out)
    _channels(x)
    _ffn_same(x)
    _drop_args(x, p, seed, stream)
    if _wants_grad(x):
        return _ff.guard_capture(_be.Dropout.apply(_FFNOps(x.device), p, stream, x, seed))
    return _FFNOps(x.device).run("dropout", x=x, p=p, seed=seed, stream=stream)


def _widest(*tensors):
    """The tensors in the widest of their floating types."""
    wide = None
    for t in tensors:
        if t is not None:
            wide = t.dtype if wide is None else torch.promote_types(wide, t.dtype)
    return tuple(t if t is None or t.dtype == wide else t.to(wide) for t in tensors)


def _boundary_check(x, y, weight, post_weight, gate) -> None:
    _channels(x)
    _ffn_same(x, y=y, weight=weight, post_weight=post_weight, gate=gate)
    _ffn_shape("y", y, x.shape)
    for name, t in (("weight", weight), ("post_weight", post_weight), ("gate", gate)):
        _ffn_shape(name, t, x.shape[-1:])


def dispatch_residual_norm(x, y=None, weight=None, post_weight=None, gate=None, scale: float = 1.0, p: float = 0.0, seed=None,
                           stream: int = 0, eps: float = 1e-6) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """The boundary between two sub-layers: ``(x_out, h)`` with

    ``x_out = x + scale * gate * dropout(z)``, ``z = RMSNorm(y) * post_weight`` (``y`` itself without post_weight), and
    ``h = RMSNorm(x_out) * weight`` (None without weight).

    x and y ``[..., C]``, weight, post_weight and gate ``[C]`` of one dtype and device; all but x are optional, and without
    y x_out is x itself.  ``p``, ``seed`` and ``stream`` as for ``dropout``.  Computed in fp32 and each result rounded once
    (h from the unrounded x_out).  Differentiable on every backend: x and y are kept for it (x for h's gradient, y also for
    post_weight's and the gate's).  Under autocast the tensors are first cast to the widest of their types.  The HIP backend takes up to
    8,192 channels."""
    dtype = _autocast_dtype(x)
    if dtype is not None:
        x, y, weight, post_weight, gate = _widest(x, y, weight, post_weight, gate)
    native = _bound("residual_norm", x)
    if native is not None:
        out = native(x, y, weight, post_weight, gate, scale, p, seed, stream, eps)
        if out is not None:
            _ff.guard_capture(out[0] if y is not None else out[1])
            return out
    _boundary_check(x, y, weight, post_weight, gate)
    _drop_args(x, p, seed, stream)
    if y is None:
        if post_weight is not None or gate is not None:
            raise ValueError("post_weight and gate go with y")
        if weight is None:
            return x, None
        p, seed, scale = 0.0, None, 1.0
    ops = _FFNOps(x.device)
    if _wants_grad(x, y, weight, post_weight, gate):
        out = _be.ResidualNorm.apply(ops, scale, p, stream, eps, x, y, weight, post_weight, gate, seed)
        if y is None:
            return x, _ff.guard_capture(out)
        return (_ff.guard_capture(out[0]), out[1]) if weight is not None else (_ff.guard_capture(out), None)
    out = ops.run("residual_norm", x=x, y=y, weight=weight, post_weight=post_weight, gate=gate, scale=scale, p=p, seed=seed,
                  stream=stream, eps=eps)
    return (x, out[1]) if y is None else out


def dispatch_residual_norm_backward(dx_out, dh, x, y=None, weight=None, post_weight=None, gate=None, scale: float = 1.0,
                                    p: float = 0.0, seed=None, stream: int = 0, eps: float = 1e-6,
                                    needs=(True, True, True, True, True)):
    """``(dx, dy, dweight, dpost_weight, dgate)`` of ``residual_norm`` for the gradients of its results, either of which
    may be None, each None where ``needs`` is false or there is no such input.  ``x`` (only its shape and type count without
    ``dh``) and ``y`` are the forward's inputs; without ``dh``, post_weight and the gate's gradient y is not read and may be
    left out.  No autograd takes part."""
    first = dx_out if dx_out is not None else dh
    if first is None:
        raise ValueError("dx_out or dh is required")
    _boundary_check(x, y, weight, post_weight, gate)
    _ffn_same(x, dx_out=dx_out, dh=dh)
    _ffn_shape("dx_out", dx_out, x.shape)
    _ffn_shape("dh", dh, x.shape)
    _drop_args(x, p, seed, stream)
    if dh is not None and weight is None:
        raise ValueError("dh goes with weight")
    if len(needs) != 5:
        raise ValueError(f"needs takes five flags (dx, dy, dweight, dpost_weight, dgate), got {needs!r}")
    if y is None and (post_weight is not None or (gate is not None and needs[4])):
        raise ValueError("post_weight and the gate's gradient need y")
    with torch.no_grad():
        return _FFNOps(x.device).run("residual_norm_backward", dx_out=dx_out, dh=dh, x=x, y=y, weight=weight,
                                         post_weight=post_weight, gate=gate, scale=scale, p=p, seed=seed, stream=stream, eps=eps,
                                         needs=tuple(needs))


# ----------------------------------------------------------------------------- token log probabilities


def _logprobs_check(logits, targets, temperature) -> None:
    _channels(logits, "logits")
    _ffn_same(logits)
    if targets.dtype != torch.int64:
        raise TypeError(f"targets must be int64, got {targets.dtype}")
    if targets.device != logits.device:
        raise RuntimeError(f"Expected all tensors to be on the same device, but got {logits.device} and {targets.device} for targets")
    _ffn_shape("targets", targets, logits.shape[:-1])
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"temperature must be positive, got {temperature}")


def dispatch_token_logprobs(logits, targets, temperature: float = 1.0, top: int = 0):
    """``(logp, entropy, lse, top_logp, top_ids)`` of the distributions ``softmax(logits / temperature)``.

    logits ``[..., V]``, targets int64 ``[...]``; logp (of the target), entropy and lse (the normaliser ``log sum exp``)
    ``[...]``, and the ``top`` likeliest tokens with their log probabilities ``[..., top]``, likeliest first, ties by the
    lower index (None for ``top=0``; the HIP backend takes up to 64).  fp32, for fp64 logits fp64.  A negative target
    stands for none: its logp is 0 and has no gradient; one of V or more gives NaN, since a GPU call cannot refuse it.  Logits
    of -inf have probability zero; a row of nothing else has lse and log probabilities -inf, entropy 0 and no gradient.
    logp, entropy and lse are differentiable on every backend (the logits are kept for it), the alternatives are not."""
    native = _bound("token_logprobs", logits)
    if native is not None:
        out = native(logits, targets, temperature, top)
        if out is not None:
            _ff.guard_capture(out[0])
            return out
    _logprobs_check(logits, targets, temperature)
    if not 0 <= top <= logits.shape[-1]:
        raise ValueError(f"top must be in [0, {logits.shape[-1]}], got {top}")
    ops = _FFNOps(logits.device)
    if _wants_grad(logits):
        out = _be.TokenLogprobs.apply(ops, temperature, top, logits, targets)
        _ff.guard_capture(out[0])
        return out
    return ops.run("token_logprobs", logits=logits, targets=targets, temperature=temperature, top=top)


def dispatch_token_logprobs_backward(dlogp, dentropy, dlse, logits, targets, lse, entropy, temperature: float = 1.0):
    """The logits' gradient of ``token_logprobs`` for the gradients of logp, entropy and lse ``[...]``, any of which may be
    None; lse and entropy as the forward returned them.  No autograd takes part."""
    _logprobs_check(logits, targets, temperature)
    wide = torch.promote_types(logits.dtype, torch.float32)
    for name, t in (("dlogp", dlogp), ("dentropy", dentropy), ("dlse", dlse), ("lse", lse), ("entropy", entropy)):
        if t is None:
            continue
        _ffn_shape(name, t, logits.shape[:-1])
        if t.dtype != wide:
            raise TypeError(f"{name} must be {wide}, got {t.dtype}")
        if t.device != logits.device:
            raise RuntimeError(f"Expected all tensors to be on the same device, but got {logits.device} and {t.device} for {name}")
    if dlogp is None and dentropy is None and dlse is None:
        raise ValueError("one of dlogp, dentropy and dlse is required")
    with torch.no_grad():
        return _FFNOps(logits.device).run("token_logprobs_backward", dlogp=dlogp, dentropy=dentropy, dlse=dlse, logits=logits,
                                          targets=targets, lse=lse, entropy=entropy, temperature=temperature)


token_logprobs = dispatch_token_logprobs
token_logprobs_backward = dispatch_token_logprobs_backward
dropout = dispatch_dropout
residual_norm = dispatch_residual_norm
residual_norm_backward = dispatch_residual_norm_backward
gated_ffn = dispatch_gated_ffn
gated_ffn_backward = dispatch_gated_ffn_backward
linear_epilogue = dispatch_linear_epilogue
linear_epilogue_backward = dispatch_linear_epilogue_backward
checkpoint_pack = dispatch_checkpoint_pack
checkpoint_unpack = dispatch_checkpoint_unpack
dgda_prefill = dispatch_dgda_prefill
dgda_step = dispatch_dgda_step
compute_centroids = dispatch_compute_centroids
index_topk = dispatch_index_topk
stream_superposition = dispatch_stream_superposition
index_topk_decode = dispatch_index_topk_decode
hca_pool = dispatch_hca_pool
maba_sa_decode = dispatch_maba_sa_decode
dgda_prologue = dispatch_dgda_prologue
maba_sa_prefill = dispatch_maba_sa_prefill
ref_dgda_prefill = _c.ref_dgda_prefill
ref_dgda_step = _c.ref_dgda_step
ref_centroids = _c.ref_centroids
ref_topk = _c.ref_topk
ref_superposition = _c.ref_superposition
