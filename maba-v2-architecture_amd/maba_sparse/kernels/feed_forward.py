"""Gradients of the feed-forward operators: autograd functions over the dispatcher's forward and
backward ops, the same on every backend.

The forward pass keeps its input (or, with ``checkpoint="e4m3"``, the input's packed form) and the
parameters; the backward op makes the pre-activations again from it.  With a checkpoint the gradients
are those at the unpacked input: the forward result is unaffected.

Calls that go to this package's own HIP kernels take the same functions natively (``csrc/torch_binding.cpp``); these
here serve the other backends, kernels registered in their place and calls that the binding declines.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from maba_sparse import _native


def _once(backward):
    """``once_differentiable`` where a second derivative may be asked for; its wrapper costs 3 us of a call."""
    wrapped = once_differentiable(backward)

    def run(ctx, grad):
        return wrapped(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)

    return run


class GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, checkpoint, x, w_gate, w_up):
        ctx.ops = ops
        if any(ctx.needs_input_grad):
            kept = ops.pack(x) if checkpoint else (x,)
            ctx.save_for_backward(w_gate, w_up, *kept)
        return ops.gated_ffn(x, w_gate, w_up)

    @staticmethod
    @_once
    def backward(ctx, dh):
        w_gate, w_up, x, *scales = ctx.saved_tensors
        grads = ctx.ops.gated_ffn_backward(dh, x, w_gate, w_up, scales[0] if scales else None, ctx.needs_input_grad[2:5])
        return (None, None, *grads)


class LinearEpilogue(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, checkpoint, activation, x, weight, bias, residual, gate):
        ctx.ops, ctx.activation = ops, activation
        dx, dw, dbias, _, dgate = ctx.needs_input_grad[3:8]
        ctx.has = (bias is not None, gate is not None)
        # x is read by dW and dgate and, with an activation, to make z again
        ctx.keeps_x = dw or dgate or ((dx or dbias) and activation != "none")
        kept = (ops.pack(x) if checkpoint else (x,)) if ctx.keeps_x else ()
        ctx.x_like = x.shape
        if dx or dw or dbias or dgate:
            ctx.save_for_backward(weight, *(t for t in (bias, gate) if t is not None), *kept)
        return ops.linear_epilogue(x, weight, bias, activation, residual, gate)

    @staticmethod
    @_once
    def backward(ctx, dy):
        dx, dw, dbias, dres, dgate = ctx.needs_input_grad[3:8]
        grads = (None, None, None, None)
        if dx or dw or dbias or dgate:
            weight, *rest = ctx.saved_tensors
            bias = rest.pop(0) if ctx.has[0] else None
            gate = rest.pop(0) if ctx.has[1] else None
            # where x is not read, a view of its shape over one weight row takes its place
            x = rest[0] if ctx.keeps_x else weight[0].expand(ctx.x_like)
            scales = rest[1] if len(rest) > 1 else None
            grads = ctx.ops.linear_epilogue_backward(dy, x, weight, bias, ctx.activation, gate, scales, (dx, dw, dbias, dgate))
        return (None, None, None, grads[0], grads[1], grads[2], dy if dres else None, grads[3])


def guard_capture(out: torch.Tensor) -> torch.Tensor:
    """Refuses to record a backward pass whose gradients would reach a leaf through an autograd node
    of another stream.  Such a node lives as long as any eager graph of that leaf does, whichever op made
    it; the engine would then make the node's stream wait inside the capture, which ends the process."""
    if out.is_cuda and out.grad_fn is not None and torch.cuda.is_current_stream_capturing():
        try:
            binding = _native.binding()
        except _native.HipLibraryMissing:                  # another backend's call, where nothing is built
            return out
        if binding.leaf_of_another_stream(out):
            raise RuntimeError(
                "a leaf of this captured call still belongs to an eager autograd graph on another stream: drop "
                "that graph's outputs first, or capture the *_backward ops, which need no autograd")
    return out
