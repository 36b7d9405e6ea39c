"""Gradients of the operators around a model's blocks: autograd functions over the dispatcher's forward and backward ops,
the same on every backend.

The boundary keeps its inputs for the backward pass, dropout its seed alone: the mask is made
again from it, so a seed must not change in between (autograd says so if it does).

Calls that go to this package's own HIP kernels take the same functions natively (``csrc/torch_binding.cpp``); these here
serve the other backends, kernels registered in their place and calls that the binding declines.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable


def _once(backward):
    """``once_differentiable`` where a second derivative may be asked for; its wrapper costs 3 us of a call."""
    wrapped = once_differentiable(backward)

    def run(ctx, *grads):
        return wrapped(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


class Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, p, stream, x, seed):
        ctx.ops, ctx.p, ctx.stream = ops, p, stream
        ctx.save_for_backward(seed)
        return ops.run("dropout", x=x, p=p, seed=seed, stream=stream)

    @staticmethod
    @_once
    def backward(ctx, dy):
        return None, None, None, ctx.ops.run("dropout", x=dy, p=ctx.p, seed=ctx.saved_tensors[0], stream=ctx.stream), None


class ResidualNorm(torch.autograd.Function):
    """``(x_out, h)``, or ``h`` alone without y, whose x_out is x itself."""

    @staticmethod
    def forward(ctx, ops, scale, p, stream, eps, x, y, weight, post_weight, gate, seed):
        ctx.ops, ctx.args = ops, dict(scale=scale, p=p, stream=stream, eps=eps)
        ctx.set_materialize_grads(False)
        x_out, h = ops.run("residual_norm", x=x, y=y, weight=weight, post_weight=post_weight, gate=gate, seed=seed, **ctx.args)
        needs = ctx.needs_input_grad[5:10]
        # x_out is made again for its norm's gradient; y is read for its own norm's and for the gate's too
        kept_y = y if weight is not None or post_weight is not None or needs[4] else None
        ctx.save_for_backward(x if weight is not None else None, kept_y, weight, post_weight, gate, seed)
        ctx.alone = y is None
        if ctx.alone:
            return h
        return (x_out, h) if h is not None else x_out

    @staticmethod
    @_once
    def backward(ctx, *grads):
        x, y, weight, post_weight, gate, seed = ctx.saved_tensors
        dx_out, dh = (None, grads[0]) if ctx.alone else (*grads, None)[:2]
        if dx_out is None and dh is None:
            return (None,) * 11
        out = ctx.ops.run("residual_norm_backward", dx_out=dx_out, dh=dh, x=x if x is not None else dx_out, y=y,
                          weight=weight, post_weight=post_weight, gate=gate, seed=seed, needs=tuple(ctx.needs_input_grad[5:10]),
                          **ctx.args)
        return (None,) * 5 + tuple(out) + (None,)


class TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ops, temperature, top, logits, targets):
        ctx.ops, ctx.temperature = ops, temperature
        ctx.set_materialize_grads(False)
        logp, entropy, lse, top_logp, top_ids = ops.run("token_logprobs", logits=logits, targets=targets, temperature=temperature, top=top)
        ctx.save_for_backward(logits, targets, lse, entropy)
        if top:
            ctx.mark_non_differentiable(top_logp, top_ids)
        return logp, entropy, lse, top_logp, top_ids

    @staticmethod
    @_once
    def backward(ctx, dlogp, dentropy, dlse, *_):
        if dlogp is None and dentropy is None and dlse is None:
            return (None,) * 5
        logits, targets, lse, entropy = ctx.saved_tensors
        d = ctx.ops.run("token_logprobs_backward", dlogp=dlogp, dentropy=dentropy, dlse=dlse, logits=logits, targets=targets, lse=lse,
                        entropy=entropy, temperature=ctx.temperature)
        return None, None, None, d, None
