"""What the autograd functions of the token operators share: they have first derivatives, backwards.

A tangent (forward mode) or a second derivative has no formula in their kernels.  An answer without it would be a wrong one, so
both are refused.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
from torch.autograd import forward_ad


def tracked(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a call goes through its autograd function: a tensor requires a gradient, or tangents are about (the function
    raises for an input that has one)."""
    if forward_ad._current_level >= 0:
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def wanted(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a derivative would have to pass through a call: a tensor requires a gradient where gradients are taken, or has a
    tangent."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


class _First(torch.autograd.Function):
    @staticmethod
    def forward(ctx, name, grad, *of):
        ctx.name = name
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.name} has no second derivative")


def first_only(name: str):
    """For a ``backward`` whose gradients depend on the saved tensors, on ``ctx.linked`` (inputs that it does not read itself, so
    that they may be overwritten) and the gradients that come in: with ``create_graph`` they depend on those in the graph too,
    and a derivative of them raises."""
    def decorate(backward):
        @functools.wraps(backward)
        def run(ctx, *grads):
            if not torch.is_grad_enabled():
                return backward(ctx, *grads)
            with torch.no_grad():
                out = backward(ctx, *grads)
            of = [t for t in (*ctx.saved_tensors, *ctx.linked, *grads) if t is not None]
            return tuple(None if g is None else _First.apply(name, g, *of) for g in out)
        return run
    return decorate
