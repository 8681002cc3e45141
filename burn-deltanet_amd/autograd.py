"""What the package's autograd functions share: their backwards are calls into
the library, which autograd cannot differentiate again."""

from __future__ import annotations

import functools

import torch

from .abi import DeltaError


class _Last(torch.autograd.Function):
    """Gradients as they are, whose own gradients are refused."""

    @staticmethod
    def forward(ctx, *grads):
        return tuple(t.view_as(t) for t in grads)

    @staticmethod
    def backward(ctx, *_):
        raise DeltaError(-9, "a second derivative of the library's operators is not available")


def first_order(backward):
    """For a Function's `backward`: where a graph of the gradients is asked for
    (create_graph=True) they become part of one that refuses to be run, whatever
    the cotangents depend on. Without it they would count as constants."""

    @functools.wraps(backward)
    def wrapped(ctx, *cotangents):
        if not torch.is_grad_enabled():
            return backward(ctx, *cotangents)
        with torch.no_grad():
            grads = backward(ctx, *cotangents)
        there = [t for t in grads if t is not None]
        last = iter(_Last.apply(*(t.detach().requires_grad_(True) for t in there)) if there else ())
        return tuple(None if t is None else next(last) for t in grads)

    return wrapped
