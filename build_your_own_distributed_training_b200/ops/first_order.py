"""Gradients that cannot be differentiated again.

A kernel's result has no graph: under ``create_graph=True`` a term through it would count as constant and be
missing from the second derivative without a word.  :func:`first_order` lets the gradient through and makes a
differentiation of it raise, for whatever the backward's node depends on.
"""

from __future__ import annotations

import torch

from ._ext import native


class _FirstOrder(torch.autograd.Function):
    @staticmethod
    def forward(ctx, op, g, *_inputs):  # type: ignore[override]
        ctx.op = op
        return g.view_as(g)

    @staticmethod
    def backward(ctx, _g):  # type: ignore[override]
        raise RuntimeError(f"{ctx.op} has no second derivative")


def first_order(op: str, g: torch.Tensor | None, dys: tuple, *inputs: torch.Tensor) -> torch.Tensor | None:
    """``g`` as the running backward of ``op`` returns it for the gradients ``dys``.  ``inputs``: the node's
    differentiable inputs, which only the CPU path needs (the C++ side asks the node)."""
    if g is None or not torch.is_grad_enabled():
        return g
    dys = tuple(t for t in dys if t is not None)
    if g.is_cuda:
        return native().first_order(g, op, dys)
    return _FirstOrder.apply(op, g.detach(), *dys, *inputs)
