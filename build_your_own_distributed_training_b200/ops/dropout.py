"""Residual add with dropout from a counter-based generator.

``y = residual + keep * x / (1 - p)`` where element ``e`` is kept by a function of ``(seed, e)`` alone:
16 bits of Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011; key = seed, counter = ``e // 8``, field
``e % 8``) compared with ``round(p * 2^16)``.  No mask is stored: the backward makes it again, and so
does a recomputed forward, another launch shape, or a rank that holds only part of the activation
(``start`` = number of its first element).  ``p`` is rounded to a multiple of 2^-16 and the kept
values are scaled for that probability.  CUDA: ``csrc/dropout.cu``; the CPU path below makes the same
mask.  The reference drops attention probabilities only (``src/model/attention.py:147``).
"""

from __future__ import annotations

import torch

from ._ext import native

_LOW = 0xFFFFFFFF


def _cut(p: float) -> int:
    return int(p * 65536 + 0.5)


def keep_mask(n: int, p: float, seed: int, start: int = 0) -> torch.Tensor:
    """The CPU restatement of the generator: which of elements ``start .. start + n`` are kept."""
    first = start // 8
    ctr = torch.arange(first, (start + n + 7) // 8, dtype=torch.int64)
    a, b = ctr & _LOW, ctr >> 32
    c, d = torch.zeros_like(a), torch.zeros_like(a)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        m0, m1 = a * 0xD2511F53, c * 0xCD9E8D57  # the 64-bit products' bits, wrapped
        a, b, c, d = ((m1 >> 32) & _LOW) ^ b ^ k0, m1 & _LOW, ((m0 >> 32) & _LOW) ^ d ^ k1, m0 & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack((a, b, c, d), dim=1)
    bits = torch.stack((words & 0xFFFF, words >> 16), dim=2).view(-1)
    return bits[start - first * 8:start - first * 8 + n] >= _cut(p)


def _apply_cpu(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: int, start: int) -> torch.Tensor:
    keep = keep_mask(x.numel(), p, seed, start).view(x.shape)
    cut = _cut(p)
    scale = 65536.0 / (65536 - cut) if cut < 65536 else 0.0
    y = torch.where(keep, x.float() * scale, 0.0)
    return (y if residual is None else residual.float() + y).to(x.dtype)


class _DropoutAddFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, start):  # type: ignore[override]
        ctx.cfg = (p, seed, start)
        return _apply_cpu(x, residual, p, seed, start)

    @staticmethod
    def backward(ctx, g):  # type: ignore[override]
        p, seed, start = ctx.cfg
        dx = _apply_cpu(g.contiguous(), None, p, seed, start) if ctx.needs_input_grad[0] else None
        return dx, (g if ctx.needs_input_grad[1] else None), None, None, None


def dropout_add(x: torch.Tensor, residual: torch.Tensor | None, p: float, seed: int, *,
                start: int = 0) -> torch.Tensor:
    """``residual + dropout(x, p)`` (``residual`` may be ``None``); fp32, bf16 or fp16.

    ``seed``: 64 bits; draw a new one per call site and step (on the host, e.g. from torch's CPU
    generator, whose state activation checkpointing restores before it recomputes).  ``start``: the
    element number of ``x``'s first element within the whole activation.  A captured CUDA graph
    replays the seed it was captured with.  Differentiable any number of times (the mask is a constant).
    """
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p} is outside [0, 1]")
    if not 0 <= seed < 1 << 64:
        raise ValueError(f"seed {seed} does not fit 64 bits")
    if start < 0:
        raise ValueError(f"negative start {start}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} does not match x {tuple(x.shape)} {x.dtype}")
    x, residual = x.contiguous(), None if residual is None else residual.contiguous()
    if x.is_cuda:
        key = seed - (1 << 64) if seed >= 1 << 63 else seed  # the same 64 bits, signed
        return native().dropout_add(x, residual, _cut(p), key, start)
    return _DropoutAddFn.apply(x, residual, p, seed, start)
