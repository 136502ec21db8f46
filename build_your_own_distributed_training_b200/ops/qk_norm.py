"""Per-head RMSNorm of queries and keys with the rotary rotation in the same pass.

On the packed ``[q | k | v]`` projection every query and key head ``x`` becomes
``R(x * rsqrt(mean(x^2) + eps) * w)`` with one ``[head_dim]`` weight for the query heads and one
for the key heads (shared by all heads) and the rotate-half rotation ``R`` of the token's position;
the value heads are carried over.  The result is what :func:`..attention.causal_attention` reads.

With normalised queries and keys the rotation cannot ride in the projection's GEMM epilogue (the
norm comes between them), so this op takes its place.  On CUDA it is one kernel forward and two
backward (``csrc/qk_norm_rope.cu``): statistics and weight gradients in fp32, sums in a fixed order,
nothing saved but the input.  No reference counterpart: the reference's attention
(``src/model/attention.py:109-155``) rotates unnormalised heads.
"""

from __future__ import annotations

from collections.abc import Callable

import torch

from . import grad_state
from ._ext import native
from .first_order import first_order


def _rotate(u: torch.Tensor, c: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    h = u.shape[-1] // 2
    lo, hi = u[..., :h], u[..., h:]
    return torch.cat((lo * c - hi * s, hi * c + lo * s), dim=-1)


def _tables(cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor | None, tokens: int, seqlen: int,
            hd: int) -> tuple[torch.Tensor, torch.Tensor]:
    if positions is None:
        pos = torch.arange(tokens, device=cos.device) % seqlen
        return cos[pos, None, : hd // 2].float(), sin[pos, None, : hd // 2].float()
    out = ((positions < 0) | (positions >= cos.shape[0]))[:, None, None]  # no such position: NaN heads
    pos = positions.long().clamp(0, cos.shape[0] - 1)
    c, s = (t[pos, None, : hd // 2].float().masked_fill(out, float("nan")) for t in (cos, sin))
    return c, s


def qk_norm_rope_reference(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                           sin: torch.Tensor, nq: int, nkv: int, hd: int, seqlen: int, eps: float,
                           positions: torch.Tensor | None = None) -> torch.Tensor:
    """The op in plain differentiable PyTorch: fp32 math, rounded once."""
    x = qkv.float().view(qkv.shape[0], nq + 2 * nkv, hd)
    c, s = _tables(cos, sin, positions, qkv.shape[0], seqlen, hd)
    w = torch.cat((q_weight.float().expand(nq, hd), k_weight.float().expand(nkv, hd)))
    a = x[:, : nq + nkv]
    u = a * torch.rsqrt(a.pow(2).mean(-1, keepdim=True) + eps) * w
    return torch.cat((_rotate(u, c, s), x[:, nq + nkv:]), dim=1).to(qkv.dtype).view(qkv.shape)


def _backward_cpu(g, x, wq, wk, cos, sin, pos, nq, nkv, hd, seqlen, eps):
    x3 = x.float().view(-1, nq + 2 * nkv, hd)
    g3 = g.float().view(-1, nq + 2 * nkv, hd)
    c, s = _tables(cos, sin, pos, x.shape[0], seqlen, hd)
    w = torch.cat((wq.float().expand(nq, hd), wk.float().expand(nkv, hd)))
    a = x3[:, : nq + nkv]
    r = torch.rsqrt(a.pow(2).mean(-1, keepdim=True) + eps)
    n = a * r
    gu = _rotate(g3[:, : nq + nkv], c, -s)  # the transposed rotation
    gn = gu * w
    da = r * (gn - n * (gn * n).mean(-1, keepdim=True))
    dw = (gu * n).sum(0)
    dx = torch.cat((da, g3[:, nq + nkv:]), dim=1).to(x.dtype).view(x.shape)
    return dx, dw[:nq].sum(0), dw[nq:].sum(0)


class _QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, wq, wk, cos, sin, positions, nq, nkv, hd, seqlen, eps, main_grads, reduce):  # type: ignore[override]
        if qkv.is_cuda:
            y = native().qk_norm_rope_fwd(qkv, wq, wk, cos, sin, positions, nq, nkv, hd, seqlen, eps)
        else:
            y = qk_norm_rope_reference(qkv, wq, wk, cos, sin, nq, nkv, hd, seqlen, eps, positions)
        ctx.save_for_backward(qkv, wq, wk, cos, sin, positions)
        ctx.cfg = (nq, nkv, hd, seqlen, eps)
        ctx.main_grads, ctx.reduce = main_grads, reduce
        return y

    @staticmethod
    def backward(ctx, g):  # type: ignore[override]
        saved = ctx.saved_tensors  # once: recomputed under activation checkpointing
        if not g.is_cuda and ctx.main_grads is None and ctx.reduce is None:
            return _QKNormRopeFn._gradients(ctx, saved, g) + (None,) * 10  # plain differentiable operations
        with torch.no_grad():
            grads = _QKNormRopeFn._gradients(ctx, saved, g)
        return tuple(first_order("qk_norm_rope", t, (g,), *saved[:3]) for t in grads) + (None,) * 10

    @staticmethod
    def _gradients(ctx, saved, g):
        qkv, wq, wk, cos, sin, positions = saved
        nq, nkv, hd, seqlen, eps = ctx.cfg
        mgs = ctx.main_grads
        if mgs is not None:
            for mg in mgs:
                grad_state.zero_if_fresh(mg)  # the weight gradients accumulate
        # straight into the weights' own gradients, unless other ranks' parts have to be added first
        direct = mgs is not None and ctx.reduce is None
        if qkv.is_cuda:
            if g.stride(-1) != 1:
                g = g.contiguous()
            if ctx.reduce is not None:
                dw = torch.empty(2, hd, device=wq.device, dtype=torch.float32)
                dwq, dwk = dw[0], dw[1]
            else:
                dwq, dwk = mgs if direct else (torch.empty_like(wq), torch.empty_like(wk))
            dx = native().qk_norm_rope_bwd(g, qkv, wq, wk, cos, sin, positions, nq, nkv, hd, seqlen, eps,
                                           dwq, dwk, direct)
        else:
            dx, dwq, dwk = _backward_cpu(g, qkv, wq, wk, cos, sin, positions, nq, nkv, hd, seqlen, eps)
            dw = torch.stack((dwq, dwk))
        if ctx.reduce is not None:
            ctx.reduce(dw)
            dwq, dwk = dw[0], dw[1]
        if mgs is not None:
            if not (direct and qkv.is_cuda):
                mgs[0].add_(dwq)
                mgs[1].add_(dwk)
            dwq = dwk = None
        else:
            dwq, dwk = dwq.to(wq.dtype), dwk.to(wk.dtype)
        return dx, dwq, dwk


def qk_norm_rope(qkv: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
                 sin: torch.Tensor, n_q_heads: int, n_kv_heads: int, head_dim: int, seqlen: int,
                 eps: float = 1e-5, *, positions: torch.Tensor | None = None,
                 main_grads: tuple[torch.Tensor, torch.Tensor] | None = None,
                 grad_reduce: Callable[[torch.Tensor], None] | None = None) -> torch.Tensor:
    """``qkv: [tokens, (nq + 2 nkv) * hd]`` -> the same shape, q and k normalised and rotated.

    Token ``m`` is at position ``m % seqlen``, or at ``positions[m]`` (int64 or int32: packed
    sequences, decoding) of the fp32 tables ``cos``/``sin`` ``[positions, hd]``; a position outside
    the tables gives NaN and sets the device error word.  ``qkv`` is fp32, bf16 or fp16 with any row
    stride; the weights share one float type.  With ``main_grads`` (the engine's fp32 gradient views
    of the two weights) the weight gradients are added there.  On CUDA, and with ``main_grads``, second
    derivatives and tangents are refused.
    """
    if qkv.dim() != 2 or qkv.shape[1] != (n_q_heads + 2 * n_kv_heads) * head_dim:
        raise ValueError(f"qkv must be [tokens, {(n_q_heads + 2 * n_kv_heads) * head_dim}], got {tuple(qkv.shape)}")
    if head_dim % 2:
        raise ValueError(f"the rotation needs an even head_dim, got {head_dim}")
    if positions is not None:
        positions = positions.reshape(-1).contiguous()
        if positions.numel() != qkv.shape[0]:
            raise ValueError(f"{positions.numel()} positions for {qkv.shape[0]} tokens")
    if qkv.stride(1) != 1:
        qkv = qkv.contiguous()
    if qkv.is_cuda and main_grads is None and grad_reduce is None:
        return native().qk_norm_rope(qkv, q_weight, k_weight, cos, sin, positions, n_q_heads, n_kv_heads, head_dim,
                                     seqlen, eps)
    return _QKNormRopeFn.apply(qkv, q_weight, k_weight, cos, sin, positions, n_q_heads, n_kv_heads, head_dim,
                               seqlen, eps, main_grads, grad_reduce)
