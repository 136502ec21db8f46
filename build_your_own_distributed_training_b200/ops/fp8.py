"""Linear layers in 8-bit floating point with one power-of-two scale for each block of 128.

A matrix in 8 bits (:class:`Fp8Blocks`) is e4m3 codes plus e8m0 scales: ``x ~ code * scale`` with the
scale of a block the least power of two that brings its largest magnitude within 448.  Blocks are
``1 x 128`` along the summed axis (activations, gradients) or ``128 x 128`` (weights, whose codes serve
the forward and the input gradient alike).  All three products of :func:`linear_fp8` then run on the
block-scaled tensor-core kernel with fp32 accumulation (``csrc/fp8_gemm.cu``)::

    y  = q(x) q(W)^T        x in 1 x 128 blocks along features
    dx = q(dy) q(W)         dy in 1 x 128 blocks along outputs
    dW = q(dy)^T q(x)       both in 1 x 128 blocks along tokens

The operands are quantised from the same bf16 tensors, each read once for both of its uses
(``csrc/fp8_quant.cu``).  A serving program keeps its weights as :class:`Fp8Blocks`
(:func:`quantize_fp8` with ``square=True``).  No reference counterpart: the reference trains in bf16
(``src/utils/dtype.py:74-106``).
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.autograd.forward_ad as fwd

from . import grad_state
from ._ext import native
from .first_order import first_order

BLOCK = 128
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


class Fp8Blocks(NamedTuple):
    """``values``: e4m3 ``[rows, cols]``; ``scales``: e8m0 ``[rows, ceil(cols / 128)]`` (one for each
    1 x 128 block) or ``[ceil(rows / 128), ceil(cols / 128)]`` (128 x 128 blocks); ``tiles`` (optional,
    CUDA): the scales as the tensor-core kernel takes them, made by :func:`quantize_fp8` and from
    ``scales`` in each product where absent."""

    values: torch.Tensor
    scales: torch.Tensor
    tiles: torch.Tensor | None = None

    @property
    def rows_per_scale(self) -> int:
        """1 or 128; raises when the scales fit neither."""
        r, c = self.values.shape
        kb = -(-c // BLOCK)
        for gran in (BLOCK, 1):
            if tuple(self.scales.shape) == (-(-r // gran), kb):
                return gran
        raise ValueError(f"scales {tuple(self.scales.shape)} fit neither 1 x 128 nor 128 x 128 blocks of {r} x {c}")

    def dequantize(self) -> torch.Tensor:
        """The fp32 values that the codes stand for."""
        s = self.scales.float()
        if self.rows_per_scale == BLOCK:
            s = s.repeat_interleave(BLOCK, 0)[: self.values.shape[0]]
        return self.values.float() * s.repeat_interleave(BLOCK, 1)[:, : self.values.shape[1]]


def _quantize_cpu(x: torch.Tensor, rows: int) -> Fp8Blocks:
    r, c = x.shape
    br, bc = -(-r // rows), -(-c // BLOCK)
    pad = torch.zeros(br * rows, bc * BLOCK)
    pad[:r, :c] = x
    b = pad.view(br, rows, bc, BLOCK)
    amax = b.abs().amax((1, 3))
    part, power = torch.frexp(amax.nan_to_num(0.0, 0.0).clamp_min(2.0 ** -100))  # 448 = 0.875 * 2^9
    exp = torch.where(amax.isfinite(), torch.where(part > 0.875, power + 119, power + 118), 255)
    scale = exp.to(torch.uint8).view(E8M0)
    codes = (b / scale.float()[:, None, :, None]).to(E4M3)
    return Fp8Blocks(codes.view(br * rows, bc * BLOCK)[:r, :c], scale)


def _quantize(x: torch.Tensor, square: bool, plain: bool, transposed: bool) -> tuple[Fp8Blocks | None, Fp8Blocks | None]:
    """Codes as they lie and / or of the transpose, from one read of ``x``."""
    if x.is_cuda:
        q, s, t, qt, st, tt = native().fp8_quantize(x, square, plain, transposed)
        return Fp8Blocks(q, s, t) if plain else None, Fp8Blocks(qt, st, tt) if transposed else None
    a = _quantize_cpu(x.float(), BLOCK if square else 1) if plain else None
    b = _quantize_cpu(x.float().t(), BLOCK if square else 1) if transposed else None
    return a, b


def quantize_fp8(x: torch.Tensor, *, square: bool = False) -> Fp8Blocks:
    """``x [rows, cols]`` (fp32, bf16, fp16) in 8 bits, in 1 x 128 or (``square``) 128 x 128 blocks.

    A block with NaN or infinity gets a NaN scale; a block below 2^-100 the scale for 2^-100.
    """
    if x.dim() != 2:
        raise ValueError(f"quantize_fp8 takes a matrix, got {tuple(x.shape)}")
    if not x.is_floating_point() or x.dtype.itemsize not in (2, 4):
        raise ValueError(f"quantize_fp8 takes fp32, bf16 or fp16, got {x.dtype}")
    x = x.detach()  # codes have no derivative
    if x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return _quantize(x, square, True, False)[0]


def _wants_grad(t: torch.Tensor) -> bool:
    return t.requires_grad and torch.is_grad_enabled()


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, *, residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16, accumulate: bool = False) -> torch.Tensor:
    """``a [M, K] @ b [N, K]^T (+ residual)`` in bf16 or fp32; ``accumulate`` adds to the fp32 ``out``.
    Has no backward (:func:`linear_fp8` has)."""
    if a.values.shape[1] != b.values.shape[1]:
        raise ValueError(f"summed axes differ: {tuple(a.values.shape)} and {tuple(b.values.shape)}")
    for t in (a, b):
        if t.values.dtype != E4M3 or t.scales.dtype != E8M0:
            raise ValueError(f"fp8_matmul takes e4m3 codes with e8m0 scales, got {t.values.dtype} and {t.scales.dtype}")
        t.rows_per_scale  # noqa: B018 - raises when the scales do not fit
    if any(t is not None and (_wants_grad(t) or fwd.unpack_dual(t).tangent is not None) for t in (residual, out)):
        raise ValueError("fp8_matmul has no backward: call linear_fp8 for the gradient of a residual")
    shape = (a.values.shape[0], b.values.shape[0])
    if out is None:
        if accumulate:
            raise ValueError("accumulate needs the fp32 tensor to add to")
        out = torch.empty(shape, device=a.values.device, dtype=out_dtype)
    if tuple(out.shape) != shape:
        raise ValueError(f"out is {tuple(out.shape)}, the product {shape}")
    if residual is not None and tuple(residual.shape) != shape:
        raise ValueError(f"residual is {tuple(residual.shape)}, the product {shape}")
    if a.values.is_cuda:
        native().fp8_product(a.values, a.scales, a.tiles, b.values, b.scales, b.tiles, out, residual, accumulate)
        return out
    y = a.dequantize() @ b.dequantize().t()
    if residual is not None:
        y = y + residual.float()
    return out.add_(y) if accumulate else out.copy_(y)


class _LinearFp8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x2, weight, residual, main_grad, grad):  # type: ignore[override]
        # transposed codes are for the backward: none without gradients, whatever the tensors ask for
        need_x, need_w = grad and ctx.needs_input_grad[0], grad and (ctx.needs_input_grad[1] or main_grad is not None)
        xq, xt = _quantize(x2, False, True, need_w)
        # the engine's weight is a view that it fills again for the backward: keeping that costs no memory, keeping
        # codes would hold a byte of every layer's weight on every rank, so the backward makes them again
        again = need_x and main_grad is not None
        wq, wt = _quantize(weight, True, True, need_x and not again)
        y = fp8_matmul(xq, wq, residual=residual, out_dtype=x2.dtype)
        on_cpu = not x2.is_cuda  # there first_order wants what the gradients would depend on
        ctx.save_for_backward(*(xt or (None,) * 3), *(wt or (None,) * 3), weight if again or on_cpu else None,
                              x2 if on_cpu else None)
        ctx.main_grad, ctx.need = main_grad, (need_x, need_w, residual is not None)
        ctx.wshape, ctx.wdtype = weight.shape, weight.dtype
        return y

    @staticmethod
    def backward(ctx, dy):  # type: ignore[override]
        saved = ctx.saved_tensors  # once: recomputed under activation checkpointing
        with torch.no_grad():
            grads = _LinearFp8Fn._gradients(ctx, saved, dy)
        inputs = [t for t in saved[6:] if t is not None]
        dx, dw = (first_order("linear_fp8", t, (dy,), *inputs) for t in grads)
        return dx, dw, (dy if ctx.need[2] else None), None, None

    @staticmethod
    def _gradients(ctx, saved, dy):
        need_x, need_w, _ = ctx.need
        dy2 = dy.contiguous()
        dx = dw = None
        if need_x or need_w:
            g, gt = _quantize(dy2, False, need_x, need_w)
        if need_x:
            wt = Fp8Blocks(*saved[3:6]) if saved[3] is not None else _quantize(saved[6], True, False, True)[1]
            dx = fp8_matmul(g, wt, out_dtype=dy.dtype)
        if need_w:
            mg, xt = ctx.main_grad, Fp8Blocks(*saved[:3])
            if mg is not None:
                store = grad_state.take_fresh(mg)
                fp8_matmul(gt, xt, out=mg.view(ctx.wshape), accumulate=not store)
            else:
                wide = ctx.wdtype not in (torch.bfloat16, torch.float32)
                dw = fp8_matmul(gt, xt, out_dtype=torch.float32 if wide else ctx.wdtype)
                dw = dw.to(ctx.wdtype) if wide else dw
        return dx, dw


def linear_fp8(x: torch.Tensor, weight: torch.Tensor | Fp8Blocks, *, residual: torch.Tensor | None = None,
               main_grad: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight^T (+ residual)`` with both operands in 8 bits; ``x [..., K]``, ``weight [N, K]``.

    A weight tensor is quantised in the call and gets its gradient (into ``main_grad`` when given);
    kept :class:`Fp8Blocks` are for inference.  On CUDA ``x`` and ``residual`` are bf16; keep the rows
    of ``Fp8Blocks.values`` on 16-byte boundaries (:func:`quantize_fp8` does), others are copied first.

    The backward needs codes of ``x`` and of the weight along their other axes.  Those of ``x`` (a byte an
    element) are kept from the forward, and so are the weight's, unless it comes with ``main_grad``: then the
    weight itself is kept and quantised again.  The rounded product has no second derivative (refused).
    """
    K = weight.values.shape[1] if isinstance(weight, Fp8Blocks) else weight.shape[1]
    N = weight.values.shape[0] if isinstance(weight, Fp8Blocks) else weight.shape[0]
    if x.shape[-1] != K:
        raise ValueError(f"x has {x.shape[-1]} features, the weight {K}")
    if x.is_cuda and x.dtype != torch.bfloat16:
        raise ValueError(f"linear_fp8 takes bf16 activations on CUDA, got {x.dtype}")
    if residual is not None and (residual.shape != (*x.shape[:-1], N) or residual.dtype != x.dtype):
        raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} does not match {(*x.shape[:-1], N)} {x.dtype}")
    x2 = x.reshape(-1, K)
    if K > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    r2 = None if residual is None else residual.reshape(-1, N).contiguous()
    if isinstance(weight, Fp8Blocks):
        if _wants_grad(x) or (residual is not None and _wants_grad(residual)):
            raise ValueError("weights kept in 8 bits have no backward: call linear_fp8 with the weight tensor")
        if x.is_cuda:
            y = native().linear_fp8_kept(x2, *weight, r2)
        else:  # (tangents: the native call above looks for them itself)
            if any(t is not None and fwd.unpack_dual(t).tangent is not None for t in (x, residual)):
                raise ValueError("weights kept in 8 bits have no derivative: call linear_fp8 with the weight tensor")
            y = fp8_matmul(_quantize(x2, False, True, False)[0], weight, residual=r2, out_dtype=x.dtype)
    else:
        w = weight if weight.is_contiguous() else weight.contiguous()
        if x.is_cuda and main_grad is None:
            y = native().linear_fp8(x2, w, r2)
        else:
            y = _LinearFp8Fn.apply(x2, w, r2, main_grad, torch.is_grad_enabled())
    return y.view(*x.shape[:-1], N)
