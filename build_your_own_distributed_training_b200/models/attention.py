"""Causal grouped-query attention block (reference ``src/model/attention.py:70-155``).

Parameters keep the reference names ``wq, wk, wv, wo``.  The forward runs
three fused ops: the packed QKV projection with RoPE in its epilogue, flash
attention reading the packed buffer (local head counts are inferred from the
possibly TP-sharded weight shapes, as the reference's ``view(..., -1, hd)``
did), and the output projection with the residual add fused (and, under TP,
the all-reduce or reduce-scatter fused with it).

With ``qk_norm`` every query and key head is normalised before the rotation
(``q_norm.weight``, ``k_norm.weight``): the rotation then runs with the norm,
after the projection.  With ``fp8`` the projections run in 8 bits.  With
``resid_dropout`` the output is dropped out before the residual add.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from ..config import ModelConfig
from ..ops.attention import causal_attention, repeat_kv  # noqa: F401
from ..ops.fp8 import linear_fp8
from ..ops.linear import linear, linear_qkv_rope
from ..ops.qk_norm import qk_norm_rope
from ..ops.rope import rope_packed
from ..parallel import tensor_parallel as tpar
from .layers import Linear, fused_rows, main_grad_of


class HeadNorm(nn.Module):
    """The ``[head_dim]`` weight of a per-head RMSNorm (applied by :func:`..ops.qk_norm.qk_norm_rope`)."""

    def __init__(self, head_dim: int) -> None:
        super().__init__()
        self.weight = nn.Parameter(torch.ones(head_dim))


class Attention(nn.Module):
    def __init__(self, config: ModelConfig) -> None:
        super().__init__()
        assert config.n_kv_heads is not None
        self.n_heads = config.n_heads
        self.n_kv_heads = config.n_kv_heads
        self.head_dim = config.head_dim
        self.dropout_p = config.dropout
        kv = self.n_kv_heads * self.head_dim
        self.wq = Linear(config.d_model, config.d_model, config.attention_bias)
        self.wk = Linear(config.d_model, kv, config.attention_bias)
        self.wv = Linear(config.d_model, kv, config.attention_bias)
        self.wo = Linear(config.d_model, config.d_model, config.attention_bias)
        self.qk_norm = config.qk_norm
        if config.qk_norm:
            self.q_norm, self.k_norm = HeadNorm(config.head_dim), HeadNorm(config.head_dim)
        self.norm_eps = config.norm_eps
        self.resid_dropout = config.resid_dropout
        self.fp8 = False
        self.tp: tpar.TPInfo | None = None

    def _normed_qkv(self, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nq: int, nkv: int) -> torch.Tensor:
        """Normalised and rotated ``[q | k | v]`` (rotated alone without ``qk_norm``)."""
        hd, seqlen = self.head_dim, cos.shape[0]
        if not self.qk_norm:
            return rope_packed(qkv, cos, sin, (nq + nkv) * hd, hd, seqlen)
        wq, wk = self.q_norm.weight, self.k_norm.weight
        mg = (main_grad_of(wq), main_grad_of(wk))
        # a rank's heads give part of the weights' gradient: the sharding engine sums such parts under
        # sequence parallelism only
        reduce = None
        if self.tp is not None and self.tp.size > 1 and not self.tp.sequence_parallel:
            reduce = lambda g: tpar.dist.all_reduce(g, group=self.tp.group)  # noqa: E731
        return qk_norm_rope(qkv, wq, wk, cos, sin, nq, nkv, hd, seqlen, self.norm_eps,
                            main_grads=mg if mg[0] is not None else None, grad_reduce=reduce)

    def _unfused_qkv(self, x2: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, nq: int, nkv: int) -> torch.Tensor:
        """The projection apart from what follows it (8-bit weights, normalised heads)."""
        x2 = tpar.column_input(x2, self.tp)
        lin = [self.wq, self.wk, self.wv]
        w, mg = fused_rows([m.weight for m in lin])
        bias = None if self.wq.bias is None else torch.cat([m.bias for m in lin]).to(x2.dtype)
        qkv = linear_fp8(x2, w, main_grad=mg) if self.fp8 else linear(x2, w, bias=bias, main_grad=mg)
        return self._normed_qkv(qkv, cos, sin, nq, nkv)

    def forward(self, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                residual: torch.Tensor | None = None) -> torch.Tensor:
        """``x``: ``[b, s, d]`` (or local ``[tokens, d]`` under sequence parallelism)."""
        out_shape = x.shape if residual is None else residual.shape
        seqlen = cos.shape[0]
        hd = self.head_dim
        nq, nkv = self.wq.weight.shape[0] // hd, self.wk.weight.shape[0] // hd
        unfused = self.fp8 or self.qk_norm
        x2 = x.reshape(-1, x.shape[-1])
        if not unfused:
            # under sequence parallelism x2 may stay this rank's rows: the QKV GEMM gathers them
            x2, grad_comm = tpar.column_input_fused(x2, self.tp, sp_ok=self.wq.bias is None)
        if unfused:
            qkv = self._unfused_qkv(x2, cos, sin, nq, nkv)
        elif self.wq.bias is not None:
            w = torch.cat([self.wq.weight, self.wk.weight, self.wv.weight])
            b = torch.cat([self.wq.bias, self.wk.bias, self.wv.bias])
            qkv = torch.nn.functional.linear(x2, w.to(x2.dtype), b.to(x2.dtype))
            from ..ops.rope import rope_forward
            qkv = qkv.clone()
            rope_forward(qkv, cos, sin, (nq + nkv) * hd, hd, seqlen)
        else:
            w, mg = fused_rows([self.wq.weight, self.wk.weight, self.wv.weight])
            qkv = linear_qkv_rope(x2, w, cos, sin, nq, nkv, hd, seqlen, main_grad=mg, grad_comm=grad_comm)
        o = causal_attention(qkv, qkv.shape[0] // seqlen, seqlen, nq, nkv, hd,
                             self.dropout_p if self.training else 0.0)
        r2 = residual.reshape(-1, residual.shape[-1]) if residual is not None else None
        if r2 is not None and self.training and self.resid_dropout > 0:
            y = tpar.row_output_dropout(o, self.wo.weight, r2, self.tp, self.resid_dropout,
                                        main_grad=main_grad_of(self.wo.weight), bias=self.wo.bias, fp8=self.fp8)
        else:
            y = tpar.row_output_linear(o, self.wo.weight, r2, self.tp,
                                       main_grad=main_grad_of(self.wo.weight), bias=self.wo.bias, fp8=self.fp8)
        return y.view(out_shape)
