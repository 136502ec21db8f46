"""Log probabilities of given tokens, with the distribution's entropy and its top alternatives.

What likelihood scoring and policy losses need of a row of logits: ``ln p(token)``, the entropy of
``p`` and the ``top_k`` most probable tokens, all at a temperature, in one read of the logits; the
backward makes the logit gradient of both ``logprob`` and ``entropy`` in one read and one write
(``csrc/token_logprobs.cu``).  The training loss's fused head (:mod:`.loss`) gives only the mean
cross-entropy.

:func:`lm_head_token_log_probs` runs the LM head in front of it in blocks of rows, so that the fp32
logits in memory are bounded; its backward makes each block's logits again.
"""

from __future__ import annotations

import os
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import gemm, grad_state
from ._ext import native
from .first_order import first_order
from .loss import IGNORE

MAX_TOP_K = 32
# bytes of fp32 logits that lm_head_token_log_probs holds at a time
HEAD_BYTES = int(os.environ.get("DTB_LOGPROB_BYTES", str(1 << 30)))


class TokenLogProbs(NamedTuple):
    logprob: torch.Tensor                    # fp32, the tokens' shape
    entropy: torch.Tensor                    # fp32, the tokens' shape
    top_logprobs: torch.Tensor | None = None  # fp32 [..., top_k], largest first
    top_tokens: torch.Tensor | None = None    # int64 [..., top_k]; equal logits: lowest index first


def _reference(x: torch.Tensor, tokens: torch.Tensor, temperature: float, top_k: int, ignore: int):
    """``x: [M, V]`` -> (logprob, entropy, top log probabilities, top tokens, (m, kind))."""
    x = x.float()
    V = x.shape[1]
    m = x.amax(-1)
    bad = ~((tokens >= 0) & (tokens < V)) | m.isnan() | (m == float("inf"))
    skip = tokens == ignore
    empty = m == float("-inf")
    ok = ~(bad | skip | empty)
    z = torch.where(ok[:, None], (x - m[:, None]) / temperature, 0.0)
    e = z.exp()
    s = e.sum(-1)
    logp = z - s.log()[:, None]
    ent = s.log() - torch.where(e > 0, e * z, 0.0).sum(-1) / s
    lp = logp.gather(1, torch.where(ok, tokens, 0)[:, None])[:, 0]
    nan, ninf = float("nan"), float("-inf")

    def finish(v: torch.Tensor, at_empty: float, at_skip: float) -> torch.Tensor:
        v = v.clone()
        v[empty], v[bad], v[skip] = at_empty, nan, at_skip
        return v

    top_i = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :top_k]
    top_v = finish(logp.gather(1, top_i), ninf, ninf)
    top_i = top_i.masked_fill((bad | skip)[:, None], -1)
    # rows that are skipped or empty have no gradient, bad ones a NaN gradient
    kind = torch.where(skip | (empty & ~bad), 1, torch.where(bad, 2, 0))
    return finish(lp, ninf, 0.0), finish(ent, 0.0, 0.0), top_v, top_i, (m, kind)


def _reference_grad(x, tokens, state, g_lp, g_ent, temperature):
    """The logits' gradient as a function of ``x`` alone (``m`` only shifts), so that it can be differentiated again;
    excluded tokens (-inf, or so far below ``m`` that the difference is) stay out of every product."""
    m, kind = state
    ok = kind == 0
    x = x.float()
    live = ok[:, None] & ((x.detach() - m[:, None]) / temperature > float("-inf"))
    z = torch.where(live, (torch.where(live, x, 0.0) - torch.where(ok, m, 0.0)[:, None]) / temperature, 0.0)
    e = torch.where(live, z.exp(), 0.0)
    s = torch.where(ok, e.sum(-1), 1.0)
    p = e / s[:, None]
    d = torch.zeros_like(z)
    if g_lp is not None:
        d = d - p * g_lp[:, None]
        d = d.scatter_add(1, torch.where(ok, tokens, 0)[:, None], g_lp[:, None])
    if g_ent is not None:
        ent = s.log() - (e * z).sum(-1) / s
        d = d - g_ent[:, None] * (p * (z - s.log()[:, None]) + p * ent[:, None])
    d = d / temperature
    d[kind == 1], d[kind == 2] = 0.0, float("nan")
    return d


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, temperature, top_k, ignore):  # type: ignore[override]
        lp, ent, top_v, top_i, state = _reference(x, tokens, temperature, top_k, ignore)
        ctx.save_for_backward(x, tokens, *state)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(top_v, top_i)
        ctx.set_materialize_grads(False)
        return lp, ent, top_v, top_i

    @staticmethod
    def backward(ctx, g_lp, g_ent, _v, _i):  # type: ignore[override]
        x, tokens, *state = ctx.saved_tensors
        return _reference_grad(x, tokens, state, g_lp, g_ent, ctx.temperature).to(x.dtype), None, None, None, None


def _row_grad(g: torch.Tensor | None) -> torch.Tensor | None:
    return None if g is None else g.float().contiguous()


def _check(tokens: torch.Tensor, rows: torch.Size, vocab: int, temperature: float, top_k: int) -> None:
    if tokens.shape != rows:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not match the logits' rows {tuple(rows)}")
    if tokens.dtype != torch.int64:
        raise ValueError(f"tokens must be int64, got {tokens.dtype}")
    if not 2.0 ** -126 <= temperature <= 2.0 ** 126:  # fp32 holds the reciprocal
        raise ValueError(f"temperature must be positive, in [2^-126, 2^126], got {temperature}")
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise ValueError(f"top_k={top_k} is outside [0, {min(MAX_TOP_K, vocab)}]")


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, top_k: int = 0,
                    ignore_index: int = IGNORE) -> TokenLogProbs:
    """``logits [..., V]`` (fp32, bf16, fp16), ``tokens [...]`` int64 -> :class:`TokenLogProbs`.

    Differentiable in ``logprob`` and ``entropy`` (twice on the CPU alone; on CUDA second derivatives and
    tangents are refused).  Forbidden tokens may be ``-inf`` or the type's
    lowest value.  Rows whose token is ``ignore_index`` give 0, 0, alternatives ``-1`` at ``-inf``, and
    no gradient; a row with every logit at ``-inf`` gives ``-inf``, entropy 0 and no gradient; NaN or
    +inf in a row, or a token outside the vocabulary (which also sets the device error word), gives NaN.
    """
    V = logits.shape[-1]
    _check(tokens, logits.shape[:-1], V, temperature, top_k)
    if logits.is_cuda:
        return TokenLogProbs(*native().token_logprobs(logits, tokens, temperature, top_k, ignore_index))
    lp, ent, top_v, top_i = _TokenLogProbsFn.apply(logits.reshape(-1, V), tokens.reshape(-1), float(temperature),
                                                   int(top_k), int(ignore_index))
    return _shaped(lp, ent, top_v, top_i, tokens.shape, top_k)


def _shaped(lp, ent, top_v, top_i, shape, top_k) -> TokenLogProbs:
    if not top_k:
        return TokenLogProbs(lp.view(shape), ent.view(shape))
    return TokenLogProbs(lp.view(shape), ent.view(shape), top_v.view(*shape, top_k), top_i.view(*shape, top_k))


def _row_blocks(rows: int, vocab: int) -> list[tuple[int, int]]:
    step = max(128, HEAD_BYTES // (4 * vocab) // 128 * 128)
    return [(r, min(rows, r + step)) for r in range(0, rows, step)]


def _whole_rows(w: torch.Tensor) -> torch.Tensor:
    """The head's weight with rows of zeros up to a multiple of 8, which the products' 16-byte rows of
    logits need; the log probabilities read the vocabulary's columns alone."""
    return F.pad(w, (0, 0, 0, -w.shape[0] % 8)) if w.shape[0] % 8 else w


class _HeadLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, tokens, temperature, top_k, ignore, main_grad):  # type: ignore[override]
        outs = []
        V, wp = w.shape[0], _whole_rows(w)
        for r0, r1 in _row_blocks(h.shape[0], V):
            logits = gemm.mm_nt(h[r0:r1], wp, out_dtype=torch.float32)[:, :V]
            outs.append(native().token_logprobs_fwd(logits, tokens[r0:r1], temperature, top_k, ignore, True))
        lp, ent, *top, state = (torch.cat(t) if len(outs) > 1 else t[0] for t in zip(*outs))
        top_v, top_i = top or (None, None)
        ctx.save_for_backward(h, w, tokens, state)
        ctx.temperature, ctx.main_grad = temperature, main_grad
        if top:
            ctx.mark_non_differentiable(*top)
        ctx.set_materialize_grads(False)
        return lp, ent, top_v, top_i

    @staticmethod
    def backward(ctx, g_lp, g_ent, _v, _i):  # type: ignore[override]
        with torch.no_grad():
            dh, dw = _HeadLogProbsFn._gradients(ctx, g_lp, g_ent)
        dh, dw = (first_order("lm_head_token_log_probs", t, (g_lp, g_ent)) for t in (dh, dw))
        return dh, dw, None, None, None, None, None

    @staticmethod
    def _gradients(ctx, g_lp, g_ent):
        h, w, tokens, state = ctx.saved_tensors
        g_lp, g_ent, mg = _row_grad(g_lp), _row_grad(g_ent), ctx.main_grad
        need_w = mg is not None or w.requires_grad
        dh = torch.empty_like(h)
        V, wp = w.shape[0], _whole_rows(w)
        direct = mg is not None and wp is w  # products straight into the engine's gradient
        store = grad_state.take_fresh(mg) if direct else True
        acc = mg.view(w.shape) if direct else (
            torch.empty(wp.shape, device=w.device, dtype=torch.float32) if need_w else None)
        for r0, r1 in _row_blocks(h.shape[0], V):
            hb = h[r0:r1]
            logits = gemm.mm_nt(hb, wp, out_dtype=torch.float32)[:, :V]
            dl = torch.empty(r1 - r0, wp.shape[0], device=h.device, dtype=h.dtype)
            if wp is not w:
                dl[:, V:] = 0
            native().token_logprobs_bwd(logits, tokens[r0:r1], state[r0:r1], None if g_lp is None else g_lp[r0:r1],
                                        None if g_ent is None else g_ent[r0:r1], ctx.temperature, dl[:, :V])
            gemm.mm_nn(dl, wp, out=dh[r0:r1])
            if acc is not None:
                gemm.mm_tn_acc(dl, hb, acc, store=store)
                store = False
        if mg is not None and not direct:
            grad_state.zero_if_fresh(mg)
            mg.view(w.shape).add_(acc[:V])
        dw = acc[:V].to(w.dtype) if mg is None and need_w else None
        return dh, dw


def lm_head_token_log_probs(h: torch.Tensor, weight: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0,
                            top_k: int = 0, ignore_index: int = IGNORE,
                            main_grad: torch.Tensor | None = None) -> TokenLogProbs:
    """:func:`token_log_probs` of ``h @ weight^T`` for ``h: [M, d]``, ``tokens: [M]``.

    On CUDA ``h`` and ``weight`` are bf16 and ``d`` a multiple of 8; the logits are fp32.  A vocabulary that is
    no multiple of 8 costs a padded copy of the weight in each direction.
    """
    _check(tokens, h.shape[:1], weight.shape[0], temperature, top_k)
    if not h.is_cuda:
        from .linear import linear
        return token_log_probs(linear(h, weight, main_grad=main_grad), tokens, temperature=temperature, top_k=top_k,
                               ignore_index=ignore_index)
    if h.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16:
        raise ValueError(f"the scoring head takes bf16 on CUDA, got {h.dtype} and {weight.dtype}")
    if h.shape[1] % 8:
        raise ValueError(f"the scoring head needs a hidden size that is a multiple of 8 on CUDA, got {h.shape[1]}")
    if h.shape[0] == 0:  # no rows: nothing for the products, zero gradients
        logits = F.linear(h, weight.detach() if main_grad is not None else weight).float()
        return token_log_probs(logits, tokens, temperature=temperature, top_k=top_k, ignore_index=ignore_index)
    lp, ent, top_v, top_i = _HeadLogProbsFn.apply(h.contiguous(), weight, tokens.contiguous(), float(temperature),
                                                  int(top_k), int(ignore_index), main_grad)
    return _shaped(lp, ent, top_v, top_i, tokens.shape, top_k)
