"""Block operators on the CPU path: values and gradients against 64-bit formulas and differences, refusals."""

from __future__ import annotations

import math

import pytest
import torch

from build_your_own_distributed_training_b200 import ops
from build_your_own_distributed_training_b200.ops.logprobs import lm_head_token_log_probs
from tests import plain_ops as plain
from tests.plain_ops import rel

# fp32 arithmetic with sums of a few hundred terms: some tens of roundings of 2^-24
F32 = 64 * 2.0 ** -24


def _tables(rows, hd):
    return ops.precompute_rope_cache(hd, rows, 10000.0)


@pytest.mark.parametrize("nq,nkv,hd,tokens,seqlen", [(4, 2, 16, 6, 3), (3, 1, 10, 1, 1), (2, 2, 64, 5, 5), (7, 1, 34, 4, 2)])
@pytest.mark.parametrize("positions", [False, True])
@pytest.mark.parametrize("main", [False, True])
def test_qk_norm_rope_matches_formula(nq, nkv, hd, tokens, seqlen, positions, main):
    g = torch.Generator().manual_seed(nq * 100 + hd)
    cos, sin = _tables(50, hd)
    x = torch.randn(tokens, (nq + 2 * nkv) * hd, generator=g).requires_grad_(True)
    wq = torch.randn(hd, generator=g).requires_grad_(True)
    wk = torch.randn(hd, generator=g).requires_grad_(True)
    pos = torch.randint(0, 50, (tokens,), generator=g) if positions else None
    where = pos.tolist() if positions else [i % seqlen for i in range(tokens)]
    dy = torch.randn(x.shape, generator=g)
    mgs = (torch.ones(hd), torch.ones(hd)) if main else None
    y = ops.qk_norm_rope(x, wq, wk, cos, sin, nq, nkv, hd, seqlen, 1e-5, positions=pos, main_grads=mgs)
    y.backward(dy)
    xd, qd, kd = (t.detach().double().requires_grad_(True) for t in (x, wq, wk))
    ref = plain.qk_norm_rope(xd, qd, kd, cos, sin, nq, nkv, hd, where, 1e-5)
    ref.backward(dy.double())
    assert rel(y, ref) < F32 and rel(x.grad, xd.grad) < F32
    gq, gk = (mgs[0] - 1, mgs[1] - 1) if main else (wq.grad, wk.grad)
    assert rel(gq, qd.grad) < 4 * F32 and rel(gk, kd.grad) < 4 * F32
    assert not main or (wq.grad is None and wk.grad is None)
    # and along a direction, against differences of the 64-bit formula
    v = torch.randn(x.shape, generator=g).double()
    f = lambda t: (plain.qk_norm_rope(t, qd.detach(), kd.detach(), cos, sin, nq, nkv, hd, where, 1e-5) * dy.double()).sum()  # noqa: E731
    want = plain.slope(f, xd.detach(), v, 1e-5)
    assert abs(float((x.grad.double() * v).sum()) - want) <= 1e-5 * float(x.grad.norm() * v.norm())


def test_qk_norm_rope_refuses():
    cos, sin = _tables(8, 16)
    w = torch.ones(16)
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="tokens"):
        ops.qk_norm_rope(x, w, w, cos, sin, 3, 1, 16, 4)
    with pytest.raises(ValueError, match="even"):
        ops.qk_norm_rope(torch.zeros(4, 60), w, w, cos, sin, 2, 1, 15, 4)
    with pytest.raises(ValueError, match="positions"):
        ops.qk_norm_rope(x, w, w, cos, sin, 2, 1, 16, 4, positions=torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("n,start", [(1, 0), (7, 0), (64, 0), (129, 5), (40, (1 << 35) - 3)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_mask_is_philox_of_the_element_number(n, start, p):
    x = torch.arange(1.0, n + 1).requires_grad_(True)
    r = torch.randn(n).requires_grad_(True)
    seed = 0xDEADBEEFCAFEF00D
    y = ops.dropout_add(x, r, p, seed, start=start)
    want = plain.dropout_add(x.detach().double(), r.detach().double(), p, seed, start)
    assert rel(y, want) < F32
    y.backward(torch.ones(n))
    assert torch.equal(r.grad, torch.ones(n))
    keep = plain.keep_mask(n, p, seed, start)
    assert torch.equal(x.grad != 0, keep)


def test_dropout_rows_of_a_split_activation_see_the_whole_mask():
    x = torch.randn(12, 9)
    whole = ops.dropout_add(x, None, 0.3, 77)
    for a, b in ((0, 5), (5, 12)):
        part = ops.dropout_add(x[a:b], None, 0.3, 77, start=a * 9)
        assert torch.equal(part, whole[a:b])
    n = 1 << 16
    kept = float((ops.dropout_add(torch.ones(n), None, 0.1, 5) != 0).float().mean())
    assert abs(kept - 0.9) < 6 * math.sqrt(0.09 / n)  # six standard deviations


def test_dropout_refuses():
    x = torch.zeros(4)
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            ops.dropout_add(x, None, bad, 1)
    with pytest.raises(ValueError, match="64 bits"):
        ops.dropout_add(x, None, 0.1, 1 << 64)
    with pytest.raises(ValueError, match="negative"):
        ops.dropout_add(x, None, 0.1, 1, start=-1)
    with pytest.raises(ValueError, match="residual"):
        ops.dropout_add(x, torch.zeros(5), 0.1, 1)


@pytest.mark.parametrize("V,top_k", [(1, 1), (7, 3), (100, 32), (33, 0)])
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_token_log_probs_match_formula(V, top_k, temperature):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(2, 5, V, generator=g) * 3).requires_grad_(True)
    tok = torch.randint(0, V, (2, 5), generator=g)
    tok[1, 2] = -100
    r = ops.token_log_probs(x, tok, temperature=temperature, top_k=top_k)
    xd = x.detach().double().view(-1, V).requires_grad_(True)
    lp, ent = plain.logprobs(xd, tok.view(-1), temperature)
    assert rel(r.logprob, lp.view(2, 5)) < F32 and float((r.entropy.view(-1).double() - ent).abs().max()) < 16 * F32
    if top_k:
        for i in range(10):
            if tok.view(-1)[i] == -100:
                assert (r.top_tokens.view(10, -1)[i] == -1).all()
            else:
                assert r.top_tokens.view(10, -1)[i].tolist() == plain.top_order(xd[i].tolist(), top_k)
    else:
        assert r.top_tokens is None
    a, b = torch.randn(2, 5, generator=g), torch.randn(2, 5, generator=g)
    (r.logprob * a + r.entropy * b).sum().backward()
    (lp * a.view(-1).double() + ent * b.view(-1).double()).sum().backward()
    assert float((x.grad.view(-1, V).double() - xd.grad).abs().max()) < 64 * F32
    assert (x.grad[1, 2] == 0).all()
    if V > 1:
        v = torch.randn(10, V, generator=g).double()
        f = lambda t: sum((u * w.view(-1).double()).sum() for u, w in zip(plain.logprobs(t, tok.view(-1), temperature), (a, b)))  # noqa: E731
        want = plain.slope(f, xd.detach(), v, 1e-5)
        assert abs(float((x.grad.view(-1, V).double() * v).sum()) - want) <= 1e-5 * (1 + abs(want))


def test_token_log_probs_edge_rows():
    inf = float("inf")
    x = torch.tensor([[-inf, -inf, -inf], [0.0, -inf, 1.0], [0.0, inf, 0.0], [0.0, float("nan"), 0.0],
                      [1.0, 2.0, 3.0], [torch.finfo(torch.float32).min] * 3], requires_grad=True)
    tok = torch.tensor([0, 1, 1, 0, 3, 2])
    r = ops.token_log_probs(x, tok, top_k=2, temperature=0.5)
    assert r.logprob[0] == -inf and r.entropy[0] == 0 and r.top_tokens[0].tolist() == [0, 1]
    assert r.logprob[1] == -inf and r.entropy[1] > 0
    assert r.logprob[2:5].isnan().all() and r.entropy[2:5].isnan().all()
    assert abs(float(r.logprob[5]) + math.log(3)) < F32 and abs(float(r.entropy[5]) - math.log(3)) < 4 * F32
    g, = torch.autograd.grad((r.logprob, r.entropy), x, (torch.ones(6), torch.ones(6)))
    assert (g[0] == 0).all() and g[1].isfinite().all() and g[2:5].isnan().all() and g[5].isfinite().all()


def test_token_log_probs_refuses():
    x, t = torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="rows"):
        ops.token_log_probs(x, t[:3])
    with pytest.raises(ValueError, match="int64"):
        ops.token_log_probs(x, t.int())
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            ops.token_log_probs(x, t, temperature=bad)
    for bad in (-1, 10, 33):
        with pytest.raises(ValueError, match="top_k"):
            ops.token_log_probs(x, t, top_k=bad)


def test_lm_head_token_log_probs_matches_logits():
    g = torch.Generator().manual_seed(3)
    h = torch.randn(6, 8, generator=g).requires_grad_(True)
    w = torch.randn(24, 8, generator=g).requires_grad_(True)
    tok = torch.randint(0, 24, (6,), generator=g)
    r = lm_head_token_log_probs(h, w, tok, top_k=4)
    s = ops.token_log_probs(h @ w.t(), tok, top_k=4)
    assert torch.allclose(r.logprob, s.logprob, atol=F32) and torch.equal(r.top_tokens, s.top_tokens)
    (r.logprob.sum() + r.entropy.sum()).backward()
    assert h.grad is not None and w.grad is not None
