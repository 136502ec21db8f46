"""Block operators on the CPU path at the edge of what they take: second derivatives, tangents, positions."""

from __future__ import annotations

import pytest
import torch

from build_your_own_distributed_training_b200 import ops
from tests import plain_ops as plain
from tests.plain_ops import rel

# fp32 arithmetic with sums of a few hundred terms: some tens of roundings of 2^-24
F32 = 64 * 2.0 ** -24


def _hessian_product(f, x, v):
    """d/dx <df/dx, v>, with the other route through df/dx's graph."""
    g, = torch.autograd.grad(f(x), x, create_graph=True)
    return torch.autograd.grad((g * v).sum(), x)[0]


@pytest.mark.parametrize("what", ["logprob", "entropy", "both"])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_second_derivatives_of_log_probs(what, temperature):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 16, generator=g) * 2
    x[2, 3] = -float("inf")
    tok = torch.tensor([0, 15, 4, -100, 7])
    a, b, v = (torch.randn(*s, generator=g) for s in ((5,), (5,), (5, 16)))
    v[2, 3] = 0.0  # an excluded token has no direction
    a, b = a * (what != "entropy"), b * (what != "logprob")
    r = lambda t: ops.token_log_probs(t, tok, temperature=temperature)  # noqa: E731
    got = _hessian_product(lambda t: ((r(t).logprob * a) + (r(t).entropy * b)).sum(), x.clone().requires_grad_(True), v)
    live = [0, 1, 2, 4]
    keep = torch.ones(5, 16, dtype=torch.bool)
    keep[2, 3] = False

    def formula(t):
        total = 0.0
        for i in live:
            z = t[i][keep[i]] / temperature
            logp = z - torch.logsumexp(z, 0)
            at = int(keep[i, :tok[i]].sum())
            total = total + a[i].double() * logp[at] - b[i].double() * (logp.exp() * logp).sum()
        return total
    xd = x.double().masked_fill(~keep, 0.0).requires_grad_(True)
    want = _hessian_product(formula, xd, v.double())
    assert got[3].abs().max() == 0 and got.isfinite().all()
    # products of probabilities with factors of up to about 10, each of some tens of roundings
    assert float((got.double() - want).abs().max()) < 16 * F32 * float(want.abs().max())
    # and against differences of the first derivative
    if what == "both":
        first = lambda t: torch.autograd.grad(formula(t.requires_grad_(True)), t)[0]  # noqa: E731
        h = 1e-5
        diff = (first((xd.detach() + h * v.double())) - first(xd.detach() - h * v.double())) / (2 * h)
        assert rel(want, diff) < 1e-6


def test_log_prob_gradients_beside_the_lowest_value():
    low = torch.finfo(torch.float32).min
    x = torch.tensor([[1e38, low, 1e38, low], [0.0, low, 1.0, -float("inf")]], requires_grad=True)
    r = ops.token_log_probs(x, torch.tensor([0, 2]), temperature=0.5)
    g, = torch.autograd.grad((r.logprob + r.entropy).sum(), x, create_graph=True)
    p = torch.softmax(torch.tensor([0.0, 2.0]).double(), 0)
    ent = -(p * p.log()).sum()
    # d logprob = (onehot - p) / T, d entropy = -p (ln p + H) / T
    want = torch.tensor([[0.5, 0.0, -0.5, 0.0]]).double() / 0.5
    assert rel(g[0], want[0]) < F32
    row = torch.stack((-p[0] - p[0] * (p[0].log() + ent), 1 - p[1] - p[1] * (p[1].log() + ent))) / 0.5
    assert rel(g[1, [0, 2]], row) < F32 and (g[1, [1, 3]] == 0).all()
    assert torch.autograd.grad(g.sum(), x)[0].isfinite().all()
