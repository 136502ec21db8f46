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


def test_second_derivatives_of_the_other_operators():
    from build_your_own_distributed_training_b200.ops.linear import swiglu_packed
    from build_your_own_distributed_training_b200.ops.rope import rope_packed
    g = torch.Generator().manual_seed(2)
    x, v = torch.randn(6, 64, generator=g), torch.randn(6, 64, generator=g)
    wq, wk = torch.randn(16, generator=g), torch.randn(16, generator=g)
    cos, sin = ops.precompute_rope_cache(16, 3, 10000.0)
    mask = ops.dropout_add(torch.ones_like(x), None, 0.3, 5).double()
    pos = [0, 1, 2, 0, 1, 2]
    turn = lambda t: plain.qk_norm_rope(t, 1.0, 1.0, cos, sin, 2, 1, 16, pos, 0.0)  # noqa: E731

    def rotated(t):  # a head of unit rms is only rotated
        u = t.view(6, 4, 16)
        r = u.square().mean(-1, keepdim=True).sqrt()
        return (turn(t).view(6, 4, 16) * torch.cat((r[:, :3], torch.ones_like(r[:, 3:])), 1)).reshape(6, 64)
    for f, ref in ((lambda t: ops.qk_norm_rope(t, wq, wk, cos, sin, 2, 1, 16, 3),
                    lambda t: plain.qk_norm_rope(t, wq.double(), wk.double(), cos, sin, 2, 1, 16, pos, 1e-5)),
                   (lambda t: ops.dropout_add(t, None, 0.3, 5), lambda t: t * mask),
                   (lambda t: swiglu_packed(t, 32), lambda t: torch.nn.functional.silu(t[:, :32]) * t[:, 32:]),
                   (lambda t: rope_packed(t, cos, sin, 48, 16, 3), rotated)):
        got = _hessian_product(lambda t: f(t).pow(3).sum(), x.clone().requires_grad_(True), v)
        want = _hessian_product(lambda t: ref(t).pow(3).sum(), x.double().requires_grad_(True), v.double())
        assert rel(got, want) < 4 * F32


@pytest.mark.parametrize("name", ["linear_fp8", "linear_fp8 main_grad", "qk_norm_rope main_grads"])
def test_second_derivatives_that_do_not_exist_are_refused(name):
    """Rounded operands, and gradients that went into the engine's buffers."""
    g = torch.Generator().manual_seed(3)
    x, w, nw = (torch.randn(*s, generator=g).requires_grad_(True) for s in ((8, 64), (24, 64), (16,)))
    cos, sin = ops.precompute_rope_cache(16, 8, 10000.0)
    f, args = {"linear_fp8": (lambda: ops.linear_fp8(x, w), (x, w)),
               "linear_fp8 main_grad": (lambda: ops.linear_fp8(x, w, main_grad=torch.zeros(24 * 64)), (x,)),
               "qk_norm_rope main_grads": (lambda: ops.qk_norm_rope(x, nw, nw, cos, sin, 2, 1, 16, 8, main_grads=(
                   torch.zeros(16), torch.zeros(16))), (x,))}[name]
    first = torch.autograd.grad(f().sum(), args)
    again = torch.autograd.grad(f().sum(), args, create_graph=True)
    for a, b in zip(first, again):
        assert torch.equal(a, b.detach())
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(b.sum() + x.pow(2).sum(), x, retain_graph=True)


@pytest.mark.parametrize("name", ["qk_norm_rope", "dropout_add", "token_log_probs", "linear_fp8", "kept weights",
                                  "kept weights residual"])
def test_tangents_are_refused(name):
    import torch.autograd.forward_ad as fwd
    x, w, nw, r = torch.randn(8, 64), torch.randn(24, 64), torch.ones(16), torch.zeros(8, 24)
    cos, sin = ops.precompute_rope_cache(16, 8, 10000.0)
    kept = ops.quantize_fp8(w, square=True)
    f, t = {"qk_norm_rope": (lambda x: ops.qk_norm_rope(x, nw, nw, cos, sin, 2, 1, 16, 8), x),
            "dropout_add": (lambda x: ops.dropout_add(x, None, 0.3, 5), x),
            "token_log_probs": (lambda x: ops.token_log_probs(x, torch.arange(8)).logprob, x),
            "linear_fp8": (lambda x: ops.linear_fp8(x, w), x),
            "kept weights": (lambda x: ops.linear_fp8(x, kept), x),
            "kept weights residual": (lambda r: ops.linear_fp8(x, kept, residual=r), r)}[name]
    with fwd.dual_level():
        with pytest.raises((RuntimeError, ValueError)):
            f(fwd.make_dual(t, torch.ones_like(t)))
        assert f(t).shape[0] == 8


@pytest.mark.parametrize("grad,x_grad,w_grad,main,sets", [
    (True, True, True, False, 4), (True, False, True, False, 3), (True, True, False, False, 3), (True, True, False, True, 3),
    (False, True, True, False, 2), (False, True, False, True, 2), (True, False, False, False, 2)])
def test_transposed_codes_are_made_for_a_backward_alone(grad, x_grad, w_grad, main, sets, monkeypatch):
    from build_your_own_distributed_training_b200.ops import fp8
    made, inner = [], fp8._quantize
    monkeypatch.setattr(fp8, "_quantize", lambda x, square, plain, t: made.append(plain + t) or inner(x, square, plain, t))
    x, w = torch.randn(8, 64).requires_grad_(x_grad), torch.randn(24, 64).requires_grad_(w_grad)
    with torch.set_grad_enabled(grad):
        ops.linear_fp8(x, w, main_grad=torch.zeros(24, 64) if main else None)
    assert sum(made) == sets


@pytest.mark.parametrize("main", [True, False])
def test_the_engine_route_keeps_no_copy_of_the_weight(main):
    """The sharding engine frees gathered weights between forward and backward; codes of them would stay."""
    x, w = torch.randn(8, 256).requires_grad_(True), torch.randn(384, 256).requires_grad_(not main)
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = ops.linear_fp8(x, w, main_grad=torch.zeros(384, 256) if main else None)
    extra = sum(t.numel() * t.element_size() for t in kept if t.data_ptr() not in (x.data_ptr(), w.data_ptr()))
    codes = w.numel()
    assert extra < codes if main else extra >= codes
    y.sum().backward()


@pytest.mark.parametrize("dt", [torch.int64, torch.int32])
def test_positions_outside_the_tables_give_nan(dt):
    cos, sin = ops.precompute_rope_cache(16, 8, 10000.0)
    x, w = torch.randn(5, 64).requires_grad_(True), torch.ones(16)
    pos = torch.tensor([-1, 0, 8, 7, -9], dtype=dt)
    y = ops.qk_norm_rope(x, w, w, cos, sin, 2, 1, 16, 1, positions=pos)
    bad = torch.tensor([True, False, True, False, True])
    assert y[bad][:, :48].isnan().all() and torch.equal(y[bad][:, 48:], x[bad][:, 48:]) and y[~bad].isfinite().all()
    good = ops.qk_norm_rope(x[~bad], w, w, cos, sin, 2, 1, 16, 1, positions=pos[~bad])
    assert torch.equal(y[~bad], good)
    g, = torch.autograd.grad(y.nan_to_num(0.0).sum(), x)
    assert g[~bad].isfinite().all()


def test_products_and_codes_do_not_drop_gradients():
    """fp8_matmul and quantize_fp8 are no autograd operations: a residual that wants its gradient is refused."""
    import torch.autograd.forward_ad as fwd
    w = torch.randn(24, 64, requires_grad=True)
    a, b = ops.quantize_fp8(torch.randn(8, 64)), ops.quantize_fp8(w, square=True)
    assert not b.values.requires_grad and not b.scales.requires_grad and not b.dequantize().requires_grad
    r = torch.zeros(8, 24, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="linear_fp8"):
        ops.fp8_matmul(a, b, residual=r)
    with pytest.raises(ValueError, match="linear_fp8"):
        ops.fp8_matmul(a, b, out=r * 1.0)
    with fwd.dual_level(), pytest.raises(ValueError, match="linear_fp8"):
        ops.fp8_matmul(a, b, residual=fwd.make_dual(r.detach(), torch.ones_like(r)))
    want = ops.fp8_matmul(a, b)
    assert not want.requires_grad
    with torch.no_grad():
        assert torch.equal(ops.fp8_matmul(a, b, residual=r), want)


@pytest.mark.parametrize("temperature", [1e-46, 1e-40, 2.0 ** -127, 2.0 ** 127, 1e39, float("inf")])
def test_temperatures_whose_reciprocal_fp32_cannot_hold_are_refused(temperature):
    x, tok = torch.randn(3, 40), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature"):
        ops.token_log_probs(x, tok, temperature=temperature)
    for t in (2.0 ** -126, 2.0 ** 126):  # the ends: all on the maximum, and uniform
        x[:, 5] = -float("inf")
        r = ops.token_log_probs(x, tok, temperature=t)
        n = 1 if t < 1 else 39
        assert float((r.entropy - torch.log(torch.tensor(float(n)))).abs().max()) < 2.0 ** -18 and not r.logprob.isnan().any()
