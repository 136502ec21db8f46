"""8-bit block-scaled matrices and linear layers on the CPU path."""

from __future__ import annotations

import pytest
import torch

from build_your_own_distributed_training_b200 import ops
from build_your_own_distributed_training_b200.ops import grad_state
from tests import plain_ops as plain
from tests.plain_ops import rel

F32 = 64 * 2.0 ** -24


@pytest.mark.parametrize("R,C", [(1, 1), (3, 128), (130, 129), (128, 256), (257, 40)])
@pytest.mark.parametrize("square", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_quantize_matches_definition(R, C, square, dt):
    g = torch.Generator().manual_seed(R + C)
    x = (torch.randn(R, C, generator=g) * torch.exp2(torch.randint(-30, 30, (R, 1), generator=g).float())).to(dt)
    x[0, 0] = 448.0  # a largest magnitude that is exactly a power of two times 448
    b = ops.quantize_fp8(x, square=square)
    want, scales = plain.fp8_round(x, 128 if square else 1)
    assert torch.equal(b.dequantize().double(), want) and torch.equal(b.scales.float().double(), scales)
    assert b.rows_per_scale in (1, 128)


def test_quantize_zeros_small_and_non_finite():
    x = torch.zeros(4, 256)
    x[1, 3] = 2.0 ** -120
    x[2, 5], x[3, 200] = float("inf"), float("nan")
    b = ops.quantize_fp8(x)
    s = b.scales.view(torch.uint8)
    assert s[0].tolist() == [19, 19] and s[1, 0] == 19 and s[2].tolist() == [255, 19] and s[3].tolist() == [19, 255]
    d = b.dequantize()
    assert (d[0] == 0).all() and d[2, :128].isnan().all() and (d[2, 128:] == 0).all() and d[3, 128:].isnan().all()


@pytest.mark.parametrize("main", [False, True])
def test_linear_matches_formula(main):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 70, 200, generator=g).requires_grad_(True)
    w = torch.randn(150, 200, generator=g).requires_grad_(True)
    r = torch.randn(3, 70, 150, generator=g).requires_grad_(True)
    dy = torch.randn(3, 70, 150, generator=g)
    mg = None
    if main:
        mg = torch.full((150 * 200,), float("nan"))
        fresh = grad_state.FreshSet(mg)
        fresh.mark([(0, mg.numel())])
        mg = grad_state.tag(mg, fresh, 0)
    y = ops.linear_fp8(x, w, residual=r, main_grad=mg)
    y.backward(dy)
    x2, d2 = x.detach().view(-1, 200), dy.view(-1, 150)
    wq = plain.fp8_round(w.detach(), 128)[0]
    want = plain.fp8_round(x2, 1)[0] @ wq.t() + r.detach().double().view(-1, 150)
    assert rel(y.view(-1, 150), want) < F32
    assert rel(x.grad.view(-1, 200), plain.fp8_round(d2, 1)[0] @ wq) < F32
    dw = plain.fp8_round(d2.t().contiguous(), 1)[0] @ plain.fp8_round(x2.t().contiguous(), 1)[0].t()
    assert rel(mg.view(150, 200) if main else w.grad, dw) < F32
    assert torch.equal(r.grad, dy)
    if main:
        ops.linear_fp8(x, w, main_grad=mg).backward(dy)
        assert rel(mg.view(150, 200), 2 * dw) < F32


def test_linear_with_kept_weights():
    x, w = torch.randn(5, 200), torch.randn(33, 200)
    b = ops.quantize_fp8(w, square=True)
    assert torch.equal(ops.linear_fp8(x, b), ops.linear_fp8(x, w))
    with pytest.raises(ValueError, match="no backward"):
        ops.linear_fp8(x.requires_grad_(True), b)
    with torch.no_grad():
        ops.linear_fp8(x, b)


def test_refusals():
    x, w = torch.randn(4, 64), torch.randn(8, 64)
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w)
    with pytest.raises(ValueError, match="features"):
        ops.linear_fp8(x[:, :60], w)
    with pytest.raises(ValueError, match="residual"):
        ops.linear_fp8(x, w, residual=torch.zeros(4, 7))
    with pytest.raises(ValueError, match="summed axes"):
        ops.fp8_matmul(a, ops.quantize_fp8(torch.randn(8, 32)))
    with pytest.raises(ValueError, match="fit neither"):
        ops.fp8_matmul(ops.Fp8Blocks(a.values, a.scales[:3]), b)
    with pytest.raises(ValueError, match="e4m3"):
        ops.fp8_matmul(ops.Fp8Blocks(x, a.scales), b)
    with pytest.raises(ValueError, match="accumulate"):
        ops.fp8_matmul(a, b, accumulate=True)
    with pytest.raises(ValueError, match="matrix"):
        ops.quantize_fp8(torch.zeros(3))
    with pytest.raises(ValueError, match="fp32, bf16"):
        ops.quantize_fp8(torch.zeros(3, 3, dtype=torch.int32))
