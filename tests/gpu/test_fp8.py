"""8-bit block-scaled kernels against plain 64-bit implementations and the CPU path."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes, skipped by marker
    pytest.skip("needs a GPU", allow_module_level=True)

from build_your_own_distributed_training_b200 import ops  # noqa: E402
from build_your_own_distributed_training_b200.ops import fp8, grad_state  # noqa: E402
from build_your_own_distributed_training_b200.ops._ext import native  # noqa: E402
from tests import plain_ops as plain  # noqa: E402
from tests.plain_ops import UNIT, rel  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16
# fp32 accumulation of up to 2^14 exact products of either sign: the error of a sum grows like the square
# root of the terms, some 2^7 roundings of 2^-24
ACC = 2.0 ** -17


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert native().device_error() == 0


def _rand(r, c, seed, dt=BF, spread=12):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(r, c, device=DEV, generator=g)
    return (x * torch.exp2(torch.randint(-spread, spread + 1, (r, 1), device=DEV, generator=g).float())).to(dt)


def _same(a: ops.Fp8Blocks, b: ops.Fp8Blocks) -> bool:
    u8 = lambda t: t.cpu().contiguous().view(torch.uint8)  # noqa: E731
    return torch.equal(u8(a.values), u8(b.values)) and torch.equal(u8(a.scales), u8(b.scales))


@pytest.mark.parametrize("R,C", [(1, 1), (1, 4096), (3, 130), (127, 128), (128, 129), (129, 777), (300, 1000), (2000, 24)])
@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("square", [False, True])
def test_quantize_gives_the_defined_codes(R, C, dt, square):
    """The codes are exact by definition: every bit equals the CPU path's, as they lie and transposed."""
    x = _rand(R, C, R + C, dt, 6)
    rows = 128 if square else 1
    a, at = fp8._quantize(x, square, True, True)
    assert _same(a, fp8._quantize_cpu(x.float().cpu(), rows))
    assert _same(at, fp8._quantize_cpu(x.float().cpu().t(), rows))
    assert _same(fp8._quantize(x, square, True, False)[0], a) and _same(fp8._quantize(x, square, False, True)[1], at)
    if R * C < 50000:
        assert torch.equal(a.dequantize().double().cpu(), plain.fp8_round(x, rows)[0])


def test_quantize_strides_and_edges():
    base = torch.randn(200 * 301 + 5, device=DEV).to(BF)
    x = base.as_strided((200, 300), (301, 1), 3)
    assert _same(ops.quantize_fp8(x), ops.quantize_fp8(x.contiguous()))
    assert _same(ops.quantize_fp8(x.t()), ops.quantize_fp8(x.t().contiguous()))
    z = torch.zeros(4, 256, device=DEV)
    z[1, 3], z[2, 5], z[3, 200] = 2.0 ** -120, float("inf"), float("nan")
    for square in (False, True):
        for got, want in zip(fp8._quantize(z, square, True, True), fp8._quantize(z.cpu(), square, True, True)):
            assert torch.equal(got.scales.cpu().contiguous().view(torch.uint8), want.scales.contiguous().view(torch.uint8))
            assert torch.equal(got.dequantize().cpu().nan_to_num(7.0), want.dequantize().nan_to_num(7.0))
    e = ops.quantize_fp8(torch.empty(0, 300, device=DEV))
    assert e.values.shape == (0, 300) and e.scales.shape == (0, 3)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 4096), (7, 16, 129), (8, 130, 11008), (17, 33, 520), (64, 4096, 96),
                                   (65, 257, 100), (128, 256, 128), (300, 1000, 1000), (1000, 40, 3000), (2500, 4096, 384),
                                   (129, 24, 40000)])
@pytest.mark.parametrize("ga,gb", [(False, True), (False, False), (True, True)])
def test_matmul(M, N, K, ga, gb):
    a, b = ops.quantize_fp8(_rand(M, K, M), square=ga), ops.quantize_fp8(_rand(N, K, N + 1), square=gb)
    want = a.dequantize().double() @ b.dequantize().double().t()
    y = ops.fp8_matmul(a, b, out_dtype=F32)
    # by rows: the scales of the rows differ by many powers of two
    err = (y.double() - want).norm(dim=1) / want.norm(dim=1).clamp_min(1e-300)
    assert float(err.max()) < ACC
    h = ops.fp8_matmul(a, b)
    assert h.dtype == BF and rel(h, want) < ACC + UNIT[BF]
    r = torch.randn(M, N, device=DEV).to(BF)
    assert rel(ops.fp8_matmul(a, b, residual=r), want + r.double()) < ACC + UNIT[BF]
    acc = torch.ones(M, N, device=DEV)
    ops.fp8_matmul(a, b, out=acc, accumulate=True)
    # adding 1 to rows that are far smaller keeps the sum's roundings, not the product's
    assert float((acc.double() - 1 - want).abs().max()) < 2 * ACC * float(want.abs().max() + 1)
    assert torch.equal(ops.fp8_matmul(a, b, out_dtype=F32), y)


@pytest.mark.parametrize("M", [3, 40, 200])
def test_matmul_layouts(M):
    N, K = 72, 300
    x, w = _rand(M, K, 1), _rand(N, K, 2)
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w, square=True)
    want = ops.fp8_matmul(a, b)
    # codes whose rows do not start on 16 bytes, scales stored the other way round
    tight = lambda t: ops.Fp8Blocks(t.values.contiguous(), t.scales.contiguous())  # noqa: E731
    assert torch.equal(ops.fp8_matmul(tight(a), tight(b)), want)
    # a result with wider rows and an odd base, a residual with others
    out = torch.zeros(M, 200, device=DEV, dtype=BF)[:, 3:3 + N]
    ops.fp8_matmul(a, b, out=out)
    assert torch.equal(out, want)
    res = torch.randn(M, 99, device=DEV).to(BF)[:, :N]
    got = ops.fp8_matmul(a, b, residual=res)
    assert rel(got, ops.fp8_matmul(a, b, out_dtype=F32).double() + res.double()) < UNIT[BF] + ACC


def test_matmul_non_finite_and_empty():
    x, w = torch.randn(40, 256, device=DEV).to(BF), torch.randn(300, 256, device=DEV).to(BF)
    x[3, 7], w[150, 200] = float("nan"), float("inf")
    for M in (4, 40):
        y = ops.linear_fp8(x[:M], w)
        # the weight's 128 x 128 block is lost with its infinity, the activation's row with its NaN
        assert y[3].isnan().all() and y[:, 128:256].isnan().all()
        keep = torch.ones(M, dtype=torch.bool)
        keep[3] = False
        assert y[keep][:, :128].isfinite().all() and y[keep][:, 256:].isfinite().all()
    e = ops.linear_fp8(torch.empty(0, 256, device=DEV, dtype=BF), w)
    assert e.shape == (0, 300)
    z = ops.fp8_matmul(ops.quantize_fp8(torch.empty(5, 0, device=DEV)), ops.quantize_fp8(torch.empty(6, 0, device=DEV)))
    assert (z == 0).all() and z.shape == (5, 6)


@pytest.mark.parametrize("T,N,K", [(1, 48, 256), (70, 150, 200), (300, 1000, 770), (1024, 512, 2048)])
@pytest.mark.parametrize("wdt", [F32, BF])
@pytest.mark.parametrize("main", [False, True])
def test_linear_training(T, N, K, wdt, main):
    x = _rand(T, K, 1, spread=2).requires_grad_(True)
    w = _rand(N, K, 2, wdt, 2).requires_grad_(True)
    r = _rand(T, N, 3, spread=2).requires_grad_(True)
    dy = _rand(T, N, 4, spread=2)
    mg = None
    if main:
        buf = torch.full((N * K,), float("nan"), device=DEV)
        fresh = grad_state.FreshSet(buf)
        fresh.mark([(0, N * K)])
        mg = grad_state.tag(buf, fresh, 0)
    y = ops.linear_fp8(x, w, residual=r, main_grad=mg)
    y.backward(dy)
    deq = lambda t, square=False: ops.quantize_fp8(t.detach(), square=square).dequantize().double()  # noqa: E731
    wq = deq(w, True)
    assert rel(y, deq(x) @ wq.t() + r.detach().double()) < ACC + UNIT[BF]
    assert rel(x.grad, deq(dy) @ wq) < ACC + UNIT[BF]
    dw = deq(dy.t().contiguous()) @ deq(x.t().contiguous()).t()
    assert rel(mg.view(N, K) if main else w.grad, dw) < ACC + (0 if main else UNIT[wdt])
    assert torch.equal(r.grad, dy) and (main or w.grad.dtype == wdt)
    # the gradient of the rounded product approximates that of the exact one: e4m3 keeps 4 bits, so each
    # operand is within 2^-4 of itself, in the mean about 2^-5
    assert rel(x.grad, dy.double() @ w.detach().double()) < 2 * 2.0 ** -4
    if main:
        assert w.grad is None
        ops.linear_fp8(x, w, main_grad=mg).backward(dy)
        assert rel(mg.view(N, K), 2 * dw) < 2 * ACC


@pytest.mark.parametrize("T", [1, 5, 8, 9, 16, 40, 64, 65, 200])
@pytest.mark.parametrize("N,K", [(22016, 512), (100, 4096), (515, 640), (64, 130)])
def test_linear_with_kept_weights(T, N, K):
    x, w = _rand(T, K, T), _rand(N, K, 9, spread=3)
    b = ops.quantize_fp8(w, square=True)
    y = ops.linear_fp8(x.view(1, T, K), b)
    want = ops.quantize_fp8(x).dequantize().double() @ b.dequantize().double().t()
    err = (y[0].double() - want).norm(dim=1) / want.norm(dim=1)
    assert y.shape == (1, T, N) and float(err.max()) < ACC + UNIT[BF]
    with torch.no_grad():
        assert torch.equal(ops.linear_fp8(x, w), y[0])


def test_refusals():
    x, w = _rand(4, 64, 1), _rand(8, 64, 2)
    with pytest.raises(ValueError, match="bf16"):
        ops.linear_fp8(x.float(), w)
    a, b = ops.quantize_fp8(x), ops.quantize_fp8(w)
    out = torch.empty(4, 8, device=DEV)
    for bad in ((a.values, a.tiles, b.values, b.tiles, out.half(), None, False),       # result type
                (a.values, a.tiles, b.values[:, :60], b.tiles, out, None, False),      # shapes
                (a.values, a.tiles[:, :, :256], b.values, b.tiles, out, None, False),  # scale tiles
                (a.values, a.tiles, b.values, b.tiles, out.to(BF), None, True)):       # bf16 accumulation
        with pytest.raises(RuntimeError):
            native().fp8_gemm(*bad)
    with pytest.raises(RuntimeError):
        native().fp8_scale_tiles(a.scales, 2, 4)


def test_kept_weights_on_another_stream_and_repeats():
    x, w = _rand(300, 1024, 1), _rand(512, 1024, 2)
    b = ops.quantize_fp8(w, square=True)
    want = ops.linear_fp8(x, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.linear_fp8(x * 1.0, b) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, want) for g in got)
