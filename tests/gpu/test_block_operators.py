"""Block operators' kernels against plain 64-bit implementations, at the sizes and masks where they can go wrong."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes, skipped by marker
    pytest.skip("needs a GPU", allow_module_level=True)

from build_your_own_distributed_training_b200 import ops  # noqa: E402
from build_your_own_distributed_training_b200.ops import grad_state  # noqa: E402
from build_your_own_distributed_training_b200.ops._ext import native  # noqa: E402
from build_your_own_distributed_training_b200.ops.logprobs import lm_head_token_log_probs  # noqa: E402
from tests import plain_ops as plain  # noqa: E402
from tests.plain_ops import UNIT, rel  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def tol(dt: torch.dtype, f32: float = 2.0 ** -18) -> float:
    """fp32 arithmetic (some tens of 2^-24) and one rounding to the storage type, whose relative error
    is at most its unit."""
    return f32 + (UNIT[dt] if dt != F32 else 0.0)


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert native().device_error() == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------------ QK norm + rotation
@pytest.mark.parametrize("nq,nkv,hd,tokens,seqlen", [
    (32, 8, 128, 1, 1), (32, 8, 128, 300, 100), (12, 4, 64, 77, 77), (5, 1, 80, 33, 11), (4, 4, 16, 130, 65),
    (2, 1, 256, 9, 9), (3, 3, 34, 21, 7), (2, 2, 512, 5, 5), (1, 1, 2, 3, 3), (3, 1, 48, 2000, 1000)])
@pytest.mark.parametrize("dt", [F32, BF, HF])
def test_qk_norm_rope(nq, nkv, hd, tokens, seqlen, dt):
    g = _gen(hd + tokens)
    W = (nq + 2 * nkv) * hd
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(hd, max(seqlen, 64), 10000.0))
    x = (torch.randn(tokens, W, device=DEV, generator=g) * 2).to(dt).requires_grad_(True)
    wq, wk = ((torch.randn(hd, device=DEV, generator=g)).to(dt).requires_grad_(True) for _ in range(2))
    dy = torch.randn(tokens, W, device=DEV, generator=g).to(dt)
    y = ops.qk_norm_rope(x, wq, wk, cos, sin, nq, nkv, hd, seqlen, 1e-5)
    y.backward(dy)
    xd, qd, kd = (t.detach().double().requires_grad_(True) for t in (x, wq, wk))
    ref = plain.qk_norm_rope(xd, qd, kd, cos, sin, nq, nkv, hd, [i % seqlen for i in range(tokens)], 1e-5)
    ref.backward(dy.double())
    assert y.dtype == dt and rel(y, ref) < tol(dt) and rel(x.grad, xd.grad) < tol(dt)
    # sums over tokens and heads of terms of either sign
    assert rel(wq.grad, qd.grad) < tol(dt, 2.0 ** -14) and rel(wk.grad, kd.grad) < tol(dt, 2.0 ** -14)


@pytest.mark.parametrize("off,pitch", [(0, 1024), (8, 1032), (3, 1029)])
@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("i32", [False, True])
def test_qk_norm_rope_strides_and_positions(off, pitch, dt, i32):
    nq, nkv, hd, tokens = 8, 2, 64, 50
    W = (nq + 2 * nkv) * hd
    g = _gen(off + pitch)
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(hd, 4096, 10000.0))
    base = torch.randn(tokens * pitch + off, device=DEV, generator=g).to(dt)
    x = base.as_strided((tokens, W), (pitch, 1), off)
    pos = torch.randint(0, 4096, (tokens,), device=DEV, generator=g, dtype=torch.int32 if i32 else torch.int64)
    w = torch.ones(hd, device=DEV)
    xg = x.detach().requires_grad_(True)
    y = ops.qk_norm_rope(xg, w, w, cos, sin, nq, nkv, hd, 1, 1e-6, positions=pos)
    dy = torch.randn(W, device=DEV, generator=g).to(dt).expand(tokens, W)  # a broadcast gradient: row stride 0
    y.backward(dy)
    xd = x.double().contiguous().requires_grad_(True)
    ref = plain.qk_norm_rope(xd, w.double(), w.double(), cos, sin, nq, nkv, hd, pos.tolist(), 1e-6)
    ref.backward(dy.double())
    assert rel(y, ref) < tol(dt) and rel(xg.grad, xd.grad) < tol(dt)


def test_qk_norm_rope_main_grads_accumulate_and_repeat():
    nq, nkv, hd, tokens = 4, 2, 128, 700
    W = (nq + 2 * nkv) * hd
    g = _gen(1)
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(hd, tokens, 10000.0))
    x = torch.randn(tokens, W, device=DEV, generator=g).to(BF).requires_grad_(True)
    w = torch.ones(hd, device=DEV, dtype=BF, requires_grad=True)
    dy = torch.randn(tokens, W, device=DEV, generator=g).to(BF)
    buf = torch.full((2 * hd,), 7.0, device=DEV)
    fresh = grad_state.FreshSet(buf)
    fresh.mark([(0, hd), (hd, hd)])
    mgs = tuple(grad_state.tag(buf[i * hd:(i + 1) * hd], fresh, i * hd) for i in range(2))
    seen = []
    for _ in range(3):
        y = ops.qk_norm_rope(x, w, w, cos, sin, nq, nkv, hd, tokens, 1e-5, main_grads=mgs)
        y.backward(dy)
        seen.append(buf.clone())
    assert w.grad is None and float(seen[0].abs().max()) > 0
    assert torch.equal(seen[1], seen[0] + seen[0])  # the same bits again, added
    one = ops.qk_norm_rope(x, w, w, cos, sin, nq, nkv, hd, tokens, 1e-5)
    dw, = torch.autograd.grad(one, w, dy)
    assert rel(dw, (seen[0][:hd] + seen[0][hd:])) < 2 * UNIT[BF]


def test_qk_norm_rope_empty_zero_rows_and_bad_position():
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(64, 8, 10000.0))
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.zeros(0, 256, device=DEV, requires_grad=True)
    y = ops.qk_norm_rope(x, w, w, cos, sin, 2, 1, 64, 1)
    y.sum().backward()
    assert y.shape == (0, 256) and (w.grad == 0).all()
    z = torch.zeros(3, 256, device=DEV, requires_grad=True)
    y = ops.qk_norm_rope(z, w, w, cos, sin, 2, 1, 64, 8)
    y.sum().backward()
    assert (y == 0).all() and z.grad.isfinite().all()
    bad = ops.qk_norm_rope(torch.ones(2, 256, device=DEV), w, w, cos, sin, 2, 1, 64, 1,
                           positions=torch.tensor([1, 8], device=DEV))
    assert bad[0].isfinite().all() and bad[1, :192].isnan().all() and (bad[1, 192:] == 1).all()
    assert native().device_error() == 3
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(x, w.double(), w.double(), cos, sin, 2, 1, 64, 1)
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope(torch.zeros(4, 256, device=DEV), w, w, cos[:, :32].contiguous(), sin, 2, 1, 64, 1)
    with pytest.raises(RuntimeError):  # more positions than table rows
        ops.qk_norm_rope(torch.zeros(20, 256, device=DEV), w, w, cos, sin, 2, 1, 64, 20)


def test_qk_norm_rope_on_another_stream():
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(64, 512, 10000.0))
    w = torch.ones(64, device=DEV)
    x = torch.randn(512, 256, device=DEV)
    want = ops.qk_norm_rope(x, w, w, cos, sin, 2, 1, 64, 512)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        z = x * 1.0
        got = ops.qk_norm_rope(z, w, w, cos, sin, 2, 1, 64, 512)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (5, 9), (64, 129), (33, 4, 16)])
@pytest.mark.parametrize("start", [0, 8, 5, (1 << 35) + 3])
@pytest.mark.parametrize("dt", [F32, BF, HF])
def test_dropout_add(shape, start, dt):
    g = _gen(len(shape) + shape[0])
    x = torch.randn(shape, device=DEV, generator=g).to(dt).requires_grad_(True)
    r = torch.randn(shape, device=DEV, generator=g).to(dt).requires_grad_(True)
    dy = torch.randn(shape, device=DEV, generator=g).to(dt)
    for p, seed in ((0.1, 3), (0.5, (1 << 64) - 7), (0.0, 1), (1.0, 2)):
        for res in (r, None):
            x.grad = r.grad = None
            y = ops.dropout_add(x, res, p, seed, start=start)
            y.backward(dy)
            rd = None if res is None else r.detach().double().cpu()
            want = plain.dropout_add(x.detach().double().cpu(), rd, p, seed, start)
            back = plain.dropout_add(dy.double().cpu(), None, p, seed, start)
            assert rel(y, want) < tol(dt) and rel(x.grad, back) < tol(dt)
            assert torch.equal(x.grad.cpu() == 0, back == 0)
            assert res is None or torch.equal(r.grad, dy)


def test_dropout_layouts_and_large_counts():
    x = torch.randn(64, 40, device=DEV, dtype=BF)
    whole = ops.dropout_add(x, x, 0.3, 9)
    # a transposed input, a base off the 16-byte grid, and a broadcast gradient give the same elements
    assert torch.equal(ops.dropout_add(x.t().contiguous().t(), x, 0.3, 9), whole)
    pad = torch.empty(64 * 40 + 1, device=DEV, dtype=BF)[1:].view(64, 40)
    pad.copy_(x)
    assert torch.equal(ops.dropout_add(pad, pad, 0.3, 9), whole)
    z = x.clone().requires_grad_(True)
    ops.dropout_add(z, None, 0.3, 9).sum().backward()
    assert torch.equal(z.grad != 0, ops.dropout_add(torch.ones_like(x), None, 0.3, 9) != 0)
    # a dropped infinity or NaN is gone
    bad = torch.full((4096,), INF, device=DEV)
    y = ops.dropout_add(bad, torch.zeros_like(bad), 0.5, 4)
    assert ((y == 0) | (y == INF)).all() and (y == 0).any()
    # element numbers past 2^32 inside one call: the tail of a split activation
    s = (1 << 32) - 20
    assert torch.equal((ops.dropout_add(torch.ones(64, device=DEV), None, 0.5, 11, start=s) != 0).cpu(),
                       plain.keep_mask(64, 0.5, 11, s))
    assert ops.dropout_add(torch.empty(0, 5, device=DEV), None, 0.5, 1).shape == (0, 5)


# ------------------------------------------------------------------------------------------ token log probabilities
def _rows(M, V, dt, seed, masked=0.0):
    g = _gen(seed)
    x = torch.randn(M, V, device=DEV, generator=g) * 3
    if masked:
        x.masked_fill_(torch.rand(M, V, device=DEV, generator=g) < masked, -INF)
    tok = torch.randint(0, V, (M,), device=DEV, generator=g)
    x[torch.arange(M, device=DEV), tok] = 2.0
    return x.to(dt), tok


@pytest.mark.parametrize("M,V,k", [(1, 128256, 20), (3, 32003, 32), (1, 1, 1), (5, 31, 31), (2, 4097, 1), (300, 700, 5),
                                   (17, 16400, 0), (40, 50304, 8), (1, 9000, 2)])
@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("temperature,masked", [(1.0, 0.0), (0.7, 0.6)])
def test_token_log_probs(M, V, k, dt, temperature, masked):
    x, tok = _rows(M, V, dt, M + V, masked)
    if M > 2:
        tok[1] = -100
    x = x.requires_grad_(True)
    r = ops.token_log_probs(x, tok, temperature=temperature, top_k=k)
    xd = x.detach().double().requires_grad_(True)
    lp, ent = plain.logprobs(xd, tok, temperature)
    g = _gen(2)
    a, b = torch.randn(M, device=DEV, generator=g), torch.randn(M, device=DEV, generator=g)
    # each value is a difference of terms of up to ~ 40 / temperature, computed in fp32
    at = 64 / temperature * 2.0 ** -24
    assert float((r.logprob.double() - lp).abs().max()) < at * 4
    assert float((r.entropy.double() - ent).abs().max()) < at * 4
    if k:
        rows = x.detach().double().cpu().tolist() if V < 40000 else None
        order = torch.sort(x.detach().double(), dim=1, descending=True, stable=True)[1][:, :k]
        want = torch.where((tok == -100)[:, None], -1, order)
        assert torch.equal(r.top_tokens, want)
        if rows is not None and tok[0] != -100:
            assert r.top_tokens[0].tolist() == plain.top_order(rows[0], k)
        live = tok != -100
        got, ref = r.top_logprobs[live].double(), (xd.detach() / temperature - torch.logsumexp(
            xd.detach() / temperature, 1, keepdim=True)).gather(1, order)[live]
        assert torch.equal(got.isinf(), ref.isinf())
        assert float((got - ref)[ref.isfinite()].abs().max()) < at * 4
    (r.logprob * a + r.entropy * b).sum().backward()
    (lp * a.double() + ent * b.double()).sum().backward()
    err = (x.grad.double() - xd.grad).abs()
    # probabilities to some 2^-20, factors g_H (ln p + H) of up to ~ 100, and the storage type's rounding
    assert float((err - UNIT[dt] * xd.grad.abs()).max()) < 100 * 2.0 ** -20 / temperature + (2.0 ** -24 if dt == HF else 0)
    assert (x.grad[tok == -100] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("order", ["equal", "up", "down", "one thread", "all masked but one", "lowest"])
@pytest.mark.parametrize("V", [1000, 20001])
def test_token_log_probs_top_order(dt, order, V):
    """Rows in which the largest elements lie as badly as they can for a strided reader."""
    k = 32
    x = torch.zeros(2, V, device=DEV)
    if order == "up":
        x += torch.arange(V, device=DEV) // 64
    elif order == "down":
        x -= torch.arange(V, device=DEV) // 64
    elif order == "one thread":
        x[:, ::512] = 3.0
        x[:, 1::512] = 5.0
    elif order == "all masked but one":
        x.fill_(-INF)
        x[:, V // 2] = 1.0
    elif order == "lowest":
        x.fill_(torch.finfo(dt).min)
    x = x.to(dt)
    tok = torch.full((2,), V // 2, device=DEV)
    r = ops.token_log_probs(x, tok, top_k=k, temperature=0.5)
    want = torch.sort(x.float(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(r.top_tokens, want)
    lp, ent = plain.logprobs(x.double(), tok, 0.5)
    assert float((r.logprob.double() - lp).abs().max()) <= 2.0 ** -16 * (1 + float(lp.abs().max()))
    assert float((r.entropy.double() - ent).abs().max()) < 2.0 ** -14


@pytest.mark.parametrize("off,pitch", [(0, 1003), (3, 1024), (1, 1001)])
@pytest.mark.parametrize("dt", [F32, BF])
def test_token_log_probs_strides(off, pitch, dt):
    M, V = 9, 1000
    base = (torch.randn(M * pitch + off, device=DEV, generator=_gen(off)) * 3).to(dt)
    x = base.as_strided((M, V), (pitch, 1), off)
    tok = torch.randint(0, V, (M,), device=DEV)
    xs = x.detach().requires_grad_(True)
    xc = x.contiguous().requires_grad_(True)
    a, b = ops.token_log_probs(xs, tok, top_k=4), ops.token_log_probs(xc, tok, top_k=4)
    # where vectors start differs, and with it the order of the sums
    assert torch.allclose(a.logprob, b.logprob, atol=2.0 ** -18, rtol=0) and torch.equal(a.top_tokens, b.top_tokens)
    (a.logprob.sum() + a.entropy.sum()).backward()
    (b.logprob.sum() + b.entropy.sum()).backward()
    assert float((xs.grad.float() - xc.grad.float()).abs().max()) < 2.0 ** -15 + (UNIT[dt] * 2 if dt == BF else 0)
    y = x.t().contiguous().t()  # columns apart: taken as a copy
    assert torch.equal(ops.token_log_probs(y, tok).logprob, b.logprob)


@pytest.mark.parametrize("V", [300, 20000, 70001])
def test_token_log_probs_edge_rows(V):
    x = torch.randn(8, V, device=DEV, generator=_gen(V))
    x[0] = -INF
    x[1, 5] = -INF
    x[2, V - 1] = INF
    x[3, V // 2] = float("nan")
    tok = torch.tensor([0, 5, 1, 0, V, -1, -100, 3], device=DEV)
    x[6] = float("nan")
    x.requires_grad_(True)
    r = ops.token_log_probs(x, tok, top_k=3)
    assert native().device_error() == 3  # tokens outside the vocabulary
    assert r.logprob[0] == -INF and r.entropy[0] == 0 and r.top_tokens[0].tolist() == [0, 1, 2]
    assert r.logprob[1] == -INF and r.entropy[1] > 0
    assert r.logprob[2:6].isnan().all() and r.entropy[2:6].isnan().all() and (r.top_tokens[2:6] == -1).all()
    assert r.logprob[6] == 0 and r.entropy[6] == 0 and (r.top_tokens[6] == -1).all()
    assert r.logprob[7].isfinite()
    g, = torch.autograd.grad((r.logprob, r.entropy), x, (torch.ones(8, device=DEV), torch.ones(8, device=DEV)))
    assert (g[0] == 0).all() and g[1].isfinite().all() and g[2:6].isnan().all() and (g[6] == 0).all()
    assert g[7].isfinite().all()


def test_token_log_probs_one_gradient_empty_and_repeats():
    x, tok = _rows(64, 5000, F32, 1)
    x.requires_grad_(True)
    g1, = torch.autograd.grad(ops.token_log_probs(x, tok).logprob.sum(), x)
    g2, = torch.autograd.grad(ops.token_log_probs(x, tok).entropy.sum(), x)
    p = torch.softmax(x.detach().double(), 1)
    assert float((g1 + p).gather(1, tok[:, None]).sub(1).abs().max()) < 2.0 ** -18
    ent = -(p * p.log()).sum(1, keepdim=True)
    assert float((g2 + p * (p.log() + ent)).abs().max()) < 2.0 ** -16
    a, b = ops.token_log_probs(x, tok, top_k=7), ops.token_log_probs(x, tok, top_k=7)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    e = ops.token_log_probs(torch.empty(0, 10, device=DEV), torch.empty(0, device=DEV, dtype=torch.int64), top_k=2)
    assert e.logprob.shape == (0,) and e.top_tokens.shape == (0, 2)


def test_lm_head_token_log_probs(monkeypatch):
    from build_your_own_distributed_training_b200.ops import logprobs as mod
    monkeypatch.setattr(mod, "HEAD_BYTES", 128 * 4 * 2000)  # three blocks of rows
    g = _gen(5)
    h = torch.randn(300, 256, device=DEV, generator=g).to(BF).requires_grad_(True)
    w = (torch.randn(2000, 256, device=DEV, generator=g) * 0.1).to(BF).requires_grad_(True)
    tok = torch.randint(0, 2000, (300,), device=DEV, generator=g)
    tok[::7] = -100
    r = lm_head_token_log_probs(h, w, tok, top_k=3)
    hd, wd = h.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    lp, ent = plain.logprobs(hd @ wd.t(), tok)
    assert float((r.logprob.double() - lp).abs().max()) < 2.0 ** -16 and float((r.entropy.double() - ent).abs().max()) < 2.0 ** -16
    (r.logprob.sum() - 0.1 * r.entropy.sum()).backward()
    (lp.sum() - 0.1 * ent.sum()).backward()
    # the logit gradient is rounded to bf16 between the two products, the results once more
    assert rel(h.grad, hd.grad) < 2 * UNIT[BF] and rel(w.grad, wd.grad) < 2 * UNIT[BF]
    mg = torch.ones(2000, 256, device=DEV)
    r = lm_head_token_log_probs(h, w.detach(), tok, main_grad=mg)
    (r.logprob.sum() - 0.1 * r.entropy.sum()).backward()
    assert rel(mg - 1, wd.grad) < 2 * UNIT[BF]
