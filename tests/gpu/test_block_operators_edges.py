"""Block operators' kernels on the calls at the edge of what they take: single rows, odd vocabularies, no eps, wrong
scales, second derivatives, tangents, calls without gradients."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes, skipped by marker
    pytest.skip("needs a GPU", allow_module_level=True)

from build_your_own_distributed_training_b200 import ops  # noqa: E402
from build_your_own_distributed_training_b200.ops._ext import native  # noqa: E402
from tests import plain_ops as plain  # noqa: E402
from tests.plain_ops import UNIT, rel  # noqa: E402

DEV = torch.device("cuda", 0)
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert native().device_error() == 0


def _randn(*shape, seed=0, dt=F32):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dt)


@pytest.mark.parametrize("nq,nkv,hd", [(5, 1, 80), (1, 1, 128), (7, 3, 16), (3, 2, 34)])
@pytest.mark.parametrize("dt", [F32, BF, HF])
def test_qk_norm_rope_without_eps(nq, nkv, hd, dt):
    """Lane groups past the last head hold zeros, whose 1 / rms is infinite without eps."""
    tokens, W = 11, (nq + 2 * nkv) * hd
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(hd, tokens, 10000.0))
    x = (_randn(tokens, W, seed=hd) * 2).to(dt).requires_grad_(True)
    wq, wk = (_randn(hd, seed=i, dt=dt).requires_grad_(True) for i in (1, 2))
    dy = _randn(tokens, W, seed=3, dt=dt)
    y = ops.qk_norm_rope(x, wq, wk, cos, sin, nq, nkv, hd, tokens, 0.0)
    y.backward(dy)
    xd, qd, kd = (t.detach().double().requires_grad_(True) for t in (x, wq, wk))
    ref = plain.qk_norm_rope(xd, qd, kd, cos, sin, nq, nkv, hd, list(range(tokens)), 0.0)
    ref.backward(dy.double())
    # fp32 arithmetic (some tens of 2^-24; the weights' gradients sum terms of either sign) and one rounding
    unit = 0.0 if dt == F32 else UNIT[dt]
    assert rel(y, ref) < 2.0 ** -18 + unit and rel(x.grad, xd.grad) < 2.0 ** -18 + unit
    assert rel(wq.grad, qd.grad) < 2.0 ** -14 + unit and rel(wk.grad, kd.grad) < 2.0 ** -14 + unit


@pytest.mark.parametrize("V", [5, 2001, 32003])
@pytest.mark.parametrize("main", [False, True])
def test_scoring_head_takes_any_vocabulary(V, main, monkeypatch):
    from build_your_own_distributed_training_b200.ops import logprobs as mod
    monkeypatch.setattr(mod, "HEAD_BYTES", 128 * 4 * V)  # blocks of 128 rows
    M, d, k = 150, 256, min(V, 3)
    h = _randn(M, d, seed=1, dt=BF).requires_grad_(True)
    w = (_randn(V, d, seed=2) * 0.1).to(BF).requires_grad_(not main)
    tok = torch.randint(0, V, (M,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(3))
    tok[::7] = -100
    mg = torch.ones(V, d, device=DEV) if main else None
    r = ops.lm_head_token_log_probs(h, w, tok, top_k=k, main_grad=mg)
    hd, wd = h.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    lp, ent = plain.logprobs(hd @ wd.t(), tok)
    # fp32 logits: no rounding to bf16 before the log probabilities
    assert float((r.logprob.double() - lp).abs().max()) < 2.0 ** -16 and float((r.entropy.double() - ent).abs().max()) < 2.0 ** -16
    live = tok != -100
    assert (r.top_tokens[live] >= 0).all() and (r.top_tokens[live] < V).all() and (r.top_tokens[~live] == -1).all()
    (r.logprob.sum() - 0.1 * r.entropy.sum()).backward()
    (lp.sum() - 0.1 * ent.sum()).backward()
    # the logit gradient is rounded to bf16 between the two products, the results once more
    assert rel(h.grad, hd.grad) < 2 * UNIT[BF] and rel(mg - 1 if main else w.grad, wd.grad) < 2 * UNIT[BF]


def test_scoring_head_refusals_and_no_rows():
    w, tok = _randn(64, 32, dt=BF), torch.zeros(4, device=DEV, dtype=torch.int64)
    with pytest.raises(ValueError, match="bf16"):
        ops.lm_head_token_log_probs(_randn(4, 32), w, tok)
    with pytest.raises(ValueError, match="bf16"):
        ops.lm_head_token_log_probs(_randn(4, 32, dt=BF), w.float(), tok)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.lm_head_token_log_probs(_randn(4, 30, dt=BF), w[:, :30].contiguous(), tok)
    h, wg = _randn(0, 32, dt=BF).requires_grad_(True), w.clone().requires_grad_(True)
    for V in (64, 61):
        h.grad = wg.grad = None
        r = ops.lm_head_token_log_probs(h, wg[:V], tok[:0], top_k=2)
        assert r.logprob.shape == (0,) and r.logprob.dtype == F32 and r.top_tokens.shape == (0, 2)
        (r.logprob.sum() + r.entropy.sum()).backward()
        assert h.grad.shape == (0, 32) and (wg.grad == 0).all()


def test_model_with_an_odd_vocabulary_scores():
    from build_your_own_distributed_training_b200.config import ModelConfig, ParallelConfig
    from build_your_own_distributed_training_b200.models import TransformerBlock, build_model
    from build_your_own_distributed_training_b200.parallel.fsdp import FullyShardedModel
    torch.manual_seed(0)
    mc = ModelConfig(vocab_size=509, d_model=128, n_layers=1, n_heads=2, n_kv_heads=1, ffn_hidden_size=256,
                     max_seq_len=64, tie_embeddings=False)
    ref, model = build_model(mc), build_model(mc)
    model.load_state_dict(ref.state_dict())
    eng = FullyShardedModel(model, None, ParallelConfig(), {TransformerBlock}, device=DEV)
    model.rope_cos, model.rope_sin = model.rope_cos.to(DEV), model.rope_sin.to(DEV)
    x, y = torch.randint(0, 509, (2, 2, 50), generator=torch.Generator().manual_seed(1))
    r, c = eng(x.to(DEV), targets=y.to(DEV), top_k=2), ref(x, targets=y, top_k=2)
    # bf16 activations through one block; the logits' spread is about 0.3
    assert float((r.logprob.cpu() - c.logprob).abs().max()) < 0.1
    (-r.logprob.sum() / 100 - 0.1 * r.entropy.sum() / 100).backward()
    (-c.logprob.sum() / 100 - 0.1 * c.entropy.sum() / 100).backward()
    for (n, p), (_, q) in zip(eng.module.named_parameters(), ref.named_parameters()):
        assert rel(p.main_grad, q.grad) < 0.06, n  # some dozens of bf16 roundings


@pytest.mark.parametrize("K", [1, 15, 130, 300])
def test_single_rows_of_codes_with_any_row_length(K):
    tight = lambda b: ops.Fp8Blocks(torch.empty(b.values.shape, device=DEV, dtype=b.values.dtype).copy_(b.values),  # noqa: E731
                                    b.scales)
    one, many = ops.quantize_fp8(_randn(1, K, seed=1, dt=BF)), ops.quantize_fp8(_randn(40, K, seed=2, dt=BF))
    for a, b in ((one, many), (many, one), (one, one)):
        want = ops.fp8_matmul(a, b, out_dtype=F32)
        assert tight(one).values.stride(0) == K
        for x, y in ((tight(a), tight(b)), (tight(a), b), (a, tight(b))):
            assert torch.equal(ops.fp8_matmul(x, y, out_dtype=F32), want)
    x, w = _randn(5, K, seed=3, dt=BF), ops.quantize_fp8(_randn(1, K, seed=4), square=True)
    assert torch.equal(ops.linear_fp8(x, tight(w)), ops.linear_fp8(x, w))


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("square", [False, True])
def test_kept_weights_with_wrong_scales_are_refused(T, square):
    N, K = 200, 1000
    x, b = _randn(T, K, dt=BF), ops.quantize_fp8(_randn(N, K, seed=1), square=square)
    s = b.scales
    wide = torch.cat((s.view(torch.uint8), s.view(torch.uint8)[:, :1]), 1).view(s.dtype)
    a = ops.quantize_fp8(x)
    wrong = [s[:, :5], s[:, :7], wide, s[:1], s[:, 0]]
    for bad in wrong:
        for tiles in (None, b.tiles):
            with pytest.raises(ValueError, match="scales"):
                ops.linear_fp8(x, ops.Fp8Blocks(b.values, bad, tiles))
        with pytest.raises(ValueError, match="scales"):
            native().linear_fp8_kept(x, b.values, bad, None, None)
        with pytest.raises(ValueError, match="scales"):
            native().fp8_product(a.values, a.scales, None, b.values, bad, None, torch.empty(T, N, device=DEV), None, False)
    with pytest.raises(ValueError, match="e4m3"):
        ops.linear_fp8(x, ops.Fp8Blocks(b.values.float(), s))


@pytest.mark.parametrize("T", [1, 5, 64, 127, 128, 300])
@pytest.mark.parametrize("N,K", [(22016, 512), (100, 4096), (515, 640), (64, 130)])
@pytest.mark.parametrize("square", [False, True])
def test_kept_weights_without_tiles(T, N, K, square):
    """Weights given as codes and scales alone: the tiles are made in the call."""
    x, b = _randn(T, K, seed=T, dt=BF), ops.quantize_fp8(_randn(N, K, seed=9), square=square)
    want = ops.linear_fp8(x, b)
    assert torch.equal(ops.linear_fp8(x, ops.Fp8Blocks(b.values, b.scales)), want)
    # codes in tight rows, scales stored the other way round
    turned = b.scales.view(torch.uint8).t().contiguous().t().view(b.scales.dtype)
    assert torch.equal(ops.linear_fp8(x, ops.Fp8Blocks(b.values.contiguous(), turned)), want)
    r = _randn(T, N, seed=5, dt=BF)
    assert torch.equal(ops.linear_fp8(x, ops.Fp8Blocks(b.values, b.scales), residual=r), ops.linear_fp8(x, b, residual=r))


def _cases():
    """(name, call, differentiated inputs): each operator as a program calls it."""
    from build_your_own_distributed_training_b200.ops.linear import swiglu_packed
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(16, 8, 10000.0))
    x, w = _randn(8, 64, seed=1, dt=BF), _randn(24, 64, seed=2, dt=BF)
    nw, tok = _randn(16, seed=3, dt=BF), torch.arange(8, device=DEV)
    grads = lambda *n: [torch.zeros(m, device=DEV) for m in n]  # noqa: E731
    qk = lambda **kw: lambda x, w: ops.qk_norm_rope(x, w, w, cos, sin, 2, 1, 16, 8, **kw)  # noqa: E731
    lp = lambda r: r.logprob * 2 + r.entropy  # noqa: E731
    return {
        "qk_norm_rope": (qk(), (x, nw)),
        "qk_norm_rope main_grads": (qk(main_grads=grads(16, 16)), (x, nw)),
        "token_log_probs": (lambda x: lp(ops.token_log_probs(x, tok)), (x,)),
        "lm_head_token_log_probs": (lambda x, w: lp(ops.lm_head_token_log_probs(x, w, tok)), (x, w)),
        "linear_fp8": (lambda x, w: ops.linear_fp8(x, w), (x, w)),
        "linear_fp8 main_grad": (lambda x, w: ops.linear_fp8(x, w, main_grad=grads(24 * 64)[0]), (x, w)),
        "swiglu_packed": (lambda x: swiglu_packed(x, 32), (x,)),
    }


@pytest.mark.parametrize("name", ["qk_norm_rope", "qk_norm_rope main_grads", "token_log_probs", "lm_head_token_log_probs",
                                  "linear_fp8", "linear_fp8 main_grad", "swiglu_packed"])
def test_second_derivatives_are_refused(name):
    f, args = _cases()[name]
    args = [a.clone().requires_grad_(True) for a in args]
    first = torch.autograd.grad(f(*args).float().sum(), args, allow_unused=True)
    again = torch.autograd.grad(f(*args).float().sum(), args, create_graph=True, allow_unused=True)
    for a, b in zip(first, again):
        assert (a is None) == (b is None)
        if a is not None:
            assert torch.equal(a, b.detach())
            # a term that is added to others must not vanish
            with pytest.raises(RuntimeError, match="second derivative"):
                torch.autograd.grad((b.float().sum() + args[0].float().pow(2).sum()), args[0], retain_graph=True)


def test_second_derivatives_of_linear_operators():
    from build_your_own_distributed_training_b200.ops.rope import rope_packed
    x = _randn(6, 64, seed=1).requires_grad_(True)
    m = ops.dropout_add(torch.ones_like(x), None, 0.3, 5)
    xd = x.detach().double().requires_grad_(True)
    for f, g, z in ((lambda t: ops.dropout_add(t, t * 2, 0.3, 5), lambda t: t * 2 + t * m.double(), x),):
        a, = torch.autograd.grad(f(z).pow(3).sum(), z, create_graph=True)
        b, = torch.autograd.grad(g(xd).pow(3).sum(), xd, create_graph=True)
        v = _randn(6, 64, seed=2)
        assert rel(torch.autograd.grad((a * v).sum(), z)[0], torch.autograd.grad((b * v.double()).sum(), xd)[0]) < 2.0 ** -20
    cos, sin = (t.to(DEV) for t in ops.precompute_rope_cache(16, 3, 10000.0))
    z, v = x.detach().to(BF).requires_grad_(True), _randn(6, 64, seed=2, dt=BF)
    zd = z.detach().double().requires_grad_(True)

    def turn(t):
        u = t.view(2, 3, 4, 16)
        c, s = cos.double()[None, :, None, :8], sin.double()[None, :, None, :8]
        lo, hi = u[:, :, :3, :8], u[:, :, :3, 8:]
        return torch.cat((torch.cat((lo * c - hi * s, hi * c + lo * s), -1), u[:, :, 3:]), 2).reshape(6, 64)
    a, = torch.autograd.grad(rope_packed(z, cos, sin, 48, 16, 3).float().pow(3).sum(), z, create_graph=True)
    b, = torch.autograd.grad(turn(zd).pow(3).sum(), zd, create_graph=True)
    got, = torch.autograd.grad((a.float() * v.float()).sum(), z)
    want, = torch.autograd.grad((b * v.double()).sum(), zd)
    # four bf16 roundings on the way, one of a factor that the cube's derivative doubles
    assert rel(got, want) < 6 * UNIT[BF]


@pytest.mark.parametrize("name", ["qk_norm_rope", "qk_norm_rope main_grads", "token_log_probs", "lm_head_token_log_probs",
                                  "linear_fp8", "linear_fp8 main_grad", "swiglu_packed", "dropout_add", "residual", "kept weights",
                                  "kept weights residual"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, grad):
    """Forward-mode differentiation has no kernels here; a tangent must not get lost on the way."""
    import torch.autograd.forward_ad as fwd
    x, w, r = _randn(8, 64, seed=1, dt=BF), ops.quantize_fp8(_randn(24, 64, seed=2), square=True), _randn(8, 24, dt=BF)
    cases = dict(_cases(), **{"dropout_add": (lambda x: ops.dropout_add(x, None, 0.3, 5), (x,)),
                              "residual": (lambda x: ops.dropout_add(x.detach(), x, 0.3, 5), (x,)),
                              "kept weights": (lambda x: ops.linear_fp8(x, w), (x,)),
                              "kept weights residual": (lambda r: ops.linear_fp8(x, w, residual=r), (r,))})
    f, args = cases[name]
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        duals = [fwd.make_dual(a, torch.ones_like(a)) for a in args]
        with pytest.raises((RuntimeError, ValueError)):
            f(*duals)
        plain_call = f(*args)  # without tangents the same call goes through
        assert plain_call.shape[0] == 8


@pytest.mark.parametrize("route", ["plain", "main_grad"])
def test_a_call_without_gradients_makes_one_set_of_codes(route):
    """The transposed codes serve the backward only."""
    T, N, K = 2048, 512, 4096
    x, w = _randn(T, K, seed=1, dt=BF).requires_grad_(True), _randn(N, K, seed=2, dt=BF).requires_grad_(True)
    kw = {"main_grad": torch.zeros(N, K, device=DEV)} if route == "main_grad" else {}
    want = ops.linear_fp8(x, w, **kw).detach()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    with torch.no_grad():
        y = ops.linear_fp8(x, w, **kw)
    peak = torch.cuda.max_memory_allocated() - before
    assert torch.equal(y, want) and not y.requires_grad
    # the codes once, the result, the scales (a 128th of the codes, up to twice as tiles), allocations in 2 MB steps at most
    assert peak < T * K + N * K + 2 * T * N + (T + N) * K // 32 + (2 << 20)


def test_products_and_codes_do_not_drop_gradients():
    """fp8_matmul and quantize_fp8 are no autograd operations: a residual that wants its gradient is refused."""
    import torch.autograd.forward_ad as fwd
    w = torch.randn(24, 64, device=DEV, requires_grad=True)
    a, b = ops.quantize_fp8(torch.randn(8, 64, device=DEV)), ops.quantize_fp8(w, square=True)
    assert not b.values.requires_grad and not b.scales.requires_grad and not b.dequantize().requires_grad
    r = torch.zeros(8, 24, device=DEV, dtype=torch.bfloat16, requires_grad=True)
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
    x, tok = torch.randn(3, 40, device=DEV), torch.zeros(3, device=DEV, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature"):
        ops.token_log_probs(x, tok, temperature=temperature)
    for t in (2.0 ** -126, 2.0 ** 126):  # the ends: all on the maximum, and uniform
        x[:, 5] = -float("inf")
        r = ops.token_log_probs(x, tok, temperature=t)
        n = 1 if t < 1 else 39
        assert float((r.entropy - torch.log(torch.tensor(float(n)))).abs().max()) < 2.0 ** -18 and not r.logprob.isnan().any()


def test_native_log_probs_refuse_such_temperatures():
    x, tok = torch.randn(3, 40, device=DEV), torch.zeros(3, device=DEV, dtype=torch.int64)
    for t in (0.0, 1e-40, float("inf"), float("nan")):
        with pytest.raises(RuntimeError, match="temperature"):
            native().token_logprobs(x, tok, t, 0, -100)


@pytest.mark.parametrize("T,ffn", [(1, 1), (30, 37), (129, 1001)])
def test_packed_swiglu_of_an_odd_width(T, ffn):
    from build_your_own_distributed_training_b200.ops.linear import swiglu_packed
    gu = (_randn(T, 2 * ffn, seed=1) * 2).to(BF).requires_grad_(True)
    da = _randn(T, ffn, seed=2, dt=BF)
    act = swiglu_packed(gu, ffn)
    act.backward(da)
    gd = gu.detach().double().requires_grad_(True)
    ref = torch.nn.functional.silu(gd[:, :ffn]) * gd[:, ffn:]
    ref.backward(da.double())
    # fp32 arithmetic and one rounding
    assert rel(act, ref) < UNIT[BF] + 2.0 ** -18 and rel(gu.grad, gd.grad) < UNIT[BF] + 2.0 ** -18


@pytest.mark.parametrize("ffn", [64, 38, 37])
@pytest.mark.parametrize("off", [1, 2, 8])
def test_packed_swiglu_of_tensors_off_the_vector_grid(ffn, off):
    from build_your_own_distributed_training_b200.ops.linear import swiglu_backward, swiglu_packed
    T = 21
    shifted = lambda t: torch.empty(t.numel() + off, device=DEV, dtype=BF)[off:].view(t.shape).copy_(t)  # noqa: E731
    gu, da = (_randn(T, 2 * ffn, seed=1) * 2).to(BF), _randn(T, ffn, seed=2, dt=BF)
    want = swiglu_backward(da, gu, ffn)
    assert torch.equal(swiglu_packed(shifted(gu), ffn), swiglu_packed(gu, ffn))
    for a, b in ((shifted(da), gu), (da, shifted(gu)), (shifted(da), shifted(gu))):
        assert torch.equal(swiglu_backward(a, b, ffn), want)


def test_8_bit_model_of_an_odd_width_trains():
    from build_your_own_distributed_training_b200.config import ModelConfig, ParallelConfig
    from build_your_own_distributed_training_b200.models import TransformerBlock, build_model, set_fp8_linear
    from build_your_own_distributed_training_b200.parallel.fsdp import FullyShardedModel
    torch.manual_seed(0)
    mc = ModelConfig(vocab_size=512, d_model=128, n_layers=1, n_heads=2, n_kv_heads=1, ffn_hidden_size=301,
                     max_seq_len=64, tie_embeddings=False)
    ref, model = set_fp8_linear(build_model(mc)), set_fp8_linear(build_model(mc))
    model.load_state_dict(ref.state_dict())
    eng = FullyShardedModel(model, None, ParallelConfig(), {TransformerBlock}, device=DEV)
    model.rope_cos, model.rope_sin = model.rope_cos.to(DEV), model.rope_sin.to(DEV)
    model.return_logits = False
    x, y = torch.randint(0, 512, (2, 3, 50), generator=torch.Generator().manual_seed(1))
    _, a = eng(x.to(DEV), labels=y.to(DEV))
    a.backward()
    _, b = ref(x, labels=y)
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) < 0.01
    for (n, p), (_, q) in zip(eng.module.named_parameters(), ref.named_parameters()):
        assert rel(p.main_grad, q.grad) < 0.15, n  # roundings to 4 bits that fall differently


def test_packed_rotation_refuses_tables_it_cannot_read():
    from build_your_own_distributed_training_b200.ops.rope import rope_packed
    cos, sin = ops.precompute_rope_cache(16, 8, 10000.0)
    x, c, s = _randn(16, 64, dt=BF), cos.to(DEV), sin.to(DEV)
    for args in ((cos, sin, 48, 16, 8),                   # tables on the host
                 (c[:4], s[:4], 48, 16, 8),               # fewer rows than positions
                 (c.double(), s.double(), 48, 16, 8),
                 (c[:, :8].contiguous(), s[:, :8].contiguous(), 48, 16, 8),
                 (c, s, 80, 16, 8), (c, s, 40, 16, 8)):   # columns past the rows, half a head
        with pytest.raises(RuntimeError, match="rope"):
            rope_packed(x, *args)
    assert rope_packed(x, c, s, 48, 16, 8).isfinite().all()
    assert rope_packed(x[:4], c[:4], s[:4], 48, 16, 8).isfinite().all()  # four tokens read four rows


@pytest.mark.parametrize("score", [False, True])
def test_recomputed_blocks_give_the_same_gradients(score):
    """Activation checkpointing runs a block again in its backward: same kernels, inputs and seeds, same bits."""
    from build_your_own_distributed_training_b200.config import ModelConfig, ParallelConfig
    from build_your_own_distributed_training_b200.models import TransformerBlock, build_model, set_fp8_linear
    from build_your_own_distributed_training_b200.parallel.fsdp import FullyShardedModel, apply_activation_checkpointing
    x, y = torch.randint(0, 512, (2, 2, 64), generator=torch.Generator().manual_seed(1)).to(DEV)
    seen = []
    for ckpt in (False, True):
        torch.manual_seed(0)
        model = set_fp8_linear(build_model(ModelConfig(
            vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_hidden_size=512, max_seq_len=64,
            tie_embeddings=False, qk_norm=True, resid_dropout=0.2)))
        if ckpt:
            apply_activation_checkpointing(model, {TransformerBlock})
        eng = FullyShardedModel(model, None, ParallelConfig(), {TransformerBlock}, device=DEV)
        model.rope_cos, model.rope_sin = model.rope_cos.to(DEV), model.rope_sin.to(DEV)
        model.return_logits = False
        eng.train()
        torch.manual_seed(3)
        loss = -eng(x, targets=y).logprob.mean() if score else eng(x, labels=y)[1]
        loss.backward()
        seen.append([loss.detach()] + [p.main_grad.clone() for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*seen))
