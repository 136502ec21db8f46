"""The block operators inside the bf16 model on the GPU."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU boxes, skipped by marker
    pytest.skip("needs a GPU", allow_module_level=True)

from build_your_own_distributed_training_b200.config import ModelConfig, ParallelConfig  # noqa: E402
from build_your_own_distributed_training_b200.models import TransformerBlock, build_model, set_fp8_linear  # noqa: E402
from build_your_own_distributed_training_b200.ops._ext import native  # noqa: E402
from build_your_own_distributed_training_b200.ops.linear import swiglu_packed  # noqa: E402
from build_your_own_distributed_training_b200.ops.rope import precompute_rope_cache, rope_packed  # noqa: E402
from build_your_own_distributed_training_b200.parallel.fsdp import FullyShardedModel  # noqa: E402
from tests.plain_ops import rel  # noqa: E402

DEV = torch.device("cuda", 0)
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    assert native().device_error() == 0


def _engines(fp8: bool, drop: float):
    """The same weights as a bf16 engine on the GPU and as an fp32 module on the CPU."""
    torch.manual_seed(0)
    mc = ModelConfig(vocab_size=512, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_hidden_size=512,
                     max_seq_len=128, tie_embeddings=False, qk_norm=True, resid_dropout=drop)
    ref, model = build_model(mc), build_model(mc)
    model.load_state_dict(ref.state_dict())
    for m in (ref, model):
        set_fp8_linear(m, fp8)
    eng = FullyShardedModel(model, None, ParallelConfig(), {TransformerBlock}, device=DEV)
    model.rope_cos, model.rope_sin = model.rope_cos.to(DEV), model.rope_sin.to(DEV)
    model.return_logits = False
    return eng, ref


@pytest.mark.parametrize("fp8,drop", [(False, 0.0), (False, 0.2), (True, 0.0), (True, 0.2)])
def test_training_step_and_scoring_match_cpu(fp8, drop):
    eng, ref = _engines(fp8, drop)
    g = torch.Generator().manual_seed(1)
    x = torch.randint(0, 512, (3, 100), generator=g)
    y = torch.randint(0, 512, (3, 100), generator=g)
    y[:, :9] = -100
    torch.manual_seed(4)
    r = eng(x.to(DEV), targets=y.to(DEV), top_k=4)
    loss = -r.logprob.sum() / 273 - 0.1 * r.entropy.sum() / 273
    loss.backward()
    torch.manual_seed(4)
    c = ref(x, targets=y, top_k=4)
    want = -c.logprob.sum() / 273 - 0.1 * c.entropy.sum() / 273
    want.backward()
    # bf16 activations through two blocks; the logits' spread is about 0.3
    assert abs(float(loss.detach()) - float(want.detach())) < 0.01
    assert float((r.logprob.cpu() - c.logprob).abs().max()) < 0.1
    for (n, p), (_, q) in zip(eng.module.named_parameters(), ref.named_parameters()):
        if q.grad is not None:
            # some dozens of bf16 roundings, or roundings to 4 bits that fall differently on inputs that
            # differ in their last bf16 bit
            assert rel(p.main_grad, q.grad) < (0.15 if fp8 else 0.06), n
    _, a = eng(x.to(DEV), labels=y.to(DEV))
    assert a.isfinite()


def test_packed_rotation_and_swiglu():
    g = torch.Generator(device=DEV).manual_seed(0)
    cos, sin = (t.to(DEV) for t in precompute_rope_cache(64, 50, 10000.0))
    y = torch.randn(100, 4 * 64, device=DEV, generator=g).to(BF).requires_grad_(True)
    d = torch.randn(100, 4 * 64, device=DEV, generator=g).to(BF)
    out = rope_packed(y, cos, sin, 3 * 64, 64, 50)
    out.backward(d)
    c, s = cos.double().repeat(2, 1)[:, None, :32], sin.double().repeat(2, 1)[:, None, :32]
    yd = y.detach().double().view(100, 4, 64).requires_grad_(True)
    lo, hi = yd[:, :3, :32], yd[:, :3, 32:]
    want = torch.cat((torch.cat((lo * c - hi * s, hi * c + lo * s), -1), yd[:, 3:]), 1).reshape(100, -1)
    want.backward(d.double())
    assert rel(out, want) < 2.0 ** -8 and rel(y.grad, yd.grad.view(100, -1)) < 2.0 ** -8
    for ffn in (64, 37):
        gu = (torch.randn(30, 2 * ffn, device=DEV, generator=g) * 2).to(BF).requires_grad_(True)
        da = torch.randn(30, ffn, device=DEV, generator=g).to(BF)
        act = swiglu_packed(gu, ffn)
        gd = gu.detach().double().requires_grad_(True)
        ref = torch.nn.functional.silu(gd[:, :ffn]) * gd[:, ffn:]
        assert rel(act, ref) < 2.0 ** -8
        if ffn % 2 == 0:  # the backward kernel takes even widths
            act.backward(da)
            ref.backward(da.double())
            assert rel(gu.grad, gd.grad) < 2.0 ** -8


def test_policy_example_learns():
    import examples.policy_step as ex
    shares = ex.main(["--steps", "10"])
    assert shares[-1] > 0.9 > shares[0]
