"""The block operators inside the model: normalised heads, residual dropout, 8-bit projections, token scoring."""

from __future__ import annotations

import copy

import pytest
import torch

from build_your_own_distributed_training_b200.config import KernelConfig, TrainingConfig
from build_your_own_distributed_training_b200.models import build_model, set_fp8_linear
from build_your_own_distributed_training_b200.models.transformer import TransformerBlock
from build_your_own_distributed_training_b200.parallel.fsdp import apply_activation_checkpointing
from build_your_own_distributed_training_b200.parallel.process_groups import build_process_context
from build_your_own_distributed_training_b200.parallel.tensor_parallel import apply_tensor_parallelism
from build_your_own_distributed_training_b200.training.trainer import build_engine
from tests._dist_utils import run_distributed
from tests.helpers import tiny_config


def _batch(n=3):
    g = torch.Generator().manual_seed(1)
    t = torch.randint(0, 256, (n, 33), generator=g)
    return t[:, :-1], t[:, 1:]


def _tiny(**over):
    cfg = tiny_config(**{f"model__{k}": v for k, v in over.items()})
    torch.manual_seed(0)
    m = build_model(cfg.model)
    for n, p in m.named_parameters():  # head norms other than one, so that they matter
        if n.endswith(("q_norm.weight", "k_norm.weight")):
            torch.nn.init.normal_(p, 1.0, 0.3)
    return cfg, m


def test_defaults_keep_parameters_and_results():
    _, m = _tiny()
    assert not any("q_norm" in n or "k_norm" in n for n, _ in m.named_parameters())
    cfg = TrainingConfig()
    assert cfg.model.qk_norm is False and cfg.model.resid_dropout == 0.0 and cfg.kernels == KernelConfig()
    state = torch.get_rng_state()
    m.train()
    x, y = _batch()
    m(x, labels=y)
    assert torch.equal(state, torch.get_rng_state())  # no seed is drawn without dropout


def test_head_norm_gradients_against_differences():
    _, m = _tiny(qk_norm=True)
    x, y = _batch()
    _, loss = m(x, labels=y)
    loss.backward()
    for name in ("q_norm", "k_norm"):
        w = getattr(m.layers[0].attention, name).weight
        v = torch.randn(w.shape, generator=torch.Generator().manual_seed(2))
        with torch.no_grad():
            h, vals = 1e-2, []
            for s in (h, -2 * h):
                w.add_(s * v)
                vals.append(float(m(x, labels=y)[1]))
            w.add_(h * v)
        want = (vals[0] - vals[1]) / (2 * h)
        # fp32 losses of about 5.5 leave the difference some 2^-22 / h; its curvature adds h^2
        assert abs(float((w.grad * v).sum()) - want) < 2e-4


def test_residual_dropout_and_recompute():
    _, m = _tiny(resid_dropout=0.2, qk_norm=True)
    x, y = _batch()
    m.eval()
    plain = float(m(x, labels=y)[1])
    m.train()
    torch.manual_seed(5)
    _, a = m(x, labels=y)
    a.backward()
    grads = {n: p.grad.clone() for n, p in m.named_parameters()}
    assert abs(float(a.detach()) - plain) > 1e-6
    # recomputed blocks draw the same seeds
    r = copy.deepcopy(m)
    r.zero_grad()
    apply_activation_checkpointing(r, {TransformerBlock})
    torch.manual_seed(5)
    _, b = r(x, labels=y)
    b.backward()
    assert torch.equal(a, b)
    for n, p in r.named_parameters():
        assert torch.allclose(p.grad, grads[n], atol=1e-6), n
    torch.manual_seed(6)
    assert not torch.equal(m(x, labels=y)[1], a)


def _tp_worker(rank, world, sp, drop, fp8):
    over = {"model__qk_norm": True, "model__resid_dropout": drop, "parallel__tp_size": 2,
            "parallel__sequence_parallel": sp, "kernels__fp8_linear": fp8}
    cfg = tiny_config(**over)
    ctx = build_process_context(2, backend="gloo", verbose=False)
    cfg.validate(ctx.world_size, ctx.dims.dp_size, 2)
    eng = build_engine(cfg, ctx)
    torch.manual_seed(cfg.seed)
    ref = build_model(cfg.model)
    ref.train()
    eng.train()
    x, y = _batch(2)
    torch.manual_seed(9)
    _, a = eng(x, labels=y)
    a.backward()
    torch.manual_seed(9)
    _, b = ref(x, labels=y)
    b.backward()
    if fp8:  # the reference is not in 8 bits: e4m3 keeps 4 bits of each operand
        assert abs(float(a) - float(b)) < 0.05
        return
    assert abs(float(a) - float(b)) < 1e-5
    from build_your_own_distributed_training_b200.training.grad_utils import sharded_total_norm
    want = float(torch.sqrt(sum(p.grad.pow(2).sum() for p in ref.parameters())))
    assert abs(float(sharded_total_norm(eng)) - want) / want < 1e-4
    for i, blk in enumerate(eng.module.layers):
        for name in ("q_norm", "k_norm"):
            got = getattr(blk.attention, name).weight.main_grad
            exp = getattr(ref.layers[i].attention, name).weight.grad
            assert torch.allclose(got, exp, atol=1e-5), (i, name)


@pytest.mark.parametrize("sp,drop,fp8", [(False, 0.0, False), (True, 0.0, False), (False, 0.3, False), (True, 0.3, False),
                                         (True, 0.0, True), (False, 0.0, True)])
def test_tensor_parallel_matches_one_process(sp, drop, fp8):
    run_distributed(_tp_worker, 2, sp, drop, fp8)


def test_fp8_projections_approximate_the_model():
    _, m = _tiny(qk_norm=True)
    x, y = _batch()
    _, a = m(x, labels=y)
    a.backward()
    grads = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    set_fp8_linear(m)
    _, b = m(x, labels=y)
    b.backward()
    assert 0 < abs(float(a.detach()) - float(b.detach())) < 0.02
    for n, p in m.named_parameters():
        # three or more roundings to 4 significant bits lie between the loss and any weight
        assert float((p.grad - grads[n]).norm() / grads[n].norm()) < 0.25, n
    set_fp8_linear(m, False)
    assert torch.equal(m(x, labels=y)[1], a)


def test_scoring_is_the_loss_per_token():
    _, m = _tiny()
    x, y = _batch()
    y = y.clone()
    y[:, :4] = -100
    r = m(x, targets=y, top_k=3)
    _, loss = m(x, labels=y)
    assert r.logprob.shape == y.shape and r.top_tokens.shape == (*y.shape, 3)
    assert abs(float(-r.logprob.sum() / (y != -100).sum()) - float(loss)) < 1e-5
    (-r.logprob.sum() / (y != -100).sum()).backward()
    g = {n: p.grad.clone() for n, p in m.named_parameters()}
    m.zero_grad()
    loss.backward()
    for n, p in m.named_parameters():
        assert torch.allclose(p.grad, g[n], atol=1e-6), n
    with pytest.raises(ValueError, match="not both"):
        m(x, labels=y, targets=y)


def _score_refuses(rank, world):
    cfg = tiny_config(parallel__tp_size=2, parallel__sequence_parallel=True)
    ctx = build_process_context(2, backend="gloo", verbose=False)
    torch.manual_seed(0)
    m = build_model(cfg.model)
    apply_tensor_parallelism(m, ctx.tp_group, sequence_parallel=True)
    x, y = _batch(2)
    with pytest.raises(NotImplementedError, match="sequence_parallel"):
        m(x, targets=y)


def test_scoring_refuses_split_tokens():
    run_distributed(_score_refuses, 2)


def test_config_refuses():
    for over, what in (({"model__resid_dropout": 1.0}, "resid_dropout"), ({"model__resid_dropout": -0.1}, "resid_dropout"),
                       ({"kernels__fp8_linear": True, "model__mlp_bias": True}, "bias")):
        with pytest.raises(ValueError, match=what):
            tiny_config(**over).validate(1, 1, 1)
    with pytest.raises(ValueError, match="bias"):
        cfg = tiny_config(model__mlp_bias=True)
        set_fp8_linear(build_model(cfg.model))


def test_policy_example_learns():
    import examples.policy_step as ex
    shares = ex.main(["--cpu", "--steps", "6"])
    assert shares[-1] > 0.9 > shares[0]
