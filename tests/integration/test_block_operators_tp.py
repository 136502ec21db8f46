"""Gradients of the 8-bit projections split over tensor-parallel ranks."""

from __future__ import annotations

import pytest
import torch

from build_your_own_distributed_training_b200.models import build_model, set_fp8_linear
from build_your_own_distributed_training_b200.parallel.process_groups import build_process_context
from build_your_own_distributed_training_b200.training.trainer import build_engine
from tests._dist_utils import run_distributed
from tests.helpers import tiny_config
from tests.plain_ops import rel

# A split sum moves the next layer's inputs by some 2^-22, which flips the rounding to 4 bits of a few of its
# 16 k elements and more; each flip moves its element by 2^-4 at most, 2^-11 of the whole, and through two blocks
# some dozens of them are allowed for.
TOL = 2.0 ** -7


def _worker(rank, world, sp, qk):
    # every rank's rows and columns are whole blocks of 128, so its codes are those of the whole matrices
    cfg = tiny_config(model__d_model=256, model__n_heads=4, model__n_kv_heads=4, model__ffn_hidden_size=512,
                      model__qk_norm=qk, parallel__tp_size=2, parallel__sequence_parallel=sp, kernels__fp8_linear=True)
    ctx = build_process_context(2, backend="gloo", verbose=False)
    cfg.validate(ctx.world_size, ctx.dims.dp_size, 2)
    eng = build_engine(cfg, ctx)
    torch.manual_seed(cfg.seed)
    ref = set_fp8_linear(build_model(cfg.model))
    g = torch.Generator().manual_seed(1)
    t = torch.randint(0, cfg.model.vocab_size, (4, 65), generator=g)  # 256 tokens, 128 a rank under sequence parallelism
    x, y = t[:, :-1], t[:, 1:]
    _, a = eng(x, labels=y)
    a.backward()
    _, b = ref(x, labels=y)
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) < 1e-3
    for (n, p), (_, q) in zip(eng.module.named_parameters(), ref.named_parameters()):
        want = q.grad
        for dim in range(want.dim()):
            if p.main_grad.shape[dim] != want.shape[dim]:
                want = want.chunk(2, dim)[rank]
        assert rel(p.main_grad, want) < TOL, n


@pytest.mark.parametrize("sp", [False, True])
@pytest.mark.parametrize("qk", [False, True])
def test_fp8_gradients_under_tensor_parallelism(sp, qk):
    run_distributed(_worker, 2, sp, qk)


def _sharded_worker(rank, world, ckpt):
    cfg = tiny_config(model__d_model=256, model__n_layers=5, model__n_heads=4, model__n_kv_heads=4, model__ffn_hidden_size=512,
                      model__qk_norm=True, kernels__fp8_linear=True, parallel__activation_checkpointing=ckpt,
                      parallel__sharding_strategy="FULL_SHARD", parallel__limit_all_gathers=True)
    ctx = build_process_context(1, backend="gloo", verbose=False)
    eng = build_engine(cfg, ctx)
    assert eng.shard_world == 2 and len({u.gathered.data_ptr() for u in eng.units}) < len(eng.units)  # slots are shared
    torch.manual_seed(cfg.seed)
    ref = set_fp8_linear(build_model(cfg.model))
    t = torch.randint(0, cfg.model.vocab_size, (4, 65), generator=torch.Generator().manual_seed(1))
    x, y = t[:, :-1], t[:, 1:]  # the same tokens on both ranks, so the mean gradient is either's
    _, a = eng(x, labels=y)
    a.backward()
    _, b = ref(x, labels=y)
    b.backward()
    assert abs(float(a.detach()) - float(b.detach())) < 1e-5
    grads = dict((n, p.grad) for n, p in ref.named_parameters())
    for u in eng.units:
        want = torch.zeros(u.numel)
        for e in u.entries:
            want[e.offset:e.offset + e.numel] = grads[e.fqn].reshape(-1)
        lo, hi = u.shard_range(rank)
        assert rel(u.grad_shard, want[lo:hi]) < 2.0 ** -18, u.name


@pytest.mark.parametrize("ckpt", [False, True])
def test_fp8_gradients_with_gathered_weights_freed_in_between(ckpt):
    """Five blocks share two gather slots: the backward quantises weights that were gathered again."""
    run_distributed(_sharded_worker, 2, ckpt)
