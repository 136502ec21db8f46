"""Checkpoints of models with the block operators."""

from __future__ import annotations

import pytest

from build_your_own_distributed_training_b200.checkpointing.checkpoint import load_checkpoint, save_checkpoint
from build_your_own_distributed_training_b200.parallel.process_groups import build_process_context
from build_your_own_distributed_training_b200.training.loop import train_step
from build_your_own_distributed_training_b200.training.trainer import Trainer
from tests._dist_utils import run_distributed
from tests.helpers import tiny_config


def _run_dropout(rank, world, tmp):
    ctx = build_process_context(1, backend="gloo", verbose=False)

    def mk():
        cfg = tiny_config(tmp, run_id="resume", model__resid_dropout=0.3)
        return cfg, Trainer(cfg, ctx=ctx, gpu_type="cpu")

    def steps(t, cfg, n):
        out = []
        for _ in range(n):
            w, _ = t._next_window()
            out.append(train_step(t.model, w, t.optimizer, t.scheduler, ctx, cfg, gpu_type="cpu").loss)
            t.step += 1
        return out
    cfg, a = mk()
    steps(a, cfg, 3)
    path = save_checkpoint(a.model, a.optimizer, a.scheduler, a.step, cfg, ctx)
    want = steps(a, cfg, 3)
    cfg, b = mk()
    b.step = load_checkpoint(b.model, b.optimizer, b.scheduler, path, ctx)
    b._fast_forward_data(b.step)
    assert steps(b, cfg, 3) == want
    cfg.resume_from = path
    c = Trainer(cfg, ctx=ctx, gpu_type="cpu")
    assert c.step == 3 and steps(c, cfg, 3) == want


@pytest.mark.parametrize("world", [1, 2])
def test_resume_with_residual_dropout_is_bit_exact(tmp_path, world):
    """The masks' seeds go on where the checkpoint left them: walking the data forward draws from the same generator."""
    run_distributed(_run_dropout, world, str(tmp_path))
