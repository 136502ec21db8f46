"""Checkpoints of models with the block operators."""

from __future__ import annotations

import pytest

from build_your_own_distributed_training_b200.checkpointing.checkpoint import load_checkpoint, save_checkpoint
from build_your_own_distributed_training_b200.checkpointing.recovery import CheckpointValidationError, validate_checkpoint
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


def _norms(rank, world, tmp):
    ctx = build_process_context(1, backend="gloo", verbose=False)

    def mk(qk, resume=None):
        return Trainer(tiny_config(tmp, run_id="norms", model__qk_norm=qk, resume_from=resume), ctx=ctx, gpu_type="cpu")
    a = mk(True)
    path = save_checkpoint(a.model, a.optimizer, a.scheduler, 1, a.config, ctx)
    assert mk(True, path).step == 1
    with pytest.raises(CheckpointValidationError, match="qk_norm"):
        mk(False, path)


def test_head_norms_are_not_dropped_by_a_resume(tmp_path):
    """A checkpoint with head norms holds weights that a model without them would leave unread."""
    run_distributed(_norms, 1, str(tmp_path))


def test_checkpoints_from_before_the_key_still_validate(tmp_path):
    import json
    d = tmp_path / "step_1"
    d.mkdir()
    (d / "_SUCCESS").write_text("1")
    model = tiny_config().to_dict()["model"]
    old = {k: v for k, v in model.items() if k not in ("qk_norm", "resid_dropout")}
    (d / "meta.json").write_text(json.dumps({"step": 1, "world_size": 0, "format": "sharded", "config": {"model": old}}))
    for qk in (False, True):  # (with head norms, loading then names the weights that are missing)
        assert validate_checkpoint(str(d), expected_config={"model": dict(model, qk_norm=qk)}).is_valid
