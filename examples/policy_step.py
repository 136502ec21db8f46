"""Policy-gradient steps on a small LLaMA with normalised heads, residual dropout and 8-bit projections.

    python examples/policy_step.py [--steps 20] [--cpu]

One process, one GPU (or the CPU path).  The "answers" are random tokens whose reward is the share of even
ids, so the mean reward under the trained policy rises as the model moves its probability to even tokens.
Every step scores the sampled tokens with ``TokenLogProbs`` (log probability, entropy, top alternatives),
takes the policy gradient with an entropy bonus, and applies AdamW through the sharding engine.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from build_your_own_distributed_training_b200.config import ModelConfig, ParallelConfig  # noqa: E402
from build_your_own_distributed_training_b200.models import TransformerBlock, build_model, set_fp8_linear  # noqa: E402
from build_your_own_distributed_training_b200.parallel.fsdp import FullyShardedModel  # noqa: E402
from build_your_own_distributed_training_b200.training.optimizer import ShardedAdamW  # noqa: E402

VOCAB, SEQ, BATCH = 512, 64, 8


def build(device: torch.device) -> tuple[FullyShardedModel, ShardedAdamW]:
    torch.manual_seed(0)
    model = build_model(ModelConfig(vocab_size=VOCAB, d_model=256, n_layers=2, n_heads=4, n_kv_heads=2,
                                    ffn_hidden_size=512, max_seq_len=SEQ, tie_embeddings=False, qk_norm=True,
                                    resid_dropout=0.05))
    set_fp8_linear(model)
    cfg = ParallelConfig(param_dtype="bfloat16" if device.type == "cuda" else "float32")
    engine = FullyShardedModel(model, None, cfg, {TransformerBlock}, device=device)
    model.rope_cos, model.rope_sin = model.rope_cos.to(device), model.rope_sin.to(device)
    return engine, ShardedAdamW(engine, lr=2e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.0)


def step(engine: FullyShardedModel, opt: ShardedAdamW, gen: torch.Generator) -> tuple[float, float, float]:
    """(share of even tokens among the top alternatives, mean log probability, mean entropy)."""
    device = engine.device
    tokens = torch.randint(0, VOCAB, (BATCH, SEQ + 1), generator=gen).to(device)
    inputs, targets = tokens[:, :-1], tokens[:, 1:].clone()
    targets[:, : SEQ // 4] = -100  # the prompt is not scored
    even = (targets % 2 == 0).float()
    advantage = torch.where(targets >= 0, even - 0.5, 0.0)
    r = engine(inputs, targets=targets, top_k=5)
    scored = (targets >= 0).sum()
    loss = -(advantage * r.logprob).sum() / scored - 0.01 * r.entropy.sum() / scored
    loss.backward()
    engine.wait_reduce()
    opt.step()
    opt.zero_grad()
    best = r.top_tokens[targets >= 0]
    return (float((best % 2 == 0).float().mean()), float(r.logprob.detach().sum() / scored),
            float(r.entropy.detach().sum() / scored))


def main(argv: list[str] | None = None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--cpu", action="store_true")
    a = ap.parse_args(argv)
    device = torch.device("cpu" if a.cpu else "cuda", None if a.cpu else 0)
    engine, opt = build(device)
    engine.train()
    gen = torch.Generator().manual_seed(1)
    shares = []
    for i in range(a.steps):
        share, lp, ent = step(engine, opt, gen)
        shares.append(share)
        print(f"step {i:3d}  even among the top 5: {share:.3f}  log p {lp:.3f}  entropy {ent:.3f}", flush=True)
    return shares


if __name__ == "__main__":
    main()
