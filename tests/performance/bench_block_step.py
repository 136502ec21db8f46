"""Forward + backward of a 7B-shaped stack through the sharding engine, with the block operators off and on.

    python tests/performance/bench_block_step.py [--layers 8] [--steps 8]

One GPU, 8192 tokens (4 x 2048), random weights and tokens; CUDA events, the median of ``--steps`` after three
warm-up steps; activations and weights exceed the L2.  The optimizer step is left out: none of the operators is in
it.  ``peak`` is the allocator's peak over the timed steps.
"""

from __future__ import annotations

import argparse
import gc
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import torch  # noqa: E402

from build_your_own_distributed_training_b200.config import ModelConfig, ParallelConfig  # noqa: E402
from build_your_own_distributed_training_b200.models import TransformerBlock, build_model, set_fp8_linear  # noqa: E402
from build_your_own_distributed_training_b200.parallel.fsdp import FullyShardedModel  # noqa: E402

DEV = torch.device("cuda", 0)
VOCAB, BATCH, SEQ = 32000, 4, 2048
# name: 8-bit projections, head norms, residual dropout, token log probabilities instead of the mean cross-entropy
CASES = {"bf16": (False, False, 0.0, False), "fp8_linear": (True, False, 0.0, False), "qk_norm": (False, True, 0.0, False),
         "resid_dropout": (False, False, 0.1, False), "fp8_linear + qk_norm + resid_dropout": (True, True, 0.1, False),
         "token scoring": (False, False, 0.0, True)}


def run(fp8: bool, qk: bool, drop: float, score: bool, layers: int, steps: int) -> tuple[float, float, float]:
    """(step, forward) in ms and the peak in GiB."""
    torch.manual_seed(0)
    model = build_model(ModelConfig(vocab_size=VOCAB, d_model=4096, n_layers=layers, n_heads=32, n_kv_heads=32,
                                    ffn_hidden_size=11008, max_seq_len=SEQ, tie_embeddings=False, qk_norm=qk, resid_dropout=drop))
    set_fp8_linear(model, fp8)
    eng = FullyShardedModel(model, None, ParallelConfig(), {TransformerBlock}, device=DEV)
    model.rope_cos, model.rope_sin = model.rope_cos.to(DEV), model.rope_sin.to(DEV)
    model.return_logits = False
    eng.train()
    x, y = torch.randint(0, VOCAB, (2, BATCH, SEQ), device=DEV)
    times = []
    for i in range(steps + 3):
        if i == 3:
            torch.cuda.reset_peak_memory_stats()
        a, b, c = (torch.cuda.Event(enable_timing=True) for _ in range(3))
        torch.cuda.synchronize()
        a.record()
        if score:
            r = eng(x, targets=y)
            loss = -r.logprob.mean() - 0.01 * r.entropy.mean()
        else:
            _, loss = eng(x, labels=y)
        b.record()
        loss.backward()
        eng.wait_reduce()
        c.record()
        torch.cuda.synchronize()
        eng.zero_grad_buffers()
        if i >= 3:
            times.append((a.elapsed_time(c), a.elapsed_time(b)))
    times.sort()
    return *times[len(times) // 2], torch.cuda.max_memory_allocated() / 2 ** 30


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    for name, case in CASES.items():
        step, fwd, peak = run(*case, a.layers, a.steps)
        print(f"{name}: {step:.1f} ms (forward {fwd:.1f}), peak {peak:.1f} GiB", flush=True)
        gc.collect()  # an engine and its hooks refer to each other
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
