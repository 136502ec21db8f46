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
