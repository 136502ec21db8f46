"""Plain 64-bit implementations of the block operators, written from their formulas, for the tests."""

from __future__ import annotations

import math

import numpy as np
import torch

# unit roundoff: half the spacing of the storage type's numbers at 1
UNIT = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def rel(a: torch.Tensor, b: torch.Tensor) -> float:
    """2-norm of the difference over the 2-norm of ``b``, in 64 bits."""
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    n = float(b.norm())
    d = float((a - b).norm())
    return d / n if n else d


def qk_norm_rope(x, wq, wk, cos, sin, nq, nkv, hd, pos, eps):
    """Differentiable in float64; ``pos``: list of positions."""
    t, h = x.shape[0], hd // 2
    x3 = x.reshape(t, nq + 2 * nkv, hd)
    c, s = cos.double()[pos][:, :h], sin.double()[pos][:, :h]
    heads = []
    for i in range(nq + 2 * nkv):
        a = x3[:, i]
        if i < nq + nkv:
            a = a / torch.sqrt((a * a).sum(1, keepdim=True) / hd + eps) * (wq if i < nq else wk)
            a = torch.cat((a[:, :h] * c - a[:, h:] * s, a[:, h:] * c + a[:, :h] * s), 1)
        heads.append(a)
    return torch.stack(heads, 1).reshape(t, -1)


def philox_fields(first: int, groups: int, seed: int) -> np.ndarray:
    """The 16-bit fields of Philox4x32-10 for counters first .. first + groups, in Python integers."""
    out = np.empty((groups, 8), np.uint32)
    for g in range(groups):
        c = [(first + g) & 0xFFFFFFFF, (first + g) >> 32, 0, 0]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        for i in range(8):
            out[g, i] = (c[i // 2] >> (16 * (i % 2))) & 0xFFFF
    return out


def keep_mask(n: int, p: float, seed: int, start: int = 0) -> torch.Tensor:
    first, last = start // 8, (start + n + 7) // 8
    f = philox_fields(first, last - first, seed).reshape(-1)
    return torch.from_numpy(f[start - 8 * first:start - 8 * first + n] >= math.floor(p * 65536 + 0.5))


def dropout_add(x, residual, p, seed, start=0):
    cut = math.floor(p * 65536 + 0.5)
    keep = keep_mask(x.numel(), p, seed, start).view(x.shape)
    y = torch.where(keep, x * (65536 / (65536 - cut) if cut < 65536 else 0.0), torch.zeros_like(x))
    return y if residual is None else residual + y


def logprobs(x, tokens, temperature=1.0, ignore=-100):
    """float64 rows -> (logprob, entropy), differentiable; rows that have a distribution."""
    # the row's maximum goes first: beside a mask of -3.4e38 even 64 bits keep nothing of ln V
    z = (x - x.detach().amax(1, keepdim=True)) / temperature
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    p = logp.exp()
    ent = -(p * torch.where(p > 0, logp, torch.zeros_like(p))).sum(1)
    skip = tokens == ignore
    at = tokens.masked_fill(skip, 0)
    lp = logp.gather(1, at[:, None])[:, 0]
    return lp.masked_fill(skip, 0.0), ent.masked_fill(skip, 0.0)


def top_order(row, k: int) -> list[int]:
    """Indices of the k largest values of a list, equal values by index."""
    return sorted(range(len(row)), key=lambda i: (-row[i], i))[:k]


def slope(f, x: torch.Tensor, v: torch.Tensor, h: float) -> float:
    """Central difference of the scalar ``f`` at ``x`` along ``v``."""
    return float((f(x + h * v) - f(x - h * v)) / (2 * h))


def fp8_round(x: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(the 64-bit values that the 8-bit codes of ``x`` stand for, scales as floats) in rows x 128
    blocks, one block at a time."""
    x = x.double().cpu()
    out, scales = torch.empty_like(x), torch.empty(-(-x.shape[0] // rows), -(-x.shape[1] // 128), dtype=torch.float64)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = x[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128]
            s = 2.0 ** math.ceil(math.log2(max(float(b.abs().max()), 2.0 ** -100) / 448))
            v = (b / s).numpy()
            step = np.exp2(np.maximum(np.frexp(v)[1] - 1, -6) - 3.0)  # 4 significant bits, 2^-9 below 2^-6
            out[i * rows:(i + 1) * rows, j * 128:(j + 1) * 128] = torch.from_numpy(np.rint(v / step) * step) * s
            scales[i, j] = s
    return out, scales
