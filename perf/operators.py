"""Cases of the training-block operators, for timing and for comparison with their plain forms.

Four operators, each in the forms in which a program calls it:

* ``qk``       per-head RMSNorm of queries and keys with the position rotation, packed projection
               in, packed projection out; forward alone (decoding) or forward and backward;
* ``dropout``  residual + dropout(x) with a counter-based mask; forward and backward;
* ``logprob``  log probabilities of given tokens with entropy and top alternatives, and the
               gradient with respect to the logits;
* ``fp8``      linear layer in 8-bit floating point with a power-of-two scale for each block of 128: the forward
               with weights kept in 8 bits (serving), or forward, input and weight gradient (training).

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the
package's operators.  ``exact`` computes the definitions in 64 bits.
"""

import math

import torch

own = False

BLOCK = 128          # elements that share a scale in 8 bits
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
IGNORE = -100


def listed():
    return [
        # one decoded token of a 32/8-head model: launch latency
        {"name": "qk_decode_1", "op": "qk", "tokens": 1, "seqlen": 1, "nq": 32, "nkv": 8, "hd": 128,
         "dtype": "bfloat16", "positions": True, "train": False},
        # fp32 parameters and activations, a ragged token count and a head size off the usual powers of two
        {"name": "qk_fp32_ragged", "op": "qk", "tokens": 999, "seqlen": 333, "nq": 5, "nkv": 1, "hd": 80,
         "dtype": "float32", "positions": False, "train": True},
        # one training step's block at 8192 tokens, 32 query and 8 key heads of 128
        {"name": "qk_train_8192", "op": "qk", "tokens": 8192, "seqlen": 8192, "nq": 32, "nkv": 8, "hd": 128,
         "dtype": "bfloat16", "positions": False, "train": True},
        # a small fp32 model's residual branch, odd width
        {"name": "dropout_fp32_odd", "op": "dropout", "rows": 257, "cols": 769, "dtype": "float32", "p": 0.5},
        # the residual branch of a 4096-wide block at 8192 tokens
        {"name": "dropout_train_8192", "op": "dropout", "rows": 8192, "cols": 4096, "dtype": "bfloat16", "p": 0.1},
        # one sampled token over a 128256-entry vocabulary, with the alternatives a server returns
        {"name": "logprob_decode_1", "op": "logprob", "rows": 1, "vocab": 128256, "pad": 0, "dtype": "float32",
         "top_k": 20, "temperature": 1.0, "masked": 0.0, "train": False},
        # a policy step on packed answers: odd vocabulary inside a padded buffer, forbidden tokens, temperature
        {"name": "logprob_policy_777", "op": "logprob", "rows": 777, "vocab": 32003, "pad": 61, "dtype": "bfloat16",
         "top_k": 5, "temperature": 0.7, "masked": 0.3, "train": True},
        # log likelihood and entropy of 4096 trained tokens over 32000 entries
        {"name": "logprob_train_4096", "op": "logprob", "rows": 4096, "vocab": 32000, "pad": 0, "dtype": "float32",
         "top_k": 0, "temperature": 1.0, "masked": 0.0, "train": True},
        # one decoded token through the gate/up projection kept in 8 bits: the weights' bytes
        {"name": "fp8_serve_1", "op": "fp8", "tokens": 1, "k": 4096, "n": 22016, "train": False},
        # a short batch through the down projection
        {"name": "fp8_serve_48", "op": "fp8", "tokens": 48, "k": 11008, "n": 4096, "train": False},
        # odd sizes in every direction
        {"name": "fp8_train_odd", "op": "fp8", "tokens": 1001, "k": 770, "n": 1302, "train": True},
        # forward, input and weight gradient of a 4096 x 11008 projection at 8192 tokens
        {"name": "fp8_train_8192", "op": "fp8", "tokens": 8192, "k": 4096, "n": 11008, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; half of them multiples of 64 where that fits."""
    n = _log(rng, lo, hi)
    if rng.random() < 0.5 and n >= 64:
        n = n // 64 * 64
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["qk", "dropout", "logprob", "fp8", "fp8"])
    if op == "qk":
        hd = rng.choice([16, 32, 48, 64, 80, 96, 128, 128, 192, 256])
        nkv = rng.choice([1, 2, 4, 5, 8])
        nq = nkv * rng.choice([1, 2, 4, 7])
        most = min(8192, 8192 * 48 * 128 // ((nq + 2 * nkv) * hd))
        tokens = _log(rng, 1, most)
        batch = rng.choice([1, 2, 3]) if tokens >= 3 else 1
        tokens = tokens // batch * batch
        if (nq + 2 * nkv) * hd == 3072 or tokens == 3072:
            nq, tokens = nq + nkv, max(1, tokens // 2)
            batch = 1
        return {"op": "qk", "tokens": tokens, "seqlen": tokens // batch, "nq": nq, "nkv": nkv, "hd": hd,
                "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                "positions": rng.random() < 0.5, "train": rng.random() < 0.7}
    if op == "dropout":
        cols = _size(rng, 32, 8192)
        rows = _size(rng, 1, 33554432 // cols)
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        return {"op": "dropout", "rows": max(1, rows // 2) if dtype == "float32" else rows, "cols": cols,
                "dtype": dtype, "p": rng.choice([0.05, 0.1, 0.3, 0.5])}
    if op == "logprob":
        vocab = _size(rng, 500, 130000)
        rows = _log(rng, 1, 131072000 // vocab if vocab > 16000 else 8192)
        return {"op": "logprob", "rows": rows + 1 if rows == 3072 else rows, "vocab": vocab,
                "pad": rng.choice([0, 0, rng.randint(1, 64)]),
                "dtype": rng.choice(["float32", "bfloat16", "float16"]),
                "top_k": rng.choice([0, 1, rng.randint(2, 32)]) if rows * vocab < 40000000 else 0,
                "temperature": rng.choice([1.0, 1.0, 0.5, 1.3]), "masked": rng.choice([0.0, 0.0, 0.5]),
                "train": rng.random() < 0.6}
    k, n = _size(rng, 128, 14336), _size(rng, 128, 22016)
    n = n if n * k <= 4096 * 22016 else 4096 * 22016 // k
    if rng.random() < 0.4:
        return {"op": "fp8", "tokens": _log(rng, 1, 256), "k": k, "n": n, "train": False}
    n = n if n * k <= 4096 * 11008 else 4096 * 11008 // k
    tokens = _size(rng, 16, max(17, min(8192, 8192 * 4096 * 11008 // (k * n))))
    return {"op": "fp8", "tokens": tokens, "k": k, "n": n, "train": True}


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "qk":
        dt = getattr(torch, case["dtype"])
        t, nq, nkv, hd = case["tokens"], case["nq"], case["nkv"], case["hd"]
        width = (nq + 2 * nkv) * hd
        table = 8192 if case["positions"] else case["seqlen"]
        ang = torch.outer(torch.arange(table, device="cuda").float(),
                          1.0 / (10000.0 ** (torch.arange(0, hd, 2, device="cuda").float() / hd)))
        ang = torch.cat((ang, ang), dim=-1)
        s["cos"], s["sin"] = ang.cos(), ang.sin()
        s["qkv"] = normal(t, width, dtype=dt, scale=1.7)
        s["wq"] = (1.0 + normal(hd, scale=0.1)).to(dt)
        s["wk"] = (1.0 + normal(hd, scale=0.1)).to(dt)
        s["pos"] = (torch.randint(0, table, (t,), device="cuda", generator=gen) if case["positions"] else None)
        if case["train"]:
            for name in ("qkv", "wq", "wk"):
                s[name].requires_grad_(True)
            s["dy"] = normal(t, width, dtype=dt)
    elif case["op"] == "dropout":
        dt = getattr(torch, case["dtype"])
        shape = (case["rows"], case["cols"])
        s["x"] = normal(*shape, dtype=dt).requires_grad_(True)
        s["residual"] = normal(*shape, dtype=dt, scale=2.0).requires_grad_(True)
        s["dy"] = normal(*shape, dtype=dt)
        s["seed"] = 0x9E3779B97F4A7C15 * (int(seed) + 1) % (1 << 62)
    elif case["op"] == "logprob":
        dt = getattr(torch, case["dtype"])
        m, v = case["rows"], case["vocab"]
        buf = normal(m, v + case["pad"], scale=2.5)
        if case["masked"]:
            buf.masked_fill_(torch.rand(m, v + case["pad"], device="cuda", generator=gen) < case["masked"], -math.inf)
        tok = torch.randint(0, v, (m,), device="cuda", generator=gen)
        # the token a policy sampled is never a forbidden one
        buf.scatter_(1, tok[:, None], normal(m, 1, scale=2.5) + 4.0)
        s["logits"] = buf.to(dt)[:, :v].detach()
        if m > 4:
            tok[torch.rand(m, device="cuda", generator=gen) < 0.1] = IGNORE
        s["tokens"] = tok
        if case["train"]:
            s["logits"].requires_grad_(True)
            s["g_lp"] = normal(m)
            s["g_ent"] = normal(m, scale=0.01)
    else:
        t, k, n = case["tokens"], case["k"], case["n"]
        s["x"] = normal(t, k, dtype=torch.bfloat16)
        w = normal(n, k, dtype=torch.bfloat16, scale=0.02)
        if case["train"]:
            s["x"].requires_grad_(True)
            s["w"] = w.requires_grad_(True)
            s["dy"] = normal(t, n, dtype=torch.bfloat16, scale=1e-3)
        else:  # what a server keeps: 8-bit values and the scales of their 128 x 128 blocks
            value, scale = _blocks(w.float(), BLOCK, BLOCK)
            s["wq"], s["ws"] = value.to(torch.float8_e4m3fn), scale.to(torch.float8_e8m0fnu)
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _rotate_half(x):
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


def _rotate_half_t(x):
    h = x.shape[-1] // 2
    return torch.cat((x[..., h:], -x[..., :h]), dim=-1)


def _plain_qk(s):
    c = s["case"]
    t, nq, nkv, hd = c["tokens"], c["nq"], c["nkv"], c["hd"]
    dt = s["qkv"].dtype
    x = s["qkv"].detach().float().view(t, nq + 2 * nkv, hd)
    pos = s["pos"] if s["pos"] is not None else torch.arange(t, device="cuda") % c["seqlen"]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    w = torch.cat((s["wq"].detach().float().expand(nq, hd), s["wk"].detach().float().expand(nkv, hd)))
    a = x[:, :nq + nkv]
    r = torch.rsqrt((a * a).mean(-1, keepdim=True) + 1e-5)
    n = a * r
    u = n * w
    y = torch.cat((u * cos + _rotate_half(u) * sin, x[:, nq + nkv:]), dim=1).to(dt).view(t, -1)
    if not c["train"]:
        return y
    g = s["dy"].float().view(t, nq + 2 * nkv, hd)
    gr = g[:, :nq + nkv]
    gu = gr * cos + _rotate_half_t(gr * sin)
    gw = gu * n
    gn = gu * w
    ga = r * (gn - n * (gn * n).mean(-1, keepdim=True))
    dx = torch.cat((ga, g[:, nq + nkv:]), dim=1).to(dt).view(t, -1)
    return {"y": y, "dqkv": dx, "dwq": gw[:, :nq].sum((0, 1)).to(dt), "dwk": gw[:, nq:].sum((0, 1)).to(dt)}


def _keep(n, p, seed):
    """Which of n elements stay: element e compares 16 random bits with round(p * 2^16): the bits
    e % 8 of the 128 that Philox4x32-10 gives for the counter e // 8 and the key `seed`."""
    mask = 0xFFFFFFFF
    ctr = torch.arange(-(-n // 8), device="cuda", dtype=torch.int64)
    a, b = ctr & mask, ctr >> 32
    c, d = torch.zeros_like(a), torch.zeros_like(a)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        m0, m1 = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((m1 >> 32) & mask) ^ b ^ k0, m1 & mask, ((m0 >> 32) & mask) ^ d ^ k1, m0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack((a, b, c, d), dim=1)
    bits = torch.stack((words & 0xFFFF, words >> 16), dim=2).view(-1)[:n]
    return bits >= round(p * 65536)


def _plain_dropout(s):
    x, res, dy, p = s["x"].detach(), s["residual"].detach(), s["dy"], s["case"]["p"]
    keep = _keep(x.numel(), p, s["seed"]).view(x.shape)
    scale = 65536.0 / (65536 - round(p * 65536))
    y = (res.float() + torch.where(keep, x.float() * scale, 0.0)).to(x.dtype)
    return {"y": y, "dx": torch.where(keep, dy.float() * scale, 0.0).to(x.dtype), "dresidual": dy}


def _plain_logprob(s):
    c = s["case"]
    x, tok = s["logits"].detach().float(), s["tokens"]
    valid = tok != IGNORE
    idx = torch.where(valid, tok, 0)[:, None]
    z = (x - x.amax(-1, keepdim=True)) / c["temperature"]
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    logp = z - total.log()
    p = e / total
    plogp = torch.where(p > 0, p * logp, 0.0)
    ent = -plogp.sum(-1)
    out = {"logprob": torch.where(valid, logp.gather(1, idx)[:, 0], 0.0), "entropy": torch.where(valid, ent, 0.0)}
    if c["top_k"]:
        top = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :c["top_k"]]
        out["top_tokens"] = torch.where(valid[:, None], top, -1)
        out["top_logprobs"] = torch.where(valid[:, None], logp.gather(1, top), -math.inf)
    if c["train"]:
        g = -p * s["g_lp"][:, None] - s["g_ent"][:, None] * (plogp + p * ent[:, None])
        g.scatter_add_(1, idx, s["g_lp"][:, None])
        out["dlogits"] = torch.where(valid[:, None], g / c["temperature"], 0.0).to(s["logits"].dtype)
    return out


def _blocks(x, rows, cols):
    """x in 8-bit values with one scale for each block of rows x cols: (values in 32 bits, scales).
    A scale is the least power of two with which the block's largest magnitude stays within 448."""
    r, c = x.shape
    br, bc = -(-r // rows), -(-c // cols)
    pad = torch.zeros(br * rows, bc * cols, device=x.device, dtype=x.dtype)
    pad[:r, :c] = x
    b = pad.view(br, rows, bc, cols)
    part, power = torch.frexp(b.abs().amax((1, 3)).clamp_min(AMAX_FLOOR))  # 448 = 0.875 * 2^9
    scale = (torch.where(part > 0.875, power + 119, power + 118) << 23).view(torch.float32)
    q = (b / scale[:, None, :, None]).to(torch.float8_e4m3fn).float()
    return q.view(br * rows, bc * cols)[:r, :c].contiguous(), scale


def _spread(value, scale, rows, cols):
    r, c = value.shape
    return value * scale.repeat_interleave(rows, 0)[:r].repeat_interleave(cols, 1)[:, :c]


def _rounded(x, rows, cols):
    return _spread(*_blocks(x, rows, cols), rows, cols)


def _plain_fp8(s):
    x = s["x"].detach().float()
    if not s["case"]["train"]:
        return (_rounded(x, 1, BLOCK) @ _spread(s["wq"].float(), s["ws"].float(), BLOCK, BLOCK).t()).bfloat16()
    dy = s["dy"].float()
    w = _rounded(s["w"].detach().float(), BLOCK, BLOCK)
    y = _rounded(x, 1, BLOCK) @ w.t()
    dx = _rounded(dy, 1, BLOCK) @ w
    dw = _rounded(dy.t().contiguous(), 1, BLOCK) @ _rounded(x.t().contiguous(), 1, BLOCK).t()
    return {"y": y.bfloat16(), "dx": dx.bfloat16(), "dw": dw.bfloat16()}


# ---------------------------------------------------------------------------------------------- the operators
def _own(s):
    from build_your_own_distributed_training_b200 import ops
    c = s["case"]
    if c["op"] == "qk":
        y = ops.qk_norm_rope(s["qkv"], s["wq"], s["wk"], s["cos"], s["sin"], c["nq"], c["nkv"], c["hd"],
                             c["seqlen"], 1e-5, positions=s["pos"])
        if not c["train"]:
            return y
        dx, dwq, dwk = torch.autograd.grad(y, (s["qkv"], s["wq"], s["wk"]), s["dy"])
        return {"y": y, "dqkv": dx, "dwq": dwq, "dwk": dwk}
    if c["op"] == "dropout":
        y = ops.dropout_add(s["x"], s["residual"], c["p"], s["seed"])
        dx, dres = torch.autograd.grad(y, (s["x"], s["residual"]), s["dy"])
        return {"y": y, "dx": dx, "dresidual": dres}
    if c["op"] == "logprob":
        r = ops.token_log_probs(s["logits"], s["tokens"], temperature=c["temperature"], top_k=c["top_k"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if c["top_k"]:
            out["top_tokens"], out["top_logprobs"] = r.top_tokens, r.top_logprobs
        if c["train"]:
            out["dlogits"], = torch.autograd.grad((r.logprob, r.entropy), (s["logits"],), (s["g_lp"], s["g_ent"]))
        return out
    if not c["train"]:
        return ops.linear_fp8(s["x"], ops.Fp8Blocks(s["wq"], s["ws"]))
    y = ops.linear_fp8(s["x"], s["w"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return {"y": y, "dx": dx, "dw": dw}


def run(state):
    if own:
        return _own(state)
    return {"qk": _plain_qk, "dropout": _plain_dropout, "logprob": _plain_logprob,
            "fp8": _plain_fp8}[state["case"]["op"]](state)


def work(case):
    """Bytes: every input read once and every output written once; operations of the definition."""
    size = {"float32": 4, "bfloat16": 2, "float16": 2}.get(case.get("dtype"), 2)
    if case["op"] == "qk":
        e = case["tokens"] * (case["nq"] + 2 * case["nkv"]) * case["hd"]
        qk = case["tokens"] * (case["nq"] + case["nkv"]) * case["hd"]
        table = 8 * case["hd"] * (case["tokens"] if case["positions"] else case["seqlen"])
        if not case["train"]:
            return {"bytes": 2 * e * size + table, "flops": 8 * qk}
        # backward: dy and the queries and keys read, the gradient written
        return {"bytes": (4 * e + qk) * size + 2 * table, "flops": 26 * qk}
    if case["op"] == "dropout":
        e = case["rows"] * case["cols"]
        return {"bytes": 5 * e * size, "flops": 3 * e}  # x, residual -> y; dy -> dx
    if case["op"] == "logprob":
        e = case["rows"] * case["vocab"]
        if not case["train"]:
            return {"bytes": e * size + case["rows"] * (16 + 12 * case["top_k"]), "flops": 6 * e}
        return {"bytes": 3 * e * size + case["rows"] * (24 + 12 * case["top_k"]), "flops": 16 * e}
    t, k, n = case["tokens"], case["k"], case["n"]
    if not case["train"]:
        return {"bytes": 2 * t * k + n * k + 2 * t * n, "flops": 2 * t * k * n}
    # x, w, dy read; y, dx, dw written
    return {"bytes": 4 * (t * k + k * n + t * n), "flops": 6 * t * k * n}


# ---------------------------------------------------------------------------------------------- in 64 bits
def _exact_qk(s, c):
    t, nq, nkv, hd = c["tokens"], c["nq"], c["nkv"], c["hd"]
    h = hd // 2
    x = s["qkv"].detach().double().reshape(t, -1, hd)
    where = s["pos"].tolist() if s["pos"] is not None else [i % c["seqlen"] for i in range(t)]
    co = s["cos"].double()[where, :h].unsqueeze(1)
    si = s["sin"].double()[where, :h].unsqueeze(1)
    y, dx = x.clone(), (s["dy"].double().reshape(t, -1, hd).clone() if c["train"] else None)
    dw = {}
    for name, lo, hi in (("wq", 0, nq), ("wk", nq, nq + nkv)):
        w = s[name].detach().double()
        a = x[:, lo:hi]
        norm = a.div((a.square().sum(-1, keepdim=True) / hd + 1e-5).sqrt())
        u1, u2 = (norm * w)[..., :h], (norm * w)[..., h:]
        y[:, lo:hi, :h] = u1 * co - u2 * si
        y[:, lo:hi, h:] = u2 * co + u1 * si
        if dx is not None:
            g1, g2 = dx[:, lo:hi, :h].clone(), dx[:, lo:hi, h:].clone()
            gu = torch.cat((g1 * co + g2 * si, g2 * co - g1 * si), -1)
            dw["d" + name] = (gu * norm).sum(0).sum(0)
            gn = gu * w
            inv = 1.0 / (a.square().sum(-1, keepdim=True) / hd + 1e-5).sqrt()
            dx[:, lo:hi] = inv * gn - inv * norm * ((gn * norm).sum(-1, keepdim=True) / hd)
    if dx is None:
        return y.reshape(t, -1)
    return {"y": y.reshape(t, -1), "dqkv": dx.reshape(t, -1), **dw}


def _exact_dropout(s, c):
    import numpy as np
    n, cut = c["rows"] * c["cols"], int(c["p"] * 65536 + 0.5)
    groups = (n + 7) // 8
    word = [np.arange(groups, dtype=np.uint64), np.zeros(groups, np.uint64),
            np.zeros(groups, np.uint64), np.zeros(groups, np.uint64)]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    word[1] = word[0] >> half
    word[0] = word[0] & low
    key = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32 % 2 ** 32]
    for r in range(10):
        left, right = word[0] * np.uint64(0xD2511F53), word[2] * np.uint64(0xCD9E8D57)
        k = [np.uint64((key[0] + r * 0x9E3779B9) % 2 ** 32), np.uint64((key[1] + r * 0xBB67AE85) % 2 ** 32)]
        word = [(right >> half) ^ word[1] ^ k[0], right & low, (left >> half) ^ word[3] ^ k[1], left & low]
    shorts = np.stack(word, 1).astype("<u4").view("<u2").reshape(-1)[:n]
    kept = torch.from_numpy(shorts >= cut).cuda().view(c["rows"], c["cols"])
    f = kept.double() * (65536.0 / (65536 - cut))
    return {"y": s["residual"].detach().double() + s["x"].detach().double() * f, "dx": s["dy"].double() * f,
            "dresidual": s["dy"].double()}


def _exact_logprob(s, c):
    x = s["logits"].detach().double() / c["temperature"]
    tok, k = s["tokens"], c["top_k"]
    skip = tok == IGNORE
    at = tok.clamp_min(0)
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(logp)
    ent = torch.special.entr(p).sum(1)
    row = torch.arange(len(tok), device="cuda")
    out = {"logprob": logp[row, at].masked_fill(skip, 0.0), "entropy": ent.masked_fill(skip, 0.0)}
    if k:
        best = torch.sort(logp, dim=1, descending=True, stable=True)[0][:, :k]
        out["top_tokens"] = None
        out["top_logprobs"] = best.masked_fill(skip[:, None], -math.inf)
    if c["train"]:
        gl, ge = s["g_lp"].double()[:, None], s["g_ent"].double()[:, None]
        d = ge * (torch.special.entr(p) - p * ent[:, None]) - gl * p
        d[row, at] += gl[:, 0]
        out["dlogits"] = (d / c["temperature"]).masked_fill(skip[:, None], 0.0)
    return out


def _exact_round(x, rows, cols):
    """Each block of rows x cols divided by 2^ceil(log2(max / 448)), rounded to 4 significant bits
    (steps of 2^-9 below 2^-6), half to even, and multiplied back."""
    r, c = x.shape
    full = torch.nn.functional.pad(x, (0, -c % cols, 0, -r % rows))
    b = full.unfold(0, rows, rows).unfold(1, cols, cols)
    scale = torch.exp2(torch.ceil(torch.log2(b.abs().amax((-1, -2), keepdim=True).clamp_min(AMAX_FLOOR) / E4M3_MAX)))
    v = b / scale
    step = torch.exp2(torch.frexp(v)[1].clamp_min(-5).double() - 4)
    v = torch.round(v / step) * step * scale
    return v.permute(0, 2, 1, 3).reshape(full.shape)[:r, :c]


def _exact_fp8(s, c):
    x = s["x"].detach().double()
    if not c["train"]:
        sc, w = s["ws"].float().double(), s["wq"].double()
        i = torch.arange(c["n"], device="cuda") // BLOCK
        j = torch.arange(c["k"], device="cuda") // BLOCK
        return torch.einsum("tk,nk->tn", _exact_round(x, 1, BLOCK), w * sc[i][:, j])
    w, dy = _exact_round(s["w"].detach().double(), BLOCK, BLOCK), s["dy"].double()
    return {"y": torch.einsum("tk,nk->tn", _exact_round(x, 1, BLOCK), w),
            "dx": torch.einsum("tn,nk->tk", _exact_round(dy, 1, BLOCK), w),
            "dw": torch.einsum("nt,kt->nk", _exact_round(dy.t(), 1, BLOCK), _exact_round(x.t(), 1, BLOCK))}


def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "dropout": _exact_dropout, "logprob": _exact_logprob,
            "fp8": _exact_fp8}[case["op"]](s, case)
