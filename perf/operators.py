"""The dense-head operators' benchmark cases: layer norm, 8-bit activation checkpoints, log probabilities.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes a
case's inputs on the GPU and ``run(state)`` is one pass: through torch's elementary operations (``own`` false)
or through this package's kernels (``own`` true).  ``work(case)`` is what a pass cannot do without and
``exact(case, seed)`` the same outputs from the definitions in 64 bits.

A case's ``op`` is

- ``norm``: layer norm of [n, d]; ``train`` adds its backward (dx, dweight, dbias);
- ``ckpt``: [n, d] packed to 8 bits (a power-of-two scale for each 32 columns of a row) and read back;
- ``wgrad``: a linear layer's input [n, d] packed to 8 bits, then dW = dy^T x and db = sum dy [n, o] from it;
- ``logp``: log probabilities of ``t`` given items of each of n score rows over c items, the row's entropy and
  its ``k`` best items; ``train`` adds the backward into the scores.
"""
import importlib
import math

import torch

own = False

PACKAGE = "problem-recommender-system-using-kgat-in-codeforces_amd"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
EPS = 1e-5
BLOCK = 32  # columns that share a checkpoint scale


def listed():
    return [
        # one user's 64-wide vector: a serving call, latency alone
        {"name": "norm one row", "op": "norm", "n": 1, "d": 64, "type": "float32", "train": False},
        # every node of the Codeforces-sized graph at an odd width, half precision
        {"name": "norm nodes odd", "op": "norm", "n": 16484, "d": 1021, "type": "bfloat16", "train": False},
        # the 1M-node table at its 64 columns, a training step: short rows, a long reduction
        {"name": "norm table step", "op": "norm", "n": 1000000, "d": 64, "type": "float32", "train": True},
        # a wide hidden layer's training step
        {"name": "norm wide step", "op": "norm", "n": 8192, "d": 4096, "type": "bfloat16", "train": True},
        # a propagation layer's neighbour sums kept for the backward: 1M nodes, 128 columns
        {"name": "checkpoint table", "op": "ckpt", "n": 1000000, "d": 128, "type": "float32"},
        # NFM's hidden layer at its batch (1,024 positive and as many negative rows)
        {"name": "wgrad hidden layer", "op": "wgrad", "n": 2048, "d": 64, "o": 64, "type": "float32"},
        # many rows through a narrow layer of odd sizes
        {"name": "wgrad odd", "op": "wgrad", "n": 100003, "d": 257, "o": 131, "type": "float16"},
        # a wide layer: one large matrix product
        {"name": "wgrad wide", "op": "wgrad", "n": 16384, "d": 4096, "o": 4096, "type": "bfloat16"},
        # one user over the Codeforces-sized catalogue: a serving call
        {"name": "logp one user", "op": "logp", "n": 1, "c": 9500, "t": 1, "k": 20, "masked": 50, "type": "float32", "train": False},
        # an evaluation batch: 20 held-out items a user, train items masked, the longest cut-off
        {"name": "logp evaluation", "op": "logp", "n": 256, "c": 9500, "t": 20, "k": 100, "masked": 200, "type": "float32", "train": False},
        # three users over a million items: few rows, a long axis
        {"name": "logp long rows", "op": "logp", "n": 3, "c": 1000003, "t": 4, "k": 20, "masked": 1000, "type": "float32", "train": False},
        # the loss of a training step over a large catalogue, with an entropy term
        {"name": "logp step", "op": "logp", "n": 4096, "c": 65537, "t": 1, "k": 0, "masked": 0, "type": "bfloat16", "train": True},
    ]


def _size(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; every second one odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v |= 1
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["norm", "norm", "ckpt", "wgrad", "wgrad", "logp", "logp", "logp"])
    kind = rng.choice(sorted(TYPES))
    if op == "norm":
        d = _size(rng, 8, 16384)
        return {"op": op, "n": _size(rng, 1, max(1, min(1000000, 33000000 // d))), "d": d, "type": kind, "train": rng.random() < 0.6}
    if op == "ckpt":
        d = _size(rng, 8, 8192)
        return {"op": op, "n": _size(rng, 1, max(1, min(1000000, 64000000 // d))), "d": d, "type": kind}
    if op == "wgrad":
        d, o = _size(rng, 16, 4096), _size(rng, 16, 4096)
        most = min(500000, 60000000 // max(d, o), 90000000000 // (d * o))
        return {"op": op, "n": _size(rng, 1, max(1, most)), "d": d, "o": o, "type": kind}
    c = _size(rng, 100, 1000003)
    n = _size(rng, 1, max(1, min(8192, 100000000 // c)))
    train = rng.random() < 0.4
    return {"op": op, "n": n, "c": c, "t": rng.choice([1, 1, 4, 20]), "k": 0 if train else rng.choice([0, 1, 20, 64, 100]),
            "masked": rng.choice([0, c // 20]), "type": kind, "train": train}


def _normal(gen, *shape):
    return torch.randn(*shape, device="cuda", generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, t = case["op"], TYPES[case["type"]]
    s = {"case": case}
    if op == "logp":
        n, c = case["n"], case["c"]
        z = _normal(gen, n, c) * 2.5
        items = torch.randint(0, c, (n, case["t"]), device="cuda", generator=gen)
        held = torch.zeros(n, c, dtype=torch.bool, device="cuda").scatter_(1, items, True)
        x = z
        if case["masked"]:  # each row's seen items
            seen = torch.randint(0, c, (n, case["masked"]), device="cuda", generator=gen)
            x = z.scatter(1, seen, float("-inf"))
        x = torch.where(held, z + 4, x)  # held-out items score above the average
        if case["t"] > 1:  # shorter lists are padded with -1
            items = torch.where(torch.rand(items.shape, device="cuda", generator=gen) < 0.1, -1, items)
        s["scores"], s["items"] = x.to(t), items
        if case["train"]:
            s["dlogp"] = -(torch.rand(n, case["t"], device="cuda", generator=gen) + 0.5) / n
            s["dentropy"] = _normal(gen, n) * (0.02 / n)
        return s
    n, d = case["n"], case["d"]
    # activations: rows of different size, a mean, and a few columns that stand out
    x = _normal(gen, n, d) * (0.5 + torch.rand(n, 1, device="cuda", generator=gen)) + 0.3
    x *= 1 + 7 * (torch.rand(d, device="cuda", generator=gen) < 0.02)
    s["x"] = x.to(t)
    if op == "norm":
        s["weight"] = 1 + 0.2 * _normal(gen, d)
        s["bias"] = 0.1 * _normal(gen, d)
        if case["train"]:
            s["dy"] = _normal(gen, n, d).to(t)
    elif op == "wgrad":
        s["dy"] = (_normal(gen, n, case["o"]) * 0.1).to(t)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    xhat = xc * rstd
    y = (xhat * s["weight"] + s["bias"]).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * s["weight"]
    dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * rstd
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * xhat).sum(0, dtype=torch.float64).float(),
            "dbias": dy.sum(0, dtype=torch.float64).float()}


def _plain_values(x):
    """What the 8-bit checkpoint of x stands for, in 32 bits: round(x / 2^e) 2^e with 2^(e + 6) <= max < 2^(e + 7)."""
    n, d = x.shape
    pad = -d % BLOCK
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(n, -1, BLOCK)
    e = (torch.frexp(v.abs().amax(2, keepdim=True))[1] - 7).clamp_(min=-126)
    q = torch.ldexp(v, -e).round_().clamp_(-127, 127)
    return torch.ldexp(q, e).view(n, d + pad)[:, :d]


def _plain_wgrad(s):
    dy = s["dy"].float()
    return {"dW": dy.t() @ _plain_values(s["x"]), "db": dy.sum(0, dtype=torch.float64).float()}


def _plain_logp(s):
    case, items = s["case"], s["items"]
    z = s["scores"].float()
    m = z.amax(1, keepdim=True)
    lse = (z - m).exp().sum(1, keepdim=True).log()
    logp = (z - m) - lse
    p = logp.exp()
    h = -(p * logp.clamp_min(-1e30)).sum(1, keepdim=True)
    given, at = items >= 0, items.clamp_min(0)
    out = {"logp": torch.where(given, logp.gather(1, at), 0.0), "entropy": h[:, 0], "lse": (m + lse)[:, 0]}
    if case["k"]:
        bits = (z + 0.0).view(torch.int32)
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * (1 << 32) - torch.arange(z.shape[1], device=z.device)
        out["top_items"] = key.topk(case["k"], dim=1)[1]  # equal scores: the lowest item first
        out["top_logp"] = logp.gather(1, out["top_items"])
    if case["train"]:
        g = torch.where(given, s["dlogp"], 0.0)
        dz = -p * (g.sum(1, keepdim=True) + s["dentropy"][:, None] * (logp.clamp_min(-1e30) + h))
        out["dscores"] = dz.scatter_add_(1, at, g).to(s["scores"].dtype)
    return out


# ------------------------------------------------------------------------------------------------ this package's calls
def _own_norm(k, s):
    if not s["case"]["train"]:
        return {"y": k.layer_norm_fwd(s["x"], s["weight"], s["bias"], EPS)}
    y, mean, rstd = k.layer_norm_fwd(s["x"], s["weight"], s["bias"], EPS, stats=True)
    dx, dweight, dbias = k.layer_norm_bwd(s["dy"], s["x"], mean, rstd, s["weight"])
    return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}


def _own_logp(k, s):
    case = s["case"]
    r = k.log_prob_fwd(s["scores"], s["items"], k=case["k"])
    out = {"logp": r.logp, "entropy": r.entropy, "lse": r.lse}
    if case["k"]:
        out["top_items"], out["top_logp"] = r.top_items, r.top_logp
    if case["train"]:
        out["dscores"] = k.log_prob_bwd(s["scores"], s["items"], r.stats, s["dlogp"], s["dentropy"])
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        k = importlib.import_module(PACKAGE + ".kernels")
        if op == "norm":
            return _own_norm(k, state)
        if op == "ckpt":
            return {"x": k.act8_unpack(k.act8_pack(state["x"]), state["x"].dtype)}
        if op == "wgrad":
            dW, db = k.act8_wgrad(state["dy"], k.act8_pack(state["x"]))
            return {"dW": dW, "db": db}
        return _own_logp(k, state)
    if op == "norm":
        return _plain_norm(state)
    if op == "ckpt":
        return {"x": _plain_values(state["x"]).to(state["x"].dtype)}
    if op == "wgrad":
        return _plain_wgrad(state)
    return _plain_logp(state)


def work(case):
    op, n, b = case["op"], case["n"], BYTES[case["type"]]
    if op == "norm":
        d = case["d"]
        if not case["train"]:
            return {"bytes": 2 * n * d * b + 8 * d, "flops": 8 * n * d}
        # forward: x in, y out; backward: x and dy in, dx out (x is read again: a pass over all rows lies between)
        return {"bytes": 5 * n * d * b + 20 * d, "flops": 22 * n * d}
    if op == "ckpt":  # x in, 8 bits and scales out; both in again, x out
        d = case["d"]
        return {"bytes": 2 * n * d * b + 2 * n * (d + -(-d // BLOCK)), "flops": 6 * n * d}
    if op == "wgrad":
        d, o = case["d"], case["o"]
        return {"bytes": n * d * b + 2 * n * (d + -(-d // BLOCK)) + n * o * b + 4 * o * (d + 1), "flops": 2 * n * d * o + 4 * n * d}
    c, t, k = case["c"], case["t"], case["k"]
    small = n * (8 * t + 4 * t + 8 + 12 * k)
    if not case["train"]:
        return {"bytes": n * c * b + small, "flops": 6 * n * c}
    return {"bytes": 3 * n * c * b + small + n * (4 * t + 4), "flops": 14 * n * c}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op, f = case["op"], torch.float64
    if op == "norm":
        x, w = s["x"].to(f), s["weight"].to(f)
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sd = (var + EPS).sqrt()
        n = (x - mean) / sd
        out = {"y": torch.addcmul(s["bias"].to(f), n, w)}
        if case["train"]:
            dy = s["dy"].to(f)
            a = dy * w
            b = torch.linalg.vecdot(a, n)[:, None] / case["d"]
            out["dx"] = (a - a.sum(1, keepdim=True) / case["d"] - n * b) / sd
            out["dweight"], out["dbias"] = torch.linalg.vecdot(dy, n, dim=0), dy.sum(0)
        return out
    if op in ("ckpt", "wgrad"):
        x = s["x"].to(f)
        n, d = x.shape
        wide = x.new_zeros(n, -(-d // BLOCK) * BLOCK)
        wide[:, :d] = x
        top = wide.abs().reshape(n, -1, BLOCK).max(2).values
        step = torch.exp2((torch.floor(torch.log2(top)) - 6).clamp(min=-126)).repeat_interleave(BLOCK, 1)[:, :d]
        v = torch.clamp(torch.round(x / step), -127, 127) * step
        if op == "ckpt":
            return {"x": v}
        dy = s["dy"].to(f)
        return {"dW": torch.matmul(dy.t(), v), "db": dy.sum(0)}
    z = s["scores"].to(f)
    lse = torch.logsumexp(z, 1)
    given = s["items"] >= 0
    logp = torch.where(given, z.gather(1, s["items"].clamp(min=0)) - lse[:, None], 0.0)
    lp = z - lse[:, None]
    p = lp.exp()
    h = torch.special.entr(p).sum(1)
    out = {"logp": logp, "entropy": h, "lse": lse}
    if case["k"]:
        out["top_items"], out["top_logp"] = None, lp.topk(case["k"], dim=1).values
    if case["train"]:
        g = torch.where(given, s["dlogp"].to(f), 0.0)
        a = torch.zeros_like(z).scatter_add_(1, s["items"].clamp(min=0), g) - p * g.sum(1, keepdim=True)
        out["dscores"] = a - s["dentropy"].to(f)[:, None] * (torch.xlogy(p, p) + p * h[:, None])
    return out
