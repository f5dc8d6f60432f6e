"""Measured cases of the device operators that put a learned model on top of
leaf indices: embedding lookup with scaling (one token or a summed bag of
tokens a row), its gradient by sorted tokens, and layer norm's forward and
backward pass.

`own = False` computes them from elementary torch operations in 32 bits;
`own = True` calls xgboost.nn.
"""
import math
import os
import sys

import torch

own = False

# Bytes of a value.
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2, "int32": 4, "int64": 8}


def listed():
    return [
        # One new token of a generation step: latency alone.
        _embed("lookup_one_token", rows=1, per_row=1, vocab=32768, dim=1024, dtype="bfloat16", out="bfloat16",
               index="int64", scale=32.0, tokens="zipf"),
        # A long prompt's (or a packed batch's) tokens, odd count, scaled by sqrt(dim).
        _embed("lookup_prompt", rows=8191, per_row=1, vocab=65536, dim=2048, dtype="bfloat16", out="bfloat16",
               index="int64", scale=math.sqrt(2048.0), tokens="zipf"),
        # The leaf indices of 262,144 rows in 100 trees of depth 8, a 64-wide vector for each leaf.
        _embed("leaf_bag_rows", rows=262144, per_row=100, vocab=25600, dim=64, dtype="bfloat16", out="float32",
               index="int32", scale=0.1, tokens="leaf"),
        # A few rows served by 2,000 trees of depth 6 (10 classes, 200 rounds) with a scale for each tree,
        # some trees missing, and an odd width whose rows start at odd addresses.
        _embed("leaf_bag_serving", rows=7, per_row=2000, vocab=128000, dim=33, dtype="float32", out="float32",
               index="int32", scale=0.3, scaled=True, missing=0.1, tokens="leaf"),
        # The table's and the scales' gradient of a small batch: 100 trees of depth 6.
        _embed("leaf_bag_grad_small", grad=True, rows=41, per_row=100, vocab=6400, dim=96, dtype="float32",
               out="float32", index="int32", scale=0.3, scaled=True, missing=0.1, tokens="leaf"),
        # A training step's tokens, the frequent ones thousands of times, the gradient kept in 32 bits.
        _embed("lookup_grad_prompt", grad=True, rows=16411, per_row=1, vocab=65536, dim=2048, dtype="bfloat16",
               out="float32", index="int64", scale=math.sqrt(2048.0), tokens="zipf"),
        # The gradient of leaf_bag_rows' table: 26 million sorted tokens.
        _embed("leaf_bag_grad_rows", grad=True, rows=262144, per_row=100, vocab=25600, dim=64, dtype="bfloat16",
               out="float32", index="int32", scale=0.1, tokens="leaf"),
        # One row of a generation step.
        _norm("norm_one_row", rows=1, dim=4096, dtype="bfloat16", param="bfloat16"),
        # The widest rows of a training step.
        _norm("norm_wide", rows=32768, dim=8192, dtype="bfloat16", param="float32"),
        # Raw features: 100,000 rows of 784.
        _norm("norm_features", rows=100000, dim=784, dtype="float32", param="float32"),
        # A small batch of bag sums, backward.
        _norm("norm_grad_small", grad=True, rows=509, dim=64, dtype="float32", param="float32"),
        # A training step, backward, with the reduction of the weight's gradient over 32,768 rows.
        _norm("norm_grad_wide", grad=True, rows=32768, dim=4096, dtype="bfloat16", param="float32"),
    ]


def _embed(name, *, rows, per_row, vocab, dim, dtype, out, index, scale, tokens, grad=False, scaled=False,
           missing=0.0):
    case = {"name": name, "op": "embedding_grad" if grad else "embedding", "rows": rows, "per_row": per_row,
            "vocab": vocab, "dim": dim, "dtype": dtype, "out": out, "index": index, "scale": scale,
            "tokens": tokens, "scaled": scaled, "missing": missing}
    return case if name else {k: v for k, v in case.items() if k != "name"}


def _norm(name, *, rows, dim, dtype, param, grad=False):
    case = {"name": name, "op": "norm_grad" if grad else "norm", "rows": rows, "dim": dim, "dtype": dtype,
            "param": param, "eps": 1e-5}
    return case if name else {k: v for k, v in case.items() if k != "name"}


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm; odd and even alike."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    other = rng.choice([dtype, "float32"])
    grad = rng.random() < 0.5
    if rng.random() < 0.4:  # layer norm: rows short and long, one to many
        dim = _log(rng, 8, 16384)
        most = (134217728 if grad else 268435456) // SIZE[dtype] * 2
        return _norm("", rows=_log(rng, 1, max(1, min(262144, most // dim))), dim=dim, dtype=dtype, param=other,
                     grad=grad)
    if rng.random() < 0.5:  # a lookup
        dim = _log(rng, 16, 4096)
        vocab = _log(rng, 256, min(131072, 134217728 // dim))
        return _embed("", grad=grad, rows=_log(rng, 1, min(65536, 33554432 // dim)), per_row=1, vocab=vocab, dim=dim,
                      dtype=dtype, out=other, index=rng.choice(["int32", "int64"]), scale=math.sqrt(dim),
                      tokens=rng.choice(["zipf", "uniform"]), missing=rng.choice([0.0, 0.3]))
    per_row = _log(rng, 2, 2000)  # bags of leaves
    dim = _log(rng, 1, 256)
    vocab = per_row * rng.choice([16, 64, 256]) if per_row <= 500 else per_row * rng.choice([16, 64])
    rows = _log(rng, 1, max(1, min(262144, 26214400 // per_row, 1677721600 // 2 // (per_row * dim))))
    return _embed("", grad=grad, rows=rows, per_row=per_row, vocab=vocab, dim=dim, dtype=dtype, out=other,
                  index=rng.choice(["int32", "int64"]), scale=rng.uniform(0.05, 1.0), tokens="leaf",
                  scaled=rng.random() < 0.5, missing=rng.choice([0.0, 0.1]))


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    dtype = getattr(torch, case["dtype"])
    rows, dim = case["rows"], case["dim"]
    s = {"case": case}
    if case["op"] in ("norm", "norm_grad"):
        param = getattr(torch, case["param"])
        # Activations: features of different means and spreads, rows of different magnitude.
        x = normal(rows, dim) * (0.5 + torch.rand(dim, generator=g, device=dev)) + 0.3 * normal(dim)
        s["x"] = (x * torch.exp(0.3 * normal(rows, 1))).to(dtype)
        s["weight"] = (1.0 + 0.1 * normal(dim)).to(param)
        s["bias"] = (0.1 * normal(dim)).to(param)
        if case["op"] == "norm_grad":
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = 1.0 / torch.sqrt((x - s["mean"][:, None]).square().mean(1) + case["eps"])
            s["grad"] = normal(rows, dim).to(dtype)
        return s
    per_row, vocab = case["per_row"], case["vocab"]
    u = torch.rand(rows, per_row, generator=g, device=dev, dtype=torch.float64 if rows < 65536 else torch.float32)
    if case["tokens"] == "leaf":  # column t holds leaves of tree t, some of them common
        leaves = vocab // per_row
        k = (u ** 1.5 * leaves).long().clamp_(max=leaves - 1) + leaves * torch.arange(per_row, device=dev)
    elif case["tokens"] == "zipf":  # rank k about 1 / k, the ranks in any order
        k = torch.randperm(vocab, generator=g, device=dev)[(vocab ** u).long().sub_(1).clamp_(0, vocab - 1)]
    else:
        k = (u * vocab).long().clamp_(max=vocab - 1)
    if case["missing"]:
        k = torch.where(torch.rand(rows, per_row, generator=g, device=dev) < case["missing"], -1, k)
    s["tokens"] = k.to(getattr(torch, case["index"]))
    if per_row == 1:
        s["tokens"] = s["tokens"].reshape(rows)
    s["token_scale"] = 0.5 + torch.rand(rows, per_row, generator=g, device=dev) if case["scaled"] else None
    if case["op"] == "embedding" or case["scaled"]:
        s["table"] = (0.05 * normal(vocab, dim)).to(dtype)
    if case["op"] == "embedding_grad":
        s["grad"] = normal(rows, dim).to(dtype)
    return s


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


# -- the plain forms: 32 bits, rounded once at the end -------------------------------


def _bags(s, case):
    """Tokens as [rows, per_row], 0 where missing, and each one's factor, 0 where missing."""
    k = s["tokens"].reshape(case["rows"], case["per_row"]).long()
    factor = torch.full_like(k, case["scale"], dtype=torch.float32)
    if s["token_scale"] is not None:
        factor = factor * s["token_scale"]
    return k.clamp(min=0), torch.where(k >= 0, factor, torch.zeros_like(factor))


def _plain_embedding(s, case):
    k, factor = _bags(s, case)
    y = (s["table"][k].float() * factor[:, :, None]).sum(1)
    return y.to(getattr(torch, case["out"]))


def _plain_embedding_grad(s, case):
    k, factor = _bags(s, case)
    grad = s["grad"].float()
    terms = (grad[:, None, :] * factor[:, :, None]).reshape(-1, case["dim"])
    table = torch.zeros(case["vocab"], case["dim"], device=grad.device).index_add_(0, k.reshape(-1), terms)
    table = table.to(getattr(torch, case["out"]))
    if s["token_scale"] is None:
        return table
    by_scale = (s["table"][k].float() * grad[:, None, :]).sum(2) * case["scale"]
    valid = s["tokens"].reshape(case["rows"], case["per_row"]) >= 0
    return table, torch.where(valid, by_scale, torch.zeros_like(by_scale))


def _plain_norm(s, case):
    x = s["x"].float()
    mean = x.mean(1)
    centred = x - mean[:, None]
    rstd = 1.0 / torch.sqrt(centred.square().mean(1) + case["eps"])
    y = centred * rstd[:, None] * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean, rstd


def _plain_norm_grad(s, case):
    h = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    grad = s["grad"].float()
    gw = grad * s["weight"].float()
    dx = (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True)) * s["rstd"][:, None]
    param = s["weight"].dtype
    return dx.to(s["x"].dtype), (grad * h).sum(0).to(param), grad.sum(0).to(param)


_plain = {"embedding": _plain_embedding, "embedding_grad": _plain_embedding_grad, "norm": _plain_norm,
          "norm_grad": _plain_norm_grad}


# -- the framework's operators ----------------------------------------------------


def _nn():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xgboost-metal_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from xgboost import nn
    global _nn

    def _nn():
        return nn
    return nn


def _own_embedding(s, case):
    return _nn().embedding(s["tokens"], s["table"], scale=case["scale"], token_scale=s["token_scale"],
                           bag=case["per_row"] > 1, out_dtype=getattr(torch, case["out"]))


def _own_embedding_grad(s, case):
    bag = case["per_row"] > 1
    table = _nn().embedding_backward(s["grad"], s["tokens"], case["vocab"], scale=case["scale"],
                                     token_scale=s["token_scale"], bag=bag, out_dtype=getattr(torch, case["out"]))
    if s["token_scale"] is None:
        return table
    return table, _nn().embedding_scale_backward(s["grad"], s["tokens"], s["table"], scale=case["scale"], bag=bag)


def _own_norm(s, case):
    return _nn().layer_norm(s["x"], s["weight"], s["bias"], eps=case["eps"])


def _own_norm_grad(s, case):
    return _nn().layer_norm_backward(s["grad"], s["x"], s["mean"], s["rstd"], s["weight"])


_own = {"embedding": _own_embedding, "embedding_grad": _own_embedding_grad, "norm": _own_norm,
        "norm_grad": _own_norm_grad}


# -- what a pass cannot do without -----------------------------------------------


def work(case):
    rows, dim, e = case["rows"], case["dim"], SIZE[case["dtype"]]
    if case["op"] == "norm":
        return {"bytes": 2 * rows * dim * e + 2 * dim * SIZE[case["param"]] + 8 * rows, "flops": 8 * rows * dim}
    if case["op"] == "norm_grad":
        return {"bytes": 3 * rows * dim * e + 3 * dim * SIZE[case["param"]] + 8 * rows, "flops": 14 * rows * dim}
    count, out = rows * case["per_row"], SIZE[case["out"]]
    total = count * (SIZE[case["index"]] + (4 if case["scaled"] else 0))
    flops = 2 * count * dim
    if case["op"] == "embedding":
        total += min(case["vocab"], count) * dim * e + rows * dim * out
    else:
        total += rows * dim * e + case["vocab"] * dim * out
        if case["scaled"]:
            total += min(case["vocab"], count) * dim * e + 4 * count
            flops *= 2
    return {"bytes": total, "flops": flops}


# -- the definition in 64 bits -----------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "norm":
        x = s["x"].to(d)
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + case["eps"]).pow(-0.5)
        return torch.addcmul(s["bias"].to(d), (x - mean[:, None]) * s["weight"].to(d), rstd[:, None]), mean, rstd
    if case["op"] == "norm_grad":
        # With n = dim, by the Jacobian's three terms: dx = q w dy - q 1 (w.dy) / n - q h (w h.dy) / n.
        q = s["rstd"].to(d)[:, None]
        h = s["x"].to(d).sub_(s["mean"].to(d)[:, None]).mul_(q)
        grad, w = s["grad"].to(d), s["weight"].to(d)
        a, b = grad @ w / case["dim"], (grad * h) @ w / case["dim"]
        dw, db = torch.einsum("rn,rn->n", grad, h), torch.ones(case["rows"], dtype=d, device=q.device) @ grad
        return (grad * w - a[:, None] - h * b[:, None]) * q, dw, db
    rows, dim = case["rows"], case["dim"]
    k = s["tokens"].reshape(rows, -1).long()
    scales = s["token_scale"]
    if case["op"] == "embedding":
        table = s["table"].to(d)
        y = torch.zeros(rows, dim, dtype=d, device=k.device)
        for t in range(k.shape[1]):  # one column of tokens at a time, the present ones only
            at = (k[:, t] >= 0).nonzero()[:, 0]
            v = table.index_select(0, k[at, t])
            y[at] += v if scales is None else v * scales[at, t].to(d)[:, None]
        return y * case["scale"]
    grad = s["grad"].to(d)
    out = torch.zeros(case["vocab"], dim, dtype=d, device=k.device)
    by_scale = torch.zeros(rows, k.shape[1], dtype=d, device=k.device)
    for t in range(k.shape[1]):
        at = (k[:, t] >= 0).nonzero()[:, 0]
        g = grad[at] * case["scale"]
        if scales is not None:
            by_scale[at, t] = torch.einsum("rd,rd->r", g, s["table"][k[at, t]].to(d))
            g = g * scales[at, t].to(d)[:, None]
        out.index_add_(0, k[at, t], g)
    return out if scales is None else (out, by_scale)
