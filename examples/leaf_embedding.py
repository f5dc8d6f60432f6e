"""A learned model on top of a booster's leaves.

Trains a booster, numbers the leaves that each row reaches (xgboost.nn.leaf_tokens),
and fits a small head on the GPU in their place: a vector for every leaf, a row's
vectors summed (embedding), normalised (layer_norm) and projected to a margin. The
gradients run back through layer_norm_backward and embedding_backward; PyTorch
provides the arrays, the projection and the update (Adam).

    python examples/leaf_embedding.py [--rows 262144] [--trees 100] [--depth 8] [--dim 64] [--steps 60]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "xgboost-metal_b200"))
import xgboost as xgb  # noqa: E402
from xgboost import nn  # noqa: E402


class Head:
    """margin = layer_norm(scale * sum of the leaves' vectors) . v + c, the
    vectors in bfloat16 with a float32 copy that the updates go to."""

    def __init__(self, vocab, trees, dim, device, rate=0.02, seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        self.scale = trees ** -0.5
        self.master = torch.randn(vocab, dim, generator=g, device=device)
        self.table = self.master.to(torch.bfloat16)
        self.weight, self.bias = torch.ones(dim, device=device), torch.zeros(dim, device=device)
        self.v, self.c = torch.zeros(dim, device=device), torch.zeros((), device=device)
        self.optimizer = torch.optim.Adam((self.master, self.weight, self.bias, self.v, self.c), lr=rate)

    def forward(self, tokens):
        h = nn.embedding(tokens, self.table, scale=self.scale, bag=True, out_dtype=torch.float32)
        y, mean, rstd = nn.layer_norm(h, self.weight, self.bias)
        return y @ self.v + self.c, (tokens, h, y, mean, rstd)

    def backward(self, d_margin, saved):
        """The gradients of table, weight, bias, v and c."""
        tokens, h, y, mean, rstd = saved
        dy = torch.outer(d_margin, self.v)
        dh, d_weight, d_bias = nn.layer_norm_backward(dy, h, mean, rstd, self.weight)
        d_table = nn.embedding_backward(dh, tokens, len(self.table), scale=self.scale, bag=True)
        return d_table, d_weight, d_bias, y.t() @ d_margin, d_margin.sum()

    def step(self, tokens, labels):
        """One step down the mean logistic loss; the loss."""
        margin, saved = self.forward(tokens)
        loss = torch.nn.functional.softplus(margin) - labels * margin
        grads = self.backward((torch.sigmoid(margin) - labels) / len(labels), saved)
        for p, g in zip((self.master, self.weight, self.bias, self.v, self.c), grads):
            p.grad = g
        self.optimizer.step()
        self.table.copy_(self.master)
        return loss.mean()


def main(rows=262144, cols=32, trees=100, depth=8, dim=64, steps=60):
    """(log loss of the booster, of the head before and after its steps), on the training rows."""
    rng = np.random.default_rng(1337)
    X = rng.normal(size=(rows, cols)).astype(np.float32)
    logit = X @ rng.normal(size=cols) * 0.5 + X[:, 0] * X[:, 1]
    y = (rng.random(rows) < 1 / (1 + np.exp(-logit))).astype(np.float32)
    d = xgb.DMatrix(X, label=y)
    booster = xgb.train({"objective": "binary:logistic", "tree_method": "hist", "device": "cuda", "max_depth": depth},
                        d, trees)
    p = np.clip(booster.predict(d), 1e-7, 1 - 1e-7)
    trained = float(-np.mean(y * np.log(p) + (1 - y) * np.log(1 - p)))
    tokens, vocab = nn.leaf_tokens(booster, d)
    device = torch.device("cuda", 0)
    tokens, labels = torch.from_numpy(tokens).to(device), torch.from_numpy(y).to(device)
    head = Head(vocab, trees, dim, device)
    losses = [head.step(tokens, labels) for _ in range(steps)]
    first, last = float(losses[0]), float(losses[-1])
    print("booster %.4f, head %.4f -> %.4f (%d leaves, %d steps)" % (trained, first, last, vocab, steps))
    return trained, first, last


if __name__ == "__main__":
    a = argparse.ArgumentParser()
    for name, value in (("rows", 262144), ("trees", 100), ("depth", 8), ("dim", 64), ("steps", 60)):
        a.add_argument("--" + name, type=int, default=value)
    main(**vars(a.parse_args()))
