"""Trains a small token model whose weights are stored in FP8 or FP4.

    python examples/token_model.py [--dtype e4m3|e5m2|e2m1] [--steps N]

The model predicts each token from the one before it: an embedding table, a
residual Linear layer and the loss over the vocabulary on the same table, all on
quantized weights with fp32 masters.  One step is: lookup, Linear, loss without
stored logits, the three layers' gradients (the table's two added together),
clipping by their global norm, AdamW with re-quantization.  The data are a random
chain in which every token has four likely successors; the loss falls towards
that chain's entropy.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from novann_amd import optim  # noqa: E402
from novann_amd.module import Embedding, Linear, LinearCrossEntropy  # noqa: E402

FOLLOWERS = 4


class TokenModel:
    def __init__(self, vocab: int, width: int, dtype: str):
        def small(shape):
            return np.random.standard_normal(shape) / np.sqrt(width)
        self.embed = Embedding(vocab, width, init=small, weight_dtype=dtype,
                               factor=float(np.sqrt(width)), tied=True)
        self.mix = Linear(width, width, init=small, weight_dtype=dtype)
        self.head = LinearCrossEntropy(width, vocab, weight=self.embed.weight)

    def parameters(self):
        return self.embed.parameters() + self.mix.parameters() + self.head.parameters()

    def loss(self, tokens, targets):
        h = self.embed(tokens)
        return self.head(h + self.mix(h), targets)

    def backward(self):
        g = self.head.backward()            # sets the table's gradient,
        self.embed.backward(g + self.mix.backward(g))  # which this one adds to


def chain(rng, vocab: int):
    """The successors of each token."""
    return rng.integers(0, vocab, (vocab, FOLLOWERS))


def train(vocab=2000, width=128, batch=4096, steps=60, dtype="e4m3", lr=0.02, max_norm=1.0,
          seed=0, log=None):
    """The losses and gradient norms of the steps."""
    np.random.seed(seed)
    rng = np.random.default_rng(seed)
    after = chain(rng, vocab)
    model = TokenModel(vocab, width, dtype)
    opt = optim.AdamW(model.parameters(), lr=lr, weight_decay=0.0)
    losses, norms = [], []
    for step in range(steps):
        tokens = rng.integers(0, vocab, batch)
        targets = after[tokens, rng.integers(0, FOLLOWERS, batch)]
        loss = model.loss(torch.from_numpy(tokens).cuda(), torch.from_numpy(targets).cuda())
        model.backward()
        norms.append(optim.clip_grad_norm(model.parameters(), max_norm))
        opt.step()
        losses.append(loss)
        if log and (step % 10 == 9 or step == 0):
            log(f"step {step + 1:4d}  loss {float(loss):.3f}  gradient norm {float(norms[-1]):.3f}")
    return [float(v) for v in losses], [float(v) for v in norms]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--dtype", default="e4m3", choices=("e4m3", "e5m2", "e2m1"))
    ap.add_argument("--steps", type=int, default=60)
    a = ap.parse_args()
    train(dtype=a.dtype, steps=a.steps, log=print)
    print(f"entropy of the data: {np.log(FOLLOWERS):.3f}")
