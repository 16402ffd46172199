"""An embedding head on a binned matrix: many classes without a tree per class.

The rows of the binned matrix are lists of tokens (their global bins; a missing value has none). The head sums the
tokens' embeddings, norms the sum and takes the softmax cross entropy of a linear layer over the classes; a step of
gradient descent clips the gradients by their global norm. All of it runs in hessboost_b200.head's kernels.

    python examples/bin_head.py --rows 20000 --classes 500 --steps 60
"""

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import hessboost_b200 as H  # noqa: E402
from hessboost_b200 import head  # noqa: E402


def make_rows(rows, features, classes, seed=0):
    """Rows around one centre a class, 5% of the cells missing, and their classes."""
    rng = np.random.default_rng(seed)
    centres = rng.standard_normal((classes, features)).astype(np.float32)
    y = rng.integers(0, classes, rows)
    x = centres[y] + 0.3 * rng.standard_normal((rows, features)).astype(np.float32)
    x[rng.random(x.shape) < 0.05] = np.nan
    return x.astype(np.float32), y


class BinHead:
    """The parameters of a head on `n_tokens` global bins, and its step of gradient descent."""

    def __init__(self, n_tokens, classes, width=64, dtype=torch.float32, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)
        new = lambda *shape, by: (by * torch.randn(*shape, generator=g, device=device)).to(dtype)  # noqa: E731
        self.table = new(n_tokens, width, by=1.0)
        self.norm_weight = torch.ones(width, dtype=dtype, device=device)
        self.norm_bias = torch.zeros(width, dtype=dtype, device=device)
        self.weight = new(classes, width, by=width**-0.5)

    def parameters(self):
        return [self.table, self.norm_weight, self.norm_bias, self.weight]

    def loss(self, tokens, labels, row_ptr=None, scale=0.2):
        """Each row's loss; what the backward pass needs is kept in self.saved."""
        e = head.embed_forward(tokens, self.table, row_ptr=row_ptr, scale=scale)
        y, mean, rstd = head.layer_norm_forward(e, self.norm_weight, self.norm_bias)
        loss, lse = head.linear_xent_forward(y, self.weight, labels)
        self.saved = (tokens, row_ptr, scale, labels, e, mean, rstd, y, lse)
        return loss

    def gradients(self):
        """The gradients of the mean loss, in the parameters' order."""
        tokens, row_ptr, scale, labels, e, mean, rstd, y, lse = self.saved
        there = ((labels >= 0) & (labels < self.weight.shape[0])).sum()
        dloss = (1.0 / there.clamp(min=1).float()).expand(labels.numel())
        dy, dweight = head.linear_xent_backward(dloss, y, self.weight, labels, lse)
        de, dnorm_weight, dnorm_bias = head.layer_norm_backward(dy, e, self.norm_weight, mean, rstd)
        dtable = head.embed_backward(de, tokens, self.table.shape[0], row_ptr=row_ptr, scale=scale)
        return [dtable, dnorm_weight, dnorm_bias, dweight]

    def step(self, tokens, labels, rate, max_norm=1.0, row_ptr=None):
        """One step; the mean loss before it, on the device."""
        loss = self.loss(tokens, labels, row_ptr)
        grads = self.gradients()
        head.clip_grad_norm(grads, max_norm)
        for p, g in zip(self.parameters(), grads):
            p.add_(g, alpha=-rate)
        return loss.mean()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--rows", type=int, default=20000)
    ap.add_argument("--features", type=int, default=28)
    ap.add_argument("--classes", type=int, default=500)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--rate", type=float, default=20.0)
    ap.add_argument("--dtype", choices=("f32", "bf16"), default="f32")
    a = ap.parse_args(argv)
    x, y = make_rows(a.rows, a.features, a.classes)
    matrix = H.BinnedMatrix.from_dense(x, max_bin=32)
    tokens, row_ptr = head.bin_tokens(matrix)
    labels = torch.from_numpy(y).cuda()
    model = BinHead(int(matrix.feature_offset[-1]), a.classes, a.width,
                    torch.float32 if a.dtype == "f32" else torch.bfloat16)
    losses = []
    for step in range(a.steps):
        losses.append(model.step(tokens, labels, a.rate, row_ptr=row_ptr))
    losses = torch.stack(losses).tolist()
    for step in range(0, a.steps, max(1, a.steps // 10)):
        print(f"step {step:4d}  mean loss {losses[step]:.4f}")
    print(f"last       mean loss {losses[-1]:.4f}")
    return losses


if __name__ == "__main__":
    main()
