"""A pre-norm feed-forward block: trained with its inputs kept in 8 bits, then
served in 8 bits.

    h = x + residual;  y = h + W2 silu(W1 norm(h) + b1) + b2

Run from the repository's root:  python examples/feedforward_block.py
"""
from __future__ import annotations

import pathlib
import sys

import numpy as np

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))

import train_station_amd as T  # noqa: E402

EPS = 1e-6


def tensor(a) -> T.Tensor:
    a = np.ascontiguousarray(a, np.float32)
    return T.Tensor.from_slice(a, a.shape)


class Block:
    """The block's parameters and its two passes."""

    def __init__(self, width: int, hidden: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        self.norm = tensor(np.ones(width))
        self.w1 = tensor(rng.standard_normal((width, hidden)) * width ** -0.5)
        self.b1 = tensor(np.zeros(hidden))
        self.w2 = tensor(rng.standard_normal((hidden, width)) * hidden ** -0.5)
        self.b2 = tensor(np.zeros(width))
        for p in self.parameters():
            p.with_requires_grad()

    def parameters(self):
        return [self.norm, self.w1, self.b1, self.w2, self.b2]

    def forward(self, x: T.Tensor, residual: T.Tensor) -> T.Tensor:
        """In full, as it is trained: each layer keeps its input in 8 bits."""
        y, stream = x.add_rms_norm(residual, self.norm, EPS)
        y = y.linear(self.w1, bias=self.b1, activation="silu", checkpoint="8bit")
        return y.linear(self.w2, bias=self.b2, residual=stream, checkpoint="8bit")

    def packed(self):
        """The weights in 8 bits, laid out once for serving ([fan_out, fan_in])."""
        with T.NoGradTrack():
            return self.w1.t().contiguous().pack8(), self.w2.t().contiguous().pack8()

    def serve(self, weights, x: T.Tensor, residual: T.Tensor) -> T.Tensor:
        """In 8 bits: the norm's output and the layers' inputs and weights."""
        with T.NoGradTrack():
            y, stream = x.add_rms_norm_packed(residual, self.norm, EPS)
            y = y.linear(weights[0], bias=self.b1, activation="silu").pack8()
            return y.linear(weights[1], bias=self.b2, residual=stream)


def train(block: Block, x, residual, target, steps: int, lr: float = 1e-3):
    """Adam on the mean squared error; the losses."""
    opt = T.Adam.with_learning_rate(lr)
    opt.add_parameters(block.parameters())
    losses = []
    for _ in range(steps):
        d = block.forward(x, residual).sub_tensor(target)
        loss = d.mul_tensor(d).mean()
        loss.backward()
        opt.step(block.parameters())
        opt.zero_grad(block.parameters())
        T.clear_gradients()
        losses.append(loss.value())
    return losses


def main(width: int = 512, hidden: int = 1024, batch: int = 256, steps: int = 30):
    rng = np.random.default_rng(1)
    x, residual = (tensor(rng.standard_normal((batch, width))) for _ in range(2))
    target = tensor(rng.standard_normal((batch, width)))
    block = Block(width, hidden)
    losses = train(block, x, residual, target, steps)
    print(f"trained {steps} steps: loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    weights = block.packed()
    with T.NoGradTrack():
        full = block.forward(x, residual).data()
    served = block.serve(weights, x, residual).data()
    off = float(np.linalg.norm(served - full) / np.linalg.norm(full))
    print(f"served in 8 bits: {off:.3%} off the block in full")
    return losses, off


if __name__ == "__main__":
    main()
