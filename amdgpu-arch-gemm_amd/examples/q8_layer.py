"""Trains and serves one layer with 8-bit products: y = norm(x + r) W^T + b.

    python amdgpu-arch-gemm_amd/examples/q8_layer.py [--tokens 512] [--features 256] [--channels 192] [--steps 30]

A teacher layer gives the targets.  Each training step keeps the master weights in
float32, quantises them, and runs the layer forward and backward:

    rmsnorm            hidden = x + r, and its norm in 8 bits: the product's
                       operand, and the checkpoint for the backward pass
    gemm               y, in 8-bit integers
    grad_weight        from the checkpoint
    grad_input         from the 8-bit weights
    rmsnorm_backward   the gradients of x (and r) and of the gain

Afterwards one token at a time runs through norm and product as in decoding, and must
give the rows of the whole batch.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from shim import q8_shim as Q  # noqa: E402

EPS = 1e-5


class Layer:
    """The layer's parameters, and the device memory of a batch of at most `tokens`."""

    def __init__(self, tokens: int, features: int, channels: int, seed: int):
        rng = np.random.default_rng(seed)
        self.m, self.k, self.n = tokens, features, channels
        self.weight = rng.normal(0, features ** -0.5, (channels, features)).astype(np.float32)
        self.gain = np.ones(features, np.float32)
        self.bias = np.zeros(channels, np.float32)
        self.ops = Q.Ops()
        m, k, n = tokens, features, channels
        ldq = self.ldq = Q.row_bytes(k)
        self.hidden, self.qx = Q.Array(m, k, Q.BF16), Q.Array(m, k, "int8", ldq)
        self.sx, self.rstd = Q.Array(1, m, Q.F32), Q.Array(1, m, Q.F32)
        self.qw, self.sw = Q.Array(n, k, "int8", ldq), Q.Array(1, n, Q.F32)
        self.y, self.dn, self.dx = Q.Array(m, n, Q.BF16), Q.Array(m, k, Q.BF16), Q.Array(m, k, Q.BF16)
        self.dw, self.dgain = Q.Array(n, k, Q.F32), Q.Array(1, k, Q.F32)
        self.upload()

    def upload(self):
        """Master parameters to the device, the weights in 8 bits with a scale for each channel."""
        weight = Q.Array.of(self.weight)
        self.ops.quantize(Q.F32, weight, self.qw, self.sw, self.n, self.k, ldq=self.ldq)
        self.gain_device, self.bias_device = Q.Array.of(self.gain, Q.BF16), Q.Array.of(self.bias, Q.BF16)
        self.ops.synchronize()

    def forward(self, x: Q.Array, r: Q.Array, rows: int):
        self.ops.rmsnorm(Q.BF16, x, r, self.gain_device, self.hidden, self.qx, self.sx, self.rstd, rows, self.k, EPS,
                         ldq=self.ldq)
        self.ops.gemm(Q.BF16, self.qx, self.sx, self.qw, self.sw, self.bias_device, self.y, rows, self.n, self.k,
                      ldx=self.ldq, ldw=self.ldq)

    def backward(self, dy: Q.Array, rows: int):
        self.ops.grad_weight(Q.BF16, dy, self.qx, self.sx, Q.F32, self.dw, rows, self.n, self.k, ldx=self.ldq)
        self.ops.grad_input(Q.BF16, dy, self.qw, self.sw, self.dn, rows, self.n, self.k, ldw=self.ldq)
        self.ops.rmsnorm_backward(Q.BF16, self.dn, self.hidden, self.gain_device, self.rstd, None, self.dx, self.dgain,
                                  rows, self.k)

    def close(self):
        self.ops.close()


def train(tokens=512, features=256, channels=192, steps=30, rate=0.15, seed=0, report=print):
    """Returns the losses of the steps and the largest difference between decoding and the batch."""
    rng = np.random.default_rng(seed + 1)
    x = Q.from_bf16(Q.to_bf16(rng.normal(0, 1, (tokens, features)).astype(np.float32)))
    r = Q.from_bf16(Q.to_bf16(rng.normal(0, 1, (tokens, features)).astype(np.float32)))
    h = x + r
    normed = h / np.sqrt((h ** 2).mean(axis=1, keepdims=True) + EPS) * (1 + 0.3 * rng.normal(0, 1, features))
    target = normed @ rng.normal(0, features ** -0.5, (channels, features)).T + 0.1 * rng.normal(0, 1, channels)
    layer = Layer(tokens, features, channels, seed)
    try:
        dx_, dr_ = Q.Array.of(x, Q.BF16), Q.Array.of(r, Q.BF16)
        losses = []
        for step in range(steps):
            layer.forward(dx_, dr_, tokens)
            layer.ops.synchronize()
            error = layer.y.numpy() - target
            losses.append(float((error ** 2).mean()))
            dy = (error * (2.0 / tokens)).astype(np.float32)
            layer.backward(Q.Array.of(dy, Q.BF16), tokens)
            layer.ops.synchronize()
            layer.weight -= rate * layer.dw.numpy()
            layer.gain -= rate / features * layer.dgain.numpy()[0]
            layer.bias -= rate * 0.1 * dy.sum(axis=0)
            layer.upload()
            report(f"step {step}: loss {losses[-1]:.5f}")
        # decoding: the same rows, one at a time
        layer.forward(dx_, dr_, tokens)
        layer.ops.synchronize()
        batch = layer.y.numpy().copy()
        worst = 0.0
        for i in range(min(tokens, 4)):
            layer.forward(Q.Array.of(x[i], Q.BF16), Q.Array.of(r[i], Q.BF16), 1)
            layer.ops.synchronize()
            worst = max(worst, float(np.abs(layer.y.numpy()[0] - batch[i]).max()))
        report(f"one token at a time: largest difference from the batch {worst}")
        return losses, worst
    finally:
        layer.close()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--features", type=int, default=256)
    ap.add_argument("--channels", type=int, default=192)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--rate", type=float, default=0.15)
    a = ap.parse_args()
    losses, worst = train(a.tokens, a.features, a.channels, a.steps, a.rate)
    if not (losses[-1] < losses[0] and worst == 0.0):
        sys.exit("the layer did not learn, or decoding differs from the batch")


if __name__ == "__main__":
    main()
