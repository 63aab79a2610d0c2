"""Scores tokens with a small residual network whose inner layers have 4-bit
weights, and takes the gradient of the scores to its last norm.

    python examples/score_tokens.py [--rows 256] [--hidden 1024] [--inner 4096] [--vocabulary 50256] [--blocks 2]

Each block is  x = x + down(relu(up(norm(x))))  with the norm's output in 8 bits
and both layers in 4-bit weights:

    rms_norm_launch    x (+ the last block's result) -> int8 rows and their scales
    q4_dense_launch    up, the scales applied, bias and ReLU fused
    q4_dense_launch    down, back in f32

and at the end, in f32, the norm, the vocabulary's layer (dense_launch) and
token_logprobs_launch: log probabilities, entropy, the likeliest alternatives.
``gradient`` goes back through token_logprobs_backward_launch, the vocabulary's
layer and rms_norm_backward_launch, as a policy-gradient step on the last norm
with the 4-bit layers kept fixed does. Weights are random: no checkpoint is read.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ml-edsl_amd"))
from mlir_edsl_hip import _native, device, lm  # noqa: E402


class Scorer:
    """The network. Buffers are made once for `rows` rows; every call reuses them."""

    def __init__(self, rows, hidden, inner, vocabulary, blocks, top=5, group_size=128, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *s, by=1.0: torch.randn(*s, device="cuda", generator=g) * by  # noqa: E731
        quantized = lambda K, N: lm.q4_quantize(normal(K, N, by=K ** -0.5), group_size)  # noqa: E731
        self.norms = [1 + normal(hidden, by=0.1) for _ in range(blocks + 1)]
        self.plain = [(quantized(hidden, inner), normal(inner, by=0.1), quantized(inner, hidden)) for _ in range(blocks)]
        self.layers = [(lm.q4_pack(*up, group_size), b, lm.q4_pack(*down, group_size)) for up, b, down in self.plain]
        self.head = normal(hidden, vocabulary, by=2 * hidden ** -0.5)
        self.head_t = self.head.t().contiguous()
        self.group_size = group_size
        f32 = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        self.q, self.scales = torch.empty(rows, hidden, dtype=torch.int8, device="cuda"), f32(rows)
        self.h, self.result, self.inner = f32(rows, hidden), f32(rows, hidden), f32(rows, inner)
        self.y, self.rstd, self.logits = f32(rows, hidden), f32(rows), f32(rows, vocabulary)
        self.logprobs, self.lse, self.entropy = f32(rows), f32(rows), f32(rows)
        self.top, self.top_ids = f32(rows, top), torch.empty(rows, top, dtype=torch.int64, device="cuda")
        self.dlogits, self.dy, self.dh, self.dweight = f32(rows, vocabulary), f32(rows, hidden), f32(rows, hidden), f32(hidden)

    def score(self, X, tokens):
        """Log probabilities of `tokens` [rows] (-1: padding) after the states X [rows, hidden]."""
        x, result = X, None
        for weight, (up, bias, down) in zip(self.norms, self.layers):
            lm.rms_norm_launch(x, weight, self.q, residual=result, total=self.h, scales=self.scales)
            lm.q4_dense_launch(self.q, up, bias, self.inner, _native.EPI_BIAS_RELU, x_scales=self.scales)
            lm.q4_dense_launch(self.inner, down, None, self.result)
            x, result = self.h, self.result
        lm.rms_norm_launch(x, self.norms[-1], self.y, residual=result, total=self.h, rstd=self.rstd)
        device.dense_launch(self.y, self.head, None, self.logits, _native.EPI_NONE)
        lm.token_logprobs_launch(self.logits, tokens, self.logprobs, self.lse, self.entropy, self.top, self.top_ids)
        return self.logprobs

    def gradient(self, tokens, dlogprobs, dentropy=None):
        """After ``score``: the gradients of the last norm's weight and of the state
        before it, given those of the log probabilities and entropies."""
        lm.token_logprobs_backward_launch(self.logits, tokens, self.lse, self.dlogits, dlogprobs,
                                          self.entropy if dentropy is not None else None, dentropy)
        device.dense_launch(self.dlogits, self.head_t, None, self.dy, _native.EPI_NONE)
        lm.rms_norm_backward_launch(self.dy, self.h, self.norms[-1], self.rstd, self.dh, self.dweight)
        return self.dweight, self.dh


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("rows", 256), ("hidden", 1024), ("inner", 4096), ("vocabulary", 50256), ("blocks", 2)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = p.parse_args()
    net = Scorer(a.rows, a.hidden, a.inner, a.vocabulary, a.blocks)
    g = torch.Generator(device="cuda").manual_seed(1)
    X = torch.randn(a.rows, a.hidden, device="cuda", generator=g)
    tokens = torch.randint(0, a.vocabulary, (a.rows,), device="cuda", generator=g)
    net.score(X, tokens)
    net.gradient(tokens, torch.full((a.rows,), -1.0 / a.rows, device="cuda"))
    torch.cuda.synchronize()
    print(f"{a.rows} tokens: mean log probability {net.logprobs.mean():.4f}, entropy {net.entropy.mean():.4f}")
    print("first row's likeliest:", ", ".join(f"{i} ({v.exp():.4f})" for i, v in zip(net.top_ids[0].tolist(), net.top[0])))
    print(f"gradient of the last norm's weight: length {net.dweight.norm():.3e}")
    for name, call in (("score", lambda: net.score(X, tokens)),
                       ("gradient", lambda: net.gradient(tokens, net.logprobs))):
        for _ in range(20):
            call()
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(100):
            call()
        torch.cuda.synchronize()
        print(f"{name}: {(time.perf_counter() - start) * 1e4:.1f} us a pass")


if __name__ == "__main__":
    main()
