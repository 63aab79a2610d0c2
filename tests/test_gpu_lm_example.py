"""The operators together, as examples/score_tokens.py runs them, against 64 bits.

Tolerance: sums are 32-bit everywhere, so what is larger than their rounding is
an 8-bit code of a norm that falls to the other side of a half: it moves one of
`hidden` values by 1/127 of the row's largest, some 4 of its root mean square,
and so a block's result by 4 / (127 sqrt(hidden)) of its size, the logits (of
size 2 here) by up to that for each of the 3 blocks' terms, 4 sizes for the
largest of many: 2 * 4 * 3 * 4 / (127 sqrt(hidden)) for a flip a row and block."""
import importlib.util
import math
import os

import pytest
import torch

import lm_reference as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("score_tokens", os.path.join(ROOT, "examples", "score_tokens.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def in_64_bits(net, X, tokens, k):
    def layer(x, quantized):
        q, s, z = quantized
        at = torch.arange(q.shape[0]) // net.group_size
        return x @ ((ref.d(q) - ref.d(z)[at]) * ref.d(s)[at])

    x = ref.d(X)
    for weight, (up, b, down) in zip(net.norms, net.plain):
        y, x, _ = ref.rms_norm(x, weight)
        scale = y.abs().amax(1, keepdim=True) / 127
        y = (y / scale).round() * scale
        x = x + layer((layer(y, up) + ref.d(b)).clamp(min=0), down)
    y, h, rstd = ref.rms_norm(x, net.norms[-1])
    logits = y @ ref.d(net.head)
    return logits, h, rstd, ref.token_logprobs(logits, tokens, k)


@pytest.mark.parametrize("rows,hidden,inner,vocabulary,group", [(1, 256, 640, 1000, 128), (33, 192, 300, 777, 32)])
def test_scores_and_gradient(example, rows, hidden, inner, vocabulary, group):
    k = 5
    net = example.Scorer(rows, hidden, inner, vocabulary, blocks=2, top=k, group_size=group)
    g = torch.Generator().manual_seed(3)
    X = torch.randn(rows, hidden, generator=g).cuda()
    tokens = torch.randint(0, vocabulary, (rows,), generator=g).cuda()
    tokens[-1:] = tokens[-1:] if rows == 1 else -1
    dlogprobs, dentropy = torch.randn(rows, generator=g).cuda(), torch.randn(rows, generator=g).cuda()
    net.score(X, tokens)
    dweight, dh = net.gradient(tokens, dlogprobs, dentropy)
    logits, h, rstd, (lp, lse, entropy, top, ids) = in_64_bits(net, X, tokens, k)
    flip = 2 * 4 * 3 * 4 / (127 * math.sqrt(hidden))
    assert float((ref.d(net.logits) - logits).abs().max()) <= flip
    # A change of each logit by `flip` moves lse by that, log probabilities by twice that.
    for got, want in ((net.logprobs, lp), (net.lse, lse), (net.top, top)):
        assert float((ref.d(got) - want).abs().max()) <= 2 * flip
    assert float((ref.d(net.entropy) - entropy).abs().max()) <= 2 * flip * math.log(vocabulary)
    # From the logits and states that the network had, the rest is 32-bit arithmetic.
    dlogits = ref.token_logprobs_backward(net.logits, tokens, ref.d(net.lse), dlogprobs, net.entropy, dentropy)
    dx, dw = ref.rms_norm_backward(dlogits @ ref.d(net.head).t(), net.h, net.norms[-1], net.rstd)
    for got, want in ((dh, dx), (dweight, dw)):
        assert float((ref.d(got) - want).norm()) <= 1e-4 * float(want.norm())
    assert float((ref.d(net.h) - h).abs().max()) <= 2 * flip
