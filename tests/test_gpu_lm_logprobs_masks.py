"""Log probabilities of rows with finite masks: large negative logits in place of
-inf, by runs and at random, and rows of nothing but equal large logits.

Tolerance. A logit enters as u = scale (x - m), m the row's largest, with a few
roundings of 2^-24 of |u| (and of 8 at most, what the rounding of the product that is
taken off leaves over). Weighed by the probabilities p the |u| sum up to no more than
the entropy, and so to log V: 8 * 2^-24 * (8 + log V) for the sums, and 40 * 2^-24 of
1 + |result| for the logarithm, the products with scale and the result itself (a
token's |u| is no more than its |log probability|)."""
import math

import pytest
import torch

import lm_reference as ref
from mlir_edsl_hip import lm

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
MASKS = (-1e4, -1e8, -1e9, -1e10, -1e14, -1e20, -1e30, -1e36)


def rows(V, dtype):
    """Eight patterns for each mask, on logits of size 3, and their tokens."""
    g = torch.Generator().manual_seed(V)
    x = 3.0 * torch.randn(len(MASKS), 8, V, generator=g)
    for i, mask in enumerate(MASKS):
        x[i, 0, V // 2:] = mask
        x[i, 1, torch.rand(V, generator=g) < 0.95] = mask
        x[i, 2] = mask
        x[i, 3, 1:] = mask
        x[i, 4, :-1] = mask
        x[i, 5, : V // 3] = 2 * mask
        x[i, 6, V // 5] = -mask
        x[i, 7] = -mask
    tokens = torch.randint(0, V, (len(MASKS) * 8,), generator=g)
    return x.flatten(0, 1).to(dtype), tokens


def same(got, want, V):
    got = ref.d(got)
    assert not torch.isnan(got).any()
    worst = float(((got - want).abs() - 8 * U * (8 + math.log(V)) - 40 * U * (1 + want.abs())).max())
    assert worst <= 0, worst


@pytest.mark.parametrize("scale", [0.7, 1.0, 1.25])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,copies,k", [(777, 1, 5), (4000, 1, 0), (4000, 6, 8), (40000, 1, 8), (300000, 1, 8)])
def test_finite_masks(V, copies, k, dtype, scale):
    x, tokens = rows(V, dtype)
    want = ref.token_logprobs(x, tokens, k, scale)
    x, tokens = x.cuda().repeat(copies, 1), tokens.cuda().repeat(copies)
    M = x.shape[0]
    lp, lse, entropy = (torch.full((M,), 7.0, device="cuda") for _ in range(3))
    top = torch.full((M, k), 7.0, device="cuda") if k else None
    ids = torch.full((M, k), 77, device="cuda") if k else None
    lm.token_logprobs_launch(x, tokens, lp, lse, entropy, top, ids, scale=scale)
    if k:
        assert torch.equal(ids.cpu(), want[4].repeat(copies, 1))
        same(top, want[3].repeat(copies, 1), V)
    for got, value in ((lp, want[0]), (lse, want[1]), (entropy, want[2])):
        same(got, value.repeat(copies), V)
