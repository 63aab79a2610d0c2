"""The language-model operators in 64 bits, from their definitions, on the CPU."""
from __future__ import annotations

import math

import torch

#: Half a unit in the last place of 1, of each type: what one rounding may cost.
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
#: The smallest step of each type near zero.
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def d(t):
    return None if t is None else t.detach().cpu().double()


def as_f32(v):
    """A number argument as the entry points take it."""
    return float(torch.tensor(v, dtype=torch.float32))


def rms_norm(x, weight, residual=None, eps=1e-6):
    h = d(x) if residual is None else d(x) + d(residual)
    rstd = (h.square().mean(1) + eps) ** -0.5
    return h * rstd[:, None] * d(weight), h, rstd


def rms_norm_backward(dy, h, weight, rstd, dh=None):
    dy, h, rstd = d(dy), d(h), d(rstd)[:, None]
    t, xh = dy * d(weight), h * rstd
    dx = rstd * (t - xh * (t * xh).mean(1, keepdim=True))
    return dx if dh is None else dx + d(dh), (dy * xh).sum(0)


def token_logprobs(logits, tokens, k=0, scale=1.0):
    """logprobs, lse, entropy, top values, top ids: by the rules of
    include/edsl_hip_lm.h for masked rows, padding and rows without probabilities."""
    scale = as_f32(scale)
    x = d(logits)
    l = scale * x
    M, V = l.shape
    bad = torch.isnan(l).any(1) | (l == math.inf).any(1)
    none = ~bad & (l == -math.inf).all(1)
    logp = torch.log_softmax(torch.where((bad | none)[:, None], 0.0, l), 1)
    lse = torch.logsumexp(torch.where(bad[:, None], 0.0, l), 1)
    entropy = -torch.where(logp > -math.inf, logp.exp() * logp, 0.0).sum(1)
    logp[none], lse[none], entropy[none] = -math.inf, -math.inf, 0.0
    logp[bad], lse[bad], entropy[bad] = math.nan, math.nan, math.nan
    lp = torch.zeros(M, dtype=torch.float64)
    if tokens is not None:
        tokens = tokens.cpu().long()
        given = (tokens >= 0) & (tokens < V)
        lp = torch.where(given, logp[torch.arange(M), torch.where(given, tokens, 0)], 0.0)
    # Falling, equal ones by their index: a stable sort of no more than the values that can matter.
    ids = torch.empty(M, k, dtype=torch.int64)
    if k:
        least = torch.where(bad[:, None], 0.0, x).topk(k, 1).values[:, -1:]
        for r in range(M):
            some = (x[r] >= least[r]).nonzero()[:, 0] if not bad[r] else torch.arange(k)
            ids[r] = some[torch.sort(x[r, some], descending=True, stable=True).indices[:k]]
    top = logp.gather(1, ids) if k else torch.empty(M, 0, dtype=torch.float64)
    ids[bad] = -1
    return lp, lse, entropy, top, ids


def token_logprobs_backward(logits, tokens, lse, dlogprobs=None, entropy=None, dentropy=None, scale=1.0):
    scale = as_f32(scale)
    l, lse = scale * d(logits), d(lse)[:, None]
    M, V = l.shape
    some = lse > -math.inf
    p = torch.where(some & (l > -math.inf), (l - lse).exp(), 0.0)
    out = torch.zeros_like(l)
    if dlogprobs is not None:
        tokens = tokens.cpu()
        given = (tokens >= 0) & (tokens < V)
        g = torch.where(given, d(dlogprobs), 0.0)[:, None]
        out -= p * g
        out[torch.arange(M), torch.where(given, tokens, 0)] += g[:, 0]
    if dentropy is not None:
        out -= d(dentropy)[:, None] * torch.where(p > 0, p * (l - lse + d(entropy)[:, None]), 0.0)
    return torch.where(some, scale * out, 0.0)
