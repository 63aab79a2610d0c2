"""The 8-bit layer, the layer on groups of rows and sampling in 64 bits, from their
definitions."""
from __future__ import annotations

import math

import torch

from lm_reference import as_f32, d

ACTS = {0: "none", 1: "relu", 2: "leaky", 3: "if_relu"}


def activate(z, epilogue, alpha):
    act = ACTS[epilogue >> 1]
    if act == "none":
        return z
    if act == "leaky":
        return z.clamp(min=0) + as_f32(alpha) * z.clamp(max=0)
    if act == "relu":
        return torch.where((z > 0) | z.isnan(), z, 0.0)
    return torch.where(z > 0, z, 0.0)


def i8_dense(x, q, scales, x_scales=None, b=None, epilogue=0, alpha=0.0):
    """The result, and what its roundings are relative to."""
    z = (d(x) @ d(q)) * d(scales)
    if x_scales is not None:
        z = z * d(x_scales)[:, None]
    size = z.abs()
    if epilogue & 1:
        z, size = z + d(b), size + d(b).abs()
    return activate(z, epilogue, alpha), size


def runs(offsets):
    off = offsets.tolist()
    return [(e, slice(a, max(a, b))) for e, (a, b) in enumerate(zip(off, off[1:]))]


def grouped_dense(x, w, offsets, b=None, epilogue=0, alpha=0.0, before=None):
    """Rows of no group: as they were `before`."""
    x, w = x.double(), w.double()
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64, device=x.device)
    if before is not None:
        y.copy_(before)
    for e, r in runs(offsets):
        z = x[r] @ w[e]
        if epilogue & 1:
            z = z + b[e].double()
        y[r] = activate(z, epilogue, alpha)
    return y


def grouped_dense_backward(dy, x, w, offsets, y=None, epilogue=0, alpha=0.0, before=None):
    """dX, dW, db; dZ rounded to dY's type before the products, as documented."""
    act = ACTS[epilogue >> 1]
    dz = dy.double()
    if act != "none":
        dz = torch.where(y.double() > 0, dz, (as_f32(alpha) if act == "leaky" else 0.0) * dz)
    rounded = dz.to(dy.dtype).double()
    x, w = x.double(), w.double()
    E, K, N = w.shape
    dx = torch.zeros_like(x)
    if before is not None:
        dx.copy_(before)
    dw = torch.zeros(E, K, N, dtype=torch.float64, device=x.device)
    db = torch.zeros(E, N, dtype=torch.float64, device=x.device)
    for e, r in runs(offsets):
        dx[r] = rounded[r] @ w[e].t()
        dw[e] = x[r].t() @ rounded[r]
        db[e] = dz[r].sum(0)
    return dx, dw, db


def kept(x, temperature, top_k, top_p, min_p):
    """The kept indices of a row of finite and -inf logits, by falling logit, and their weights."""
    x = d(x)
    order = torch.sort(x, descending=True, stable=True).indices
    if 0 < top_k < len(x):
        order = order[:top_k]
    w = ((x[order] - x[order[0]]) / as_f32(temperature)).exp()
    before = w.cumsum(0) - w
    keep = torch.ones(len(w), dtype=torch.bool)
    if top_p < 1:
        keep = before < max(as_f32(top_p), 0.0) * w.sum()
        keep[0] = True
    if min_p > 0:
        keep &= w >= min(as_f32(min_p), 1.0)
    return order[keep], w[keep]


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability) of one row."""
    v = d(x)
    if v.isnan().any() or (v == math.inf).any():
        return -1, math.nan
    if (v == -math.inf).all():
        return -1, -math.inf
    if temperature == 0:
        return int((v == v.max()).nonzero()[0]), 0.0
    order, w = kept(x, temperature, top_k, top_p, min_p)
    order, at = order.sort()
    w = w[at]
    mass = w.cumsum(0)
    u = min(max(float(u), 0.0), 1.0 - 2.0 ** -53)
    i = min(int((mass <= u * mass[-1]).sum()), len(w) - 1)
    return int(order[i]), float((w[i] / mass[-1]).log())
