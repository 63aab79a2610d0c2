"""Gradients through leaky epilogues whose products with the slope are exact, 0, 1 or without end: as without that
product, infinities too. Integers, compared bit for bit."""
import math

import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import _native, lm
from test_gpu_lm_grouped import FILL, TYPES, offsets_of, same, stack, whole

pytestmark = pytest.mark.gpu


def gradients(dy, x, w, off, y, epi, alpha, grad):
    E, K, N = w.shape
    dx = torch.full(x.shape, FILL, dtype=x.dtype, device="cuda")
    dw, db = (torch.full(s, FILL, dtype=grad, device="cuda") for s in ((E, K, N), (E, N)))
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db, y, epi, alpha)
    return dx, dw, db


def operands(counts, K, N, t, order):
    E, T = len(counts), sum(counts)
    return (whole(T, N, seed=3, dtype=t, most=2), whole(T, K, seed=1, dtype=t), stack(whole(E, K, N, seed=2, dtype=t), order),
            offsets_of(counts), whole(T, N, seed=4, dtype=t, most=2))


CASES = pytest.mark.parametrize("counts,K,N", [([3, 0, 20], 40, 24), ([150, 90, 0], 131, 259), ([150, 0, 300], 264, 136)],
                                ids=str)
EACH = pytest.mark.parametrize("dtype,grad", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16"),
                                              ("f32", "f32")])


@EACH
@CASES
@pytest.mark.parametrize("order", ["kn", "nk"])
def test_slope_of_0(dtype, grad, counts, K, N, order):
    """What does not pass is 0, an infinity or NaN of dY too, in dX, dW and db alike."""
    dy, x, w, off, y = operands(counts, K, N, TYPES[dtype], order)
    down = y <= 0
    clean = torch.where(down, torch.zeros_like(dy), dy)
    lost = torch.tensor([math.inf, -math.inf, math.nan], device="cuda").to(dy.dtype)
    dy = torch.where(down, lost[torch.arange(dy.numel(), device="cuda").reshape(dy.shape) % 3], dy)
    for got, right in zip(gradients(dy, x, w, off, y, _native.EPI_BIAS_LEAKY, 0.0, TYPES[grad]),
                          layers.grouped_dense_backward(clean, x, w, off)):
        same(got, right)


@EACH
@CASES
def test_slope_of_1(dtype, grad, counts, K, N):
    """The same bits as without an activation, where x has infinities."""
    dy, x, w, off, y = operands(counts, K, N, TYPES[dtype], "kn")
    x[::7, ::5] = math.inf
    with_slope = gradients(dy, x, w, off, y, _native.EPI_LEAKY, 1.0, TYPES[grad])
    without = gradients(dy, x, w, off, None, _native.EPI_NONE, 0.0, TYPES[grad])
    for a, b in zip(with_slope, without):
        assert torch.equal(a.nan_to_num(nan=12345.0), b.nan_to_num(nan=12345.0))


@EACH
def test_slope_without_end(dtype, grad):
    """A group whose outputs are all above 0 does not meet it."""
    dy, x, w, off, y = operands([40, 60], 72, 56, TYPES[dtype], "kn")
    y[:40] = 1
    dy[dy == 0] = 1
    got = gradients(dy, x, w, off, y, _native.EPI_LEAKY, math.inf, TYPES[grad])
    want = layers.grouped_dense_backward(dy, x, w, off)
    same(got[0][:40], want[0][:40])
    same(got[1][0], want[1][0])
    same(got[2][0], want[2][0])
    want = torch.where(y > 0, dy.double(), math.inf * dy.double())[40:].sum(0)
    assert torch.equal(got[2][1].double().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
