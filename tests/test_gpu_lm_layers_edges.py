"""The layers on groups of rows and in 8-bit integers at the ends of their operands: rows that
start on 16 bytes and end inside a load, strides that are not the row's length, axes longer than a launch's.

Integer values: products and sums are exact in 32 bits, and results are compared bit for bit."""
import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import _native, last_plan, lm
from test_gpu_lm_grouped import ALPHA, FILL, TYPES, offsets_of, same, whole

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def wider(t, more):
    """The same values, `more` NaN behind each row of the last index but the very last row: nothing follows that."""
    shape, n = t.shape, t.shape[-1]
    rows = t.numel() // n
    flat = torch.full(((rows - 1) * (n + more) + n,), float("nan"), dtype=t.dtype, device="cuda")
    strides = [n + more, 1] if t.dim() == 2 else [shape[1] * (n + more), n + more, 1]
    view = flat.as_strided(shape, strides)
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("odd", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("counts", [[3, 20], [300, 150]], ids=str)
def test_rows_that_end_inside_a_load(dtype, odd, counts):
    t = TYPES[dtype]
    K, N, T, E = 64 + odd, 128 + odd, sum(counts), 2
    pad_n, pad_k = -N % 8, -K % 8
    dy, y = whole(T, N, seed=3, dtype=t, most=2), whole(T, N, seed=4, dtype=t, most=2)
    off = offsets_of(counts)
    # Forward: whole loads of x, weights whose columns end inside one.
    x, w = whole(T, 72, seed=1, dtype=t), wider(whole(E, 72, N, seed=2, dtype=t), pad_n)
    out = torch.full((T, N), FILL, dtype=t, device="cuda")
    lm.grouped_dense_launch(x, w, off, None, out)
    assert ("stream" if max(counts) < 33 else "direct") in last_plan()
    same(out, layers.grouped_dense(x, w, off))
    # Gradients: both operands of dW end inside a load.
    x, w = wider(whole(T, K, seed=1, dtype=t), pad_k), wider(whole(E, K, N, seed=2, dtype=t, most=2), pad_n)
    for epi in (_native.EPI_NONE, _native.EPI_RELU):
        grad = wider(dy, pad_n)
        dx, dw, db = torch.full((T, K), FILL, dtype=t, device="cuda"), torch.empty(E, K, N, device="cuda"), \
            torch.empty(E, N, device="cuda")
        lm.grouped_dense_backward_launch(grad, x, w, off, dx, dw, db, y, epi)
        assert "dW 128x128" in last_plan(), last_plan()
        for got, right in zip((dx, dw, db), layers.grouped_dense_backward(dy, x, w, off, y, epi, ALPHA)):
            same(got, right)
