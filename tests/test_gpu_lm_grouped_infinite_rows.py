"""dW through a slope where x or dY holds infinities and NaN: what the sum of the products is in 64 bits. Finite sums
within n + 65 roundings of 2^-23 of their terms, and of dW's type."""
import math

import pytest
import torch

import lm_layers_reference as layers
import lm_reference as ref
from mlir_edsl_hip import _native, lm
from test_gpu_lm_grouped import TYPES, offsets_of, stack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,grad", [("bf16", "f32"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("counts,K,N", [([3, 0, 20], 40, 24), ([150, 90, 0], 131, 259), ([150, 0, 300], 264, 136)], ids=str)
def test_infinities(dtype, grad, order, counts, K, N):
    t, alpha = TYPES[dtype], 0.3
    T, E, g = sum(counts), len(counts), torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    dy, x, y = r(T, N), r(T, K), r(T, N).to(t)
    dy = torch.where(dy.abs() < 0.01, 0.01, dy)  # no zeros: 0 times infinity is NaN
    # Two rows of x meet in some sums: infinities of both signs, and NaN.
    x[1, ::3], x[2, ::4], x[-1, 1::5], x[-2, 2::7] = math.inf, -math.inf, math.inf, math.nan
    dy[0, ::6], dy[-3, 1::6] = math.inf, -math.inf
    dy, x = dy.to(t), x.to(t)
    off = offsets_of(counts)
    dw = stack(torch.full((E, K, N), 7.0, dtype=TYPES[grad], device="cuda"), order)
    lm.grouped_dense_backward_launch(dy.cuda(), x.cuda(), None, off, dW=dw, Y=y.cuda(), epilogue=_native.EPI_LEAKY,
                                     alpha=alpha)
    dz = torch.where(y > 0, dy.double(), layers.as_f32(alpha) * dy.double())
    x, dw = x.double(), dw.cpu()
    for e, rows in layers.runs(off.cpu()):
        terms = x[rows][:, :, None] * dz[rows][:, None, :]
        want, size = terms.sum(0), terms.abs().sum(0)
        got = dw[e].double()
        assert torch.equal(got.isnan(), want.isnan())
        fine = want.isfinite()
        assert torch.equal(got[~fine].nan_to_num(nan=0.0), want[~fine].nan_to_num(nan=0.0))
        bound = (max(counts) + 65) * 2.0 ** -23 * size + ref.HALF_ULP[dw.dtype] * want.abs() + ref.TINY[dw.dtype]
        assert bool(((got - want).abs() <= bound)[fine].all())
