"""dW in f32 through a leaky epilogue: of 16-bit gradients times a slope that is no power of two, with no rounding
of their products, so that what is left is the sums' own. And small f16 gradients, whose products with the slope f16 does not hold."""
import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import _native, last_plan, lm
from test_gpu_lm_grouped import TYPES, offsets_of, stack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("alpha", [0.01, 0.3, 0.0, 1.0])
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("counts,K,N", [([3, 0, 20], 40, 24), ([150, 90, 0], 131, 259), ([150, 0, 300], 264, 136),
                                        ([1700, 1500], 4096, 2304), ([0, 0], 8, 8)], ids=str)
@pytest.mark.parametrize("size", [1.0, 1e-5])
def test_slope(dtype, alpha, order, counts, K, N, size):
    t, T, E, g = TYPES[dtype], sum(counts), len(counts), torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    dy, x, w, y = (size * r(T, N)).to(t).cuda(), r(T, K).to(t).cuda(), stack(r(E, K, N).to(t).cuda(), order), r(T, N).to(t).cuda()
    off = offsets_of(counts)
    dx, dw, db = torch.empty_like(x), stack(torch.full((E, K, N), 7.0, device="cuda"), order), torch.empty(E, N, device="cuda")
    lm.grouped_dense_backward_launch(dy, x, w, off, dx, dw, db, y, _native.EPI_BIAS_LEAKY, alpha)
    assert "dW" in last_plan()
    alone = torch.empty_like(dw)
    lm.grouped_dense_backward_launch(dy, x, None, off, dW=alone, Y=y, epilogue=_native.EPI_BIAS_LEAKY, alpha=alpha)
    assert torch.equal(alone, dw)
    # Sums of at most n terms in 32 bits, n + 64 roundings of 2^-23 of the terms' absolute sum; the slope's is one more.
    dz = torch.where(y > 0, dy.double(), layers.as_f32(alpha) * dy.double())
    n = max(counts)
    for e, rows in layers.runs(off):
        for got, want, terms in ((dw[e], x[rows].double().t() @ dz[rows], x[rows].double().abs().t() @ dz[rows].abs()),
                                 (db[e], dz[rows].sum(0), dz[rows].abs().sum(0))):
            assert float(((got.double() - want).abs() - (n + 65) * 2.0 ** -23 * terms).max()) <= 0
    # dX: dz rounded to its type, and its result.
    rounded = dz.to(t).double()
    for e, rows in layers.runs(off):
        want, terms = rounded[rows] @ w[e].double().t(), rounded[rows].abs() @ w[e].double().abs().t()
        bound = (N + 64) * 2.0 ** -23 * terms + torch.finfo(t).eps / 2 * want.abs() + torch.finfo(t).tiny * torch.finfo(t).eps
        if rows.stop > rows.start:
            assert float(((dx[rows].double() - want).abs() - bound).max()) <= 0
