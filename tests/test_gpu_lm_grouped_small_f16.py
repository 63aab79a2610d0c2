"""dW in f16 through a slope, of gradients whose products with it f16 does not hold: of the unrounded products in 64
bits within the sums' own roundings, n + 65 of 2^-23 of their terms, and the result's one, half a step of 2^-24 where it is
small."""
import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import _native, lm
from test_gpu_lm_grouped import F16, offsets_of, stack

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("alpha", [0.01, 0.3, 0.9, 0.0, 1.0])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-5])
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("counts,K,N", [([3, 0, 20], 40, 24), ([150, 90, 0], 131, 259), ([150, 0, 300], 264, 136),
                                        ([1700, 1500], 1024, 512)], ids=str)
def test_small_gradients(alpha, size, order, counts, K, N):
    T, E, g = sum(counts), len(counts), torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    dy, x, y = (size * r(T, N)).to(F16).cuda(), r(T, K).to(F16).cuda(), r(T, N).to(F16).cuda()
    off, dw = offsets_of(counts), stack(torch.full((E, K, N), 7.0, dtype=F16, device="cuda"), order)
    lm.grouped_dense_backward_launch(dy, x, None, off, dW=dw, Y=y, epilogue=_native.EPI_BIAS_LEAKY, alpha=alpha)
    dz = torch.where(y > 0, dy.double(), layers.as_f32(alpha) * dy.double())
    for e, rows in layers.runs(off):
        want, terms = x[rows].double().t() @ dz[rows], x[rows].double().abs().t() @ dz[rows].abs()
        bound = (max(counts) + 65) * 2.0 ** -23 * terms + 2.0 ** -11 * want.abs() + 2.0 ** -25
        assert float(((dw[e].double() - want).abs() - bound).max()) <= 0
