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


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_captured(dtype):
    """A captured call whose rows, groups and infinities change between its replays: the eager call's bits."""
    t, T, E, K, N = TYPES[dtype], 160, 3, 72, 136
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(t).cuda()  # noqa: E731
    dy, x, y, w, off = r(T, N), r(T, K), r(T, N), r(E, K, N), offsets_of([100, 20, 40])
    outs = [torch.zeros(T, K, dtype=t, device="cuda"), torch.zeros(E, K, N, dtype=t if dtype == "f16" else torch.float32,
                                                                   device="cuda"), torch.zeros(E, N, device="cuda")]

    def step(outs):
        lm.grouped_dense_backward_launch(dy, x, w, off, *outs, y, _native.EPI_BIAS_LEAKY, 0.3)
    step(outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs)
    for i, counts in enumerate(([0, 160, 0], [1, 30, 129], [60, 60, 40], [10, 5, 2])):
        dy.copy_(r(T, N))
        x.copy_(r(T, K))
        x[i, ::3], x[150 - i, ::4] = math.inf, math.nan if i % 2 else -math.inf
        off.copy_(offsets_of(counts))
        for out in outs:
            out.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.full_like(out, -7.0) for out in outs]
        step(eager)
        for got, want in zip(outs, eager):
            assert torch.equal(got.double().nan_to_num(nan=12345.0), want.double().nan_to_num(nan=12345.0))
