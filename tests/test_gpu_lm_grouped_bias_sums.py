"""db of a group of very many rows. Rows are summed by 32 in 32 bits and those sums in 64: at most 31 roundings of 2^-24
of the terms' absolute sum, one of the slope's product and one of the result, whatever the number of rows."""
import pytest
import torch

import lm_layers_reference as layers
from mlir_edsl_hip import _native, lm
from test_gpu_lm_grouped import TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("slope", [None, 0.3])
@pytest.mark.parametrize("T", [(1 << 20) - 5, 300001])
def test_one_large_group(dtype, slope, T):
    t, N, first = TYPES[dtype], 72, 1000
    g = torch.Generator(device="cuda").manual_seed(T)
    dy = torch.rand(T, N, generator=g, device="cuda")
    dy[:, ::2] = 0.1  # sums whose roundings all go one way
    dy, y = dy.to(t), None
    if slope is not None:
        y = torch.randn(T, N, generator=g, device="cuda").to(t)
    off = torch.tensor([0, first, first, T], dtype=torch.int64, device="cuda")
    db = torch.full((3, N), 7.0, device="cuda")
    lm.grouped_dense_backward_launch(dy, None, None, off, db=db, Y=y, epilogue=_native.EPI_NONE if y is None else
                                     _native.EPI_LEAKY, alpha=slope or 0.0)
    dz = dy.double()
    if y is not None:
        dz = torch.where(y > 0, dz, layers.as_f32(slope) * dz)
    for e, rows in enumerate((slice(0, first), slice(0, 0), slice(first, T))):
        want = dz[rows].sum(0)
        assert float(((db[e].double() - want).abs() - 34 * 2.0 ** -24 * dz[rows].abs().sum(0)).max()) <= 0


def test_more_columns_than_an_axis_of_a_launch():
    """64 columns a workgroup, 2^20 workgroups along an axis: sums of small integers, exact."""
    T, N = 3, (1 << 26) + 77
    dy = torch.randint(-3, 4, (T, N), dtype=torch.int8, device="cuda").to(TYPES["bf16"])
    off = torch.tensor([0, 1, T], dtype=torch.int32, device="cuda")
    db = torch.full((2, N), 7.0, device="cuda")
    lm.grouped_dense_backward_launch(dy, None, None, off, db=db)
    assert torch.equal(db[0], dy[0].float()) and torch.equal(db[1], dy[1].float() + dy[2].float())
