"""Rows of x with an infinity or NaN, under every epilogue: NaN in all of the row,
0 where the epilogue selects what is above 0. The other rows are those of the same
call without them, bit for bit."""
import math

import pytest
import torch

from mlir_edsl_hip import lm
from test_gpu_lm_q4 import ALPHA, BF16, E4M3, EPI, F16, F32, make_weights, make_x

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("epi", list(EPI))
@pytest.mark.parametrize("dtype", [F32, BF16, F16, E4M3])
@pytest.mark.parametrize("M", [3, 20, 70])
def test_epilogues(M, dtype, epi):
    K, N = 300, 90
    q, s, z = make_weights(K, N, 64)
    W, b = lm.q4_pack(q, s, z, group_size=64), torch.randn(N, device="cuda")
    x = make_x(M, K, dtype)
    y = torch.empty(M, N, device="cuda")
    lm.q4_dense_launch(x, W, b, y, EPI[epi], ALPHA)
    want = y.clone()
    assert not torch.isnan(want).any()
    x[0, 0] = math.nan
    if dtype != E4M3:  # which has no infinities
        x[1, K - 1] = -math.inf
    lm.q4_dense_launch(x, W, b, y, EPI[epi], ALPHA)
    bad = 1 if dtype == E4M3 else 2
    if epi.endswith("if_relu"):
        assert (y[:bad] == 0).all()
    else:
        assert torch.isnan(y[:bad]).all()
    assert torch.equal(y[bad:], want[bad:])
