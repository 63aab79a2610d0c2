"""The 4-bit layer on so many rows that the sums of x of a block's four groups lie
more than 2^32 bytes apart from one another's end. Tolerance: that of
test_gpu_lm_q4.py, by its check of sampled rows."""
import pytest
import torch

from mlir_edsl_hip import last_plan, lm
from test_gpu_lm_large import normal, q4_check, q4_weights

pytestmark = pytest.mark.gpu


def test_sums_of_x_past_32_bits():
    M, K, N, group = 358_000_000 + 65, 128, 2, 32  # x: 92e9 bytes; 12 bytes a row and block of sums: past 2^32
    q, s = q4_weights(K, N, group)
    W = lm.q4_pack(q, s, group_size=group)
    X = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, 77, M // 3, M // 2, M - 66, M - 2, M - 1], device="cuda")
    X[rows] = 1 + normal(len(rows), K, seed=1, dtype=torch.bfloat16).cuda()
    Y = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    lm.q4_dense_launch(X, W, None, Y)
    assert last_plan().startswith("q4_prep+q4_tile"), last_plan()
    q4_check(Y[rows], X[rows], q, s, group)
    assert bool((Y[2:77] == 0).all()) and not bool(Y.isnan().any())
    del X, Y
    torch.cuda.empty_cache()
