"""What last_plan() says of a 4-bit layer on up to 32 rows is what ran: fewer than
eight waves are of up to 16 rows."""
import pytest
import torch

from mlir_edsl_hip import last_plan
from test_gpu_lm_q4 import BF16, F32, I8, layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,K,N,dtype,waves", [
    (16, 1024, 8192, BF16, 4), (17, 1024, 8192, BF16, 8), (20, 1024, 8192, I8, 8), (32, 448, 16384, BF16, 8),
    (16, 448, 16400, F32, 4), (3, 448, 33000, BF16, 2)])
def test_waves(M, K, N, dtype, waves):
    layer(M, K, N, 128, dtype)
    plan = last_plan()
    assert plan.startswith("q4_small") and "cols=32" in plan, plan
    assert (f" waves={waves}" in plan) if waves < 8 else ("waves" not in plan), plan
